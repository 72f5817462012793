"""Arguments of the MXFP4 linear-layer load are checked before any HIP call."""

import pytest

from gpumon.ops.load import SyntheticLoad


@pytest.mark.parametrize("kw,msg", [({"mx_rows": 0}, "at least 1"), ({"mx_n": -1}, "at least 1"), ({"mx_k": 0}, "at least 1"),
                                    ({"duty": 0.0}, "duty"), ({"mx_k": 1 << 29}, "limits"),
                                    ({"mx_n": 1 << 22, "mx_k": 1 << 16}, "limits")])
def test_bad_arguments_are_refused_before_the_gpu(kw, msg):
    with pytest.raises(ValueError, match=msg):
        SyntheticLoad(kind="mxlinear", **kw)
