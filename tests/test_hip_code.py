"""What the compiler made of the HIP sources, read from the libraries that were built here."""

import glob
import os

import pytest

from gfx_code import disassembly

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIP = glob.glob(os.path.join(ROOT, "gpumon", "_hip*.so"))


@pytest.fixture(scope="module")
def tmp(tmp_path_factory):
    return str(tmp_path_factory.mktemp("code"))


def test_loads_to_lds_are_checked_over_their_whole_offset(tmp):
    """The product's loads run past the last piece of k, and after the last tile past a buffer of no bytes,
    and count on getting zeros without a read. The check against the buffer's size does not count an
    instruction's scalar offset, so there must be none: `buffer_load_dwordx4 voffset, resource, 0 offen lds`."""
    (lib,) = HIP
    loads = [(k, i) for k, lines in disassembly(lib, tmp).items() for i in lines
             if i.startswith("buffer_load") and i.split()[-1] == "lds"]
    assert len(loads) > 100
    bad = [(k, i) for k, i in loads if i.split(",")[2].split()[0] != "0"]
    assert not bad, (len(bad), bad[:5])


@pytest.mark.parametrize("lib", ["gpumon/_hip*.so", "lib/libgpumon_probe.so", "build/obj/hip/probe_gfx950.hsaco"])
def test_no_packed_f32_arithmetic(tmp, lib):
    """Some forms of the packed f32 instructions have given wrong results: everything is compiled without."""
    for path in glob.glob(os.path.join(ROOT, lib)) or pytest.skip(f"{lib} is not built"):
        packed = {k for k, lines in disassembly(path, tmp).items()
                  for i in lines if i.startswith(("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))}
        assert not packed, packed
