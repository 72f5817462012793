"""The MXFP4 linear-layer load (``gpumon load --kind mxlinear``) on a real MI355X."""

import json
import os
import subprocess
import sys
import time

import pytest

from gpumon.ops.load import SyntheticLoad

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_load_counts_whole_layers_and_runs_again():
    rows, n, k = 100, 300, 700
    load = SyntheticLoad(0, "mxlinear", mx_rows=rows, mx_n=n, mx_k=k)
    for _ in range(2):
        with load:
            time.sleep(0.3)
            s = load.stats()
        assert s["launches"] > 0 and s["busy_s"] > 0
        assert s["mfma_s"] == s["hbm_s"] == s["busy_s"]
    done = load.stats()
    assert done["flops"] == done["launches"] * 2.0 * rows * n * k
    assert done["bytes"] == pytest.approx(done["launches"] * (2 * rows * k + 17 / 32 * n * k + 2 * rows * n))


def test_few_rows_stream_and_many_rows_multiply():
    with SyntheticLoad(0, "mxlinear", mx_rows=1) as load:
        time.sleep(1.0)
        few = load.stats()
    with SyntheticLoad(0, "mxlinear", mx_rows=4096) as load:
        time.sleep(1.0)
        many = load.stats()
    print(f"\nmxlinear: 1 row {few['tbps']:.2f} TB/s, 4096 rows {many['tflops']:.0f} TFLOP/s")
    assert few["tbps"] > 2.0 and few["tflops"] < 100
    assert many["tflops"] > 1500


def test_duty():
    with SyntheticLoad(0, "mxlinear", mx_rows=256, duty=0.3) as load:
        time.sleep(0.5)
        a = load.stats()
        time.sleep(1.5)
        b = load.stats()
    busy = SyntheticLoad.rates(a, b)["busy"]
    assert 0.1 < busy < 0.6, busy


def test_cli_prints_the_stats():
    r = subprocess.run([sys.executable, "-m", "gpumon", "load", "--kind", "mxlinear", "--rows", "8", "--seconds", "1"],
                       cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    assert json.loads(r.stdout)["bytes"] > 0


def test_the_matrix_counter_agrees_with_the_layers():
    """gpu_mfma_tflops{dtype="f6f4"} under real products (whole tiles, so no padding is counted): the
    layers' own rate, and nothing on another path's counter."""
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tools/mfma_dtypes.py"), "mxlinear"], capture_output=True,
                       text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-2000:]
    d = json.loads(r.stdout.strip().splitlines()[-1])["mxlinear"]
    (name, tf), = d["pmc_tflops"].items()
    assert name == "f6f4", d
    assert abs(tf - d["event_tflops"]) < 0.05 * d["event_tflops"], d
