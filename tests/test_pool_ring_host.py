"""The ring of stages of kg_pool_attend_dev's kernels (katgpt-rs_b200/csrc/kg_pool_ring.h, their own source) on host threads."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_wait_that_runs_out(tmp_path):
    exe = tmp_path / "pool_ring_host"
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-pthread", os.path.join(ROOT, "tests", "host", "pool_ring_host.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout
