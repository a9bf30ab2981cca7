"""The number of parts of kg_pool_attend_dev's work (katgpt-rs_b200/csrc/kg_pool_sched.h, the kernels' own source) on the CPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_parts_hold_work_and_few_cut_items(tmp_path):
    exe = tmp_path / "pool_parts_host"
    r = subprocess.run(["g++", "-O1", "-std=c++17", os.path.join(ROOT, "tests", "host", "pool_parts_host.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout
