"""CPU: which lane of a warp stores which sum (csrc/lane_sums.cuh), enumerated."""
import os
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_sum_is_stored_by_one_lane(tmp_path):
    exe = str(tmp_path / "model")
    subprocess.run([shutil.which("g++") or "g++", "-std=c++17", "-O1", "-I" + os.path.join(ROOT, "hdla_impl_b200", "csrc"),
                    os.path.join(ROOT, "tests", "model", "lane_sums_model.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], stdout=subprocess.PIPE, text=True, timeout=60)
    assert r.returncode == 0, r.stdout[-2000:]
