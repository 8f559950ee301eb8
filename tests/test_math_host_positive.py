"""exp_neg_p (mxs_math.h) for positive arguments, built with the host compiler:
a beam selection's sums meet some, where their unit moves between rounded
values of nearly the same maximum."""
import subprocess
from pathlib import Path

HERE = Path(__file__).resolve().parent


def test_exp_neg_p_of_positive_arguments(tmp_path):
    exe = tmp_path / "check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-fno-fast-math",
                    str(HERE / "math_host_check_positive.cpp"), "-o", str(exe), "-lm"], check=True)
    fail, cases = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert cases > 1000000 and fail == 0
