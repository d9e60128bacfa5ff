"""CPU: what a backward pass of the microscaled operators does for its sizes (forms, parts, workspace)."""
import os
import subprocess

from conftest import ROOT


def test_backward_plans(tmp_path):
    exe = str(tmp_path / "grad_plan_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-o", exe,
                    os.path.join(ROOT, "tests", "grad_plan_check.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "PLAN_OK" in out.stdout, out.stdout + out.stderr
