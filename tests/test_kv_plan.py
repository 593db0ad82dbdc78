"""How the attention kernels cut their work, checked on the CPU (native/kv_plan_check.cpp)."""
import os
import subprocess

from _util import ROOT


def test_spans_and_parts(tmp_path):
    exe = str(tmp_path / "kv_plan_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                    "-o", exe, os.path.join(ROOT, "tests", "native", "kv_plan_check.cpp")], check=True)
    got = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "ok", got.stdout + got.stderr
