"""How the paged cache's attention shares a batch out between workgroups, on the host: the arithmetic that the kernel uses
(ggml-compiler_amd/csrc/paged_plan.h), over thousands of batches."""

import re
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def test_every_item_and_row_has_a_workgroup(tmp_path):
    exe = tmp_path / "paged_plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT / 'ggml-compiler_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cpp" / "paged_plan.cpp"), "-o", str(exe)], check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stdout
    found = [int(x) for x in re.findall(r"\d+", out.stdout.splitlines()[-1])]
    assert min(found[:3]) > 0 and found[3] == 0, out.stdout  # the batches in question are among them
