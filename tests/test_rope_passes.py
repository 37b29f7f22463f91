"""How the heads of rows are given to waves, without a GPU."""

from __future__ import annotations

import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_every_pass_has_heads_and_every_head_a_pass(tmp_path):
    exe = tmp_path / "heads_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'nnc-py_amd' / 'csrc'}", str(ROOT / "tests" / "native" / "heads_check.cpp"), "-o", str(exe)],
                   check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout == "ok\n", res.stdout + res.stderr
