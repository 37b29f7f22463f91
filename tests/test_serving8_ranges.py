"""The 8-bit serving operators at the ends of what include/nnc_hip.h allows:
windows, scales and values of any size. Plain float64 forms: serving8.py."""

from __future__ import annotations

import subprocess
from pathlib import Path

import numpy as np
import pytest

import serving8 as s8
from serving8 import F16, F32, I8, I32
from test_serving8 import CACHE, cache_arrays, check_attention, dev, ragged, run_attention, tables  # noqa: F401 (dev: fixture)

ROOT = Path(__file__).resolve().parent.parent


# ---------------------------------------------------------------------------
# windows
# ---------------------------------------------------------------------------

def test_keys_under_windows_of_any_size(tmp_path):
    exe = tmp_path / "window_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'nnc-py_amd' / 'csrc'}", str(ROOT / "tests" / "native" / "window_check.cpp"), "-o", str(exe)],
                   check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout == "ok\n", res.stdout + res.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30, 33])
@pytest.mark.parametrize("heads,kv,rows", [(4, 2, [8, 5, 1]), (128, 32, [90, 45, 40])])
def test_windows_of_any_size_with_rows_without_a_position(heads, kv, rows, window, t, dev):  # noqa: F811
    """Sequences with three rows and more than they have positions, in both
    kernels: rows that have positions see them all under a window that is as
    good as none."""
    rng = np.random.default_rng(heads)
    run_attention(dev, rng, [5, 2, 40], rows, heads, kv, 64, 16, t, window=window, garbage=True, tile=128 if heads == 128 else None)
