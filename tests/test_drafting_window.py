"""Windows of nnc_hip_kv_tree_attention: the kernel is chosen by the keys that a
window leaves."""

from __future__ import annotations

import subprocess
from pathlib import Path

import numpy as np
import pytest

from serving8 import F16
from test_drafting import run_tree, wide
from test_serving8 import dev  # noqa: F401 (fixture)
from test_serving8_kernels import ran

ROOT = Path(__file__).resolve().parent.parent
JOIN = "nnc_hip_kv_tree_attention_join"  # of the kernel for 256 rows alone


def test_keys_that_a_window_leaves(tmp_path):
    exe = tmp_path / "window_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'nnc-py_amd' / 'csrc'}", str(ROOT / "tests" / "native" / "window_check.cpp"), "-o", str(exe)],
                   check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout == "ok\n", res.stdout + res.stderr


# a table as wide as the kernel for 256 rows asks for; the keys that a window
# leaves are fewer than that, or as many
@pytest.mark.gpu
@pytest.mark.parametrize("window,many", [(0, True), (1, False), (100, False), (1000, False), (2 ** 31 - 1, True)])
def test_kernel_by_the_keys_that_a_window_leaves(window, many, dev):  # noqa: F811
    rng = np.random.default_rng(3)
    table = ran(lambda: run_tree(dev, rng, [2500, 1700], [80, 70], 4, 1, 64, 32, F16, window=window, garbage=False, width=wide(2, 1, 32)))
    assert (JOIN in table) == many and "nnc_hip_kv_tree_attention" in table


@pytest.mark.gpu
@pytest.mark.parametrize("window", [3300, 4200])
def test_many_rows_behind_long_windows(window, dev):  # noqa: F811
    """The kernel for 256 rows with keys that its window hides: [6 sequences of
    up to 140 drafts, 32 heads over 4 of 32] has 24 times 64 keys a CU from a
    window of 3200 on."""
    rng = np.random.default_rng(window)
    lengths, rows = [6000, 5003, 4400, 140, 5200, 900], [140, 139, 140, 140, 140, 140]
    table = ran(lambda: run_tree(dev, rng, lengths, rows, 32, 4, 32, 48, F16, window=window, max_length=6000, garbage=False))
    assert JOIN in table
