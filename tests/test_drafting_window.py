"""Windows of nnc_hip_kv_tree_attention: the kernel is chosen by the keys that a
window leaves, and masks can say what a window of positions means for drafts that
reach further than it."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

import drafting as dr
import serving8 as s8
from serving8 import F16, F32
from test_drafting import run_tree, wide
from test_serving8 import CACHE, cache_arrays, check_attention, dev, ragged, tables  # noqa: F401 (dev: fixture)
from test_serving8_kernels import ran

ROOT = Path(__file__).resolve().parent.parent
JOIN = "nnc_hip_kv_tree_attention_join"  # of the kernel for 256 rows alone


def test_keys_that_a_window_leaves(tmp_path):
    exe = tmp_path / "draft_window_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'nnc-py_amd' / 'csrc'}", str(ROOT / "tests" / "native" / "draft_window_check.cpp"), "-o", str(exe)],
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


def chain_masks(rows, window, total):
    """Chains of drafts whose rows name the last `window` of those that lead to them."""
    return dr.masks([[list(range(max(0, i - window + 1), i + 1)) for i in range(n)] for n in rows], -(-max(rows) // 32), total)


CHAINS = [([200, 9, 30, 77], [20, 9, 30, 1], w) for w in (1, 2, 7, 19, 20, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("lengths,rows,window", CHAINS)
def test_chains_longer_than_the_window(lengths, rows, window, t, dev):  # noqa: F811
    """A chain whose masks stop a window back sees what a run of tokens does."""
    rng = np.random.default_rng(window)
    starts, total = ragged(rows)
    table, pages = tables(rng, lengths, 16)
    cache = s8.Cache(rng, pages, 2, 16, 64, table)
    q = (rng.standard_normal((total, 4 * 64)) * 2).astype(t)
    d = dev({"q": q, **cache_arrays(cache, starts, lengths), "tree": chain_masks(rows, window, total), "out": np.zeros((total, 256), t)})
    d.call("nnc_hip_kv_tree_attention", "q", *CACHE, "starts", "lengths", "tree", "out", 0, 4, 0.125, window, 0)
    check_attention(d.get("out"), q.reshape(total, 4, 64), cache, starts, lengths, F32(0.125), window)


@pytest.mark.parametrize("lengths,rows,window", CHAINS)
def test_chains_longer_than_the_window_on_the_oracle(lengths, rows, window, oracle_lib, abi):
    rng = np.random.default_rng(window)
    starts, total = ragged(rows, 0)
    table, pages = tables(rng, lengths, 16)
    cache = s8.Cache(rng, pages, 2, 16, 32, table)
    arrays = {"q": rng.standard_normal((total, 4 * 32)).astype(F32), **cache_arrays(cache, starts, lengths),
              "tree": chain_masks(rows, window, total), "out": np.zeros((total, 128), F32), "want": np.zeros((total, 128), F32)}
    kept = {n: (abi.make_tensor(a.ctypes.data, abi.NUMPY_TO_NNC[a.dtype.name], a.shape, a.nbytes), a) for n, a in
            ((n, np.ascontiguousarray(a)) for n, a in arrays.items())}
    T = lambda *names: [ctypes.pointer(kept[n][0][0]) for n in names]  # noqa: E731
    oracle_lib.nnc_hip_kv_tree_attention(*T("q", *CACHE, "starts", "lengths", "tree", "out"), 0, 4, 0.125, window, 0)
    oracle_lib.nnc_hip_kv_attention(*T("q", *CACHE, "starts", "lengths", "want"), 0, 4, 0.125, window, 0)
    np.testing.assert_array_equal(kept["out"][1], kept["want"][1])
    assert kept["out"][1].any()
