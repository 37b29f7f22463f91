"""The 8-bit serving operators at the ends of what include/nnc_hip.h allows:
windows, scales and values of any size. Plain float64 forms: serving8.py."""

from __future__ import annotations

import subprocess
from pathlib import Path

import numpy as np
import pytest

import serving8 as s8
from serving8 import F16, F32, I32
from test_serving8 import CACHE, cache_arrays, check_attention, check_norm, dev, run_attention, tables  # noqa: F401 (dev: fixture)

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


# ---------------------------------------------------------------------------
# value scales
# ---------------------------------------------------------------------------

# name: scales (powers of two) of a sequence's pages in turn, None a page of zeros
SCALES = {
    "zeros among 2^90": [90, None],
    "zeros among 2^114": [114, None, None, 113],
    "zeros among 2^-100": [-100, None],
    "zeros among the smallest": [-107, None, -106],
    "zeros and both ends": [100, None, -107, 0],
    "zeros alone": [None],
    "zeros first": [None, None, None, None, None, -3],
    "the smallest first": [-107, -107, -107, -107, -107, 110],
    "the largest first": [110, -107, -107, -107, -107, -107],
    "a step up each page": list(range(-100, 110, 15)),
    "a step down each page": list(range(110, -100, -15)),
    "far apart in turn": [-60, 60, -20, 100, -100],
}


# and such as float16 outputs can hold
SCALES16 = {"zeros among 2^7": [7, None], "zeros first": [None, None, None, None, None, -3], "the smallest first": [-107] * 5 + [7],
            "far apart in turn": [-60, 7, -20, -100], "zeros alone": [None]}


def far_bound(out, dim, about, t):
    """Scales far from 1: the logarithm of a scale under 2^128 is off by its
    last bit (2^-17), its sum with the scores and the maximum by half of one
    each; a weight by ln 2 times that, and the divisor's weights need not be off
    alike. A row whose weight is all on a page of zeros may have a result below
    float32's smallest step, 2^-149: it is rounded to a whole number of them."""
    size = about[0]
    return s8.attention_bound(t, dim, out, *about) + 2 * 0.6932 * 2.0 ** -16 * size + 2.0 ** -150


@pytest.mark.gpu
@pytest.mark.parametrize("sharp", [0.0, 0.3, 4.0, 60.0])
@pytest.mark.parametrize("name,t", [(n, F32) for n in SCALES] + [(n, F16) for n in SCALES16])
@pytest.mark.parametrize("rows,heads,kv,dim,length", [(1, 2, 1, 32, 9000), (1, 8, 2, 64, 700), (3, 4, 2, 256, 700), (700, 64, 1, 32, 700),
                                                      (200, 128, 32, 64, 300)])
def test_attention_over_pages_of_any_scale(rows, heads, kv, dim, length, name, t, sharp, dev):  # noqa: F811
    """Pages whose value scales lie anywhere from 2^-107 up, with pages of
    zeros among them: each key has its weight in the divisor however small its
    page's values are beside another's. Flat scores, and such as pick a page."""
    powers = (SCALES if t == F32 else SCALES16)[name]
    rng = np.random.default_rng(rows + dim)
    page = 16
    table, pages = tables(rng, [length], page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    for slot, p in enumerate(table[0]):
        power = powers[slot % len(powers)]
        if power is None:
            cache.vs[p] = 0
            if slot % 3:  # values are whole numbers times 0 either way
                cache.v[p] = 0
        else:
            cache.vs[p] = (rng.uniform(1, 2, kv) * 2.0 ** power).astype(F32)
    starts = np.array([0, rows], I32)
    q = (rng.standard_normal((rows, heads * dim)) * sharp).astype(t)
    scale = F32(dim ** -0.5)
    d = dev({"q": q, **cache_arrays(cache, starts, [length]), "out": np.full((rows, heads * dim), 7, t)})
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", 0, heads, float(scale), 0, 0)
    got = d.get("out").astype(np.float64)
    some = slice(None) if rows < 50 else slice(0, heads, 9)  # every head's answer has the same code
    shown = np.arange(rows) if rows < 50 else np.unique(np.linspace(0, rows - 1, 40).astype(int))
    out, about = attention_of(q.reshape(rows, heads, dim), cache, length, scale, shown, some)
    bound = far_bound(out, dim, about, t)
    off = np.abs(got.reshape(rows, heads, dim)[shown][:, some] - out)
    bad = ~(off <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), off[bad][:4], out[bad][:4])


def attention_of(q, cache, length, scale, shown, some):
    """serving8.attention for some rows and heads of one sequence whose rows
    are all `length` positions' last: out and what its bound needs."""
    rows, heads, dim = q.shape
    group = heads // cache.kv
    k, v, u, _ = cache.values(0, length)
    pos = length - rows + shown
    see = np.arange(length) <= pos[:, None]
    hs = np.arange(heads)[some]
    out, size = np.zeros((2, len(shown), len(hs), dim))
    reach, seen, peak = np.zeros((3, len(shown), len(hs)))
    for i, h in enumerate(hs):
        kk, vv, uu = k[h // group], v[h // group], u[h // group]
        x = q[shown, h].astype(np.float64)
        s = np.where(see, float(scale) * (x @ kk.T), -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, i], size[:, i] = p @ vv, p @ np.abs(vv)
        peak[:, i] = (p * uu).max(1)
        reach[:, i] = np.where(see, float(scale) * (np.abs(x) @ np.abs(kk).T), 0).max(1)
        seen[:, i] = see.sum(1)
    return out, (size, reach, seen, peak)


# ---------------------------------------------------------------------------
# norms of large values
# ---------------------------------------------------------------------------

def large_rows(rng, rows, width, power):
    """Rows around 2^power (one of ordinary size, one of zeros but for one
    element), below the largest number with a residual of a quarter."""
    x = rng.uniform(-1, 1, (rows, width)) * 2.0 ** power
    res = rng.uniform(-0.25, 0.25, (rows, width)) * 2.0 ** power
    if rows > 2:
        x[1], res[1] = x[1] * 2.0 ** -power, res[1] * 2.0 ** -power
        x[2], res[2] = 0, 0
        x[2, width // 2] = 2.0 ** power
    return x.astype(F32), res.astype(F32), rng.uniform(0.1, 0.5, width).astype(F32)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [55, 60, 64, 90, 126, 127])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 256), (5, 4096), (4, 1345), (3, 8192), (3, 8200), (2, 40000), (4100, 64),
                                        (4100, 500), (4097, 1000)])
def test_rms_norm_of_large_values(rows, width, int8, power, dev):  # noqa: F811
    """Squares that pass the largest float32 number: the root is finite and
    every output has its value, in the kernel of each width and row count."""
    rng = np.random.default_rng(rows + width + power)
    x, res, w = large_rows(rng, rows, width, power)
    check_norm(dev, x, None, w, int8)
    check_norm(dev, x, res, w, int8, alias=rows > 4000)
    if rows < 10:
        check_norm(dev, x, res, w, int8, shift={"x": 4})


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [3e38, 1e30, 1e-30, 1e-38])
def test_rms_norm_of_any_epsilon(eps, dev):  # noqa: F811
    rng = np.random.default_rng(1)
    eps = float(F32(eps))
    for power in (-40, 0, 62, 127):
        x, res, w = large_rows(rng, 4, 700, power)
        for int8 in (False, True):
            check_norm(dev, x, res, w, int8, eps=eps)


# ---------------------------------------------------------------------------
# query sizes
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("q_power,k_power", [(-125, 126), (-120, 124), (-100, 97), (60, -60), (104, -105), (101, -104)])
@pytest.mark.parametrize("rows,heads,kv", [(1, 4, 2), (200, 128, 32)])
def test_queries_and_key_scales_far_from_one(rows, heads, kv, q_power, k_power, dev):  # noqa: F811
    """Scores of ordinary size from queries and keys that are not."""
    rng = np.random.default_rng(rows)
    page, dim, length = 16, 64, 300
    table, pages = tables(rng, [length], page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    cache.ks = (rng.uniform(0.004, 0.02, cache.ks.shape) * 2.0 ** k_power).astype(F32)
    starts = np.array([0, rows], I32)
    q = (rng.standard_normal((rows, heads * dim)) * 2.0 ** q_power).astype(F32)
    scale = F32(0.125)
    d = dev({"q": q, **cache_arrays(cache, starts, [length]), "out": np.zeros((rows, heads * dim), F32)})
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", 0, heads, float(scale), 0, 0)
    some = slice(None) if rows == 1 else slice(0, heads, 9)
    shown = np.unique(np.linspace(0, rows - 1, 20).astype(int))
    out, about = attention_of(q.reshape(rows, heads, dim), cache, length, scale, shown, some)
    off = np.abs(d.get("out").reshape(rows, heads, dim)[shown][:, some].astype(np.float64) - out)
    assert (off <= s8.attention_bound(F32, dim, out, *about)).all(), off.max()


# ---------------------------------------------------------------------------
# caches of more than 4 GiB
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("lengths,rows,heads", [([40, 17, 33], [40, 1, 2], 16), ([300, 250], [250, 250], 64)])
def test_pages_behind_four_gib(lengths, rows, heads, t, hip, abi):
    """Pages at the far end of a cache: written, read back and attended to, by
    both attention kernels, as by a small cache that holds them alone."""
    from nnc_py_amd import runtime
    runtime.clear_error()
    kv, page, dim, pages = 8, 16, 128, 280000
    assert pages * kv * page * dim > 2 ** 32
    rng = np.random.default_rng(len(lengths))
    table, used = tables(rng, lengths, page, extra=0)
    small = s8.Cache(rng, used, kv, page, dim, table, filled=False)
    far = np.concatenate([np.arange(pages - used + 1, pages), [0]]).astype(I32)  # the small cache's page -> the large one's
    far_table = np.where(table < used, far[np.minimum(table, used - 1)], table).astype(I32)
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(I32)
    total = int(starts[-1])
    x = rng.standard_normal((total, (heads + 2 * kv) * dim)).astype(t)
    d = s8.Dev(hip, abi, runtime, {"x": x, "table": far_table, "starts": starts, "lengths": np.array(lengths, I32),
                                   "k_scale": np.zeros((pages, kv), F32), "v_scale": np.zeros((pages, kv), F32),
                                   "kr": np.zeros((total, kv * dim), t), "vr": np.zeros((total, kv * dim), t),
                                   "out": np.zeros((total, heads * dim), t)})
    big = [runtime.DeviceBuffer.empty((pages, kv, *s), np.int8) for s in ((page, dim), (dim, page))]
    try:
        for name, b in zip(("k_cache", "v_cache"), big):
            d.desc[name], shape = b.tensor()
            d.kept.append(shape)
        before = [n - min(n, r) for n, r in zip(lengths, rows)]
        if any(before):  # the positions before the rows
            b_starts = np.concatenate([[0], np.cumsum(before)]).astype(I32)
            y = rng.standard_normal((int(b_starts[-1]), 2 * kv * dim)).astype(t)
            e = s8.Dev(hip, abi, runtime, {"x": y, "starts": b_starts, "lengths": np.array(before, I32)})
            args = [d.t(n) for n in CACHE]
            hip.nnc_hip_kv_write(e.t("x"), e.t("x"), *args, e.t("starts"), e.t("lengths"), 0, kv * dim)
            runtime.sync()
            small.write(y[:, :kv * dim].reshape(-1, kv, dim), y[:, kv * dim:].reshape(-1, kv, dim), b_starts, before)
            e.free()
        k_col, v_col = heads * dim, (heads + kv) * dim
        d.call("nnc_hip_kv_write", "x", "x", *CACHE, "starts", "lengths", k_col, v_col)
        parts = x.reshape(total, heads + 2 * kv, dim)
        small.write(parts[:, heads:heads + kv], parts[:, heads + kv:], starts, lengths)
        d.call("nnc_hip_kv_read", *CACHE, "starts", "lengths", "kr", "vr", 0, 0)
        kr, vr = (d.get(n).reshape(total, kv, dim) for n in ("kr", "vr"))
        for b, n in enumerate(lengths):
            for i in range(max(0, rows[b] - n), rows[b]):
                pos = n - rows[b] + i
                p = small.page_of(b, pos)
                np.testing.assert_array_equal(kr[starts[b] + i], (small.k[p, :, pos % page].astype(F32) * small.ks[p][:, None]).astype(t))
                np.testing.assert_array_equal(vr[starts[b] + i], (small.v[p, :, :, pos % page].astype(F32) * small.vs[p][:, None]).astype(t))
        d.call("nnc_hip_kv_attention", "x", *CACHE, "starts", "lengths", "out", 0, heads, float(F32(dim ** -0.5)), 0, 0)
        check_attention(d.get("out"), parts[:, :heads], small, starts, lengths, F32(dim ** -0.5), 0)
    finally:
        d.free()
        for b in big:
            b.free()
