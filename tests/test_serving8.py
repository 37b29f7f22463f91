"""The 8-bit serving operators (include/nnc_hip.h: nnc_hip_rms_norm,
nnc_hip_quantize_rows, nnc_hip_dequantize_rows, nnc_hip_matmul_i8,
nnc_hip_kv_write, nnc_hip_kv_read, nnc_hip_kv_attention) against plain
float64 forms (serving8.py). Whole numbers, scales of rows that are not
normalised and everything read back are equal; the rest is off by no more than
the counted roundings."""

from __future__ import annotations

import threading

import numpy as np
import pytest

import serving8 as s8
from serving8 import F16, F32, I8, I32, SUB16, U16, U32

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(hip, abi):
    from nnc_py_amd import runtime
    runtime.clear_error()
    made = []

    def make(arrays, shift=None):
        made.append(s8.Dev(hip, abi, runtime, arrays, shift))
        return made[-1]
    yield make
    for d in made:
        d.free()


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------

def norm_inputs(rng, rows, width, t, residual):
    x = rng.standard_normal((rows, width)).astype(t)
    res = None
    if residual:
        res = (rng.standard_normal((rows, width)) * 2).astype(t)
        res[:, ::97] *= t(8)
    return x, res, (1 + 0.1 * rng.standard_normal(width)).astype(t)


def norm_rel(width):
    """r is off by its sum of squares' roundings, halved by the root (a
    thread's run of at most width / 64 + 2 terms, the joins under 16), the
    mean, eps, root and quotient (5); y adds two products."""
    return (0.5 * (width / 64 + 18) + 8) * U32


def check_norm(dev, x, res, w, int8, eps=1e-6, shift=None, alias=False):
    t = x.dtype.type
    arrays = {"x": x, "w": w, "out": np.zeros(x.shape, I8 if int8 else t)}
    if res is not None:
        arrays["res"] = res
        if not alias:
            arrays["sum"] = np.zeros_like(x)
    if int8:
        arrays["scale"] = np.zeros(x.shape[:-1], F32)
    d = dev(arrays, shift)
    total = None if res is None else "res" if alias else "sum"
    d.call("nnc_hip_rms_norm", "x", "res" if res is not None else None, "w", total, "out", "scale" if int8 else None, eps)
    s, tw, r, y = s8.rms_norm(x, res, w, eps)
    if res is not None:
        np.testing.assert_array_equal(d.get(total), s)
    rel = norm_rel(x.shape[-1])
    if int8:
        unit = s8.unit8(s8.absmax(tw, -1))
        np.testing.assert_array_equal(d.get("out"), s8.whole8(tw, unit[..., None]))
        want = r[..., 0] * unit
        np.testing.assert_allclose(d.get("scale"), want, rtol=rel + U32, atol=0)
    else:
        got = d.get("out").astype(np.float64)
        bound = rel * np.abs(y) + (U16 * np.abs(y) * (1 + rel) + SUB16 if t == F16 else 0)
        assert (np.abs(got - y) <= bound).all(), np.max(np.abs(got - y) / np.maximum(bound, 1e-300))


NORM_SHAPES = [(1, 1), (1, 4096), (3, 33), (8, 4096), (37, 1345), (5, 8192), (2, 16400), (300, 64), (65, 520), (9, 1000)]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("rows,width", NORM_SHAPES)
def test_rms_norm(rows, width, int8, t, dev):
    rng = np.random.default_rng(rows * 31 + width)
    for residual in (False, True):
        x, res, w = norm_inputs(rng, rows, width, t, residual)
        check_norm(dev, x, res, w, int8)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("int8", [False, True])
def test_rms_norm_sum_over_residual_and_unaligned(int8, t, dev):
    """The sum written over the residual, rows in three extents, buffers that
    start on no 16-byte boundary."""
    rng = np.random.default_rng(5)
    x, res, w = norm_inputs(rng, 12, 512, t, True)
    check_norm(dev, x.reshape(3, 4, 512), res.reshape(3, 4, 512), w, int8, alias=True)
    e = x.dtype.itemsize
    check_norm(dev, x, res, w, int8, shift={"x": e, "res": 2 * e, "w": e, "out": 1 if int8 else e, "sum": e, "scale": 4})
    check_norm(dev, x, res, w, int8, shift={"out": 4})


@pytest.mark.parametrize("t", [F32, F16])
def test_rms_norm_output_over_input(t, dev):
    rng = np.random.default_rng(6)
    x, _, w = norm_inputs(rng, 7, 640, t, False)
    d = dev({"x": x, "w": w})
    d.call("nnc_hip_rms_norm", "x", None, "w", None, "x", None, 1e-5)
    y = s8.rms_norm(x, None, w, 1e-5)[3]
    bound = norm_rel(640) * np.abs(y) + (U16 * 1.01 * np.abs(y) + SUB16 if t == F16 else 0)
    assert (np.abs(d.get("x") - y) <= bound).all()


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("width", [48, 777, 4096])
def test_rows_that_are_zero_or_not_finite(width, t, dev):
    rng = np.random.default_rng(width)
    x = rng.standard_normal((6, width)).astype(t)
    x[1] = 0
    x[2, width // 2] = np.nan
    x[3, width - 1] = np.inf
    x[4, 0] = -np.inf
    w = np.ones(width, t)
    d = dev({"x": x, "w": w, "q": np.full(x.shape, 99, I8), "s": np.zeros(6, F32), "y": np.zeros_like(x)})
    for call in (("nnc_hip_quantize_rows", "x", "q", "s"), ("nnc_hip_rms_norm", "x", None, "w", None, "q", "s", 1e-6)):
        d.call(*call)
        q, s = d.get("q"), d.get("s")
        assert not q[1:5].any() and s[1] == 0 and np.isnan(s[2:5]).all()
        assert np.isfinite(s[[0, 5]]).all() and (np.abs(q[[0, 5]]).max(1) == 127).all()
        d.call("nnc_hip_dequantize_rows", "q", "s", "y")
        y = d.get("y")
        assert not y[1].any() and np.isnan(y[2:5]).all() and np.isfinite(y[[0, 5]]).all()


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 31), (8, 4096), (33, 1345), (3, 14336), (200, 96)])
def test_quantize_and_dequantize_rows(rows, width, t, dev):
    rng = np.random.default_rng(width)
    x = (rng.standard_normal((rows, width)) * rng.uniform(1e-3, 1e3, (rows, 1))).astype(t)
    # ties: multiples of half a step of a row whose largest value is 127
    if width > 8:
        x[-1] = (rng.integers(-253, 254, width) * 0.5).astype(t)
        x[-1, 3] = 127
    if t == F32:
        x[0] *= F32(2.0 ** -90)
    d = dev({"x": x, "q": np.zeros(x.shape, I8), "s": np.zeros(rows, F32), "y": np.zeros_like(x)})
    d.call("nnc_hip_quantize_rows", "x", "q", "s")
    unit = s8.unit8(s8.absmax(x.astype(F32), 1))
    q = s8.whole8(x.astype(F32), unit[:, None])
    np.testing.assert_array_equal(d.get("s"), unit)
    np.testing.assert_array_equal(d.get("q"), q)
    d.call("nnc_hip_dequantize_rows", "q", "s", "y")
    np.testing.assert_array_equal(d.get("y"), (q.astype(F32) * unit[:, None]).astype(t))


def test_empty_rows_do_nothing(dev):
    d = dev({"x": np.zeros((0, 64), F32), "q": np.zeros((0, 64), I8), "s": np.zeros(0, F32), "w": np.ones(64, F32)})
    d.call("nnc_hip_quantize_rows", "x", "q", "s")
    d.call("nnc_hip_dequantize_rows", "q", "s", "x")
    d.call("nnc_hip_rms_norm", "x", None, "w", None, "q", "s", 1e-6)


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------

def check_product(dev, rng, m, n, k, t, bias=True, shift=None, lead=None, full=False):
    a = rng.integers(-128 if full else -127, 128, (m, k)).astype(I8)
    w = rng.integers(-128 if full else -127, 128, (n, k)).astype(I8)
    if full:
        a[0], w[0] = -128, -128
    sa, sw = rng.uniform(0.001, 0.02, m).astype(F32), rng.uniform(0.001, 0.02, n).astype(F32)
    b = (rng.standard_normal(n) * 3).astype(F32)
    lead = lead or (m,)
    d = dev({"a": a.reshape(*lead, k), "sa": sa, "w": w, "sw": sw, "b": b, "out": np.full((*lead, n), 7, t)}, shift)
    d.call("nnc_hip_matmul_i8", "a", "sa", "w", "sw", "b" if bias else None, "out")
    acc = a.astype(np.float64) @ w.astype(np.float64).T
    p = acc * sa[:, None].astype(np.float64) * sw.astype(np.float64)
    y = p + b if bias else p
    # the sum to float32, the scales' product, the product, the bias
    bound = 3 * U32 * np.abs(p) + U32 * np.abs(y)
    if t == F16:
        bound = bound + U16 * np.abs(y) * 1.001 + SUB16
    got = d.get("out").reshape(m, n).astype(np.float64)
    bad = ~(np.abs(got - y) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], y[bad][:4])


PRODUCTS = [(1, 1, 1), (1, 32, 32), (1, 4096, 4096), (3, 5, 7), (8, 1024, 4096), (13, 33, 16), (16, 48, 1040), (17, 300, 512),
            (33, 64, 64), (64, 64, 128), (37, 101, 77), (100, 257, 1345), (128, 128, 1024), (130, 520, 272), (257, 129, 640),
            (300, 1000, 96), (512, 512, 48), (777, 1001, 345), (1, 7, 20000), (5, 4097, 64), (260, 2050, 2064)]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul_i8(m, n, k, t, dev):
    check_product(dev, np.random.default_rng(m + 7 * n + 13 * k), m, n, k, t, bias=(m + n) % 2 == 0)


@pytest.mark.parametrize("m,n,k", [(4, 96, 256), (48, 80, 320), (300, 400, 512)])
def test_matmul_i8_unaligned_leading_extents_and_full_range(m, n, k, dev):
    rng = np.random.default_rng(k)
    check_product(dev, rng, m, n, k, F32, lead=(2, m // 2))
    check_product(dev, rng, m, n, k, F16, shift={"a": 1, "w": 3, "sa": 4, "sw": 8, "b": 4, "out": 2})
    check_product(dev, rng, m, n, k, F32, shift={"a": 4, "w": 16, "out": 4})
    check_product(dev, rng, m, n, k, F32, full=True)


def test_matmul_i8_extreme_sums(dev):
    """The longest rows of the lowest value: the sum is just under 2^31."""
    k = 131071
    a, w = np.full((2, k), -128, I8), np.full((3, k), -128, I8)
    one = np.ones(3, F32)
    d = dev({"a": a, "sa": one[:2], "w": w, "sw": one, "out": np.zeros((2, 3), F32)})
    d.call("nnc_hip_matmul_i8", "a", "sa", "w", "sw", None, "out")
    assert (d.get("out") == F32(128 * 128 * k)).all()


@pytest.mark.parametrize("m", [1, 8, 40, 300])
def test_matmul_i8_keeps_to_its_rows(m, dev):
    """Integers that float32 holds come out exactly; a scale that is not
    finite stays in its row or column."""
    rng = np.random.default_rng(m)
    k, n = 144, 90
    a, w = rng.integers(-9, 10, (m, k)).astype(I8), rng.integers(-9, 10, (n, k)).astype(I8)
    sa, sw = np.ones(m, F32), np.ones(n, F32)
    sw[7] = np.nan
    if m > 1:
        sa[1] = np.nan
    d = dev({"a": a, "sa": sa, "w": w, "sw": sw, "out": np.zeros((m, n), F32)})
    d.call("nnc_hip_matmul_i8", "a", "sa", "w", "sw", None, "out")
    want = (a.astype(F32) @ w.astype(F32).T) * sa[:, None] * sw
    np.testing.assert_array_equal(d.get("out"), want)


# ---------------------------------------------------------------------------
# cache
# ---------------------------------------------------------------------------

def ragged(rows, pad=0):
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(I32)
    return starts, int(starts[-1]) + pad


def tables(rng, lengths, page, extra=2, width=None):
    """A table of scattered pages, unused slots full of numbers that are no page."""
    used = [-(-n // page) for n in lengths]
    width = width or max(1, max(used, default=1))
    pages = sum(used) + extra
    order = rng.permutation(pages).astype(I32)
    table = np.full((len(lengths), width), 123456789, I32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def cache_arrays(cache, starts, lengths):
    return {**cache.tensors(), "starts": starts, "lengths": np.asarray(lengths, I32)}


CACHE = ("k_cache", "v_cache", "k_scale", "v_scale", "table")


def check_cache(d, cache):
    for name, want in (("k_scale", cache.ks), ("v_scale", cache.vs), ("k_cache", cache.k), ("v_cache", cache.v)):
        np.testing.assert_array_equal(d.get(name), want, err_msg=name)


KV_SIZES = [(1, 16, 32), (2, 16, 128), (3, 48, 64), (2, 64, 64), (1, 128, 128), (2, 256, 256), (5, 32, 64), (1, 240, 32)]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("kv,page,dim", KV_SIZES)
def test_kv_write_and_read(kv, page, dim, t, dev):
    write_and_read(kv, page, dim, t, dev, 1, 3, 4, 7)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("kv,page,dim", KV_SIZES + [(3, 16, 64), (1, 112, 64), (2, 128, 256), (1, 64, 128),
                                                     (1, 256, 128), (1, 176, 256)])
def test_kv_write_and_read_aligned(kv, page, dim, t, dev):
    write_and_read(kv, page, dim, t, dev, 0, 8, 8, 8)


def write_and_read(kv, page, dim, t, dev, k_shift, v_shift, back_col, back_pad):
    """Ragged rows: new sequences, rows that begin inside a page, at its first
    and last position, none, a sequence of one position; rows of a fused
    projection; padding behind the last."""
    rng = np.random.default_rng(page + dim)
    lengths = [page + 3, 1, page, 0, 2 * page + 5, page - 1, 3 * page, 2 * page]
    rows = [page + 3, 1, 1, 0, 4, 0, page + 2, page]
    starts, total = ragged(rows, pad=3)
    table, pages = tables(rng, lengths, page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    heads = 2
    x = rng.standard_normal((total, (heads + 2 * kv) * dim + (5 if k_shift else 8))).astype(t)
    x[2] *= 20  # scales that grow
    k_col, v_col = heads * dim + k_shift, (heads + kv) * dim + v_shift
    back_rows = [min(n, r + page - 1) for n, r in zip(lengths, rows)]
    back, back_total = ragged(back_rows, pad=2)
    d = dev({"x": x, **cache_arrays(cache, starts, lengths), "back": back,
             "kr": np.full((back_total, kv * dim), 9, t), "vr": np.full((back_total, kv * dim + back_pad), 9, t)})
    d.call("nnc_hip_kv_write", "x", "x", *CACHE, "starts", "lengths", k_col, v_col)
    want = cache.copy()
    want.write(x[:, k_col:k_col + kv * dim].reshape(total, kv, dim), x[:, v_col:v_col + kv * dim].reshape(total, kv, dim), starts, lengths)
    check_cache(d, want)
    # once more: nothing changes
    d.call("nnc_hip_kv_write", "x", "x", *CACHE, "starts", "lengths", k_col, v_col)
    check_cache(d, want)
    d.call("nnc_hip_kv_read", *CACHE, "back", "lengths", "kr", "vr", 0, back_col)
    kr, vr = np.full((back_total, kv * dim), 9, t), np.full((back_total, kv * dim + back_pad), 9, t)
    for b, n in enumerate(lengths):
        for i in range(back_rows[b]):
            pos = n - back_rows[b] + i
            p = want.page_of(b, pos)
            kr[back[b] + i] = (want.k[p, :, pos % page].astype(F32) * want.ks[p][:, None]).reshape(-1).astype(t)
            vr[back[b] + i, back_col:back_col + kv * dim] = (want.v[p, :, :, pos % page].astype(F32) * want.vs[p][:, None]).reshape(-1).astype(t)
    np.testing.assert_array_equal(d.get("kr"), kr)
    np.testing.assert_array_equal(d.get("vr"), vr)


@pytest.mark.parametrize("t", [F32, F16])
def test_kv_write_token_by_token(t, dev):
    """A sequence written one row at a time over two pages, its scale growing
    now and then, among sequences that get none in that call."""
    rng = np.random.default_rng(3)
    page, kv, dim, steps = 16, 2, 64, 37
    table = np.array([[2, 0, 3], [4, 4, 4]], I32)
    cache = s8.Cache(rng, 5, kv, page, dim, table)
    x = (rng.standard_normal((steps, 2 * kv * dim)) * rng.uniform(0.5, 2, (steps, 1))).astype(t)
    d = dev({"x": np.zeros((1, 2 * kv * dim), t), **cache_arrays(cache, np.array([0, 1, 1], I32), [0, 7])})
    for i in range(steps):
        d.set("x", x[i:i + 1])
        d.set("lengths", np.array([i + 1, 7], I32))
        d.call("nnc_hip_kv_write", "x", "x", *CACHE, "starts", "lengths", 0, kv * dim)
        cache.write(x[i:i + 1, :kv * dim].reshape(1, kv, dim), x[i:i + 1, kv * dim:].reshape(1, kv, dim), [0, 1, 1], [i + 1, 7])
        check_cache(d, cache)


def test_kv_write_values_that_are_not_finite(dev):
    """An infinity or a NaN makes its page and head read as NaN, nothing else;
    a page that starts over is well again. Zeros have scale 0."""
    rng = np.random.default_rng(4)
    page, kv, dim = 16, 2, 32
    cache = s8.Cache(rng, 4, kv, page, dim, np.array([[0, 1, 2]], I32))
    x = rng.standard_normal((2 * page, kv * dim)).astype(F32)
    x[3, 5] = np.inf       # head 0, first page
    x[page + 1, 40] = np.nan  # head 1, second page
    y = np.zeros_like(x)
    d = dev({"x": x, "y": y, **cache_arrays(cache, np.array([0, 2 * page], I32), [2 * page]),
             "kr": np.zeros((2 * page, kv * dim), F32), "vr": np.ones((2 * page, kv * dim), F32)})
    d.call("nnc_hip_kv_write", "x", "y", *CACHE, "starts", "lengths", 0, 0)
    d.call("nnc_hip_kv_read", *CACHE, "starts", "lengths", "kr", "vr", 0, 0)
    kr = d.get("kr").reshape(2, page, kv, dim)
    assert np.isnan(kr[0, :, 0]).all() and np.isnan(kr[1, :, 1]).all()
    assert np.isfinite(kr[0, :, 1]).all() and np.isfinite(kr[1, :, 0]).all()
    assert not d.get("vr").any() and not d.get("v_scale")[:2].any()
    x[:] = 1
    d.set("x", x)
    d.call("nnc_hip_kv_write", "x", "y", *CACHE, "starts", "lengths", 0, 0)
    d.call("nnc_hip_kv_read", *CACHE, "starts", "lengths", "kr", "vr", 0, 0)
    assert np.isfinite(d.get("kr")).all()


def test_kv_calls_with_bad_tables_and_lengths(dev):
    """Page numbers outside the cache, lengths outside the table, rows without
    positions: nothing is written for them, the rest is as ever."""
    rng = np.random.default_rng(8)
    page, kv, dim = 16, 2, 64
    table = np.array([[-1, 0], [1, 7], [2, 3], [4, 5]], I32)  # pages 0..5
    cache = s8.Cache(rng, 6, kv, page, dim, table)
    lengths = [20, 32, 1000, -5]
    starts = np.array([0, 20, 25, 30, 40], I32)
    x = rng.standard_normal((40, kv * dim)).astype(F32)
    d = dev({"x": x, **cache_arrays(cache, starts, lengths), "r": np.full((40, kv * dim), 5, F32),
             "s": np.full((40, kv * dim), 5, F32), "out": np.full((40, kv * dim), 5, F32)})
    d.call("nnc_hip_kv_write", "x", "x", *CACHE, "starts", "lengths", 0, 0)
    clamped = [20, 32, 32, 0]
    want = cache.copy()
    want.write(x.reshape(40, kv, dim), x.reshape(40, kv, dim), starts, clamped)
    check_cache(d, want)
    d.call("nnc_hip_kv_read", *CACHE, "starts", "lengths", "r", "s", 0, 0)
    r = d.get("r")
    assert (r[0:16] == 5).all() and (r[20:25] == 5).all() and (r[30:] == 5).all()
    assert (r[16:20] != 5).any() and (r[25:30] != 5).any()
    d.call("nnc_hip_kv_attention", "x", *CACHE, "starts", "lengths", "out", 0, kv, 0.125, 0, 0)
    check_attention(d.get("out"), x.reshape(40, kv, dim), want, starts, clamped, 0.125, 0)
    assert not d.get("out")[:16].any() and not d.get("out")[30:].any()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def check_attention(got, q, cache, starts, lengths, scale, window):
    rows, heads, dim = q.shape
    out, about = s8.attention(q, cache, starts, lengths, scale, window)
    owned = ~np.isnan(out[:, 0, 0])
    bound = s8.attention_bound(got.dtype.type, dim, out, *about)
    off = np.abs(got.reshape(out.shape).astype(np.float64) - out)
    bad = ~(off <= bound) & owned[:, None, None]
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), off[bad][:4], bound[bad][:4])
    return owned


def run_attention(dev, rng, lengths, rows, heads, kv, dim, page, t, window=0, max_length=0, pad=2, sharp=2.0, width=None, garbage=False, tile=None, spread=0):
    starts, total = ragged(rows, pad)
    table, pages = tables(rng, lengths, page, width=width)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    if garbage:  # everything that no row sees
        for b, n in enumerate(lengths):
            if n % page:
                p = cache.page_of(b, n - 1)
                cache.k[p, :, n % page:] = -128
                cache.v[p, :, :, n % page:] = -128
        used = {cache.page_of(b, t) for b, n in enumerate(lengths) for t in range(n)}
        for p in set(range(pages)) - used:
            cache.ks[p] = cache.vs[p] = np.nan
    if spread:
        cache.vs *= (2.0 ** rng.integers(-spread, spread + 1, cache.vs.shape)).astype(F32)
        if t == F16:
            cache.vs = np.minimum(cache.vs, F32(300))
        cache.v[table[0, 1]] = cache.k[table[0, 1]] = 0
        cache.vs[table[0, 1]] = cache.ks[table[0, 1]] = 0
    q_col = 3
    qrows = (rng.standard_normal((total, heads * dim + 6)) * sharp).astype(t)
    scale = dim ** -0.5
    d = dev({"q": qrows, **cache_arrays(cache, starts, lengths), "out": np.full((total, heads * dim), 7, t)})
    if tile:
        from nnc_py_amd import runtime
        runtime.profile_reset()
        runtime.profile_enable(True)
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", q_col, heads, scale, window, max_length)
    if tile:
        names = [r["name"] for r in runtime.profile_table()]
        runtime.profile_enable(False)
        assert names == [f"nnc_hip_kv_attention_{tile}"]
    got = d.get("out")
    q = qrows[:, q_col:q_col + heads * dim].reshape(total, heads, dim)
    owned = check_attention(got, q, cache, starts, lengths, F32(scale), window)
    assert (got[~owned] == 7).all()
    return got


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,page", [(1, 1, 32, 16), (4, 4, 64, 16), (8, 2, 128, 16), (6, 2, 64, 48), (7, 1, 128, 64),
                                               (4, 2, 256, 32), (20, 1, 64, 128), (40, 2, 32, 256)])
def test_kv_attention_single_tokens(heads, kv, dim, page, t, dev):
    rng = np.random.default_rng(heads + dim + page)
    lengths = [1, 15, 16, 17, 0, 63, 64, 65, 200, 333]
    run_attention(dev, rng, lengths, [1] * 10, heads, kv, dim, page, t, garbage=True)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,page", [(2, 2, 64, 16), (4, 1, 128, 32), (3, 3, 32, 16), (2, 1, 256, 64), (5, 1, 64, 48)])
def test_kv_attention_runs_of_tokens(heads, kv, dim, page, t, dev):
    """Prompts, chunks behind a cached context, none, single tokens, more rows
    than positions; padding behind."""
    rng = np.random.default_rng(heads * dim)
    run_attention(dev, rng, [70, 9, 140, 40, 3, 0, 129], [70, 2, 33, 0, 5, 4, 1], heads, kv, dim, page, t, garbage=True)


PROMPTS = {128: ([130, 70, 40, 9, 0, 33], [130, 33, 3, 12, 4, 0], 32), 256: ([200, 130], [190, 110], 64)}


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("tile,dim,page", [(128, 32, 16), (128, 64, 48), (128, 128, 16), (128, 256, 64), (256, 32, 64), (256, 64, 16), (256, 128, 32)])
def test_kv_attention_prompts(tile, dim, page, t, dev):
    """Enough rows and heads for the kernels of 128 and 256 rows: whole
    prompts, chunks, more rows than positions, none; windows; scores that pick
    single keys; value scales from page to page 2^20 up and down, a page of
    zeros; what no row sees is garbage."""
    rng = np.random.default_rng(tile + dim)
    lengths, rows, kv = PROMPTS[tile]
    for window, sharp, spread in ((0, 2.0, 0), (37, 1.0, 0), (100, 30.0, 0), (0, 1.0, 20), (0, 0.0, 3)):
        run_attention(dev, rng, lengths, rows, 128, kv, dim, page, t, window=window, garbage=True, tile=tile, sharp=sharp, spread=spread)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("tile", [128, 256])
def test_kv_attention_prompts_with_pages_that_cannot_be_read(tile, t, dev):
    """Page numbers outside the cache inside a prompt: their keys are unseen."""
    rng = np.random.default_rng(tile)
    lengths, rows, kv = PROMPTS[tile]
    starts, total = ragged(rows, 0)
    table, pages = tables(rng, lengths, 16)
    table[0, 2], table[0, 7], table[1, 0] = -1, pages, 2 ** 31 - 1
    cache = s8.Cache(rng, pages, kv, 16, 64, table)
    q = (rng.standard_normal((total, 128 * 64)) * 2).astype(t)
    d = dev({"q": q, **cache_arrays(cache, starts, lengths), "out": np.zeros((total, 128 * 64), t)})
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", 0, 128, 0.125, 0, 0)
    check_attention(d.get("out"), q.reshape(total, 128, 64), cache, starts, lengths, F32(0.125), 0)


def test_kv_attention_prompts_without_a_table(dev):
    """A table of no width: no row sees anything."""
    rng = np.random.default_rng(0)
    cache = s8.Cache(rng, 2, 32, 16, 64, np.zeros((2, 0), I32))
    starts = np.array([0, 100, 190], I32)
    d = dev({"q": np.ones((190, 128 * 64), F32), **cache_arrays(cache, starts, [40, 0]), "out": np.ones((190, 128 * 64), F32)})
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", 0, 128, 0.125, 0, 0)
    assert not d.get("out").any()


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("window", [1, 16, 37, 64, 100, 1000])
def test_kv_attention_window(window, t, dev):
    rng = np.random.default_rng(window)
    run_attention(dev, rng, [1, 130, 200, 97, 300], [1, 1, 90, 3, 1], 4, 2, 64, 16, t, window=window, garbage=True)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("max_length", [0, 1, 3000, 5000])
def test_kv_attention_long_axis(max_length, t, dev):
    """A few rows over a long context: the keys are divided, and joined; the
    hint may be wrong."""
    rng = np.random.default_rng(1)
    run_attention(dev, rng, [5000, 3, 2049], [1, 1, 2], 8, 2, 64, 32, t, max_length=max_length, pad=0)


@pytest.mark.parametrize("t", [F32, F16])
def test_kv_attention_wide_table(t, dev):
    """A table for far longer sequences than there are."""
    rng = np.random.default_rng(2)
    run_attention(dev, rng, [40, 7, 0], [1, 1, 1], 4, 2, 128, 16, t, width=4000)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows", [1, 40])
def test_kv_attention_sharp_and_flat(rows, t, dev):
    """Scores that pick single keys, and queries of zero (a plain mean)."""
    rng = np.random.default_rng(3)
    run_attention(dev, rng, [400, 90], [rows, rows], 4, 4, 64, 16, t, sharp=30.0)
    run_attention(dev, rng, [400, 90], [rows, rows], 4, 4, 64, 16, t, sharp=0.0)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows", [1, 33])
def test_kv_attention_pages_of_different_size(rows, t, dev):
    """Scales that differ by 2^40 from page to page, pages of zeros (scale 0)."""
    rng = np.random.default_rng(9)
    page, kv, dim, heads, length = 16, 2, 64, 4, 200
    table, pages = tables(rng, [length], page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    cache.vs *= (2.0 ** rng.integers(-20, 21, cache.vs.shape)).astype(F32)
    cache.ks *= (2.0 ** rng.integers(-3, 2, cache.ks.shape)).astype(F32)
    for name in ("v", "k"):
        getattr(cache, name)[table[0, 3]] = 0
        getattr(cache, name + "s")[table[0, 3]] = 0
    if t == F16:
        cache.vs = np.minimum(cache.vs, F32(300))
    starts = np.array([0, rows], I32)
    q = (rng.standard_normal((rows, heads * dim)) * 2).astype(t)
    d = dev({"q": q, **cache_arrays(cache, starts, [length]), "out": np.zeros((rows, heads * dim), t)})
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", 0, heads, 0.125, 0, 0)
    check_attention(d.get("out"), q.reshape(rows, heads, dim), cache, starts, [length], F32(0.125), 0)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("batch,kv,several", [(40, 8, False), (70, 4, False), (256, 2, False), (256, 8, False), (300, 1, False),
                                              (600, 4, False), (90, 4, True)])
@pytest.mark.parametrize("dim", [32, 128])
def test_kv_attention_many_sequences(dim, batch, kv, several, t, dev):
    """More workgroups than fit at once, of different sizes: every sequence answered once, in
    whatever order, those without rows or positions among them; with one
    sequence of several tiles too."""
    rng = np.random.default_rng(batch)
    lengths = rng.integers(0, 150, batch)
    lengths[:3] = [700, 0, 1]
    rows = rng.integers(0, 5, batch) > 0
    rows = [int(r) for r in rows]
    rows[0] = 1
    if several:
        rows[5] = 20
    run_attention(dev, rng, [int(n) for n in lengths], rows, 2 * kv, kv, dim, 16, t, garbage=True)


@pytest.mark.parametrize("rows,heads,length", [(1, 4, 9000), (600, 64, 700)])
@pytest.mark.parametrize("power", [-100, 90])
def test_kv_attention_values_very_small_and_large(power, rows, heads, length, dev):
    """Values from the smallest that the cache holds to far beyond a product's:
    neither the sums nor the divisor overflow or vanish."""
    rng = np.random.default_rng(abs(power) + rows)
    table, pages = tables(rng, [length], 64)
    cache = s8.Cache(rng, pages, 1, 64, 32, table)
    cache.vs = (rng.uniform(1, 4, cache.vs.shape) * 2.0 ** power).astype(F32)
    starts = np.array([0, rows], I32)
    q = rng.standard_normal((rows, heads * 32)).astype(F32)
    d = dev({"q": q, **cache_arrays(cache, starts, [length]), "out": np.zeros((rows, heads * 32), F32)})
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", 0, heads, 0.1, 0, 0)
    check_attention(d.get("out"), q.reshape(rows, heads, 32), cache, starts, [length], F32(0.1), 0)


def test_kv_attention_query_sizes(dev):
    """fp32 queries from very small to very large: the pieces hold 22 bits of
    each row at any size; a row that is not finite stays by itself."""
    rng = np.random.default_rng(10)
    page, kv, dim, heads = 16, 1, 64, 1
    lengths = [50] * 6
    table, pages = tables(rng, lengths, page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    q = rng.standard_normal((6, dim)).astype(F32)
    q *= np.array([1e-30, 1e-6, 1.0, 1.0, 1e6, 1.0], F32)[:, None]
    cache.ks[table[4, :4]] *= F32(1e-6)
    q[3, 7] = np.nan
    starts = np.arange(7, dtype=I32)
    d = dev({"q": q, **cache_arrays(cache, starts, lengths), "out": np.zeros((6, dim), F32)})
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", 0, heads, 0.125, 0, 0)
    got = d.get("out")
    assert np.isnan(got[3]).all() and np.isfinite(np.delete(got, 3, 0)).all()
    fine = np.delete(np.arange(6), 3)
    out, about = s8.attention(np.where(np.isnan(q), 0, q).reshape(6, 1, dim), cache, starts, lengths, 0.125, 0)
    bound = s8.attention_bound(F32, dim, out, *about)
    assert (np.abs(got.reshape(6, 1, dim) - out) <= bound)[fine].all()


# ---------------------------------------------------------------------------
# as they are used
# ---------------------------------------------------------------------------

def decode_setup(rng, t, batch=3, steps=5):
    page, kv, dim, heads = 16, 2, 64, 4
    context = [30, 1, 15][:batch]
    most = [n + steps for n in context]
    table, pages = tables(rng, most, page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    x = rng.standard_normal((steps, batch, (heads + 2 * kv) * dim)).astype(t)
    return page, kv, dim, heads, context, cache, x


def test_captured_decode_step_replayed(dev, hip):
    """kv_write and kv_attention captured once and replayed for every token,
    rows and lengths changing between the replays, with a synchronisation and
    an eager call in between."""
    from nnc_py_amd import runtime
    rng = np.random.default_rng(12)
    page, kv, dim, heads, context, cache, x = decode_setup(rng, F16)
    steps, batch, _ = x.shape
    starts = np.arange(batch + 1, dtype=I32)
    d = dev({"x": x[0], **cache_arrays(cache, starts, context), "out": np.zeros((batch, heads * dim), F16)})
    k_col, v_col = heads * dim, (heads + kv) * dim
    runtime.check(hip.nnc_hip_graph_begin(), "begin")
    hip.nnc_hip_kv_write(d.t("x"), d.t("x"), *(d.t(n) for n in CACHE), d.t("starts"), d.t("lengths"), k_col, v_col)
    hip.nnc_hip_kv_attention(d.t("x"), *(d.t(n) for n in CACHE), d.t("starts"), d.t("lengths"), d.t("out"), 0, heads, 0.125, 0, 60)
    runtime.check(hip.nnc_hip_graph_end(), "end")
    for i in range(steps):
        lengths = [n + i + 1 for n in context]
        d.set("x", x[i])
        d.set("lengths", np.array(lengths, I32))
        runtime.check(hip.nnc_hip_graph_launch(), "launch")
        runtime.sync()
        rows = x[i].reshape(batch, heads + 2 * kv, dim)
        cache.write(rows[:, heads:heads + kv], rows[:, heads + kv:], starts, lengths)
        check_cache(d, cache)
        got = d.get("out")
        check_attention(got, rows[:, :heads], cache, starts, lengths, F32(0.125), 0)
        d.call("nnc_hip_kv_attention", "x", *CACHE, "starts", "lengths", "out", 0, heads, 0.125, 0, 60)
        np.testing.assert_array_equal(d.get("out"), got)
    hip.nnc_hip_graph_destroy()


def test_two_threads_and_the_second_stream(dev, hip):
    """Divided attention from two host threads at once and on the side stream:
    each has its own workspace."""
    from nnc_py_amd import runtime
    rng = np.random.default_rng(13)
    jobs = []
    for n in (4000, 2500):
        table, pages = tables(rng, [n], 16)
        cache = s8.Cache(rng, pages, 2, 16, 64, table)
        q = rng.standard_normal((1, 4 * 64)).astype(F32)
        d = dev({"q": q, **cache_arrays(cache, np.array([0, 1], I32), [n]), "out": np.zeros((1, 256), F32)})
        jobs.append((d, q, cache, n))

    def run(d, times):
        for _ in range(times):
            hip.nnc_hip_kv_attention(d.t("q"), *(d.t(c) for c in CACHE), d.t("starts"), d.t("lengths"), d.t("out"), 0, 4, 0.125, 0, 0)
        runtime.sync()
    threads = [threading.Thread(target=run, args=(j[0], 20)) for j in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    first = [j[0].get("out") for j in jobs]
    for j, got in zip(jobs, first):
        check_attention(got, j[1].reshape(1, 4, 64), j[2], [0, 1], [j[3]], F32(0.125), 0)
    runtime.check(hip.nnc_hip_stream_fork(), "fork")
    runtime.check(hip.nnc_hip_stream_select(1), "select")
    run(jobs[0][0], 1)
    runtime.check(hip.nnc_hip_stream_select(0), "select")
    run(jobs[1][0], 1)
    runtime.check(hip.nnc_hip_stream_join(), "join")
    runtime.sync()
    for j, got in zip(jobs, first):
        np.testing.assert_array_equal(j[0].get("out"), got)
