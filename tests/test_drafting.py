"""Rotary positions, tree attention and token log probabilities
(include/nnc_hip.h: nnc_hip_rope, nnc_hip_rope_kv_write,
nnc_hip_kv_tree_attention, nnc_hip_token_logprobs) against plain float64 forms
(drafting.py). What goes into the cache and the tokens named are equal; the rest
is off by no more than the counted roundings."""

from __future__ import annotations

import threading

import numpy as np
import pytest

import drafting as dr
import serving8 as s8
from serving8 import F16, F32, I32, SUB16, U16, U32
from test_serving8 import CACHE, cache_arrays, check_cache, dev, ragged, tables  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# rotation
# ---------------------------------------------------------------------------

def turn_table(rng, places, rot):
    a = rng.uniform(-4, 4, (places, rot // 2))
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(F32)


def run_rope(dev, rng, rows, heads, dim, rot, interleaved, norm, t, places=50, col=0, pad=0, out_col=0, out_pad=0, shift=None, in_place=False, each=False):
    width = heads * dim
    x = (rng.standard_normal((rows, col + width + pad)) * 3).astype(t)
    w = (1 + 0.2 * rng.standard_normal((heads, dim) if each else dim)).astype(t) if norm else None
    table = turn_table(rng, places, rot) if rot else None
    at = rng.integers(-3, places + 3, rows).astype(I32)
    arrays = {"x": x, "out": np.full((rows, out_col + width + out_pad), 7, t)}
    if norm:
        arrays["w"] = w
    if rot:
        arrays.update(angles=table, at=at)
    d = dev(arrays, shift)
    out, to = ("x", col) if in_place else ("out", out_col)
    eps = 1e-5
    d.call("nnc_hip_rope", "x", "w" if norm else None, "angles" if rot else None, "at" if rot else None, out, col, to, heads, dim, int(interleaved), eps)
    got = d.get(out)
    y, size = dr.rope(x[:, col:col + width].reshape(rows, heads, dim), w, table, at, interleaved, eps)
    mine = got[:, to:to + width].reshape(y.shape).astype(np.float64)
    bound = dr.rope_bound(t, y, size)
    assert (np.abs(mine - y) <= bound).all(), np.max(np.abs(mine - y) / bound)
    other = np.delete(got, np.s_[to:to + width], 1)
    np.testing.assert_array_equal(other, np.delete(x, np.s_[col:col + width], 1) if in_place else np.full_like(other, 7))
    return got


ROPE = [(1, 1, 2, 2), (1, 1, 64, 64), (5, 3, 128, 128), (3, 5, 96, 48), (17, 40, 128, 64), (2, 7, 80, 80), (300, 2, 64, 32), (4, 2, 256, 256),
        (9, 6, 112, 56), (3, 1, 192, 20), (6, 3, 33, 14), (5, 2, 7, 6), (70, 10, 32, 32), (2, 3, 1000, 500), (1000, 1, 16, 16), (3, 64, 128, 2)]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,dim,rot", ROPE)
def test_rope(rows, heads, dim, rot, interleaved, t, dev):
    rng = np.random.default_rng(rows * 7 + dim)
    for norm in (False, True):
        run_rope(dev, rng, rows, heads, dim, rot, interleaved, norm, t, each=norm and heads > 2)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("heads,dim,rot", [(6, 64, 64), (3, 128, 32), (5, 40, 12), (9, 256, 128)])
def test_rope_in_place_columns_and_alignment(heads, dim, rot, t, dev):
    rng = np.random.default_rng(dim + rot)
    e = np.dtype(t).itemsize
    for interleaved in (False, True):
        run_rope(dev, rng, 37, heads, dim, rot, interleaved, True, t, col=dim, pad=2 * dim, in_place=True, each=True)
        run_rope(dev, rng, 37, heads, dim, rot, interleaved, True, t, col=8, pad=8, out_col=16, out_pad=24)
        run_rope(dev, rng, 37, heads, dim, rot, interleaved, True, t, col=3, pad=2, out_col=1, out_pad=4)
        run_rope(dev, rng, 11, heads, dim, rot, interleaved, True, t, col=1, pad=0, in_place=True)
        run_rope(dev, rng, 11, heads, dim, rot, interleaved, True, t, shift={"x": e, "out": 2 * e, "w": e, "angles": 4, "at": 4})
        run_rope(dev, rng, 11, heads, dim, rot, interleaved, True, t, shift={"w": e})
        run_rope(dev, rng, 11, heads, dim, rot, interleaved, False, t, shift={"angles": 4})


@pytest.mark.parametrize("t", [F32, F16])
def test_rope_norm_without_rotation_and_nothing(t, dev):
    rng = np.random.default_rng(3)
    run_rope(dev, rng, 20, 6, 64, 0, False, True, t)
    run_rope(dev, rng, 20, 6, 50, 0, True, True, t, each=True)
    got = run_rope(dev, rng, 20, 6, 64, 0, False, False, t)  # a copy
    assert got.any()


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("dim,rot", [(64, 64), (48, 10)])
def test_rope_values_of_any_size(dim, rot, t, dev):
    """Heads of zeros, of the type's largest and smallest values, and ones that
    are not finite, beside others that they must not reach."""
    rng = np.random.default_rng(dim)
    x = rng.standard_normal((8, 2, dim)).astype(t)
    big, small = np.finfo(t).max, np.finfo(t).smallest_subnormal
    x[0, 0], x[1, 0], x[2, 0] = 0, big, small
    x[3, 0, 3], x[4, 0, 1] = np.nan, np.inf
    table = np.concatenate([np.ones((1, rot // 2)), np.zeros((1, rot // 2))], 1).astype(F32)  # no turn: the type's largest stays
    w = np.ones(dim, t)
    for norm in (True, False):
        d = dev({"x": x.reshape(8, -1), "w": w, "angles": table, "at": np.zeros(8, I32), "out": np.zeros((8, 2 * dim), t)})
        d.call("nnc_hip_rope", "x", "w" if norm else None, "angles", "at", "out", 0, 0, 2, dim, 0, 1e-6)
        got = d.get("out").reshape(x.shape)
        with np.errstate(invalid="ignore"):
            y, size = dr.rope(x, w if norm else None, table, np.zeros(8, int), False, 1e-6)
        fine = np.ones((8, 2), bool)
        fine[3, 0] = fine[4, 0] = False
        assert (np.abs(got[fine] - y[fine]) <= dr.rope_bound(t, y, size)[fine]).all()
        assert not got[0, 0].any() and np.isfinite(got[fine]).all() and np.isnan(got[3, 0, 3])
        assert np.isnan(got[3, 0]).all() or not norm


def test_rope_far_positions(dev):
    """Angles of far positions come from the table: its last rows, and what is
    beyond clamped to the last."""
    from nnc_py_amd import rotary
    rng = np.random.default_rng(8)
    at = np.array([0, 1, 99999, 131071, 131072, 2 ** 31 - 1, -1, -2 ** 31], I32)
    table = rotary.angles(131072, 8)
    x = rng.standard_normal((8, 64)).astype(F32)
    d = dev({"x": x, "angles": table, "at": at, "out": np.zeros_like(x)})
    d.call("nnc_hip_rope", "x", None, "angles", "at", "out", 0, 0, 1, 64, 0, 0.0)
    y, size = dr.rope(x[:, None], None, table, at.astype(np.int64), False, 0.0)
    assert (np.abs(d.get("out") - y[:, 0]) <= dr.rope_bound(F32, y, size)[:, 0]).all()


# ---------------------------------------------------------------------------
# into the cache
# ---------------------------------------------------------------------------

def run_rope_kv_write(dev, rng, lengths, rows, heads, kv, dim, page, rot, interleaved, norm, t, positions=False, in_place=False, pad=2, col=0,
                      tail=0, queries=True, shift=None, each=False):
    """One call against the plain forms, and against the three calls that it is."""
    starts, total = ragged(rows, pad)
    table, pages = tables(rng, lengths, page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    most = max(max(lengths), 1)
    x = (rng.standard_normal((total, col + (heads + 2 * kv) * dim + tail)) * 2).astype(t)
    angles = turn_table(rng, most, rot) if rot else None
    at = rng.integers(0, most, total).astype(I32)
    arrays = {"x": x, **cache_arrays(cache, starts, lengths), "q": np.full((total, heads * dim), 7, t)}
    if norm:
        arrays["qw"] = (1 + 0.2 * rng.standard_normal((heads, dim) if each else dim)).astype(t)
        arrays["kw"] = (1 + 0.2 * rng.standard_normal((kv, dim) if each else dim)).astype(t)
    if rot:
        arrays["angles"] = angles
    if positions:
        arrays["at"] = at
    d = dev(arrays, shift)
    q_col, k_col = col, col + heads * dim
    v_col = k_col + kv * dim
    d.call("nnc_hip_rope_kv_write", "x" if queries else None, "x", "x", "qw" if norm and queries else None, "kw" if norm else None,
           "angles" if rot else None, "at" if positions else None, None if in_place or not queries else "q", *CACHE, "starts", "lengths",
           q_col, heads, k_col, v_col, int(interleaved), 1e-6)
    place, owned = np.zeros(total, int), np.zeros(total, bool)
    for b, n in enumerate(lengths):
        place[starts[b]:starts[b + 1]] = np.arange(n - rows[b], n)
        owned[starts[b]:starts[b + 1]] = True
    if positions:
        place = at
    got = d.get("x")
    rowed = x[:, col:col + (heads + 2 * kv) * dim].reshape(total, heads + 2 * kv, dim)
    if queries:
        y, size = dr.rope(rowed[:, :heads], arrays.get("qw"), angles, place, interleaved, 1e-6)
        q = got[:, q_col:k_col] if in_place else d.get("q")
        bound = dr.rope_bound(t, y, size)
        assert (np.abs(q.reshape(y.shape).astype(np.float64) - y) <= bound)[owned].all()
        before = x[:, q_col:k_col] if in_place else np.full_like(q, 7)
        np.testing.assert_array_equal(q[~owned], before[~owned])
    if not in_place or not queries:
        np.testing.assert_array_equal(got, x)
        assert queries or (d.get("q") == 7).all()
    else:
        np.testing.assert_array_equal(np.delete(got, np.s_[q_col:k_col], 1), np.delete(x, np.s_[q_col:k_col], 1))
    # the cache: the whole numbers of the plain form, and of the calls one by one
    k, _ = dr.rope(rowed[:, heads:heads + kv], arrays.get("kw"), angles, place, interleaved, 1e-6)
    after = cache.copy()
    after.write(k.astype(F32).astype(t), rowed[:, heads + kv:], starts, lengths)
    check_cache(d, after)
    e = dev({"x": x, **cache_arrays(cache, starts, lengths), "k": np.zeros((total, kv * dim), t), "place": np.asarray(place, I32),
             **{n: arrays[n] for n in ("kw", "angles") if n in arrays}})
    e.call("nnc_hip_rope", "x", "kw" if norm else None, "angles" if rot else None, "place" if rot else None, "k", k_col, 0, kv, dim, int(interleaved), 1e-6)
    e.call("nnc_hip_kv_write", "k", "x", *CACHE, "starts", "lengths", 0, v_col)
    for n in CACHE[:4]:
        np.testing.assert_array_equal(e.get(n), d.get(n))
    return d


APPEND = [(1, 1, 32, 16, 32), (8, 2, 128, 16, 128), (6, 2, 64, 48, 32), (4, 4, 64, 64, 64), (7, 1, 128, 128, 64), (4, 2, 256, 32, 256), (3, 3, 32, 256, 16),
          (2, 1, 256, 256, 256), (5, 5, 64, 16, 10)]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,dim,page,rot", APPEND)
def test_rope_kv_write(heads, kv, dim, page, rot, interleaved, t, dev):
    """Prompts, chunks behind a cached context, none, single tokens, more rows
    than positions; padding behind."""
    rng = np.random.default_rng(heads * dim + page)
    lengths, rows = [70, 9, 140, 40, 3, 0, 129, page, 2 * page + 1], [70, 2, 33, 0, 5, 4, 1, page, 1]
    for norm in (False, True):
        run_rope_kv_write(dev, rng, lengths, rows, heads, kv, dim, page, rot, interleaved, norm, t, positions=norm, each=norm and interleaved)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("dim,page,rot", [(64, 16, 64), (128, 32, 64), (128, 16, 128)])
def test_rope_kv_write_in_place_columns_and_alignment(dim, page, rot, t, dev):
    rng = np.random.default_rng(dim + rot)
    lengths, rows = [40, 0, 19, 66], [7, 0, 1, 50]
    e = np.dtype(t).itemsize
    run = lambda **kw: run_rope_kv_write(dev, rng, lengths, rows, 4, 2, dim, page, rot, kw.pop("interleaved", False), True, t, **kw)  # noqa: E731
    run(in_place=True)
    run(in_place=True, interleaved=True, positions=True, col=16, tail=24)
    run(queries=False)
    run(col=3, tail=2)
    run(in_place=True, col=1, interleaved=True)
    run(shift={"x": e, "q": e, "qw": e, "kw": e, "angles": 4})
    run(shift={"kw": e})
    run(shift={"angles": 4})
    run_rope_kv_write(dev, rng, lengths, rows, 4, 2, dim, page, 0, False, True, t)
    run_rope_kv_write(dev, rng, lengths, rows, 4, 2, dim, page, 0, False, False, t, in_place=True)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("batch", [1, 63, 64, 65, 130, 4097])
def test_rope_kv_write_many_sequences(batch, t, dev):
    """Each row's sequence among few and many, sequences without rows between."""
    rng = np.random.default_rng(batch)
    rows = [int(r) for r in rng.integers(0, 3, batch)]
    rows[-1] = 2
    lengths = [r + int(n) for r, n in zip(rows, rng.integers(0, 30, batch))]
    run_rope_kv_write(dev, rng, lengths, rows, 2, 1, 32, 16, 32, False, True, t, pad=3)


def test_rope_kv_write_token_by_token(dev):
    """Scales that grow while a page fills, one token after the other."""
    rng = np.random.default_rng(4)
    page, kv, dim, heads, steps = 16, 2, 64, 2, 20
    table, pages = tables(rng, [steps + 3] * 2, page)
    cache = s8.Cache(rng, pages, kv, page, dim, table, filled=False)
    starts = np.arange(3, dtype=I32)
    angles = turn_table(rng, 64, 64)
    d = dev({"x": np.zeros((2, (heads + 2 * kv) * dim), F16), **cache_arrays(cache, starts, [0, 0]), "angles": angles})
    for i in range(steps):
        x = (rng.standard_normal((2, heads + 2 * kv, dim)) * 1.3 ** i).astype(F16)
        lengths = [i + 1, i + 4]
        d.set("x", x.reshape(2, -1))
        d.set("lengths", np.array(lengths, I32))
        d.call("nnc_hip_rope_kv_write", "x", "x", "x", None, None, "angles", None, None, *CACHE, "starts", "lengths", 0, heads, heads * dim,
               (heads + kv) * dim, 0, 0.0)
        k, _ = dr.rope(x[:, heads:heads + kv], None, angles, np.array([i, i + 3]), False, 0.0)
        cache.write(k.astype(F32).astype(F16), x[:, heads + kv:], starts, lengths)
        check_cache(d, cache)


@pytest.mark.parametrize("shift", [0, 2])
def test_rope_kv_write_values_that_are_not_finite(shift, dev):
    """A NaN or an infinity among a page's keys makes that page's scale NaN, one
    among the values theirs; other heads and pages stay."""
    rng = np.random.default_rng(6)
    page, kv, dim = 16, 2, 64
    lengths, rows = [33, 20], [33, 20]
    starts, total = ragged(rows)
    table, pages = tables(rng, lengths, page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    x = rng.standard_normal((total, 3 * kv, dim)).astype(F16)
    x[3, kv, 5] = np.nan       # a key of page 0 of sequence 0, head 0
    x[20, 2 * kv + 1, 7] = np.inf  # a value of page 1, head 1
    x[40, kv + 1] = 0
    angles = turn_table(rng, 64, dim)
    w = np.ones(dim, F16)
    d = dev({"x": x.reshape(total, -1), **cache_arrays(cache, starts, lengths), "angles": angles, "w": w, "q": np.zeros((total, kv * dim), F16)}, {"x": shift})
    d.call("nnc_hip_rope_kv_write", "x", "x", "x", "w", "w", "angles", None, "q", *CACHE, "starts", "lengths", 0, kv, kv * dim, 2 * kv * dim, 0, 1e-6)
    place = np.concatenate([np.arange(33), np.arange(20)])
    with np.errstate(invalid="ignore"):
        k, _ = dr.rope(x[:, kv:2 * kv], w, angles, place, False, 1e-6)
        cache.write(k.astype(F32).astype(F16), x[:, 2 * kv:], starts, lengths)
    check_cache(d, cache)
    ks, vs = d.get("k_scale"), d.get("v_scale")
    assert np.isnan(ks[table[0, 0], 0]) and np.isnan(vs[table[0, 1], 1]) and np.isnan(ks).sum() == 1 and np.isnan(vs).sum() == 1


def test_rope_kv_write_with_bad_tables_and_lengths(dev):
    """Pages that are none, lengths that are too long or negative, starts out of
    order: nothing is touched that is not there."""
    rng = np.random.default_rng(7)
    page, kv, dim = 16, 1, 32
    cache = s8.Cache(rng, 5, kv, page, dim, np.array([[0, -1], [9, 1], [2, 3], [4, 4]], I32))
    starts = np.array([0, 20, 25, 30, 400], I32)
    x = rng.standard_normal((40, 3 * dim)).astype(F32)
    angles = turn_table(rng, 8, dim)
    for bad in ([20, 1000, 32, -5], [20, 5, 32, 0]):
        d = dev({"x": x, **cache_arrays(cache, starts, bad), "angles": angles, "q": np.full((40, dim), 7, F32)})
        d.call("nnc_hip_rope_kv_write", "x", "x", "x", None, None, "angles", None, "q", *CACHE, "starts", "lengths", 0, 1, dim, 2 * dim, 0, 0.0)
        clamped = [min(max(n, 0), 32) for n in bad]
        want = cache.copy()
        rows = x.reshape(40, 3, dim)
        place = np.concatenate([np.arange(n - r, n) for n, r in zip(clamped, (20, 5, 5, 10))])
        k, _ = dr.rope(rows[:, 1:2], None, angles, place, False, 0.0)
        want.write(k.astype(F32), rows[:, 2:], np.minimum(starts, 40), clamped)
        check_cache(d, want)
    d.set("starts", np.array([7, 3, -9, 2 ** 31 - 1, 0], I32))
    d.call("nnc_hip_rope_kv_write", "x", "x", "x", None, None, "angles", None, None, *CACHE, "starts", "lengths", 0, 1, dim, 2 * dim, 0, 0.0)
    for n in CACHE:
        d.get(n)  # nothing written outside


def test_rope_kv_write_without_pages(dev):
    """A table of no columns: nothing is cached, the queries are turned all the same."""
    rng = np.random.default_rng(12)
    starts, total = ragged([3, 4], 2)
    cache = s8.Cache(rng, 2, 1, 16, 64, np.zeros((2, 0), I32))
    x = rng.standard_normal((total, 4, 64)).astype(F16)
    angles = turn_table(rng, 40, 64)
    at = rng.integers(0, 40, total).astype(I32)
    d = dev({"x": x.reshape(total, -1), **cache_arrays(cache, starts, [0, 0]), "angles": angles, "at": at, "q": np.full((total, 128), 7, F16)})
    d.call("nnc_hip_rope_kv_write", "x", "x", "x", None, None, "angles", "at", "q", *CACHE, "starts", "lengths", 0, 2, 128, 192, 0, 0.0)
    want, _ = dr.rope(x[:7, :2], None, angles, at[:7], False, 0.0)
    got = d.get("q").reshape(total, 2, 64)
    np.testing.assert_array_equal(got[:7], want.astype(F32).astype(F16))
    assert (got[7:] == 7).all()
    check_cache(d, cache)


# ---------------------------------------------------------------------------
# attention of drafts
# ---------------------------------------------------------------------------

def run_tree(dev, rng, lengths, rows, heads, kv, dim, page, t, window=0, max_length=0, pad=2, sharp=2.0, width=None, garbage=True, spread=0, words=None,
             lines=None, q_col=3):
    starts, total = ragged(rows, pad)
    table, pages = tables(rng, lengths, page, width=width)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    lines = dr.trees(rng, rows) if lines is None else lines
    tree = dr.masks(lines, words or max(1, -(-max(rows) // 32)), total)
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
    qrows = (rng.standard_normal((total, heads * dim + 2 * q_col)) * sharp).astype(t)
    scale = dim ** -0.5
    d = dev({"q": qrows, **cache_arrays(cache, starts, lengths), "tree": tree, "out": np.full((total, heads * dim), 7, t)})
    d.call("nnc_hip_kv_tree_attention", "q", *CACHE, "starts", "lengths", "tree", "out", q_col, heads, scale, window, max_length)
    got = d.get("out")
    q = qrows[:, q_col:q_col + heads * dim].reshape(total, heads, dim)
    dr.check_tree(got, q, cache, starts, lengths, tree, F32(scale), window)
    owned = np.zeros(total, bool)
    owned[starts[0]:starts[-1]] = True
    assert (got[~owned] == 7).all()
    return got.reshape(total, heads, dim), d


TREE = [(1, 1, 32, 16), (4, 4, 64, 16), (8, 2, 128, 16), (6, 2, 64, 48), (7, 1, 128, 64), (4, 2, 256, 32), (20, 1, 64, 128), (40, 2, 32, 256),
        (64, 1, 128, 16), (2, 2, 256, 64)]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,page", TREE)
def test_tree_attention(heads, kv, dim, page, t, dev):
    """Trees behind contexts of any length and behind none, single drafts, none,
    more rows than positions; masks of several words; padding behind."""
    rng = np.random.default_rng(heads + dim + page)
    run_tree(dev, rng, [70, 9, 140, 40, 3, 0, 333, 65, 16], [12, 9, 33, 0, 5, 4, 1, 64, 1], heads, kv, dim, page, t)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (4, 4, 64, 64), (3, 1, 32, 16), (2, 1, 256, 48)])
@pytest.mark.parametrize("rows", [1, 2, 5, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 130])
def test_tree_attention_of_any_rows(rows, heads, kv, dim, page, t, dev):
    rng = np.random.default_rng(rows * heads)
    run_tree(dev, rng, [rows + 117], [rows], heads, kv, dim, page, t, pad=0, q_col=0 if rows % 2 else 4)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("first", [0, 1, 15, 16, 17, 31, 33, 47, 63, 64, 65, 127, 250])
def test_tree_attention_first_draft_anywhere(first, t, dev):
    """Where the context ends within 16 keys, 64, a page."""
    rng = np.random.default_rng(first)
    run_tree(dev, rng, [first + 20, first + 40], [20, 40], 4, 2, 64, 48, t)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 399, 400, 2 ** 30, 2 ** 31 - 1])
def test_tree_attention_window(window, t, dev):
    rng = np.random.default_rng(window % 1000)
    run_tree(dev, rng, [400, 30, 90, 0, 7], [20, 9, 40, 3, 9], 4, 2, 64, 32, t, window=window, garbage=False)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("max_length", [0, 20000])
def test_tree_attention_long_axis(max_length, t, dev):
    rng = np.random.default_rng(11)
    run_tree(dev, rng, [20000], [24], 4, 1, 64, 64, t, max_length=max_length)
    run_tree(dev, rng, [9000, 5, 300], [3, 2, 40], 8, 2, 128, 16, t, max_length=max_length and 9000)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("batch,kv,dim", [(70, 4, 64), (256, 2, 32), (300, 1, 128)])
def test_tree_attention_many_sequences(batch, kv, dim, t, dev):
    rng = np.random.default_rng(batch)
    lengths = [int(n) for n in rng.integers(0, 150, batch)]
    rows = [int(r) for r in rng.integers(0, 7, batch)]
    lengths[:4], rows[:4] = [900, 0, 1, 300], [9, 0, 1, 70]
    run_tree(dev, rng, lengths, rows, 2 * kv, kv, dim, 16, t)


def test_tree_attention_masks(dev):
    """Masks that see nothing, everything, only others, rows that there are not;
    more words than rows, fewer than rows need."""
    rng = np.random.default_rng(1)
    rows, lengths = [6, 40, 3], [6, 240, 3]
    lines = [[[], [0, 1, 2, 3, 4, 5], [5], [0, 2, 4], [], [5]], [list(range(40)) for _ in range(40)], [[0, 17, 31], [31], [1, 2]]]
    for words in (1, 2, 5):
        got, _ = run_tree(dev, rng, lengths, rows, 4, 2, 64, 16, F32, words=words, lines=lines)
        assert not got[0].any() and not got[4].any() and got[1].any() and not got[47].any()
    chain = [[list(range(i + 1)) for i in range(n)] for n in rows]
    got, d = run_tree(dev, rng, lengths, rows, 4, 2, 64, 16, F32, lines=chain, words=2, q_col=0)
    d.call("nnc_hip_kv_attention", "q", *CACHE, "starts", "lengths", "out", 0, 4, 0.125, 0, 0)
    want = d.get("out").reshape(got.shape)
    np.testing.assert_allclose(got[:49], want[:49], rtol=0, atol=2e-5)  # a chain is a run of tokens: values up to 127 * 0.02, both off by 1e-6 of them


@pytest.mark.parametrize("t", [F32, F16])
def test_tree_attention_pages_that_cannot_be_read(t, dev):
    rng = np.random.default_rng(2)
    lengths, rows = [200, 90], [20, 90]
    starts, total = ragged(rows)
    table, pages = tables(rng, lengths, 16)
    cache = s8.Cache(rng, pages, 2, 16, 64, table)
    cache.table[0, 3], cache.table[0, 11], cache.table[1, :5] = -1, pages, [2 ** 31 - 1, -2 ** 31, pages + 5, -1, -7]
    tree = dr.masks(dr.trees(rng, rows), 3, total)
    q = rng.standard_normal((total, 4 * 64)).astype(t)
    d = dev({"q": q, **cache_arrays(cache, starts, lengths), "tree": tree, "out": np.full((total, 256), 7, t)})
    d.call("nnc_hip_kv_tree_attention", "q", *CACHE, "starts", "lengths", "tree", "out", 0, 4, 0.125, 0, 0)
    dr.check_tree(d.get("out"), q.reshape(total, 4, 64), cache, starts, lengths, tree, F32(0.125), 0)
    # nothing to read at all
    d.set("table", np.full_like(cache.table, -1))
    d.call("nnc_hip_kv_tree_attention", "q", *CACHE, "starts", "lengths", "tree", "out", 0, 4, 0.125, 0, 0)
    assert not d.get("out")[:starts[-1]].any()
    # lengths and starts that cannot be
    for s, n in (([0, 20, 1000], [10 ** 9, -4]), ([0, -5, 7], [200, 90]), ([50, 20, 10], [3, 200])):
        d.set("starts", np.array(s, I32))
        d.set("lengths", np.array(n, I32))
        d.call("nnc_hip_kv_tree_attention", "q", *CACHE, "starts", "lengths", "tree", "out", 0, 4, 0.125, 0, 0)
        assert np.isfinite(d.get("out")).all()


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows", [4, 40])
def test_tree_attention_pages_of_different_size(rows, t, dev):
    """Scales of values far apart, pages of zeros, sharp and flat scores."""
    rng = np.random.default_rng(rows)
    run_tree(dev, rng, [700, 300], [rows, 3], 4, 1, 64, 16, t, garbage=False, spread=9 if t == F16 else 60)
    run_tree(dev, rng, [700, 300], [rows, 3], 4, 1, 64, 16, t, sharp=200.0)
    run_tree(dev, rng, [700, 300], [rows, 3], 4, 1, 64, 16, t, sharp=0.0)


def test_tree_attention_hidden_drafts_that_are_not_finite(dev):
    """Neighbours that a draft does not see do not reach it, whatever they hold."""
    rng = np.random.default_rng(3)
    lengths, rows = [80], [32]
    starts, total = ragged(rows)
    table, pages = tables(rng, lengths, 16)
    cache = s8.Cache(rng, pages, 1, 16, 64, table)
    cache.ks[table[0, 4]] = np.nan  # positions 64 .. 79: drafts 16 .. 31
    cache.vs[table[0, 4]] = np.nan
    lines = [[[i] if i >= 16 else list(range(i + 1)) for i in range(32)]]
    tree = dr.masks(lines, 1, total)
    q = rng.standard_normal((total, 64)).astype(F16)
    d = dev({"q": q, **cache_arrays(cache, starts, lengths), "tree": tree, "out": np.zeros((total, 64), F16)})
    d.call("nnc_hip_kv_tree_attention", "q", *CACHE, "starts", "lengths", "tree", "out", 0, 1, 0.125, 0, 0)
    got = d.get("out")
    assert np.isfinite(got[:16]).all() and np.isnan(got[16:32]).all()


# Many rows for a cached head behind contexts that are cut, some with few in
# their last tile; tables that could hold more than the kernel for 256 rows asks
# for
MANY = [([1500, 1200, 4000, 3000, 2047, 40], [16, 1, 40, 0, 3, 9]), ([1500, 1200, 4000, 64, 2047, 70], [130, 64, 70, 65, 33, 5]),
        ([1700, 1, 4000, 2048, 1025, 260], [300, 1, 64, 0, 2, 257])]


def wide(batch, kv, page):
    return 1 + 24 * 256 * 64 // (batch * kv * page)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (4, 1, 64, 64), (16, 1, 32, 48), (6, 2, 128, 256)])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_tree_attention_many_rows_of_long_contexts(which, heads, kv, dim, page, t, dev):
    rng = np.random.default_rng(dim + which)
    lengths, rows = MANY[which]
    run_tree(dev, rng, lengths, rows, heads, kv, dim, page, t, q_col=4 if which == 1 else 3, width=wide(6, kv, page))


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows", [9, 16, 17, 31, 32, 33, 63, 64, 65, 130])
def test_tree_attention_many_rows_of_one_long_context(rows, t, dev):
    rng = np.random.default_rng(rows)
    run_tree(dev, rng, [9000 + rows], [rows], 4, 1, 128, 64, t, pad=0, width=wide(1, 1, 64))
    run_tree(dev, rng, [1025], [rows], 8, 2, 64, 16, t, pad=3, width=wide(1, 2, 16), max_length=1030 if rows % 2 else 0)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("window", [1, 64, 700, 1500, 3999])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_tree_attention_many_rows_window(which, window, t, dev):
    rng = np.random.default_rng(window + which)
    run_tree(dev, rng, *MANY[which], 4, 1, 64, 32, t, window=window, garbage=False, width=wide(6, 1, 32))


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("batch,most", [(70, 30), (70, 200), (140, 160)])
def test_tree_attention_many_rows_of_many_sequences(batch, most, t, dev):
    rng = np.random.default_rng(batch)
    lengths = [int(n) for n in rng.integers(0, 1800, batch)]
    rows = [int(r) for r in rng.integers(0, most, batch)]
    lengths[:4], rows[:4] = [2500, 0, 1, 300], [9, 0, 1, 200]
    run_tree(dev, rng, lengths, rows, 4, 2, 32, 16, t, width=wide(batch, 2, 16) + 200)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows", [40, 100, 300])
def test_tree_attention_many_rows_pages_of_different_size(rows, t, dev):
    rng = np.random.default_rng(rows)
    lengths, all_rows = [2700, 1300], [rows, 30]
    width = wide(2, 1, 16)
    run_tree(dev, rng, lengths, all_rows, 2, 1, 64, 16, t, garbage=False, spread=9 if t == F16 else 60, width=width)
    run_tree(dev, rng, lengths, all_rows, 2, 1, 64, 16, t, sharp=200.0, width=width)
    run_tree(dev, rng, lengths, all_rows, 2, 1, 64, 16, t, sharp=0.0, width=width)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows", [[40, 20], [100, 90], [300, 90]])
def test_tree_attention_many_rows_that_see_little(rows, t, dev):
    """Masks of nothing, pages that cannot be read, drafts that are not finite
    and that the others do not see, lengths and starts that cannot be."""
    rng = np.random.default_rng(4)
    lengths, kv, dim = [3000, 1290], 1, 64
    starts, total = ragged(rows)
    table, pages = tables(rng, lengths, 16, width=wide(2, kv, 16))
    cache = s8.Cache(rng, pages, kv, 16, dim, table)
    cache.table[0, 3], cache.table[0, 111], cache.table[1, :35] = -1, pages, [2 ** 31 - 1, -2 ** 31, pages + 5, -1, -7] * 7
    lines = dr.trees(rng, rows)
    lines[0][7] = []
    tree = dr.masks(lines, -(-max(rows) // 32), total)
    q = rng.standard_normal((total, 2 * dim)).astype(t)
    d = dev({"q": q, **cache_arrays(cache, starts, lengths), "tree": tree, "out": np.full((total, 2 * dim), 7, t)})

    def run():
        d.call("nnc_hip_kv_tree_attention", "q", *CACHE, "starts", "lengths", "tree", "out", 0, 2, 0.125, 0, 0)
        return d.get("out")
    want = run()
    dr.check_tree(want, q.reshape(total, 2, dim), cache, starts, lengths, tree, F32(0.125), 0)
    d.set("table", np.full_like(cache.table, -1))
    assert not run()[:starts[-1]].any()
    for s, n in (([0, 20, 1000], [10 ** 9, -4]), ([0, -5, 7], [200, 90]), ([50, 20, 10], [3, 3000]), ([0, 10 ** 9, 5], [3000, 3000]), ([0, 30, 2 ** 31 - 1], [3000, 1290])):
        d.set("starts", np.array(s, I32))
        d.set("lengths", np.array(n, I32))
        assert np.isfinite(run()).all()
    # the last 8 drafts, those of the last page, are not finite, and the others do not see them
    cache.table[0, 3], cache.table[0, 111] = table[0, 3], table[0, 111]
    last = cache.page_of(0, 2999)
    cache.ks[last], cache.vs[last] = np.nan, np.nan
    d.set("starts", starts), d.set("lengths", np.array(lengths, I32)), d.set("table", cache.table)
    d.set("k_scale", cache.ks), d.set("v_scale", cache.vs)
    alone = [[[j for j in line if j < n - 9] if i < n - 9 else line for i, line in enumerate(own)] for own, n in zip(lines, rows)]
    d.set("tree", dr.masks(alone, -(-max(rows) // 32), total))
    got = run()
    assert np.isfinite(got[:rows[0] - 9]).all() and np.isnan(got[rows[0] - 1]).all()


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------

def run_logprobs(dev, x, top=5, scale=1.0, tokens=None, shift=None, what=("logprob", "entropy", "top"), rng=None):
    rows, vocab = x.shape
    rng = rng or np.random.default_rng(rows)
    tokens = rng.integers(0, vocab, rows).astype(I32) if tokens is None else tokens
    arrays = {"x": x, "tokens": tokens, "logprob": np.full(rows, 7, F32), "entropy": np.full(rows, 7, F32)}
    if top:
        arrays.update(index=np.full((rows, top), 7, I32), values=np.full((rows, top), 7, F32))
    d = dev(arrays, shift)
    lp, h = "logprob" in what, "entropy" in what
    best = top and "top" in what
    d.call("nnc_hip_token_logprobs", "x", "tokens" if lp else None, "logprob" if lp else None, "entropy" if h else None, "index" if best else None,
           "values" if best else None, scale)
    p, entropy, off, off_h = dr.logprobs(x, scale)
    ok = np.isfinite(entropy)

    def near(got, want, off):
        got, fine = got.astype(np.float64), np.isfinite(want)
        np.testing.assert_array_equal(got[~fine], want[~fine])
        bad = ~(np.abs(got[fine] - want[fine]) <= off[fine] + U32 * 1.001 * np.abs(want[fine]))
        assert not bad.any(), (got[fine][bad][:4], want[fine][bad][:4], off[fine][bad][:4])
    if lp:
        inside = (tokens >= 0) & (tokens < vocab)
        want = np.where(inside, p[np.arange(rows), np.clip(tokens, 0, vocab - 1)], np.nan)
        near(d.get("logprob"), want, off)
    else:
        assert (d.get("logprob") == 7).all()
    if h:
        near(d.get("entropy"), entropy, off_h)
    else:
        assert (d.get("entropy") == 7).all()
    if best:
        n = min(top, vocab)
        order = dr.ranking(np.where(ok[:, None], x, 0), n)
        index, values = d.get("index"), d.get("values")
        np.testing.assert_array_equal(index[ok][:, :n], order[ok])
        assert (index[ok][:, n:] == -1).all() and (index[~ok] == -1).all()
        assert np.isnan(values[~ok]).all() and (values[ok][:, n:] == -np.inf).all()
        near(values[:, :n], np.where(ok[:, None], np.take_along_axis(p, order, 1), np.nan), np.repeat(off[:, None], n, 1))
    return d


def logits(rng, rows, vocab, t):
    x = rng.standard_normal((rows, vocab)) * 2.2
    for i in range(rows):
        x[i, rng.integers(0, vocab, min(vocab, 6))] += rng.uniform(0, 16)
    return x.astype(t)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 64), (4, 65), (3, 255), (2, 1000), (7, 4099), (3, 8192), (1, 32000), (5, 50257), (2, 128256),
                                        (300, 513), (1200, 96), (40, 20000), (1, 262147)])
def test_token_logprobs(rows, vocab, t, dev):
    rng = np.random.default_rng(rows + vocab)
    x = logits(rng, rows, vocab, t)
    for top in (0, 1, 5, 20, 64):
        run_logprobs(dev, x, top, rng=rng)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("vocab", [130, 3001, 40000])
def test_token_logprobs_ties(vocab, t, dev):
    """Equal values: the earlier token first, whether a few are equal or all."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(-3, 4, (6, vocab)).astype(t)
    x[1] = 2
    x[2] = 0
    x[2, ::2] = -0.0
    x[3] = np.arange(vocab) // 50 % 60
    x[4] = -np.inf
    x[4, vocab // 2] = 1
    x[5] = np.sort(x[5])
    for top in (3, 64):
        run_logprobs(dev, x, top)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_token_logprobs_rising_and_falling(vocab, t, dev):
    """The likeliest at the end, at the start, side by side."""
    x = np.zeros((5, vocab), t)
    x[0] = np.linspace(-5, 5, vocab)
    x[1] = np.linspace(5, -5, vocab)
    x[2, vocab // 3:vocab // 3 + 64] = np.linspace(1, 9, 64)[:max(0, min(64, vocab - vocab // 3))]
    x[3, ::64] = 3
    x[4, 5::16] = 4
    run_logprobs(dev, x, 64)
    run_logprobs(dev, x, 20)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("vocab", [50, 2000, 40001])
def test_token_logprobs_rows_that_are_not_finite(vocab, t, dev):
    rng = np.random.default_rng(vocab)
    x = logits(rng, 9, vocab, t)
    x[1] = -np.inf
    x[2, vocab - 1] = np.inf
    x[3, vocab // 2] = np.nan
    x[4, 1:] = -np.inf
    x[5, ::2] = -np.inf
    x[6] = np.finfo(t).min
    x[6, 3] = 0
    x[7] = np.finfo(t).max
    x[8, : vocab // 2] = np.finfo(t).min
    tokens = np.array([0, 1, 2, 3, 0, 0, 3, vocab - 1, 1], I32)
    run_logprobs(dev, x, 10, tokens=tokens)
    tokens = np.array([-1, 1, 2, 3, 1, 1, 0, vocab, 2 ** 31 - 1], I32)
    run_logprobs(dev, x, 64, tokens=tokens)


@pytest.mark.parametrize("t", [F32, F16])
def test_token_logprobs_parts_alignment_and_scale(t, dev):
    rng = np.random.default_rng(5)
    x = logits(rng, 6, 3000, t)
    e = x.dtype.itemsize
    for what in (("logprob",), ("entropy",), ("top",), ("logprob", "top"), ("entropy", "top"), ("logprob", "entropy")):
        run_logprobs(dev, x, 4, what=what)
    run_logprobs(dev, x, 4, shift={"x": e, "tokens": 4, "logprob": 4, "entropy": 4, "index": 4, "values": 4})
    run_logprobs(dev, x, 4, shift={"x": 8})
    for scale in (0.25, 1.7, 20.0, 1e-3):
        run_logprobs(dev, x, 4, scale=scale)


def test_token_logprobs_of_certain_rows(dev):
    """One token far above the rest: what is left of the others is what its log
    probability and the entropy are made of."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((6, 5000)).astype(F32)
    x[np.arange(6), 77] = [12, 18, 25, 30, 60, 200]
    d = run_logprobs(dev, x, 3, tokens=np.full(6, 77, I32))
    assert (d.get("logprob")[:4] < 0).all() and (d.get("entropy")[:4] > 0).all()


def test_token_logprobs_behind_four_gib(hip, abi, dev):
    """Rows at the far end of logits of more than 4 GiB."""
    from nnc_py_amd import runtime
    rows, vocab = 17000, 128256
    assert rows * vocab * 2 > 2 ** 32
    rng = np.random.default_rng(1)
    big = runtime.DeviceBuffer.empty((rows, vocab), F16)
    try:
        some = [0, 1, 8000, rows - 2, rows - 1]
        x = logits(rng, len(some), vocab, F16)
        for i, r in enumerate(some):
            runtime.check(hip.nnc_hip_memcpy_h2d(big.ptr + r * vocab * 2, np.ascontiguousarray(x[i]).ctypes.data, vocab * 2), "upload")
        d = dev({"tokens": np.full(rows, 9, I32), "lp": np.zeros(rows, F32), "h": np.zeros(rows, F32), "i": np.zeros((rows, 4), I32), "v": np.zeros((rows, 4), F32)})
        d.desc["x"], shape = big.tensor()
        d.kept.append(shape)
        d.call("nnc_hip_token_logprobs", "x", "tokens", "lp", "h", "i", "v", 1.0)
        p, h, off, off_h = dr.logprobs(x, 1.0)
        assert (np.abs(d.get("h")[some] - h) <= off_h + 2 * U32 * h).all()
        assert (np.abs(d.get("lp")[some] - p[:, 9]) <= off + 2 * U32 * np.abs(p[:, 9])).all()
        np.testing.assert_array_equal(d.get("i")[some], dr.ranking(x, 4))
    finally:
        big.free()


# ---------------------------------------------------------------------------
# as they are used
# ---------------------------------------------------------------------------

def step_setup(rng, t, batch=3, steps=4, drafts=5):
    page, kv, dim, heads, vocab = 16, 2, 64, 4, 777
    context = [30, 1, 15][:batch]
    table, pages = tables(rng, [n + drafts * steps for n in context], page)
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    x = rng.standard_normal((steps, batch * drafts, (heads + 2 * kv) * dim)).astype(t)
    head = rng.integers(-127, 128, (vocab, heads * dim)).astype(np.int8)
    return page, kv, dim, heads, vocab, context, cache, x, head


def test_captured_draft_step_replayed(dev, hip):
    """Rotation into the cache, attention of a tree, product and log
    probabilities captured once and replayed for every set of drafts, rows,
    masks, positions and lengths changing between the replays, with a
    synchronisation and eager calls in between."""
    from nnc_py_amd import runtime
    rng = np.random.default_rng(12)
    page, kv, dim, heads, vocab, context, cache, x, head = step_setup(rng, F16)
    steps, total, _ = x.shape
    drafts = total // 3
    starts = np.arange(4, dtype=I32) * drafts
    angles = turn_table(rng, 100, dim)
    w = (1 + 0.1 * rng.standard_normal(dim)).astype(F16)
    d = dev({"x": x[0], **cache_arrays(cache, starts, context), "q": np.zeros((total, heads * dim), F16), "out": np.zeros((total, heads * dim), F16),
             "angles": angles, "at": np.zeros(total, I32), "w": w, "tree": np.zeros((total, 1), I32), "a8": np.zeros((total, heads * dim), np.int8),
             "as": np.zeros(total, F32), "head": head, "hs": np.full(vocab, 0.002, F32), "logits": np.zeros((total, vocab), F16),
             "tokens": np.arange(total, dtype=I32), "lp": np.zeros(total, F32), "h": np.zeros(total, F32), "i": np.zeros((total, 3), I32),
             "v": np.zeros((total, 3), F32)})
    T = lambda *names: [d.t(n) for n in names]  # noqa: E731

    def calls():
        hip.nnc_hip_rope_kv_write(*T("x", "x", "x", "w", "w", "angles", "at", "q", *CACHE, "starts", "lengths"), 0, heads, heads * dim, (heads + kv) * dim, 0, 1e-6)
        hip.nnc_hip_kv_tree_attention(*T("q", *CACHE, "starts", "lengths", "tree", "out"), 0, heads, 0.125, 0, 0)
        hip.nnc_hip_quantize_rows(*T("out", "a8", "as"))
        hip.nnc_hip_matmul_i8(*T("a8", "as", "head", "hs", None, "logits"))
        hip.nnc_hip_token_logprobs(*T("logits", "tokens", "lp", "h", "i", "v"), 1.0)
    runtime.check(hip.nnc_hip_graph_begin(), "begin")
    calls()
    runtime.check(hip.nnc_hip_graph_end(), "end")
    names = ("q", "out", "lp", "h", "i", "v") + CACHE[:4]
    for i in range(steps):
        lengths = [n + drafts * (i + 1) for n in context]
        lines = dr.trees(rng, [drafts] * 3)
        at = np.array([n - drafts + len(line) - 1 for n, seq in zip(lengths, lines) for line in seq], I32)
        tree = dr.masks(lines, 1)
        for name, a in (("x", x[i]), ("lengths", np.array(lengths, I32)), ("at", at), ("tree", tree)):
            d.set(name, a)
        runtime.check(hip.nnc_hip_graph_launch(), "launch")
        runtime.sync()
        rows = x[i].reshape(total, heads + 2 * kv, dim)
        k, _ = dr.rope(rows[:, heads:heads + kv], w, angles, at, False, 1e-6)
        cache.write(k.astype(F32).astype(F16), rows[:, heads + kv:], starts, lengths)
        check_cache(d, cache)
        got = {n: d.get(n) for n in names}
        dr.check_tree(got["out"], got["q"].reshape(total, heads, dim), cache, starts, lengths, tree, F32(0.125), 0)
        p, h, off, off_h = dr.logprobs(d.get("logits"), 1.0)
        assert (np.abs(got["h"] - h) <= off_h + 2 * U32 * h).all()
        np.testing.assert_array_equal(got["i"], dr.ranking(d.get("logits"), 3))
        calls()  # again, outside the graph: the rows are in the cache already
        runtime.sync()
        for n in names:
            np.testing.assert_array_equal(d.get(n), got[n])
    hip.nnc_hip_graph_destroy()


def test_two_threads_and_the_second_stream(dev, hip):
    """Every call from two host threads at once and on the side stream: each has
    its own scratch."""
    from nnc_py_amd import runtime
    rng = np.random.default_rng(13)
    jobs = []
    for n, rows in ((4000, 9), (2500, 17)):
        table, pages = tables(rng, [n], 16)
        cache = s8.Cache(rng, pages, 2, 16, 64, table)
        q = rng.standard_normal((rows, 8 * 64)).astype(F32)
        lines = dr.trees(rng, [rows])
        d = dev({"q": q, **cache_arrays(cache, np.array([0, rows], I32), [n]), "tree": dr.masks(lines, 1), "out": np.zeros((rows, 256), F32),
                 "angles": turn_table(rng, n, 64), "x": logits(rng, 3, 40000, F32), "h": np.zeros(3, F32), "i": np.zeros((3, 20), I32),
                 "v": np.zeros((3, 20), F32), "turned": np.zeros((rows, 256), F32)})
        jobs.append((d, rows))
    names = ("out", "turned", "h", "i", "v") + CACHE[:4]

    def run(d, times):
        T = lambda *a: [d.t(n) for n in a]  # noqa: E731
        for _ in range(times):
            hip.nnc_hip_rope_kv_write(*T("q", "q", "q", None, None, "angles", None, "turned", *CACHE, "starts", "lengths"), 0, 4, 256, 384, 1, 0.0)
            hip.nnc_hip_kv_tree_attention(*T("turned", *CACHE, "starts", "lengths", "tree", "out"), 0, 4, 0.125, 0, 0)
            hip.nnc_hip_token_logprobs(*T("x", None, None, "h", "i", "v"), 1.0)
        runtime.sync()
    for d, _ in jobs:
        run(d, 1)
    first = [{n: d.get(n) for n in names} for d, _ in jobs]
    threads = [threading.Thread(target=run, args=(d, 20)) for d, _ in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()

    def same():
        for (d, _), want in zip(jobs, first):
            for n in names:
                np.testing.assert_array_equal(d.get(n), want[n])
    same()
    runtime.check(hip.nnc_hip_stream_fork(), "fork")
    runtime.check(hip.nnc_hip_stream_select(1), "select")
    run(jobs[0][0], 1)
    runtime.check(hip.nnc_hip_stream_select(0), "select")
    run(jobs[1][0], 1)
    runtime.check(hip.nnc_hip_stream_join(), "join")
    runtime.sync()
    same()
    assert runtime.last_error()[0] == 0


def test_many_rows_captured_and_replayed(dev, hip):
    """The kernel for 256 rows in a graph: lengths, trees and queries change
    between the replays, an eager call of another shape uses the same scratch."""
    from nnc_py_amd import runtime
    rng = np.random.default_rng(21)
    heads, kv, dim, page, rows = 8, 2, 64, 32, [90, 70]
    starts, total = ragged(rows)
    table, pages = tables(rng, [2600, 2000], page, width=wide(2, kv, page))
    cache = s8.Cache(rng, pages, kv, page, dim, table)
    d = dev({"q": np.zeros((total, heads * dim), F16), **cache_arrays(cache, starts, [0, 0]), "tree": np.zeros((total, 3), I32),
             "out": np.zeros((total, heads * dim), F16), "other": np.zeros((total, heads * dim), F16)})
    T = lambda *names: [d.t(n) for n in names]  # noqa: E731

    def call(out, longest=0):
        hip.nnc_hip_kv_tree_attention(*T("q", *CACHE, "starts", "lengths", "tree", out), 0, heads, 0.125, 0, longest)
    call("out")
    runtime.sync()
    runtime.check(hip.nnc_hip_graph_begin(), "begin")
    call("out")
    runtime.check(hip.nnc_hip_graph_end(), "end")
    for lengths in ([2600, 2000], [90, 1999], [0, 71], [1500, 1300], [1500, 1300]):
        q = rng.standard_normal((total, heads * dim)).astype(F16)
        tree = dr.masks(dr.trees(rng, rows), 3, total)
        for name, a in (("q", q), ("tree", tree), ("lengths", np.array(lengths, I32))):
            d.set(name, a)
        call("other", 2600)  # by the other kernel
        runtime.check(hip.nnc_hip_graph_launch(), "launch")
        runtime.sync()
        got, other = d.get("out"), d.get("other")
        for x in got, other:
            dr.check_tree(x, q.reshape(total, heads, dim), cache, starts, lengths, tree, F32(0.125), 0)
        call("out")
        runtime.sync()
        np.testing.assert_array_equal(d.get("out"), got)
    hip.nnc_hip_graph_destroy()


@pytest.mark.parametrize("dim", [64, 18])
def test_rope_behind_four_gib(dim, hip, dev):
    """Rows at the far end of a matrix of more than 4 GiB, in place."""
    from nnc_py_amd import runtime
    rows, ld, heads, col = 1100000, 2048, 2, 1800
    assert rows * ld * 2 > 2 ** 32
    rng = np.random.default_rng(dim)
    big = runtime.DeviceBuffer.empty((rows, ld), F16)
    try:
        some = [0, 5, rows // 2, rows - 2, rows - 1]
        x = rng.standard_normal((len(some), ld)).astype(F16)
        for i, r in enumerate(some):
            runtime.check(hip.nnc_hip_memcpy_h2d(big.ptr + r * ld * 2, np.ascontiguousarray(x[i]).ctypes.data, ld * 2), "upload")
        at = rng.integers(0, 99, rows).astype(I32)
        angles = turn_table(rng, 99, dim)
        d = dev({"at": at, "angles": angles})
        d.desc["x"], shape = big.tensor()
        d.kept.append(shape)
        d.call("nnc_hip_rope", "x", None, "angles", "at", "x", col, col, heads, dim, 1, 0.0)
        want = x.copy()
        y, _ = dr.rope(x[:, col:col + heads * dim].reshape(-1, heads, dim), None, angles, at[some], True, 0.0)
        want[:, col:col + heads * dim] = y.astype(F32).astype(F16).reshape(len(some), -1)
        for i, r in enumerate(some):
            got = np.empty(ld, F16)
            runtime.check(hip.nnc_hip_memcpy_d2h(got.ctypes.data, big.ptr + r * ld * 2, ld * 2), "download")
            np.testing.assert_array_equal(got, want[i])
    finally:
        big.free()


def test_cache_behind_four_gib(hip, dev):
    """Pages at the far end of caches of more than 4 GiB each: written, and
    attended by few rows and by many."""
    from nnc_py_amd import runtime
    rng = np.random.default_rng(5)
    page, kv, dim, heads, pages = 128, 4, 128, 8, 70000
    assert pages * kv * page * dim > 2 ** 32
    lengths, rows = [300, 700], [40, 150]
    starts, total = ragged(rows)
    table, held = tables(rng, lengths, page)
    cache = s8.Cache(rng, held, kv, page, dim, table)
    far = pages - held
    scales = np.zeros((2, pages, kv), F32)
    scales[0, far:], scales[1, far:] = cache.ks, cache.vs
    big = [runtime.DeviceBuffer.empty((pages, kv, page, dim), np.int8), runtime.DeviceBuffer.empty((pages, kv, dim, page), np.int8)]
    try:
        bytes_of = page * kv * dim
        for buf, a in zip(big, (cache.k, cache.v)):
            runtime.check(hip.nnc_hip_memcpy_h2d(buf.ptr + far * bytes_of, np.ascontiguousarray(a).ctypes.data, a.nbytes), "upload")
        x = rng.standard_normal((total, heads + 2 * kv, dim)).astype(F16)
        angles = turn_table(rng, 900, dim)
        tree = dr.masks(dr.trees(rng, rows), 5, total)
        wide_table = np.full((2, wide(2, kv, page)), -1, I32)
        wide_table[:, :table.shape[1]] = np.where(table < held, table + far, -1)
        d = dev({"x": x.reshape(total, -1), "k_scale": scales[0], "v_scale": scales[1], "table": wide_table, "starts": starts, "lengths": np.array(lengths, I32),
                 "angles": angles, "q": np.zeros((total, heads * dim), F16), "tree": tree, "out": np.zeros((total, heads * dim), F16)})
        for name, buf in zip(("k_cache", "v_cache"), big):
            d.desc[name], shape = buf.tensor()
            d.kept.append(shape)
        d.call("nnc_hip_rope_kv_write", "x", "x", "x", None, None, "angles", None, "q", *CACHE, "starts", "lengths", 0, heads, heads * dim, (heads + kv) * dim, 0, 0.0)
        place = np.concatenate([np.arange(n - r, n) for n, r in zip(lengths, rows)])
        own = slice(starts[0], starts[-1])
        k, _ = dr.rope(x[own, heads:heads + kv], None, angles, place, False, 0.0)
        keys = np.zeros((total, kv, dim), F16)
        keys[own] = k.astype(F32).astype(F16)
        cache.write(keys, x[:, heads + kv:], starts, lengths)
        for buf, a in zip(big, (cache.k, cache.v)):
            got = np.empty_like(a)
            runtime.check(hip.nnc_hip_memcpy_d2h(got.ctypes.data, buf.ptr + far * bytes_of, a.nbytes), "download")
            np.testing.assert_array_equal(got, a)
        np.testing.assert_array_equal(d.get("k_scale")[far:], cache.ks)
        q = d.get("q").reshape(total, heads, dim)
        for longest in (0, 700):  # by the kernel for 256 rows, and by the other
            d.call("nnc_hip_kv_tree_attention", "q", *CACHE, "starts", "lengths", "tree", "out", 0, heads, 0.09, 0, longest)
            dr.check_tree(d.get("out"), q, cache, starts, lengths, tree, F32(0.09), 0)
    finally:
        for buf in big:
            buf.free()


def test_token_logprobs_of_many_rows_and_of_one_long(dev):
    """More rows than one launch takes; a row of several hundred segments."""
    rng = np.random.default_rng(8)
    run_logprobs(dev, rng.standard_normal(((1 << 22) + 3, 3)).astype(F16), top=1, rng=rng)
    run_logprobs(dev, logits(rng, 1, 3000017, F32), top=64, rng=rng)
