"""nnc_hip_token_logprobs held to the roundings that its kernel makes, no more:
bounds for rows that one workgroup has and for rows that several share."""

from __future__ import annotations

import re

import numpy as np
import pytest

import drafting as dr
from serving8 import F16, F32, I32
from test_drafting import logits
from test_serving8 import dev  # noqa: F401 (fixture)

U = 2.0 ** -24  # float32's half step
LOG2E = F32(1.4426950408889634)
LN2 = np.log(2.0)


def joins(vocab, t):
    """The most times that a term is scaled where segments of a row are joined:
    the smallest segment is 1024 packs of 16 bytes, a lane takes every 64th and
    six steps join the lanes. None for a row of one segment."""
    segments = -(-(vocab * np.dtype(t).itemsize // 16 + 2) // 1024)
    return 0 if segments == 1 else 6 + -(-segments // 64) - 1


def bounds(x, scale, count):
    """log p and entropies in float64, and how far each row's may be off before
    they are rounded to float32.

    A term is 2^t, t = c (x - m) and c = scale * log2 e in float32: log2 e is
    rounded (0.23 U) and so is the product (U). t is one rounding of c x - (c m),
    U of it, or of x - m and of its product with c, 2 U, where c m is 4096 and
    more; so t and with it the natural exponent d is off by 2.23 U |d|, or 3.23 U
    |d|. What c m is rounded by is put back to within its square, 0.25 U. The
    exponential is good to its last place, 2 U. Two packs are 16 values in
    float16 and 8 in float32, added in four sums of up to four and these two by
    two: 5 roundings; from there on sums are float64. A term t 2^t is one more
    product, and t's own error. Each join multiplies by an exponential (2 U)
    whose own argument is a difference times c, 3.23 U of it. Terms below 2^-126
    are 0. The largest is counted."""
    x = x.astype(np.float64)
    top = x.max(1, keepdims=True)
    d = np.float64(F32(scale)) * (x - top)
    e = np.exp(d)
    total = e.sum(1)
    rest = np.where(d == 0, 0, e) if not count else e
    far = np.abs(top) * float(F32(scale) * LOG2E) >= 4095
    slope = np.where(far | (count > 0), 3.23, 2.23) * U
    with np.errstate(invalid="ignore"):
        size = np.where(e > 0, np.abs(d), 0)
    term = (2 + 5 + 0.25 + 2 * count) * U + slope * size
    small = x.shape[1] * 2.0 ** -126 + 2.0 ** -45
    off = (term * rest).sum(1) / total * (1 + 2.0 ** -18) + small
    mean = (size * e).sum(1) / total
    off_h = ((term + slope + U) * size * rest).sum(1) / total * (1 + 2.0 ** -18) + off * (1 + mean) + small
    return d - np.log(total)[:, None], np.log(total) + mean, off, off_h


def rows_of(rng, vocab, t):
    """Spread logits, flat ones (all terms near 1, where only the sums' roundings
    count), steps of equal values, one token above the rest."""
    x = np.concatenate([logits(rng, 3, vocab, t).astype(np.float64), rng.uniform(-0.05, 0, (2, vocab)), rng.integers(-4, 1, (1, vocab)) / 4.0,
                        rng.standard_normal((1, vocab))])
    x[-1, rng.integers(0, vocab)] += 14
    return x.astype(t)


ONE = {F32: [1, 2, 9, 64, 513, 1000, 2047, 4080], F16: [1, 3, 16, 130, 1025, 4099, 8170]}  # rows of one segment
MANY = [20000, 32000, 50257, 128256, 262147]


def run(dev, x, scale):
    rows, vocab = x.shape
    tokens = np.random.default_rng(rows).integers(0, vocab, rows).astype(I32)
    n = min(8, vocab)
    d = dev({"x": x, "tokens": tokens, "lp": np.zeros(rows, F32), "h": np.zeros(rows, F32), "i": np.zeros((rows, n), I32), "v": np.zeros((rows, n), F32)})
    p, h, off, off_h = bounds(x, scale, joins(vocab, x.dtype))
    for top in (True, False):
        d.call("nnc_hip_token_logprobs", "x", "tokens", "lp", "h", "i" if top else None, "v" if top else None, scale)
        for got, want, by in [(d.get("lp"), p[np.arange(rows), tokens], off), (d.get("h"), h, off_h)] + (
                [(d.get("v"), np.take_along_axis(p, dr.ranking(x, n), 1), off[:, None])] if top else []):
            bound = by + U * 1.001 * np.abs(want)
            assert (np.abs(got.astype(np.float64) - want) <= bound).all(), np.max(np.abs(got - want) / bound)


@pytest.mark.gpu
@pytest.mark.parametrize("t,vocab", [(t, n) for t in (F32, F16) for n in ONE[t] + MANY])
def test_roundings_of_a_row(t, vocab, dev):  # noqa: F811
    rng = np.random.default_rng(vocab)
    for scale in (1.0, 0.7, 30.0):
        run(dev, rows_of(rng, vocab, t), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("t,vocab", [(F32, 3000), (F16, 6000), (F16, 50257)])
def test_roundings_of_logits_far_from_zero(t, vocab, dev):  # noqa: F811
    """A largest logit whose exponent is 4096 and more, and just below it."""
    rng = np.random.default_rng(vocab)
    x = rows_of(rng, vocab, t).astype(np.float64)
    for shift in (2800.0, 2900.0, -20000.0):
        run(dev, (x + shift).astype(t), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, F16])
def test_roundings_of_many_short_rows(t, dev):  # noqa: F811
    """A wave to a row."""
    rng = np.random.default_rng(7)
    for rows, vocab in ((1500, 100), (600, 1017), (600, 1900)):
        run(dev, (rng.uniform(-0.05, 0, (rows, vocab)) * rng.choice([1.0, 100.0], (rows, 1))).astype(t), 1.0)


# on the host: what the bound lets pass

def kernel_like(x, scale, off_by=0.0):
    """A row of one segment as the kernel computes it; off_by: planted, relative,
    in every term."""
    x = x.astype(F32)
    c = F32(F32(scale) * LOG2E)
    m = x.max()
    shift = F32(m * c)
    lost = float(m) * float(c) - float(shift)
    t = (x.astype(np.float64) * float(c) - float(shift)).astype(F32)
    e = (np.exp2(t.astype(np.float64)) * (1 + off_by)).astype(F32)
    one = x == m
    e, w = np.where(one, F32(0), e), np.where(one, F32(0), (e * np.maximum(t, F32(-1000))).astype(F32))

    def sums(v):
        v = np.concatenate([v, np.zeros(-len(v) % 16, F32)]).reshape(-1, 4, 4)
        four = v[:, 0]
        for i in range(1, 4):
            four = four + v[:, i]
        return ((four[:, 0] + four[:, 1]) + (four[:, 2] + four[:, 3])).astype(np.float64).sum()
    a = 1 - LN2 * lost
    rest, weighted = sums(e), sums(w)
    weighted, rest = a * (weighted - lost * rest), a * rest
    total = rest + one.sum()
    return np.log(total), np.log(total) - weighted / total * LN2


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("vocab", [9, 1000, 4000])
def test_the_bound_holds_for_the_roundings_and_not_for_more(vocab, t):
    rng = np.random.default_rng(vocab)
    for scale in (1.0, 0.7, 30.0):
        x = rows_of(rng, vocab, t)
        p, h, off, off_h = bounds(x, scale, 0)
        for i, row in enumerate(x):
            log_sum, entropy = kernel_like(row, scale)
            assert abs(-log_sum - p[i].max()) <= off[i] and abs(entropy - h[i]) <= off_h[i]
    # flat rows whose terms are all off by 2^-20
    x = rng.uniform(-0.05, 0, (2, 4000)).astype(t)
    p, h, off, off_h = bounds(x, 1.0, 0)
    for i, row in enumerate(x):
        log_sum, _ = kernel_like(row, 1.0, 2.0 ** -20)
        assert abs(-log_sum - p[i].max()) > off[i]


def test_the_library_has_the_kernels_that_calls_reach(pkg):
    """(waves, packs a lane, with the likeliest tokens) of each type; without
    tokens 8 packs, with them 16."""
    from nnc_py_amd import runtime
    if not runtime.LIB_PATH.exists():
        pytest.fail("libnnc_hip.so is not built: run __graft_entry__.build()")
    found = set(re.findall(rb"logprobs_kI(DF16_|f)Li(\d+)ELi(\d+)ELb(\d)EEE", runtime.LIB_PATH.read_bytes()))
    each = [(1, 4, 0), (1, 4, 1), (1, 8, 0), (1, 8, 1), (4, 4, 0), (4, 4, 1), (4, 8, 0), (4, 16, 1)]
    assert found == {(t, *(b"%d" % n for n in k)) for t in (b"DF16_", b"f") for k in each}
