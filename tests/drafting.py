"""Plain float64 forms of rotary positions, tree attention and token log
probabilities, with what their bounds need."""

from __future__ import annotations

import numpy as np

import serving8 as s8
from serving8 import F16, F32, I32, SUB16, U16, U32


def rope(x, weight, angles, places, interleaved, eps):
    """x [rows][heads][dim] -> y in float64, and the size of each result's two
    terms (what its own roundings are relative to)."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt(np.mean(y ** 2, -1, keepdims=True) + np.float64(F32(eps))) * weight.astype(np.float64)
    if angles is None:
        return y, np.abs(y)
    rot = angles.shape[1]
    a = angles[np.clip(places, 0, len(angles) - 1)].astype(np.float64)[:, None]
    c, s = a[..., :rot // 2], a[..., rot // 2:]
    one, other = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out, size = y.copy(), np.abs(y)
    out[..., one], out[..., other] = y[..., one] * c - y[..., other] * s, y[..., other] * c + y[..., one] * s
    size[..., one] = np.abs(y[..., one] * c) + np.abs(y[..., other] * s)
    size[..., other] = np.abs(y[..., other] * c) + np.abs(y[..., one] * s)
    return out, size


def rope_bound(t, y, size):
    """Float64 roundings (under 2^-44 with a sum of up to 256 squares), then
    one to float32 and, for float16, one more."""
    return 2.0 ** -44 * size + U32 * np.abs(y) * 1.001 + 2.0 ** -150 + ((U16 * 1.001) * np.abs(y) + SUB16 if t == F16 else 0)


def trees(rng, rows, branch=4):
    """For each sequence the drafts that lead to each of its drafts, itself last."""
    out = []
    for n in rows:
        lines = []
        for i in range(n):
            p = int(rng.integers(max(-1, i - branch), i)) if i else -1
            lines.append((lines[p] if p >= 0 else []) + [i])
        out.append(lines)
    return out


def masks(lines, words, total=None):
    """[rows][words] int32 of the lists of drafts that each row sees."""
    flat = [line for seq in lines for line in seq]
    m = np.zeros((total if total is not None else len(flat), words), np.uint32)
    for i, line in enumerate(flat):
        for d in line:
            if d < 32 * words:
                m[i, d // 32] |= np.uint32(1 << d % 32)
    return m.view(I32)


def tree_attention(q, cache, starts, lengths, tree, scale, window):
    """As serving8.attention, each row seeing the positions before its
    sequence's rows (the last of them, by its own position, under a window) and
    the rows that its mask names."""
    rows, heads, dim = q.shape
    out = np.full((rows, heads, dim), np.nan)
    size, (reach, seen, peak) = np.zeros((rows, heads, dim)), np.zeros((3, rows, heads))
    group = heads // cache.kv
    bits = tree.view(np.uint32)
    for b, length in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        if n <= 0:
            continue
        k, v, u, ok = cache.values(b, length)
        first = length - n
        see = np.zeros((n, length), bool)
        for i in range(n):
            mine = np.array([m < 32 * tree.shape[1] and bool(bits[starts[b] + i, m // 32] >> np.uint32(m % 32) & np.uint32(1)) for m in range(n)])
            j = np.arange(length)
            at = first + mine.sum() - 1
            see[i] = np.where(j < first, (j > at - window) if window else True, mine[np.clip(j - first, 0, n - 1)]) & ok
        some = see.any(1) if length else np.zeros(n, bool)
        rs = slice(starts[b], starts[b] + n)
        out[rs] = 0
        if not some.any():
            continue
        for h in range(heads):
            kk, vv, uu = k[h // group], v[h // group], u[h // group]
            x = q[rs, h].astype(np.float64)
            s = np.where(see, scale * (x @ kk.T), -np.inf)
            top = np.where(some, s.max(1, initial=-np.inf), 0)
            p = np.exp(s - top[:, None])
            p /= np.where(some, p.sum(1), 1)[:, None]
            out[rs, h], size[rs, h] = p @ vv, p @ np.abs(vv)
            peak[rs, h] = (p * uu).max(1)
            reach[rs, h] = np.where(see, scale * (np.abs(x) @ np.abs(kk).T), 0).max(1)
            seen[rs, h] = see.sum(1)
    return out, (size, reach, seen, peak)


def check_tree(got, q, cache, starts, lengths, tree, scale, window):
    out, about = tree_attention(q, cache, starts, lengths, tree, scale, window)
    got = got.astype(np.float64).reshape(out.shape)
    mine = ~np.isnan(out)
    bound = s8.attention_bound(q.dtype.type, q.shape[2], out, *about)
    bad = mine & ~(np.abs(got - out) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.max(np.where(mine, np.abs(got - out) / np.maximum(bound, 1e-300), 0))))


def logprobs(x, scale):
    """log p in float64, entropies, and for each row how far its sum may be off,
    relative, and its entropy besides.

    A term e^d is off by the exponential's last place (2^-23), by what rounding
    the difference, log2 e times the scale, their product and log2 e itself does
    to d (3.5 * 2^-24 of it) and by the float32 sum of the 32 values that a lane
    takes at once, two by two (5 * 2^-24): together under 2^-21 + 2^-22 |d|. It is
    scaled once for each time that a larger maximum turns up in its lane and
    where lanes (6 steps), waves and segments are joined, each off by 2^-23: 20
    times at most here. The largest, e^0, is counted."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        top = x.max(1, keepdims=True)
        ok = np.isfinite(top[:, 0])
        d = np.float64(F32(scale)) * (x - top)
        e = np.exp(d)
        total = e.sum(1)
        lp = np.where(ok[:, None], d - np.log(total)[:, None], np.nan)
        de = np.where(e > 0, np.abs(d) * e, 0)
        h = np.where(ok, np.log(total) + de.sum(1) / total, np.nan)
        term = np.where(e > 0, (2.0 ** -21 + 20 * 2.0 ** -23 + 2.0 ** -22 * np.where(e > 0, np.abs(d), 0)) * e, 0)
        off = (np.where(d == 0, 0, term)).sum(1) / total + 2.0 ** -45
        off_h = (np.where(e > 0, (np.abs(d) * term + 2.0 ** -22 * de), 0)).sum(1) / total + off * (1 + de.sum(1) / total)
    return lp, h, off, off_h


def ranking(x, n):
    """The n likeliest tokens of each row, the earlier of equal ones first."""
    return np.argsort(-x.astype(np.float64), 1, kind="stable")[:, :n]
