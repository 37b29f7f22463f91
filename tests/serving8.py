"""Plain float64 forms of the 8-bit serving operators, inputs for them, and a
runner for their calls on device memory."""

from __future__ import annotations

import ctypes

import numpy as np

F32, F16, I8, I32 = np.float32, np.float16, np.int8, np.int32
U32 = 2.0 ** -24  # half a step of float32, relative
U16 = 2.0 ** -11  # of float16
SUB16 = 2.0 ** -25  # half a step of float16 below its normal numbers


def half_step(t):
    return U16 if t == F16 else U32


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------

def unit8(top):
    """The step for values up to `top` (array), float32."""
    top = np.asarray(top, F32)
    with np.errstate(invalid="ignore", over="ignore"):
        u = (top.astype(np.float64) / 127).astype(F32)
    u = np.where(top < F32(2.0 ** -100), F32(0), u)
    return np.where(np.isfinite(top), u, F32(np.nan)).astype(F32)


def whole8(x, unit):
    """Nearest whole numbers to x / unit, ties to even (rint of a float64
    quotient: float32 operands cannot come closer to a tie without being one)."""
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.rint(x.astype(np.float64) / unit.astype(np.float64))
    return np.where(unit > 0, q, 0).astype(I8)


def absmax(x, axis):
    return np.max(np.abs(x), axis=axis, initial=0)  # NaN if any is


def rms_norm(x, res, w, eps):
    """(s in the type, s * w in float32, r in float64, y in float64)."""
    s = x if res is None else (x.astype(F32) + res.astype(F32)).astype(x.dtype)
    s64 = s.astype(np.float64)
    r = 1 / np.sqrt(np.mean(s64 ** 2, axis=-1, keepdims=True) + eps)
    t = s.astype(F32) * w.astype(F32)
    return s, t, r, s64 * r * w.astype(np.float64)


# ---------------------------------------------------------------------------
# cache
# ---------------------------------------------------------------------------

class Cache:
    """A paged cache on the host; table entries outside the pages allowed."""

    def __init__(self, rng, pages, kv, page, dim, table, filled=True):
        self.page, self.kv, self.dim = page, kv, dim
        self.table = np.ascontiguousarray(table, I32)
        q = rng.integers(-127, 128, (2, pages, kv, page, dim)).astype(I8) if filled else np.zeros((2, pages, kv, page, dim), I8)
        self.k, self.v = q[0].copy(), np.ascontiguousarray(q[1].transpose(0, 1, 3, 2))
        self.ks, self.vs = (rng.uniform(0.004, 0.02, (2, pages, kv)) if filled else np.zeros((2, pages, kv))).astype(F32)

    def copy(self):
        c = object.__new__(Cache)
        c.__dict__ = {k: (v.copy() if isinstance(v, np.ndarray) else v) for k, v in self.__dict__.items()}
        return c

    def page_of(self, b, t):
        p = int(self.table[b, t // self.page])
        return p if 0 <= p < self.k.shape[0] else -1

    def tensors(self):
        return {"k_cache": self.k, "v_cache": self.v, "k_scale": self.ks, "v_scale": self.vs, "table": self.table}

    def write(self, k, v, starts, lengths):
        """k, v: [rows][kv][dim]."""
        for b, length in enumerate(lengths):
            n = starts[b + 1] - starts[b]
            first = max(length - n, 0)
            for slot in range(first // self.page, -(-length // self.page) if n > 0 else 0):
                begin = slot * self.page
                lo, hi = max(first, begin), min(length, begin + self.page)
                p = self.page_of(b, begin)
                if p < 0 or lo >= hi:
                    continue
                rows = slice(starts[b + 1] - length + lo, starts[b + 1] - length + hi)
                for x, q, s, turned in ((k, self.k, self.ks, False), (v, self.v, self.vs, True)):
                    new = x[rows].transpose(1, 0, 2).astype(F32)
                    unit = unit8(absmax(new, (1, 2)))
                    held = q[p].transpose(0, 2, 1) if turned else q[p]
                    if lo > begin:
                        old = s[p].copy()
                        unit = np.maximum(unit, old)  # NaN if either is
                        grown = ~(unit == old)
                        kept = held[:, :lo - begin].astype(np.float64) * old[:, None, None].astype(np.float64)
                        with np.errstate(invalid="ignore", divide="ignore"):
                            again = np.where(unit[:, None, None] > 0, np.rint(kept / unit[:, None, None].astype(np.float64)), 0)
                        held[:, :lo - begin] = np.where(grown[:, None, None], np.nan_to_num(again), held[:, :lo - begin])
                    held[:, lo - begin:hi - begin] = whole8(new, unit[:, None, None])
                    s[p] = unit

    def values(self, b, length):
        """K and V [kv][length][dim] and V's scales [kv][length] in float64,
        and which positions can be read."""
        k, v = np.zeros((2, self.kv, length, self.dim))
        u = np.zeros((self.kv, length))
        ok = np.zeros(length, bool)
        for t in range(length):
            p = self.page_of(b, t)
            if p >= 0:
                ok[t] = True
                u[:, t] = self.vs[p]
                k[:, t] = self.k[p, :, t % self.page] * self.ks[p].astype(np.float64)[:, None]
                v[:, t] = self.v[p, :, :, t % self.page] * self.vs[p].astype(np.float64)[:, None]
        return k, v, u, ok


def attention(q, cache, starts, lengths, scale, window):
    """q [rows][heads][dim] -> out and what its bound needs: sum_j p_j |v_j|,
    the largest scale * sum_d |q_d k_jd| of a seen key, the number of seen keys
    and the largest p_j u_j (u the scale of key j's value), each
    [rows][heads](...); out is NaN in rows of no sequence."""
    rows, heads, dim = q.shape
    out = np.full((rows, heads, dim), np.nan)
    size, (reach, seen, peak) = np.zeros((rows, heads, dim)), np.zeros((3, rows, heads))
    group = heads // cache.kv
    for b, length in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        if n <= 0:
            continue
        k, v, u, ok = cache.values(b, length)
        j = np.arange(length)
        pos = length - n + np.arange(n)[:, None]
        see = ok & (j <= pos) & ((j > pos - window) if window else True)
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


def attention_bound(t, dim, out, size, reach, seen, peak):
    """How far a result of type t may be off, each element.

    Scores, in powers of two, are off by their operands' pieces (fp32: q cut to
    22 bits; f16: exact), the running sum of dim products and the two scales,
    relative to the sum of the products' sizes (reach), and by the rounding of
    the sum with the scale's logarithm (its size under 2 reach + 32). A
    weight is off by ln 2 times that and the exponential's last bits; both the
    sum of weighted values and of weights see it. The weights' rounding for the
    second product: two f16 pieces, or one; its sums: one rounding per 32 keys
    and for each join (under 64). A weight times its value's scale is rounded
    as a multiple of 2^-12 of the row's largest, and f16 has steps of 2^-24
    at its smallest: each is off by half of 2^-36 of the largest besides, and
    stands before a whole number of up to 128."""
    score = (2.0 ** -22 + (dim / 4 + 4) * U32) * reach * 1.4427 + 2 * U32 * (2 * reach + 32)
    weight = 2 * (score * 0.6932 + 2.0 ** -21)
    weight = weight + (U16 if t == F16 else 2.0 ** -21) + (seen / 32 + 64) * 2 * U32
    least = seen * 2.0 ** -37 * peak * 128
    return weight[..., None] * size + least[..., None] + half_step(t) * np.abs(out) + (SUB16 if t == F16 else 0)


# ---------------------------------------------------------------------------
# calls
# ---------------------------------------------------------------------------

class Dev:
    """Device copies of named arrays, each `shift` bytes past an allocation's
    start, with a guard behind that has to stay as it was."""

    GUARD = 64

    def __init__(self, lib, abi, runtime, arrays, shift=None):
        self.lib, self.abi, self.rt = lib, abi, runtime
        self.kept, self.bufs, self.desc = [], {}, {}
        for name, a in arrays.items():
            a = np.ascontiguousarray(a)
            s = (shift or {}).get(name, 0)
            raw = np.full(s + a.nbytes + self.GUARD, 0xA5, np.uint8)
            raw[s:s + a.nbytes] = a.reshape(-1).view(np.uint8)
            buf = runtime.DeviceBuffer.from_array(raw)
            self.bufs[name] = (buf, a.shape, a.dtype, s, a.nbytes)
            t, shape = abi.make_tensor(buf.ptr + s, abi.NUMPY_TO_NNC[a.dtype.name], a.shape, a.nbytes)
            self.kept.append(shape)
            self.desc[name] = t

    def t(self, name):
        return None if name is None else ctypes.pointer(self.desc[name])

    def call(self, fn, *args):
        """Strings are tensors, None a NULL one."""
        getattr(self.lib, fn)(*[self.t(a) if a is None or isinstance(a, str) else a for a in args])
        self.rt.sync()
        code, msg = self.rt.last_error()
        assert code == 0, msg

    def get(self, name):
        buf, shape, dtype, s, n = self.bufs[name]
        raw = buf.to_array()
        assert (raw[:s] == 0xA5).all() and (raw[s + n:] == 0xA5).all(), f"{name}: written outside"
        return raw[s:s + n].view(dtype).reshape(shape).copy()

    def set(self, name, a):
        buf, shape, dtype, s, n = self.bufs[name]
        raw = buf.to_array()
        raw[s:s + n] = np.ascontiguousarray(a, dtype).reshape(-1).view(np.uint8)
        buf.upload(raw)

    def free(self):
        for b, *_ in self.bufs.values():
            b.free()
