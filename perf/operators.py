"""The 8-bit serving operators as cases that can be timed: what one layer of a
decoder does with its activations, weights and cache.

  norm       RMS norm with the residual's addition; its output as floats, or in
             8 bits with a scale for each row, read back as the values held
  product    8-bit activations by 8-bit weights, a scale for each token and
             each channel
  cache      new keys and values written to a paged 8-bit cache (a scale for
             each page and head), and rows of the cache read back
  attention  queries over such a cache: one token of every sequence, or runs
             of tokens behind a cached context

A cache holds K as [pages][kv_heads][page][head_dim] and V as
[pages][kv_heads][head_dim][page], with float scales [pages][kv_heads] each.
Sequence b's rows are starts[b] .. starts[b + 1] of the activations; they are
its last positions, lengths[b] being its length with them.

`own` false: the operators in elementary torch operations, in 32 bits (64 for
the roundings to whole numbers). `own` true: the calls of the library.
"""

from __future__ import annotations

import ctypes
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
TYPES = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2}
TINY = 2.0 ** -100  # a row or page whose largest value is below holds zeros


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one token of a few requests: latency of the smallest norm
        {"name": "norm_decode", "kind": "norm", "rows": 8, "width": 4096, "type": "f16", "residual": True, "q8": True},
        # odd extents of an fp32 program; float output
        {"name": "norm_ragged", "kind": "norm", "rows": 777, "width": 1345, "type": "f32", "residual": True, "q8": False},
        # a prompt batch: the streaming rate
        {"name": "norm_prompt", "kind": "norm", "rows": 16384, "width": 4096, "type": "f16", "residual": True, "q8": True},
        # decoding: the weights are read once for a handful of rows
        {"name": "product_decode", "kind": "product", "m": 8, "n": 4096, "k": 4096, "type": "f16", "bias": False},
        # rows that start on no 16-byte boundary, bias, fp32 output
        {"name": "product_ragged", "kind": "product", "m": 777, "n": 1001, "k": 1345, "type": "f32", "bias": True},
        # a prompt against a square weight: the matrix units' rate
        {"name": "product_prompt", "kind": "product", "m": 8192, "n": 4096, "k": 4096, "type": "f16", "bias": False},
        # one new token in each of 32 sequences, somewhere inside a page
        {"name": "cache_decode", "kind": "cache", "batch": 32, "rows": 1, "length": 2048, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "type": "f16", "ragged": True},
        # prompts written whole; pages of 64, fp32 rows
        {"name": "cache_prompt", "kind": "cache", "batch": 8, "rows": 1024, "length": 1024, "heads": 16, "kv_heads": 16,
         "head_dim": 64, "page": 64, "type": "f32", "ragged": True},
        # single tokens in fp32, one query head for each cached head, short
        # odd contexts: latency
        {"name": "attention_small", "kind": "attention", "batch": 4, "rows": 1, "length": 333, "heads": 8, "kv_heads": 8,
         "head_dim": 64, "page": 16, "type": "f32", "window": 0, "ragged": True},
        # a serving batch: single tokens, contexts of very different length
        {"name": "attention_batch", "kind": "attention", "batch": 64, "rows": 1, "length": 8192, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "type": "f16", "window": 0, "ragged": True},
        # one request with a very long context: the axis has to be split
        {"name": "attention_long", "kind": "attention", "batch": 1, "rows": 1, "length": 131072, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "type": "f16", "window": 0, "ragged": False},
        # the second half of two prompts, behind the first half in the cache
        {"name": "attention_prompt", "kind": "attention", "batch": 2, "rows": 2048, "length": 4096, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "type": "f16", "window": 0, "ragged": False},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cache_shape(rng):
    dim = rng.choice([32, 64, 64, 128, 128, 256])
    kv = _spread(rng, 1, 16)
    return {"heads": kv * rng.choice([1, 1, 2, 4, 7, 8]), "kv_heads": kv, "head_dim": dim,
            "page": rng.choice([16, 16, 32, 48, 64, 128]), "type": rng.choice(["f32", "f16"]), "ragged": rng.random() < 0.8}


def draw(rng):
    kind = rng.choice(["norm", "product", "product", "cache", "attention", "attention", "attention"])
    most = {}
    for c in listed():
        w = work(c)
        for k in w:
            most[k] = max(most.get(k, 0), w[k])
    while True:
        if kind == "norm":
            c = {"kind": kind, "rows": _spread(rng, 1, 16384), "width": _spread(rng, 33, 8192),
                 "type": rng.choice(["f32", "f16"]), "residual": rng.random() < 0.7, "q8": rng.random() < 0.7}
            if rng.random() < 0.6:
                c["width"] = -(-c["width"] // 64) * 64
        elif kind == "product":
            c = {"kind": kind, "m": _spread(rng, 1, 8192), "n": _spread(rng, 32, 8192), "k": _spread(rng, 32, 8192),
                 "type": rng.choice(["f32", "f16"]), "bias": rng.random() < 0.5}
            if rng.random() < 0.6:  # widths that a model has; the others fall anywhere
                c["n"], c["k"] = -(-c["n"] // 64) * 64, -(-c["k"] // 64) * 64
        elif kind == "cache":
            c = {"kind": kind, "batch": _spread(rng, 1, 64), "rows": rng.choice([1, 1, _spread(rng, 2, 1024)]), **_cache_shape(rng)}
            c["length"] = c["rows"] + rng.choice([0, rng.randint(0, 2000)])
        else:
            c = {"kind": kind, "batch": _spread(rng, 1, 64), "rows": rng.choice([1, 1, 1, rng.randint(2, 8), _spread(rng, 9, 2048)]),
                 **_cache_shape(rng)}
            c["length"] = c["rows"] + _spread(rng, 1, 8192) - 1
            c["window"] = rng.choice([0, 0, 0, rng.randint(1, 2 * c["length"])])
            if 4 * c["batch"] * c["heads"] * c["rows"] * c["length"] > 2.2e9:  # the plain form holds the scores
                continue
            if 4 * c["batch"] * c["kv_heads"] * c["length"] * c["head_dim"] > 2.2e9:  # and the keys
                continue
        w = work(c)
        if all(w[k] <= most[k] for k in w):
            return c


def _extent(case):
    """Every sequence's length and new rows, as lists: a program's scheduler has
    them on the host. Ragged batches are spread from the full length down, and
    hold a sequence without new rows and one with nothing at all."""
    c = case
    if not c["ragged"]:
        return [c["length"]] * c["batch"], [c["rows"]] * c["batch"]
    rng = random.Random(1000003 * c["batch"] + 31 * c["length"] + c["rows"])
    rows, lengths = [], []
    for b in range(c["batch"]):
        n = c["rows"] if c["rows"] == 1 or b == 0 else rng.randint(1, c["rows"])
        rows.append(n)
        lengths.append(c["length"] if b == 0 else rng.randint(n, max(n, c["length"] - (c["rows"] - n))))
    if c["batch"] >= 3 and c["rows"] > 1:
        rows[1] = 0
        rows[2] = lengths[2] = 0
    return lengths, rows


def work(case):
    c = case
    e = SIZE[c["type"]]
    if c["kind"] == "norm":
        n = c["rows"] * c["width"]
        return {"bytes": n * e * (2 + 2 * c["residual"]) + c["width"] * e + (4 * c["rows"] if c["q8"] else 0),
                "flops": 8.0 * n}
    if c["kind"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k + n * k + m * n * e + 4 * (m + n) + (4 * n if c["bias"] else 0), "flops": 2.0 * m * n * k}
    lengths, rows = _extent(c)
    row = c["kv_heads"] * c["head_dim"]
    if c["kind"] == "cache":
        back = sum(_back(c, lengths, rows))
        return {"bytes": 2 * row * (sum(rows) * (e + 1) + back * e), "flops": 6.0 * row * (sum(rows) + back)}
    pairs = sum(min(p + 1, c["window"] or p + 1) for n, r in zip(lengths, rows) for p in range(n - r, n))
    seen = sum(min(n, (c["window"] or n) + r - 1) if r else 0 for n, r in zip(lengths, rows))
    return {"bytes": 2 * row * seen + 2 * e * c["heads"] * c["head_dim"] * sum(rows),
            "flops": 4.0 * c["heads"] * c["head_dim"] * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class State:
    """A program's tensors for one case, on the GPU."""

    def __init__(self, case, **tensors):
        self.case = case
        self.calls = None  # the library's argument descriptors, made by the first pass that needs them
        for name, value in tensors.items():
            setattr(self, name, value)


def _back(c, lengths, rows):
    """How many of each sequence's last positions the pass reads back: the new
    ones, and enough before them to cover the page that they began in."""
    return [min(n, r + c["page"] - 1) if r else 0 for n, r in zip(lengths, rows)]


def _starts(rows):
    total = [0]
    for r in rows:
        total.append(total[-1] + r)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def _norm_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 1)
    t = TYPES[c["type"]]
    x = torch.randn((c["rows"], c["width"]), generator=g, device="cuda").to(t)
    # a residual stream: larger, a few channels much larger than the rest
    res = torch.randn((c["rows"], c["width"]), generator=g, device="cuda") * 2
    res[:, :: 97] *= 8
    w = (1 + 0.1 * torch.randn((c["width"],), generator=g, device="cuda")).to(t)
    return x, res.to(t) if c["residual"] else None, w


def _rows8(x):
    s = x.abs().amax(1) / 127
    return torch.round(x / s[:, None]).to(torch.int8), s


def _product_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 2)
    a = _rows8(torch.randn((c["m"], c["k"]), generator=g, device="cuda"))
    w = _rows8(torch.randn((c["n"], c["k"]), generator=g, device="cuda") * c["k"] ** -0.5)
    bias = torch.randn((c["n"],), generator=g, device="cuda") * 0.1 if c["bias"] else None
    return a, w, bias


def _cache_inputs(c, seed):
    """Rows of a fused projection (queries, keys, values), and a cache that
    holds every sequence up to its new rows, its pages scattered."""
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 3)
    lengths, rows = _extent(c)
    page, kv, dim = c["page"], c["kv_heads"], c["head_dim"]
    width = max(1, -(-max(lengths) // page))
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + 1  # the last page belongs to nobody
    order = torch.randperm(pages - 1, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["batch"], width), pages - 1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n

    def held(*shape):
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16).mul_(35)
        return x.round_().clamp_(-127, 127).to(torch.int8)

    def scales():
        return 0.02 + 0.02 * torch.rand((pages, kv), generator=g, device="cuda")
    qkv = torch.randn((max(1, sum(rows)), (c["heads"] + 2 * kv) * dim), generator=g, device="cuda")
    qkv[:, :c["heads"] * dim] *= 2
    return {"lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "starts": _starts(rows),
            "most_rows": max(rows), "most_length": max(lengths), "table": table, "k_scale": scales(), "v_scale": scales(),
            "k_cache": held(pages, kv, page, dim), "v_cache": held(pages, kv, dim, page), "qkv": qkv.to(TYPES[c["type"]])}


def prepare(case, seed):
    c = case
    t = TYPES[c["type"]]
    if c["kind"] == "norm":
        x, res, w = _norm_inputs(c, seed)
        s = State(c, x=x, res=res, w=w, sum=torch.empty_like(x) if c["residual"] else None, out=torch.empty_like(x),
                  q=torch.empty_like(x, dtype=torch.int8) if c["q8"] else None,
                  scale=torch.empty((c["rows"],), device="cuda") if c["q8"] else None)
    elif c["kind"] == "product":
        (a, sa), (w, sw), bias = _product_inputs(c, seed)
        s = State(c, a=a, sa=sa, w=w, sw=sw, bias=bias, out=torch.empty((c["m"], c["n"]), dtype=t, device="cuda"))
    else:
        s = State(c, **_cache_inputs(c, seed))
        row = c["kv_heads"] * c["head_dim"]
        if c["kind"] == "cache":
            back = _back(c, *_extent(c))
            s.back = _starts(back)
            s.k_out, s.v_out = (torch.empty((sum(back), row), dtype=t, device="cuda") for _ in range(2))
        else:
            s.out = torch.zeros((s.qkv.shape[0], c["heads"] * c["head_dim"]), dtype=t, device="cuda")
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------

EPS = 1e-6


def _library():
    if "nnc_py_amd" not in sys.modules:
        pkg = ROOT / "nnc-py_amd"
        spec = importlib.util.spec_from_file_location("nnc_py_amd", pkg / "__init__.py",
                                                      submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["nnc_py_amd"] = mod
        spec.loader.exec_module(mod)
    from nnc_py_amd import abi, runtime
    return runtime.init(0), abi


def _calls(s):
    """The pass's calls with their Tensor descriptors, which a program keeps
    beside its buffers."""
    lib, abi = _library()
    c = s.case

    def d(t):
        if t is None:
            return None
        name = str(t.dtype).replace("torch.", "")
        desc, shape = abi.make_tensor(t.data_ptr(), abi.NUMPY_TO_NNC[name], tuple(t.shape), t.numel() * t.element_size())
        desc.kept = shape
        return ctypes.pointer(desc)
    if c["kind"] == "norm":
        if not c["q8"]:
            return [(lib.nnc_hip_rms_norm, (d(s.x), d(s.res), d(s.w), d(s.sum), d(s.out), None, EPS))]
        return [(lib.nnc_hip_rms_norm, (d(s.x), d(s.res), d(s.w), d(s.sum), d(s.q), d(s.scale), EPS)),
                (lib.nnc_hip_dequantize_rows, (d(s.q), d(s.scale), d(s.out)))]
    if c["kind"] == "product":
        return [(lib.nnc_hip_matmul_i8, (d(s.a), d(s.sa), d(s.w), d(s.sw), d(s.bias), d(s.out)))]
    cache = (d(s.k_cache), d(s.v_cache), d(s.k_scale), d(s.v_scale), d(s.table))
    if c["kind"] == "cache":
        k_col = c["heads"] * c["head_dim"]
        v_col = k_col + c["kv_heads"] * c["head_dim"]
        return [(lib.nnc_hip_kv_write, (d(s.qkv), d(s.qkv), *cache, d(s.starts), d(s.lengths), k_col, v_col)),
                (lib.nnc_hip_kv_read, (*cache, d(s.back), d(s.lengths), d(s.k_out), d(s.v_out), 0, 0))]
    return [(lib.nnc_hip_kv_attention, (d(s.qkv), *cache, d(s.starts), d(s.lengths), d(s.out), 0, c["heads"],
                                        c["head_dim"] ** -0.5, c["window"], s.most_length))]


def _run_own(s):
    if s.calls is None:
        s.calls = _calls(s)
    for fn, args in s.calls:
        fn(*args)
    kind = s.case["kind"]
    if kind == "norm":
        return {"sum": s.sum, "out": s.out, "scale": s.scale}
    if kind == "cache":
        return {"k": s.k_out, "v": s.v_out, "k_scale": s.k_scale, "v_scale": s.v_scale}
    return s.out


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _unit(largest):
    """What one step of the 8 bits stands for: a 127th, rounded to 32 bits once."""
    return torch.where(largest < TINY, torch.zeros_like(largest), (largest.double() / 127).float())


def _whole(x, unit):
    """x / unit as whole numbers, ties to even; 64 bits decide next to a tie."""
    q = torch.round(x.double() / unit.double())
    return torch.where(unit > 0, q, torch.zeros_like(q)).float()


def _norm(s):
    c, t = s.case, TYPES[s.case["type"]]
    x = s.x if s.res is None else (s.x.float() + s.res.float()).to(t)
    f, w = x.float(), s.w.float()
    r = torch.rsqrt(f.square().mean(1, keepdim=True) + EPS)
    total = None if s.res is None else x
    if not c["q8"]:
        return {"sum": total, "out": (f * r * w).to(t), "scale": None}
    v = f * w
    unit = _unit(v.abs().amax(1, keepdim=True))
    scale = r * unit
    return {"sum": total, "out": (_whole(v, unit) * scale).to(t), "scale": scale[:, 0]}


def _product(s):
    out = (s.a.float() @ s.w.float().t()) * (s.sa[:, None] * s.sw[None, :])
    if s.bias is not None:
        out = out + s.bias
    return out.to(s.out.dtype)


def _owner(starts, total):
    """Which sequence each row belongs to, and its place there."""
    row = torch.arange(total, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(starts[1:].contiguous(), row, right=True).clamp_(max=starts.numel() - 2)
    return b, row - starts[b]


def _write(s):
    """Every page that a sequence's new rows touch, as [batch, pages each,
    kv_heads, head_dim, page]; slots that are none address the spare page and
    give it what it held."""
    c = s.case
    page, kv, dim = c["page"], c["kv_heads"], c["head_dim"]
    n = s.starts[1:] - s.starts[:-1]
    first = s.lengths - n
    slots = min(s.table.shape[1], (s.most_rows + page - 2) // page + 1)
    slot = first[:, None] // page + torch.arange(slots, device="cuda")
    begins = slot * page
    touched = (begins < s.lengths[:, None]) & (n > 0)[:, None]
    at = torch.where(touched, s.table.gather(1, slot.clamp(max=s.table.shape[1] - 1).long()),
                     torch.full_like(slot, s.k_scale.shape[0] - 1, dtype=torch.int32)).long()
    pos = begins[..., None] + torch.arange(page, device="cuda")
    fresh = ((pos >= first[:, None, None]) & (pos < s.lengths[:, None, None]) & touched[..., None])[:, :, None, None, :]
    kept = ((pos < first[:, None, None]) & touched[..., None])[:, :, None, None, :]
    row = (s.starts[:-1, None, None] + pos - first[:, None, None]).clamp(0, s.qkv.shape[0] - 1)
    col = c["heads"] * dim
    for cache, scale, turned in ((s.k_cache, s.k_scale, False), (s.v_cache, s.v_scale, True)):
        x = s.qkv[row, col:col + kv * dim].float().view(*row.shape, kv, dim).permute(0, 1, 3, 4, 2)
        x = torch.where(fresh, x, torch.zeros_like(x))
        held = cache[at] if turned else cache[at].transpose(3, 4)
        before = torch.where((begins < first[:, None])[..., None], scale[at], torch.zeros_like(scale[at]))
        unit = torch.maximum(before, _unit(x.abs().amax((3, 4))))
        old, new = before[..., None, None], unit[..., None, None]
        again = torch.where(new > old, _whole(held.double() * old.double(), new), held.float())
        q = torch.where(fresh, _whole(x, new), torch.where(kept, again, held.float())).to(torch.int8)
        cache[at] = q if turned else q.transpose(3, 4)
        scale[at] = torch.where(touched[..., None], unit, scale[at])
        col += kv * dim


def _read(s):
    c = s.case
    b, i = _owner(s.back, s.k_out.shape[0])
    pos = s.lengths[b] - (s.back[b + 1] - s.back[b]) + i
    at = s.table[b, pos // c["page"]].long()
    k = s.k_cache[at, :, pos % c["page"], :].float() * s.k_scale[at][..., None]
    v = s.v_cache[at, :, :, pos % c["page"]].float() * s.v_scale[at][..., None]
    return {"k": k.flatten(1).to(s.k_out.dtype), "v": v.flatten(1).to(s.k_out.dtype), "k_scale": s.k_scale, "v_scale": s.v_scale}


def _attention(s):
    c = s.case
    kv, dim = c["kv_heads"], c["head_dim"]
    group = c["heads"] // kv
    batch, width = s.table.shape
    length = width * c["page"]
    table = s.table.long()
    k = (s.k_cache[table].float() * s.k_scale[table][..., None, None]).transpose(1, 2).reshape(batch, kv, length, dim)
    v = (s.v_cache[table].float() * s.v_scale[table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(batch, kv, length, dim)
    n = s.starts[1:] - s.starts[:-1]
    i = torch.arange(s.most_rows, device="cuda")
    row = (s.starts[:-1, None] + i).clamp(max=s.qkv.shape[0] - 1)
    q = s.qkv[:, :c["heads"] * dim][row].float().view(batch, -1, kv, group, dim).permute(0, 2, 1, 3, 4)
    scores = q.reshape(batch, kv, -1, dim) @ k.transpose(2, 3).contiguous()
    del k
    scores = scores.view(batch, kv, s.most_rows, group, length).mul_(dim ** -0.5)
    pos = (s.lengths - n)[:, None] + i
    j = torch.arange(length, device="cuda")
    seen = (j <= pos[..., None]) & (i < n[:, None])[..., None]
    if c["window"]:
        seen &= j > pos[..., None] - c["window"]
    seen = seen[:, None, :, None, :]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.view(batch, kv, -1, length) @ v).view(batch, kv, s.most_rows, group, dim)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 2, 1, 3, 4).reshape(batch, s.most_rows, -1).to(s.out.dtype)
    b, at = _owner(s.starts, s.qkv.shape[0])
    return out[b, at]


def run(state):
    if own:
        return _run_own(state)
    kind = state.case["kind"]
    if kind == "norm":
        return _norm(state)
    if kind == "product":
        return _product(state)
    if kind == "cache":
        _write(state)
        return _read(state)
    return _attention(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_norm(c, seed):
    t = TYPES[c["type"]]
    x, res, w = _norm_inputs(c, seed)
    s = x.double() if res is None else (x.double() + res.double()).to(t).double()
    w = w.double()
    r = 1 / (s.pow(2).sum(1, keepdim=True) / c["width"] + EPS).sqrt()
    total = s if res is not None else None
    if not c["q8"]:
        return {"sum": total, "out": s * w * r, "scale": None}
    # what is quantised, and the step, are 32-bit values by definition
    v = (s * w).float().double()
    step = (v.abs().max(1, keepdim=True).values / 127).float().double()
    q = (v / step.clamp(min=1e-300)).round() * (step > 0)
    return {"sum": total, "out": q * (step * r), "scale": (step * r)[:, 0]}


def _exact_product(c, seed):
    (a, sa), (w, sw), bias = _product_inputs(c, seed)
    out = []
    for at in range(0, c["m"], 1024):
        y = (a[at:at + 1024].double() @ w.double().t()) * sa[at:at + 1024].double()[:, None] * sw.double()
        out.append(y if bias is None else y + bias.double())
    return torch.cat(out)


def _exact_cache(c, seed):
    """Page by page, as the rule for one page reads."""
    s = _cache_inputs(c, seed)
    lengths, rows = _extent(c)
    page, kv, dim = c["page"], c["kv_heads"], c["head_dim"]
    table, starts = s["table"].tolist(), s["starts"].tolist()
    back = _back(c, lengths, rows)
    out = {}
    for name, col in (("k", c["heads"] * dim), ("v", (c["heads"] + kv) * dim)):
        held = s[name + "_cache"].double()
        held = held if name == "k" else held.transpose(2, 3).contiguous()
        scale = s[name + "_scale"].double()
        x = s["qkv"][:, col:col + kv * dim].double().view(-1, kv, dim).transpose(0, 1)
        for b, (length, n) in enumerate(zip(lengths, rows)):
            at = length - n
            while at < length:
                p, lo = table[b][at // page], at % page
                hi = min(page, lo + length - at)
                new = x[:, starts[b] + at - (length - n):starts[b] + at - (length - n) + hi - lo]
                step = (new.abs().amax((1, 2)) / 127).float().double()
                if lo:
                    step = torch.maximum(step, scale[p])
                    held[p, :, :lo] = torch.where((step > scale[p])[:, None, None],
                                                  (held[p, :, :lo] * scale[p][:, None, None] / step[:, None, None]).round(),
                                                  held[p, :, :lo])
                held[p, :, lo:hi] = (new / step[:, None, None]).round()
                scale[p] = step
                at += hi - lo
        got = []
        for b, (length, n) in enumerate(zip(lengths, back)):
            if n:
                flat = held[s["table"][b].long()] * scale[s["table"][b].long()][..., None, None]
                got.append(flat.transpose(1, 2).reshape(-1, kv * dim)[length - n:length])
        out[name], out[name + "_scale"] = torch.cat(got), scale
    return out


def _exact_attention(c, seed):
    s = _cache_inputs(c, seed)
    lengths, rows = _extent(c)
    kv, dim = c["kv_heads"], c["head_dim"]
    group = c["heads"] // kv
    out = torch.zeros((s["qkv"].shape[0], c["heads"] * dim), dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist()
    for b, (length, n) in enumerate(zip(lengths, rows)):
        if not n:
            continue
        mine = s["table"][b].long()
        for h in range(kv):
            k = (s["k_cache"][mine, h].double() * s["k_scale"][mine, h, None, None].double()).reshape(-1, dim)[:length]
            v = (s["v_cache"][mine, h].double() * s["v_scale"][mine, h, None, None].double()).transpose(1, 2).reshape(-1, dim)[:length]
            k = k.t().contiguous()
            for first in range(0, n, 512):
                m = min(512, n - first)
                at = starts[b] + first
                q = s["qkv"][at:at + m, h * group * dim:(h + 1) * group * dim].double().reshape(m * group, dim)
                x = (q @ k).view(m, group, length) / math.sqrt(dim)
                pos = torch.arange(length - n + first, length - n + first + m, device="cuda")[:, None, None]
                j = torch.arange(length, device="cuda")
                hidden = (j > pos) | ((j <= pos - c["window"]) if c["window"] else torch.zeros_like(j > pos))
                x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
                out[at:at + m, h * group * dim:(h + 1) * group * dim] = (x.view(m * group, length) @ v).view(m, group * dim)
    return out


def exact(case, seed):
    with torch.no_grad():
        return {"norm": _exact_norm, "product": _exact_product, "cache": _exact_cache,
                "attention": _exact_attention}[case["kind"]](case, seed)
