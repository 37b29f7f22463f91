"""What a decoder that drafts several tokens ahead does between its products, as
cases that can be timed:

  rope      norms of query and key heads and their rotation by position, in one
            pass over the rows of a fused projection
  append    the same for a call's queries and keys, the keys and values going
            into a paged 8-bit cache; rows of the cache read back
  tree      attention of drafted tokens over such a cache: each sees the tokens
            before the drafts, and those of the drafts that lead to it
  logprobs  log probabilities of given tokens, entropy, the likeliest tokens

A cache holds K as [pages][kv_heads][page][head_dim] and V as
[pages][kv_heads][head_dim][page], with float scales [pages][kv_heads] each.
Sequence b's rows are starts[b] .. starts[b + 1] of the activations; they are
its last positions, lengths[b] being its length with them. Angles are a table
[positions][rot]: rot / 2 cosines, then the sines.

`own` false: the operators in elementary torch operations, in 32 bits (64 for
what is rounded to whole numbers, and for sums over a vocabulary). `own` true:
the calls of the library.
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
TINY = 2.0 ** -100  # a page whose largest value is below holds zeros
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one token of a few requests: latency
        {"name": "rope_decode", "kind": "rope", "rows": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "rot": 128,
         "interleaved": False, "norm": True, "type": "f16", "table": 32768},
        # heads that are no power of two, half of each turned, neighbours as pairs; fp32
        {"name": "rope_part", "kind": "rope", "rows": 777, "heads": 12, "kv_heads": 4, "head_dim": 96, "rot": 48,
         "interleaved": True, "norm": False, "type": "f32", "table": 4096},
        # a prompt batch: the streaming rate
        {"name": "rope_prompt", "kind": "rope", "rows": 16384, "heads": 32, "kv_heads": 8, "head_dim": 128, "rot": 128,
         "interleaved": False, "norm": True, "type": "f16", "table": 32768},
        # one new token in each of 32 sequences, somewhere inside a page
        {"name": "append_decode", "kind": "append", "batch": 32, "rows": 1, "length": 2048, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot": 128, "interleaved": False, "norm": True, "drafts": False, "page": 16, "type": "f16", "ragged": True},
        # drafted tokens of 16 sequences, fp32, half of each head turned; several share a position
        {"name": "append_drafts", "kind": "append", "batch": 16, "rows": 24, "length": 1500, "heads": 16, "kv_heads": 16,
         "head_dim": 64, "rot": 32, "interleaved": True, "norm": False, "drafts": True, "page": 64, "type": "f32", "ragged": True},
        # prompts written whole
        {"name": "append_prompt", "kind": "append", "batch": 8, "rows": 2048, "length": 2048, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot": 128, "interleaved": False, "norm": True, "drafts": False, "page": 64, "type": "f16", "ragged": False},
        # a few drafts behind short odd contexts, fp32, one query head for each cached head: latency
        {"name": "tree_small", "kind": "tree", "batch": 4, "rows": 5, "length": 333, "heads": 8, "kv_heads": 8,
         "head_dim": 64, "page": 16, "type": "f32", "window": 0, "ragged": True},
        # a serving batch, contexts of very different length
        {"name": "tree_batch", "kind": "tree", "batch": 32, "rows": 16, "length": 8192, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "type": "f16", "window": 0, "ragged": True},
        # one request with a wide tree behind a long context
        {"name": "tree_long", "kind": "tree", "batch": 1, "rows": 64, "length": 65536, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "type": "f16", "window": 0, "ragged": False},
        # the answers of a few requests: latency
        {"name": "logprobs_decode", "kind": "logprobs", "rows": 8, "vocab": 32000, "top": 5, "type": "f32"},
        # a vocabulary whose rows start on no 16-byte boundary; scores only
        {"name": "logprobs_odd", "kind": "logprobs", "rows": 301, "vocab": 50257, "top": 0, "type": "f32"},
        # every draft of a serving batch, many alternatives
        {"name": "logprobs_drafts", "kind": "logprobs", "rows": 512, "vocab": 128256, "top": 20, "type": "f16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, dims):
    dim = rng.choice(dims)
    kv = _spread(rng, 1, 16)
    return {"heads": kv * rng.choice([1, 1, 2, 4, 7, 8]), "kv_heads": kv, "head_dim": dim, "type": rng.choice(["f32", "f16"])}


def _turn(rng, dim):
    return {"rot": rng.choice([dim, dim, dim // 2, dim // 4 * 2, 2 * rng.randint(1, dim // 2)]), "interleaved": rng.random() < 0.4,
            "norm": rng.random() < 0.5}


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "tree", "tree", "tree", "logprobs", "logprobs"])
    most = {}
    for c in listed():
        if c["kind"] == kind:
            w = work(c)
            for k in w:
                most[k] = max(most.get(k, 0), w[k])
    while True:
        if kind == "rope":
            c = {"kind": kind, "rows": _spread(rng, 1, 16384), **_heads(rng, [32, 64, 80, 96, 128, 128, 192, 256])}
            c.update(_turn(rng, c["head_dim"]), table=_spread(rng, 64, 65536))
        elif kind == "append":
            c = {"kind": kind, "batch": _spread(rng, 1, 64), "rows": rng.choice([1, 1, rng.randint(2, 64), _spread(rng, 65, 2048)]),
                 **_heads(rng, [32, 64, 64, 128, 128, 256]), "page": rng.choice([16, 16, 32, 48, 64, 128]), "ragged": rng.random() < 0.8}
            c.update(_turn(rng, c["head_dim"]), drafts=1 < c["rows"] <= 64 and rng.random() < 0.6)
            c["length"] = c["rows"] + rng.choice([0, rng.randint(0, 2000)])
        elif kind == "tree":
            c = {"kind": kind, "batch": _spread(rng, 1, 64), "rows": rng.choice([1, rng.randint(2, 8), _spread(rng, 9, 100)]),
                 **_heads(rng, [32, 64, 64, 128, 128, 256]), "page": rng.choice([16, 16, 32, 48, 64, 128]), "ragged": rng.random() < 0.8}
            c["length"] = c["rows"] + _spread(rng, 1, 16384) - 1
            c["window"] = rng.choice([0, 0, 0, rng.randint(1, 2 * c["length"])])
            if 4 * c["batch"] * c["heads"] * c["rows"] * c["length"] > 2.2e9:  # the plain form holds the scores
                continue
            if 4 * c["batch"] * c["kv_heads"] * c["length"] * c["head_dim"] > 2.2e9:  # and the keys
                continue
        else:
            c = {"kind": kind, "rows": _spread(rng, 1, 1024), "vocab": _spread(rng, 401, 262144), "top": rng.choice([0, 1, 5, 20, rng.randint(2, 64)]),
                 "type": rng.choice(["f32", "f16"])}
            if rng.random() < 0.5:
                c["vocab"] = -(-c["vocab"] // 64) * 64
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


def _trees(case, seed):
    """For each sequence its drafts' parents: -1, or an earlier draft."""
    rng = random.Random(int(seed) * 31 + 5)
    return [[rng.randint(max(-1, i - 5), i - 1) for i in range(n)] for n in _extent(case)[1]]


def _lines(parents):
    """For each draft the drafts that lead to it, itself the last."""
    lines = []
    for i, p in enumerate(parents):
        lines.append((lines[p] if p >= 0 else []) + [i])
    return lines


def work(case):
    c = case
    e = SIZE[c["type"]]
    if c["kind"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * e + c["rows"] * (12 + 8 * c["top"]), "flops": 6.0 * n}
    heads, kv, dim = c["heads"], c["kv_heads"], c["head_dim"]
    if c["kind"] == "rope":
        n = c["rows"] * (heads + kv) * dim
        return {"bytes": 2 * n * e + 4 * min(c["rows"], c["table"]) * c["rot"] + ((heads + kv) * dim * e if c["norm"] else 0), "flops": 8.0 * n}
    lengths, rows = _extent(c)
    row = kv * dim
    if c["kind"] == "append":
        back = sum(_back(c, lengths, rows))
        angles = 4 * c["rot"] * min(sum(rows), max(lengths))
        return {"bytes": 2 * e * sum(rows) * heads * dim + 2 * row * (sum(rows) * (e + 1) + back * e) + angles,
                "flops": sum(rows) * (8.0 * heads * dim + 14.0 * row) + 6.0 * 2 * row * back}
    # the context, and of the drafts the mean line: a third of them at most
    pairs = sum(r * (min(n - r, c["window"] or n) + min(r, 1 + r / 3)) for n, r in zip(lengths, rows))
    seen = sum(min(n, (c["window"] or n) + r - 1) if r else 0 for n, r in zip(lengths, rows))
    return {"bytes": 2 * row * seen + 2 * e * heads * dim * sum(rows), "flops": 4.0 * heads * dim * pairs}


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


def _generator(seed, what):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + what)


def _angles(positions, rot):
    """Cosines and sines, in 64 bits until they are rounded."""
    f = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _head_weights(c, g, heads):
    return (1 + 0.2 * torch.randn((heads, c["head_dim"]), generator=g, device="cuda")).to(TYPES[c["type"]]) if c["norm"] else None


def _rope_inputs(c, seed):
    g = _generator(seed, 1)
    heads, dim = c["heads"] + c["kv_heads"], c["head_dim"]
    x = torch.randn((c["rows"], (heads + c["kv_heads"]) * dim), generator=g, device="cuda") * 2  # a fused projection's rows
    positions = torch.randint(0, c["table"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
    run = torch.arange(c["rows"], device="cuda", dtype=torch.int32)  # consecutive, from somewhere
    positions = (positions[:1] + run) % c["table"]
    return {"x": x.to(TYPES[c["type"]]), "positions": positions, "weight": _head_weights(c, g, heads), "angles": _angles(c["table"], c["rot"])}


def _cache_inputs(c, seed):
    """A cache that holds every sequence up to its length, its pages scattered."""
    g = _generator(seed, 3)
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
    s = {"lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "starts": _starts(rows),
         "most_rows": max(rows), "most_length": max(lengths), "table": table, "k_scale": scales(), "v_scale": scales(),
         "k_cache": held(pages, kv, page, dim), "v_cache": held(pages, kv, dim, page), "qkv": qkv.to(TYPES[c["type"]])}
    if c["kind"] == "append":
        s.update(q_weight=_head_weights(c, g, 1), k_weight=_head_weights(c, g, 1), angles=_angles(max(lengths), c["rot"]), positions=None)
        if c["drafts"]:
            at = [n - r + len(line) - 1 for n, r, p in zip(lengths, rows, _trees(c, seed)) for line in _lines(p)]
            s["positions"] = torch.tensor(at or [0], dtype=torch.int32, device="cuda")
    else:
        words = -(-s["most_rows"] // 32)
        bits = []
        for parents in _trees(c, seed):
            for line in _lines(parents):
                mask = sum(1 << i for i in line)
                bits.append([_signed(mask >> 32 * w) for w in range(words)])
        s["tree"] = torch.tensor(bits or [[0] * words], dtype=torch.int32, device="cuda")
    return s


def _signed(word):
    """32 bits as torch's int32 holds them."""
    word &= 0xffffffff
    return word - (1 << 32) if word >> 31 else word


def _logits_inputs(c, seed):
    """Logits as a head makes them: a wide bell, a few tokens far above it in
    most rows, tokens that a grammar rules out in every fourth."""
    g = _generator(seed, 4)
    rows, vocab = c["rows"], c["vocab"]
    x = torch.randn((rows, vocab), generator=g, device="cuda") * 2.2
    some = min(vocab, 12)
    at = torch.randint(0, vocab, (rows, some), generator=g, device="cuda")
    x.scatter_add_(1, at, torch.rand((rows, some), generator=g, device="cuda") * 16)
    ruled = torch.rand((vocab,), generator=g, device="cuda") < 0.6
    x[::4, ruled] = -math.inf
    x[::4, 0] = 1.0  # something is left
    tokens = torch.where(torch.rand((rows,), generator=g, device="cuda") < 0.7, at[:, 0],
                         torch.randint(0, vocab, (rows,), generator=g, device="cuda"))
    return x.to(TYPES[c["type"]]), tokens.to(torch.int32)


def prepare(case, seed):
    c = case
    t = TYPES[c["type"]]
    if c["kind"] == "rope":
        s = State(c, **_rope_inputs(c, seed))
        s.out = torch.empty((c["rows"], (c["heads"] + c["kv_heads"]) * c["head_dim"]), dtype=t, device="cuda")
    elif c["kind"] == "logprobs":
        logits, tokens = _logits_inputs(c, seed)
        s = State(c, logits=logits, tokens=tokens, top_index=None, top_logprob=None)
        s.logprob, s.entropy = (torch.empty((c["rows"],), device="cuda") for _ in range(2))
        if c["top"]:
            s.top_index = torch.empty((c["rows"], c["top"]), dtype=torch.int32, device="cuda")
            s.top_logprob = torch.empty((c["rows"], c["top"]), device="cuda")
    else:
        s = State(c, **_cache_inputs(c, seed))
        row = c["kv_heads"] * c["head_dim"]
        s.out = torch.zeros((s.qkv.shape[0], c["heads"] * c["head_dim"]), dtype=t, device="cuda")
        if c["kind"] == "append":
            back = _back(c, *_extent(c))
            s.back = _starts(back)
            s.k_out, s.v_out = (torch.empty((sum(back), row), dtype=t, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------

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
    if c["kind"] == "logprobs":
        return [(lib.nnc_hip_token_logprobs, (d(s.logits), d(s.tokens), d(s.logprob), d(s.entropy), d(s.top_index), d(s.top_logprob), 1.0))]
    if c["kind"] == "rope":
        return [(lib.nnc_hip_rope, (d(s.x), d(s.weight), d(s.angles), d(s.positions), d(s.out), 0, 0, c["heads"] + c["kv_heads"],
                                    c["head_dim"], int(c["interleaved"]), EPS))]
    cache = (d(s.k_cache), d(s.v_cache), d(s.k_scale), d(s.v_scale), d(s.table))
    if c["kind"] == "append":
        k_col = c["heads"] * c["head_dim"]
        v_col = k_col + c["kv_heads"] * c["head_dim"]
        return [(lib.nnc_hip_rope_kv_write, (d(s.qkv), d(s.qkv), d(s.qkv), d(s.q_weight), d(s.k_weight), d(s.angles), d(s.positions), d(s.out),
                                             *cache, d(s.starts), d(s.lengths), 0, c["heads"], k_col, v_col, int(c["interleaved"]), EPS)),
                (lib.nnc_hip_kv_read, (*cache, d(s.back), d(s.lengths), d(s.k_out), d(s.v_out), 0, 0))]
    return [(lib.nnc_hip_kv_tree_attention, (d(s.qkv), *cache, d(s.starts), d(s.lengths), d(s.tree), d(s.out), 0, c["heads"],
                                             c["head_dim"] ** -0.5, c["window"], s.most_length))]


def _run_own(s):
    if s.calls is None:
        s.calls = _calls(s)
    for fn, args in s.calls:
        fn(*args)
    return _results(s)


def _results(s):
    kind = s.case["kind"]
    if kind == "append":
        return {"q": s.out, "k": s.k_out, "v": s.v_out, "k_scale": s.k_scale, "v_scale": s.v_scale}
    if kind == "logprobs":
        return {"logprob": s.logprob, "entropy": s.entropy, "top_index": s.top_index, "top_logprob": s.top_logprob}
    return s.out


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _turned(x, weight, angles, positions, rot, interleaved):
    """x [rows][heads][dim]: norm of each head, rotation of its first dims; in 64
    bits, what follows may round it to whole numbers."""
    y = x.double()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.double()
    a = angles[positions.long().clamp(0, angles.shape[0] - 1)].double()[:, None]
    c, s = a[..., :rot // 2], a[..., rot // 2:]
    first, second = (y[..., :rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    u, v = first * c - second * s, second * c + first * s
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, y[..., rot:]], -1).float()


def _rope(s):
    c = s.case
    heads = c["heads"] + c["kv_heads"]
    x = s.x[:, :heads * c["head_dim"]].view(c["rows"], heads, c["head_dim"])
    return _turned(x, s.weight, s.angles, s.positions, c["rot"], c["interleaved"]).flatten(1).to(s.out.dtype)


def _unit(largest):
    """What one step of the 8 bits stands for: a 127th, rounded to 32 bits once."""
    return torch.where(largest < TINY, torch.zeros_like(largest), (largest.double() / 127).float())


def _whole(x, unit):
    """x / unit as whole numbers, ties to even; 64 bits decide next to a tie."""
    q = torch.round(x.double() / unit.double())
    return torch.where(unit > 0, q, torch.zeros_like(q)).float()


def _owner(starts, total):
    """Which sequence each row belongs to, and its place there."""
    row = torch.arange(total, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(starts[1:].contiguous(), row, right=True).clamp_(max=starts.numel() - 2)
    return b, row - starts[b]


def _write(s, fresh_rows):
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
    for cache, scale, turned, rows in ((s.k_cache, s.k_scale, False, fresh_rows[0]), (s.v_cache, s.v_scale, True, fresh_rows[1])):
        x = rows[row].float().permute(0, 1, 3, 4, 2)
        x = torch.where(fresh, x, torch.zeros_like(x))
        held = cache[at] if turned else cache[at].transpose(3, 4)
        before = torch.where((begins < first[:, None])[..., None], scale[at], torch.zeros_like(scale[at]))
        unit = torch.maximum(before, _unit(x.abs().amax((3, 4))))
        old, new = before[..., None, None], unit[..., None, None]
        again = torch.where(new > old, _whole(held.double() * old.double(), new), held.float())
        q = torch.where(fresh, _whole(x, new), torch.where(kept, again, held.float())).to(torch.int8)
        cache[at] = q if turned else q.transpose(3, 4)
        scale[at] = torch.where(touched[..., None], unit, scale[at])


def _append(s):
    c = s.case
    heads, kv, dim = c["heads"], c["kv_heads"], c["head_dim"]
    b, i = _owner(s.starts, s.qkv.shape[0])
    place = s.positions
    if place is None:
        place = s.lengths[b] - (s.starts[b + 1] - s.starts[b]) + i
    x = s.qkv.view(-1, heads + 2 * kv, dim)
    turn = (s.angles, place, c["rot"], c["interleaved"])
    q = _turned(x[:, :heads], s.q_weight, *turn).flatten(1).to(s.out.dtype)
    k = _turned(x[:, heads:heads + kv], s.k_weight, *turn).to(s.out.dtype)
    _write(s, (k, x[:, heads + kv:]))
    b, i = _owner(s.back, s.k_out.shape[0])
    pos = s.lengths[b] - (s.back[b + 1] - s.back[b]) + i
    at = s.table[b, pos // c["page"]].long()
    k = s.k_cache[at, :, pos % c["page"], :].float() * s.k_scale[at][..., None]
    v = s.v_cache[at, :, :, pos % c["page"]].float() * s.v_scale[at][..., None]
    return {"q": q, "k": k.flatten(1).to(q.dtype), "v": v.flatten(1).to(q.dtype), "k_scale": s.k_scale, "v_scale": s.v_scale}


def _tree(s):
    c = s.case
    kv, dim = c["kv_heads"], c["head_dim"]
    group = c["heads"] // kv
    batch, width = s.table.shape
    length = width * c["page"]
    table = s.table.long()
    k = (s.k_cache[table].float() * s.k_scale[table][..., None, None]).transpose(1, 2).reshape(batch, kv, length, dim)
    v = (s.v_cache[table].float() * s.v_scale[table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(batch, kv, length, dim)
    n = s.starts[1:] - s.starts[:-1]
    first = s.lengths - n
    i = torch.arange(s.most_rows, device="cuda")
    row = (s.starts[:-1, None] + i).clamp(max=s.qkv.shape[0] - 1)
    q = s.qkv[:, :c["heads"] * dim][row].float().view(batch, -1, kv, group, dim).permute(0, 2, 1, 3, 4)
    scores = q.reshape(batch, kv, -1, dim) @ k.transpose(2, 3).contiguous()
    del k
    scores = scores.view(batch, kv, s.most_rows, group, length).mul_(dim ** -0.5)
    # drafts that each draft sees, [batch][draft][draft], and its position
    sees = (s.tree[:, i // 32] >> (i % 32) & 1).bool()[row] & (i < n[:, None])[:, None]
    pos = first[:, None] + sees.sum(2) - 1
    j = torch.arange(length, device="cuda")
    seen = (j < first[:, None])[:, None].expand(batch, s.most_rows, length)
    if c["window"]:
        seen = seen & (j > pos[..., None] - c["window"])
    draft = (j - first[:, None])[:, None].expand(batch, s.most_rows, length)
    own_rows = (draft >= 0) & (draft < n[:, None, None])
    seen = seen | (own_rows & sees.gather(2, draft.clamp(0, s.most_rows - 1)))
    seen = (seen & (i < n[:, None])[..., None])[:, None, :, None, :]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.view(batch, kv, -1, length) @ v).view(batch, kv, s.most_rows, group, dim)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 2, 1, 3, 4).reshape(batch, s.most_rows, -1).to(s.out.dtype)
    b, at = _owner(s.starts, s.qkv.shape[0])
    return out[b, at]


def _ranked(x):
    """Whole numbers ordered as the values are, the earlier of equal ones first."""
    bits = x.float().add(0.0).view(torch.int32)  # (-0 becomes 0)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    return (order << 32) - torch.arange(x.shape[1], device="cuda")


def _logprobs(s):
    c = s.case
    x = s.logits.float()
    shifted = x - x.amax(1, keepdim=True)
    e = shifted.exp()
    total = e.sum(1, dtype=torch.float64)
    weighted = torch.where(e > 0, shifted * e, torch.zeros_like(e)).sum(1, dtype=torch.float64)
    log = total.log()
    logprob = shifted.gather(1, s.tokens.long()[:, None])[:, 0].double() - log
    out = {"logprob": logprob.float(), "entropy": (log - weighted / total).float(), "top_index": None, "top_logprob": None}
    if c["top"]:
        at = torch.topk(_ranked(x), min(c["top"], c["vocab"]), dim=1).indices
        out["top_logprob"] = (shifted.gather(1, at).double() - log[:, None]).float()
        out["top_index"] = at.to(torch.int32)
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"rope": _rope, "append": _append, "tree": _tree, "logprobs": _logprobs}[state.case["kind"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_turned(c, x, weight, angles, positions):
    """Pair by pair of a head's dims, as complex numbers."""
    rot = c["rot"]
    y = x.double()
    if weight is not None:
        y = y * weight.double() / (y.pow(2).sum(-1, keepdim=True) / c["head_dim"] + EPS).sqrt()
    out = y.clone()
    one = torch.arange(0, rot, 2, device="cuda") if c["interleaved"] else torch.arange(rot // 2, device="cuda")
    other = one + 1 if c["interleaved"] else one + rot // 2
    a = angles[positions.long()].double()
    turn = torch.complex(a[:, :rot // 2], a[:, rot // 2:])[:, None]
    z = torch.complex(y[..., one].contiguous(), y[..., other].contiguous()) * turn
    out[..., one], out[..., other] = z.real, z.imag
    return out


def _exact_rope(c, seed):
    s = _rope_inputs(c, seed)
    heads = c["heads"] + c["kv_heads"]
    out = []
    for at in range(0, c["rows"], 2048):
        x = s["x"][at:at + 2048, :heads * c["head_dim"]].reshape(-1, heads, c["head_dim"])
        out.append(_exact_turned(c, x, s["weight"], s["angles"], s["positions"][at:at + 2048]).flatten(1))
    return torch.cat(out)


def _exact_append(c, seed):
    """Page by page, as the rule for one page reads."""
    s = _cache_inputs(c, seed)
    lengths, rows = _extent(c)
    page, heads, kv, dim = c["page"], c["heads"], c["kv_heads"], c["head_dim"]
    table, starts = s["table"].tolist(), s["starts"].tolist()
    back = _back(c, lengths, rows)
    place = s["positions"]
    if place is None:
        place = torch.cat([torch.arange(n - r, n, device="cuda") for n, r in zip(lengths, rows)] or [torch.zeros(1, device="cuda")])
    total = sum(rows)
    place = place[:total]
    x = s["qkv"][:total].view(total, heads + 2 * kv, dim)
    q = torch.zeros((s["qkv"].shape[0], heads * dim), dtype=torch.float64, device="cuda")
    q[:total] = _exact_turned(c, x[:, :heads], s["q_weight"], s["angles"], place).flatten(1)
    # a turned key is a value of the activations' type by definition
    k = _exact_turned(c, x[:, heads:heads + kv], s["k_weight"], s["angles"], place).float().to(TYPES[c["type"]])
    out = {"q": q}
    for name, fresh in (("k", k), ("v", x[:, heads + kv:])):
        held = s[name + "_cache"].double()
        held = held if name == "k" else held.transpose(2, 3).contiguous()
        scale = s[name + "_scale"].double()
        fresh = fresh.double().transpose(0, 1)
        for b, (length, n) in enumerate(zip(lengths, rows)):
            at = length - n
            while at < length:
                p, lo = table[b][at // page], at % page
                hi = min(page, lo + length - at)
                new = fresh[:, starts[b] + at - (length - n):starts[b] + at - (length - n) + hi - lo]
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


def _exact_tree(c, seed):
    s = _cache_inputs(c, seed)
    lengths, rows = _extent(c)
    kv, dim = c["kv_heads"], c["head_dim"]
    group = c["heads"] // kv
    out = torch.zeros((s["qkv"].shape[0], c["heads"] * dim), dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist()
    for b, (length, n, parents) in enumerate(zip(lengths, rows, _trees(c, seed))):
        if not n:
            continue
        mine = s["table"][b].long()
        first = length - n
        see = torch.zeros((n, length), dtype=torch.bool)
        for i, line in enumerate(_lines(parents)):
            see[i, max(0, first + len(line) - c["window"]) if c["window"] else 0:first] = True
            see[i, [first + m for m in line]] = True
        see = see.cuda()
        for h in range(kv):
            k = (s["k_cache"][mine, h].double() * s["k_scale"][mine, h, None, None].double()).reshape(-1, dim)[:length]
            v = (s["v_cache"][mine, h].double() * s["v_scale"][mine, h, None, None].double()).transpose(1, 2).reshape(-1, dim)[:length]
            q = s["qkv"][starts[b]:starts[b] + n, h * group * dim:(h + 1) * group * dim].double().reshape(n * group, dim)
            x = (q @ k.t().contiguous()).view(n, group, length) / math.sqrt(dim)
            x = torch.softmax(x.masked_fill(~see[:, None], -math.inf), -1)
            out[starts[b]:starts[b] + n, h * group * dim:(h + 1) * group * dim] = (x.view(n * group, length) @ v).view(n, group * dim)
    return out


def _exact_logprobs(c, seed):
    x, tokens = _logits_inputs(c, seed)
    out = {"logprob": [], "entropy": [], "top_index": [], "top_logprob": []}
    for at in range(0, c["rows"], 128):
        p = torch.log_softmax(x[at:at + 128].double(), 1)
        out["logprob"].append(p.gather(1, tokens[at:at + 128].long()[:, None])[:, 0])
        out["entropy"].append(-torch.where(p > -math.inf, p.exp() * p, torch.zeros_like(p)).sum(1))
        if c["top"]:
            best, order = torch.sort(x[at:at + 128].float(), dim=1, descending=True, stable=True)
            out["top_index"].append(order[:, :c["top"]].to(torch.int32))
            out["top_logprob"].append(p.gather(1, order[:, :c["top"]]))
    return {k: torch.cat(v) if v else None for k, v in out.items()}


def exact(case, seed):
    with torch.no_grad():
        return {"rope": _exact_rope, "append": _exact_append, "tree": _exact_tree, "logprobs": _exact_logprobs}[case["kind"]](case, seed)
