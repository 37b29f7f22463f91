"""Rotary positions, drafted trees and token log probabilities as graph nodes,
together, as a decoder that drafts uses them: prompts written with their
positions, then trees of drafts behind them, each draft's log probability,
entropy and alternatives out of a head's logits. Every node's result is held
against float64 forms of what the node itself read, so no tolerance has to cover
a chain of roundings. On the host's oracle here, on the device under the gpu
marker."""

from __future__ import annotations

import re
import subprocess
from pathlib import Path

import numpy as np
import pytest

import drafting as dr
import serving8 as s8
from serving8 import F32, I8, I32, U32
from test_serving8_graph import near

ROOT = Path(__file__).resolve().parent.parent

LAYERS, BATCH, WIDTH, HEADS, KV, DIM, PAGE, VOCAB, TOP, PLACES = 2, 3, 96, 4, 2, 32, 16, 201, 4, 64
FUSED = (HEADS + 2 * KV) * DIM
LENGTHS = [PAGE + 5, 1, PAGE]  # of the prompts
DRAFTS = [6, 3, 1]
STEPS = 3


def decoder(rows, table_width, drafts, seed=5):
    """One run's program: rows in 8 bits in, the rows' log probabilities out;
    with `drafts` attention by masks and positions that are given."""
    from nnc_py_amd.compiler.builder import GraphBuilder
    rng = np.random.default_rng(seed)
    b = GraphBuilder("drafts")

    def weight(name, n, k):
        return (b.const(name, rng.integers(-127, 128, (n, k)).astype(I8)),
                b.const(f"{name}_scale", rng.uniform(0.5, 1.5, n).astype(F32) / F32(70 * k ** 0.5)))

    def norm(name, width=WIDTH):
        return b.const(name, (1 + 0.1 * rng.standard_normal(width)).astype(F32))
    x8, xs = b.input("x8", (rows, WIDTH), "int8"), b.input("x_scale", (rows,))
    place = [b.input("table", (BATCH, table_width), "int32"), b.input("starts", (BATCH + 1,), "int32"),
             b.input("lengths", (BATCH,), "int32")]
    tokens = b.input("tokens", (rows,), "int32")
    at = b.input("positions", (rows,), "int32") if drafts else None
    tree = b.input("tree", (rows, 1), "int32") if drafts else None
    angles = b.rope_angles("angles", PLACES, DIM // 2, base=500.0, factor=2.0)
    pages = BATCH * table_width
    x = b.dequantize_rows(x8, xs)
    for i in range(LAYERS):
        cache = b.kv_cache(f"cache{i}", pages, KV, PAGE, DIM)
        q, s = b.rms_norm(x, norm(f"norm{i}"), int8=True)
        qkv = b.matmul_i8(q, s, *weight(f"qkv{i}", FUSED, WIDTH))
        q = b.rope_kv_write(qkv, qkv, qkv, cache, *place, heads=HEADS, angles=angles, positions=at, q_weight=norm(f"q_norm{i}", DIM),
                            k_weight=norm(f"k_norm{i}", DIM) if i else None, k_col=HEADS * DIM, v_col=(HEADS + KV) * DIM, interleaved=bool(i))
        window = PAGE + 2 if i else 0
        a = (b.kv_tree_attention(q, cache, *place, tree, heads=HEADS, window=window) if drafts
             else b.kv_attention(q, cache, *place, heads=HEADS, window=window))
        o = b.matmul_i8(*b.quantize_rows(a), *weight(f"out{i}", WIDTH, HEADS * DIM))
        x = b.add(x, o)
    logits = b.matmul_i8(*b.quantize_rows(b.rms_norm(x, norm("norm_out"))), *weight("head", VOCAB, WIDTH))
    for t in b.token_logprobs(logits, tokens, top=TOP, scale=1.5):
        b.output(t)
    return b.build()


def check_node(node, get, was, starts, lengths, angles):
    """One node's outputs against what it read; `was`: its cache before."""
    at = node.attrs
    rows = lambda: np.concatenate([np.arange(n - (starts[b + 1] - starts[b]), n) for b, n in enumerate(lengths)])  # noqa: E731
    opt = lambda i: get(node.inputs[i]) if node.inputs[i] else None  # noqa: E731
    if node.op_type == "RopeKvWrite":
        q, k, v = (get(n) for n in node.inputs[:3])
        places = rows() if opt(6) is None else opt(6)
        k = k[:, at["k_col"]:at["k_col"] + KV * DIM].reshape(-1, KV, DIM)
        v = v[:, at["v_col"]:at["v_col"] + KV * DIM].reshape(-1, KV, DIM)
        y, size = dr.rope(q[:, at["q_col"]:at["q_col"] + HEADS * DIM].reshape(-1, HEADS, DIM), opt(3), angles, places, at["interleaved"], at["epsilon"])
        near(get(node.outputs[0]).reshape(y.shape), y, dr.rope_bound(F32, y, size))
        was.write(dr.rope(k, opt(4), angles, places, at["interleaved"], at["epsilon"])[0].astype(F32), v, starts, lengths)
        for n, want in zip(node.outputs[1:], (was.k, was.v, was.ks, was.vs)):
            np.testing.assert_array_equal(get(n), want)
    elif node.op_type in ("KvTreeAttention", "KvAttention"):
        q = get(node.inputs[0]).reshape(-1, HEADS, DIM)
        more = (get(node.inputs[-1]),) if node.op_type == "KvTreeAttention" else ()
        form = dr.tree_attention if more else s8.attention
        out, about = form(q, was, starts, lengths, *more, F32(at["scale"]), at["window"])
        near(get(node.outputs[0]).reshape(out.shape), out, s8.attention_bound(F32, DIM, out, *about))
    elif node.op_type == "TokenLogprobs":
        x, tokens = get(node.inputs[0]), get(node.inputs[1])
        p, h, off, off_h = dr.logprobs(x, at["scale"])
        want = p[np.arange(len(x)), tokens]
        near(get(node.outputs[0]), want, off + 2 * U32 * np.abs(want))
        near(get(node.outputs[1]), h, off_h + 2 * U32 * h)
        order = dr.ranking(x, TOP)
        np.testing.assert_array_equal(get(node.outputs[2]), order)
        best = np.take_along_axis(p, order, 1)
        near(get(node.outputs[3]), best, off[:, None] + 2 * U32 * np.abs(best))
    else:
        return 0
    return 1


def run_together(device, lib, replay=False):
    """The prompts through one program, then drafts through another that was
    given its cache, at opt level 0 and 3; after each set of drafts the longest
    line stays and the rest is written over."""
    from nnc_py_amd.compiler.executor import Executor, build_program
    rng = np.random.default_rng(9)
    width = -(-(max(LENGTHS) + STEPS * max(DRAFTS)) // PAGE)
    table = rng.permutation(BATCH * width).astype(I32).reshape(BATCH, width)
    held, before, ran = None, None, False
    lengths = list(LENGTHS)
    for step in range(STEPS + 1):
        drafts = step > 0
        rows = DRAFTS if drafts else LENGTHS
        if drafts:
            lengths = [n + r for n, r in zip(lengths, rows)]
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(I32)
        total = int(starts[-1])
        if step < 2:
            graph = decoder(total, width, drafts)
            ex, fast = (Executor(build_program(graph if level == 0 else decoder(total, width, drafts), level), device, lib) for level in (0, 3))
            assert sum(c.op == "nnc_hip_rope_kv_write" for c in fast.prog.calls) == LAYERS
            if held is None:
                held = {n.inputs[7]: s8.Cache(np.random.default_rng(0), graph.tensors[n.inputs[7]].shape[0], KV, PAGE, DIM, table, filled=False)
                        for n in graph.nodes if n.op_type == "RopeKvWrite"}
            else:  # the cache moves on
                for name in graph.constants:
                    if name.startswith("cache"):
                        ex._write(name, before.get(name))
                        fast._write(name, before.get(name))
            before, ran = ex, False
        lines = dr.trees(rng, rows)
        feeds = {"x8": rng.integers(-127, 128, (total, WIDTH)).astype(I8), "x_scale": rng.uniform(0.005, 0.02, total).astype(F32), "table": table,
                 "starts": starts, "lengths": np.array(lengths, I32), "tokens": rng.integers(0, VOCAB, total).astype(I32)}
        if drafts:
            feeds["tree"] = dr.masks(lines, 1)
            feeds["positions"] = np.array([n - r + len(line) - 1 for n, r, seq in zip(lengths, rows, lines) for line in seq], I32)
        for e in (ex, fast):
            for name, a in feeds.items():
                e.set_input(name, a)
        ex.run()
        if replay and drafts:
            if not ran:
                fast.capture()
                ran = True
            fast.replay()
        else:
            fast.run()
        checked = sum(check_node(n, ex.get, next((held[i] for i in n.inputs if i in held), None), starts, lengths, graph.tensors["angles"].data)
                      for n in graph.topological_sort())
        assert checked == 2 * LAYERS + 1
        for name in graph.outputs:
            np.testing.assert_array_equal(fast.get(name), ex.get(name))
        if drafts:  # the longest line is kept: here as many positions
            lengths = [n - r + max(len(line) for line in seq) for n, r, seq in zip(lengths, rows, lines)]


def test_drafting_on_the_oracle(oracle_lib, pkg):
    run_together(False, oracle_lib)


@pytest.mark.gpu
@pytest.mark.parametrize("replay", [False, True])
def test_drafting_on_the_device(replay, hip):
    from nnc_py_amd import runtime
    runtime.clear_error()
    run_together(True, hip, replay)
    code, msg = runtime.last_error()
    assert code == 0, msg
    if replay:
        hip.nnc_hip_graph_destroy()


def rope_graph():
    from nnc_py_amd.compiler.builder import GraphBuilder
    rng = np.random.default_rng(3)
    b = GraphBuilder("rope")
    x, at = b.input("x", (5, 3 * 40 + 8)), b.input("at", (5,), "int32")
    w = b.const("w", (1 + 0.1 * rng.standard_normal((3, 40))).astype(F32))
    b.output(b.rope(x, 3, 40, b.rope_angles("angles", 20, 24), at, w, col=8, interleaved=True, out="y"))
    b.output(b.rope(x, 3, 40, weight=w, out="normed"))
    return b.build()


def check_rope(ex, graph):
    rng = np.random.default_rng(4)
    x, at = rng.standard_normal((5, 128)).astype(F32), np.array([0, 19, 7, 25, -1], I32)
    ex.set_input("x", x)
    ex.set_input("at", at)
    ex.run()
    w = graph.tensors["w"].data
    y, size = dr.rope(x[:, 8:].reshape(5, 3, 40), w, graph.tensors["angles"].data, at, True, 1e-6)
    near(ex.get("y").reshape(y.shape), y, dr.rope_bound(F32, y, size))
    y, size = dr.rope(x[:, :120].reshape(5, 3, 40), w, None, None, False, 1e-6)
    near(ex.get("normed").reshape(y.shape), y, dr.rope_bound(F32, y, size))


def test_rope_node_on_the_oracle(oracle_lib, pkg):
    from nnc_py_amd.compiler.executor import Executor, build_program
    for level in (0, 3):
        graph = rope_graph()
        check_rope(Executor(build_program(graph, level), False, oracle_lib), graph)


@pytest.mark.gpu
def test_rope_node_on_the_device(hip):
    from nnc_py_amd.compiler.executor import Executor, build_program
    graph = rope_graph()
    check_rope(Executor(build_program(graph, 3), True, hip), graph)


def test_oracle_logprobs_of_rows_that_are_not_finite(oracle_lib, abi):
    import ctypes
    x = np.array([[0, 1, 1, -np.inf], [np.nan, 0, 0, 0], [-np.inf] * 4, [np.inf, 0, 0, 0]], F32)
    arrays = [x, np.array([1, 0, 0, 9], I32), np.zeros(4, F32), np.zeros(4, F32), np.zeros((4, 6), I32), np.zeros((4, 6), F32)]
    kept = [abi.make_tensor(a.ctypes.data, abi.NUMPY_TO_NNC[a.dtype.name], a.shape, a.nbytes) for a in arrays]
    oracle_lib.nnc_hip_token_logprobs(*[ctypes.pointer(t) for t, _ in kept], 1.0)
    p, h, _, _ = dr.logprobs(x, 1.0)
    assert abs(arrays[2][0] - p[0, 1]) < 1e-7 and np.isnan(arrays[2][1:]).all() and abs(arrays[3][0] - h[0]) < 1e-6
    assert arrays[4][0].tolist() == [1, 2, 0, 3, -1, -1] and (arrays[4][1:] == -1).all() and arrays[5][0, 3] == -np.inf and np.isnan(arrays[5][1:]).all()


def test_a_rotated_write_stays_where_no_node_reads_the_cache(pkg):
    from nnc_py_amd.compiler.builder import GraphBuilder
    from nnc_py_amd.compiler.executor import build_program
    b = GraphBuilder("write")
    x = b.input("x", (2, KV * DIM))
    cache = b.kv_cache("cache", 2, KV, PAGE, DIM)
    place = [b.input("table", (1, 2), "int32"), b.input("starts", (2,), "int32"), b.input("lengths", (1,), "int32")]
    b.rope_kv_write(x, x, x, cache, *place, heads=KV)
    b.output(b.relu(x))
    for opt in (0, 1, 3):
        assert sorted(c.op for c in build_program(b.build(), opt).calls) == ["nnc_hip_rope_kv_write", "nnc_relu"]


def test_generated_program_compiles(tmp_path, pkg):
    from nnc_py_amd.compiler.compiler import Compiler
    Compiler(target="mi355x", opt_level=3).compile(decoder(10, 3, True), str(tmp_path), entry_point="draft")
    text = (tmp_path / "model.c").read_text()
    order = re.findall(r"^    (nnc_hip_(?:rope|kv|token)_\w+)\(", text, re.M)
    assert order == ["nnc_hip_rope_kv_write", "nnc_hip_kv_tree_attention"] * LAYERS + ["nnc_hip_token_logprobs"]
    for src in ("model.c", "tensors.c", "constants_loader.c"):
        subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-D_GNU_SOURCE", f"-I{ROOT / 'include'}", "-c", str(tmp_path / src),
                        "-o", str(tmp_path / (src + ".o"))], check=True, capture_output=True, text=True)


def test_cost_model_prices_the_calls(pkg):
    from nnc_py_amd import costmodel
    from nnc_py_amd.compiler.executor import build_program
    names = costmodel.estimate(build_program(decoder(10, 3, True), 3)).by_name()
    for call in ("nnc_hip_rope_kv_write", "nnc_hip_kv_tree_attention", "nnc_hip_token_logprobs"):
        assert names[call].us > 0
