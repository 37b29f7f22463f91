"""The 8-bit serving operators as graph nodes, together, as a decoder uses
them: token ids' rows kept in 8 bits, two layers of norm, products, cache and
attention, prompts of different length and then one token at a time, the cache
staying in the program. Every node's result is held against float64 forms of
what the node itself read, so no tolerance has to cover a chain of roundings.
On the host's oracle here, on the device under the gpu marker."""

from __future__ import annotations

import re
import subprocess
from pathlib import Path

import numpy as np
import pytest

import serving8 as s8
from serving8 import F32, I8, I32, U32

ROOT = Path(__file__).resolve().parent.parent

LAYERS, BATCH, WIDTH, HEADS, KV, DIM, PAGE, INNER = 2, 3, 96, 4, 2, 32, 16, 160
FUSED = (HEADS + 2 * KV) * DIM
LENGTHS = [PAGE + 5, 1, PAGE]  # of the prompts
STEPS = 4


def decoder(rows, table_width, seed=5):
    from nnc_py_amd.compiler.builder import GraphBuilder
    rng = np.random.default_rng(seed)
    b = GraphBuilder("decoder8")

    def weight(name, n, k):
        return (b.const(name, rng.integers(-127, 128, (n, k)).astype(I8)),
                b.const(f"{name}_scale", rng.uniform(0.5, 1.5, n).astype(F32) / F32(70 * k ** 0.5)))

    def norm(name):
        return b.const(name, (1 + 0.1 * rng.standard_normal(WIDTH)).astype(F32))
    x8, xs = b.input("x8", (rows, WIDTH), "int8"), b.input("x_scale", (rows,))
    place = [b.input("table", (BATCH, table_width), "int32"), b.input("starts", (BATCH + 1,), "int32"),
             b.input("lengths", (BATCH,), "int32")]
    pages = BATCH * table_width
    x = b.dequantize_rows(x8, xs)
    for i in range(LAYERS):
        cache = b.kv_cache(f"cache{i}", pages, KV, PAGE, DIM)
        q, s = b.rms_norm(x, norm(f"norm{i}a"), int8=True)
        qkv = b.matmul_i8(q, s, *weight(f"qkv{i}", FUSED, WIDTH))
        b.kv_write(qkv, qkv, cache, *place, k_col=HEADS * DIM, v_col=(HEADS + KV) * DIM)
        a = b.kv_attention(qkv, cache, *place, heads=HEADS, window=PAGE + 2 if i else 0)
        o = b.matmul_i8(*b.quantize_rows(a), *weight(f"out{i}", WIDTH, HEADS * DIM))
        q, s, h = b.rms_norm(o, norm(f"norm{i}b"), residual=x, int8=True)
        up = b.matmul_i8(q, s, *weight(f"up{i}", INNER, WIDTH), b.const(f"bias{i}", rng.standard_normal(INNER).astype(F32)))
        down = b.matmul_i8(*b.quantize_rows(b.relu(up)), *weight(f"down{i}", WIDTH, INNER))
        x = b.add(h, down)
    b.output(b.rms_norm(x, norm("norm_out"), out="y"))
    return b.build()


def calls_for(steps):
    """(rows, starts, lengths) of the prompts' run and of each token's."""
    starts = np.concatenate([[0], np.cumsum(LENGTHS)]).astype(I32)
    yield starts, np.array(LENGTHS, I32)
    for i in range(steps):
        yield np.arange(BATCH + 1, dtype=I32), np.array(LENGTHS, I32) + I32(i + 1)


def near(got, want, bound):
    bad = ~(np.abs(got.astype(np.float64) - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())


def check_node(node, get, was, starts, lengths):
    """One node's outputs against what it read; `was`: its cache before."""
    at = node.attrs
    if node.op_type == "DequantizeRows":
        q, s = (get(n) for n in node.inputs)
        np.testing.assert_array_equal(get(node.outputs[0]), q.astype(F32) * s[:, None])
    elif node.op_type == "QuantizeRows":
        x = get(node.inputs[0])
        unit = s8.unit8(s8.absmax(x, 1))
        np.testing.assert_array_equal(get(node.outputs[1]), unit)
        np.testing.assert_array_equal(get(node.outputs[0]), s8.whole8(x, unit[:, None]))
    elif node.op_type == "RmsNormalization":
        x, w = get(node.inputs[0]), get(node.inputs[1])
        res = get(node.inputs[2]) if len(node.inputs) > 2 else None
        s, t, r, y = s8.rms_norm(x, res, w, at["epsilon"])
        if res is not None:
            np.testing.assert_array_equal(get(node.outputs[-1]), s)
        rel = (0.5 * (x.shape[1] / 64 + 18) + 8) * U32  # the sum of squares, root and products
        if at["int8"]:
            unit = s8.unit8(s8.absmax(t, 1))
            np.testing.assert_array_equal(get(node.outputs[0]), s8.whole8(t, unit[:, None]))
            np.testing.assert_allclose(get(node.outputs[1]), r[:, 0] * unit, rtol=rel + U32, atol=0)
        else:
            near(get(node.outputs[0]), y, rel * np.abs(y))
    elif node.op_type == "MatMulRows8":
        a, sa, w, sw = (get(n) for n in node.inputs[:4])
        p = (a.astype(np.float64) @ w.astype(np.float64).T) * sa[:, None].astype(np.float64) * sw.astype(np.float64)
        y = p + (get(node.inputs[4]) if len(node.inputs) > 4 else 0)
        near(get(node.outputs[0]), y, 3 * U32 * np.abs(p) + U32 * np.abs(y))
    elif node.op_type == "KvWrite":
        rows = [get(n) for n in node.inputs[:2]]
        k, v = (x[:, at[c]:at[c] + KV * DIM].reshape(len(x), KV, DIM) for x, c in zip(rows, ("k_col", "v_col")))
        was.write(k, v, starts, lengths)
        for n, want in zip(node.outputs, (was.k, was.v, was.ks, was.vs)):
            np.testing.assert_array_equal(get(n), want)
    elif node.op_type == "KvAttention":
        q = get(node.inputs[0])[:, at["q_col"]:at["q_col"] + HEADS * DIM].reshape(-1, HEADS, DIM)
        out, about = s8.attention(q, was, starts, lengths, F32(at["scale"]), at["window"])
        near(get(node.outputs[0]).reshape(out.shape), out, s8.attention_bound(F32, DIM, out, *about))


class Caches:
    """The cache tensors of a graph on the host."""

    def __init__(self, graph, table):
        self.table, self.held = table, {}
        for n in graph.nodes:
            if n.op_type == "KvWrite":
                c = s8.Cache(np.random.default_rng(0), graph.tensors[n.inputs[2]].shape[0], KV, PAGE, DIM, table, filled=False)
                self.held[n.inputs[2]] = c

    def of(self, node):
        return next((self.held[i] for i in node.inputs if i in self.held), None)


def run_together(device, lib, abi, replay=False):
    """The prompts through one program, then tokens through another that was
    given its cache; at opt level 0, every tensor in a place of its own."""
    from nnc_py_amd.compiler.executor import Executor, build_program
    rng = np.random.default_rng(9)
    width = -(-(max(LENGTHS) + STEPS) // PAGE)
    table = rng.permutation(BATCH * width).astype(I32).reshape(BATCH, width)
    caches, ran, before, results = None, None, None, []
    for step, (starts, lengths) in enumerate(calls_for(STEPS)):
        rows = int(starts[-1])
        if step < 2:
            graph = decoder(rows, width)
            fast = Executor(build_program(decoder(rows, width), 3), device, lib)
            ex = Executor(build_program(graph, 0), device, lib)
            assert sum(c.op == "nnc_hip_kv_write" for c in fast.prog.calls) == LAYERS
            if caches is None:
                caches = Caches(graph, table)
            else:  # the cache moves on
                for name in graph.constants:
                    if name.startswith("cache"):
                        ex._write(name, before.get(name))
                        fast._write(name, before.get(name))
            before, ran = ex, False
        x8, xs = rng.integers(-127, 128, (rows, WIDTH)).astype(I8), rng.uniform(0.005, 0.02, rows).astype(F32)
        for e in (ex, fast):
            for name, a in (("x8", x8), ("x_scale", xs), ("table", table), ("starts", starts), ("lengths", lengths)):
                e.set_input(name, a)
        ex.run()
        if replay and step >= 1:
            if not ran:
                fast.capture()
                ran = True
            fast.replay()
        else:
            fast.run()
        y = ex.get("y")
        np.testing.assert_array_equal(fast.get("y"), y)
        for node in graph.topological_sort():
            check_node(node, ex.get, caches.of(node), starts, lengths)
        assert np.isfinite(y).all()
        results.append(y)
    return results


def test_decoder_on_the_oracle(oracle_lib, abi, pkg):
    run_together(False, oracle_lib, abi)


@pytest.mark.gpu
@pytest.mark.parametrize("replay", [False, True])
def test_decoder_on_the_device(replay, hip, abi):
    from nnc_py_amd import runtime
    runtime.clear_error()
    run_together(True, hip, abi, replay)
    code, msg = runtime.last_error()
    assert code == 0, msg
    if replay:
        hip.nnc_hip_graph_destroy()


def test_cache_read_on_the_oracle(oracle_lib, abi):
    """What is read back is whole numbers times scales, for the last rows."""
    import ctypes
    rng = np.random.default_rng(2)
    lengths, rows = [PAGE + 3, 0, 2 * PAGE], [5, 0, 2 * PAGE]
    table = rng.permutation(6).astype(I32).reshape(3, 2)
    c = s8.Cache(rng, 6, KV, PAGE, DIM, table)
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(I32)
    k, v = np.zeros((2, int(starts[-1]), KV * DIM), F32)
    arrays = [c.k, c.v, c.ks, c.vs, c.table, starts, np.array(lengths, I32), k, v]
    kept = [abi.make_tensor(a.ctypes.data, abi.NUMPY_TO_NNC[a.dtype.name], a.shape, a.nbytes) for a in arrays]
    oracle_lib.nnc_hip_kv_read(*[ctypes.pointer(t) for t, _ in kept], 0, 0)
    for b, n in enumerate(lengths):
        for i in range(rows[b]):
            t = n - rows[b] + i
            p = c.page_of(b, t)
            np.testing.assert_array_equal(k[starts[b] + i].reshape(KV, DIM), c.k[p, :, t % PAGE].astype(F32) * c.ks[p][:, None])
            np.testing.assert_array_equal(v[starts[b] + i].reshape(KV, DIM), c.v[p, :, :, t % PAGE].astype(F32) * c.vs[p][:, None])


def test_a_write_stays_where_no_node_reads_the_cache(pkg):
    from nnc_py_amd.compiler.builder import GraphBuilder
    from nnc_py_amd.compiler.executor import build_program
    b = GraphBuilder("write")
    x = b.input("x", (2, KV * DIM))
    cache = b.kv_cache("cache", 2, KV, PAGE, DIM)
    place = [b.input("table", (1, 2), "int32"), b.input("starts", (2,), "int32"), b.input("lengths", (1,), "int32")]
    b.kv_write(x, x, cache, *place)
    b.output(b.relu(x))
    for opt in (0, 1, 3):
        calls = [c.op for c in build_program(b.build(), opt).calls]
        assert sorted(calls) == ["nnc_hip_kv_write", "nnc_relu"]


def test_generated_decoder_compiles(tmp_path, pkg):
    from nnc_py_amd.compiler.compiler import Compiler
    Compiler(target="mi355x", opt_level=3).compile(decoder(3, 2), str(tmp_path), entry_point="decode")
    text = (tmp_path / "model.c").read_text()
    order = re.findall(r"^    (nnc_hip_kv_\w+)\(", text, re.M)
    assert order == ["nnc_hip_kv_write", "nnc_hip_kv_attention"] * LAYERS
    for src in ("model.c", "tensors.c", "constants_loader.c"):
        subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-D_GNU_SOURCE", f"-I{ROOT / 'include'}", "-c", str(tmp_path / src),
                        "-o", str(tmp_path / (src + ".o"))], check=True, capture_output=True, text=True)
