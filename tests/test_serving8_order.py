"""Graphs that write a cache: every node sees the cache as it stood where the
node was added, at each optimisation level, whatever the passes fuse and the
sort defers. Level 0 runs the nodes as they were added; the oracle's results at
the other levels are held against it, over two runs, the cache staying."""

from __future__ import annotations

import numpy as np
import pytest

KV, PAGE, DIM, PAGES, ROWS = 2, 16, 32, 4, 2
WIDTH = KV * DIM
F32, I32 = np.float32, np.int32


class Made:
    """A builder with a cache of one sequence, its new rows the last ROWS."""

    def __init__(self, as_inputs=False):
        from nnc_py_amd.compiler.builder import GraphBuilder
        self.b = b = GraphBuilder("order")
        self.feeds = {"table": np.array([[2, 0]], I32), "starts": np.array([0, ROWS], I32), "lengths": np.array([PAGE + 3], I32)}
        self.lasting = {}
        if as_inputs:
            shapes = ((PAGES, KV, PAGE, DIM), (PAGES, KV, DIM, PAGE), (PAGES, KV), (PAGES, KV))
            self.cache = tuple(b.input(f"c{i}", s, "int8" if i < 2 else "float32") for i, s in enumerate(shapes))
            self.lasting = {n: np.zeros(s, np.int8 if i < 2 else F32) for i, (n, s) in enumerate(zip(self.cache, shapes))}
        else:
            self.cache = b.kv_cache("cache", PAGES, KV, PAGE, DIM)
        self.place = [b.input("table", (1, 2), "int32"), b.input("starts", (2,), "int32"), b.input("lengths", (1,), "int32")]

    def input(self, name, shape=(ROWS, WIDTH)):
        rng = np.random.default_rng(len(self.feeds))
        self.feeds[name] = rng.standard_normal(shape).astype(F32)
        return self.b.input(name, shape)

    def write(self, x):
        self.b.kv_write(x, x, self.cache, *self.place)

    def attend(self, q):
        return self.b.kv_attention(q, self.cache, *self.place, heads=KV)

    @property
    def k_scale(self):
        return self.cache[2]


def keys_behind_a_fused_residual(m):
    """The rows come from a convolution with a residual that is computed after
    it; the attention's query is there from the start."""
    b = m.b
    img, y = m.input("img", (1, ROWS, 8, 8)), m.input("y", (1, ROWS, 8, 8))
    w = b.const("w", np.random.default_rng(7).standard_normal((ROWS, ROWS, 1, 1)).astype(F32))
    x = b.relu(b.add(b.conv(img, w), b.exp(y)))
    m.write(b.reshape(x, (ROWS, WIDTH)))
    b.output(m.attend(m.input("q")))


def a_read_on_either_side(m):
    b = m.b
    z = m.input("z", (PAGES, KV))
    old = b.mul(m.k_scale, z)
    m.write(m.input("x"))
    b.output(b.sub(m.k_scale, old))


def a_chain_that_starts_before_the_write(m):
    b = m.b
    z = m.input("z", (PAGES, KV))
    old = b.add(m.k_scale, z)
    m.write(m.input("x"))
    b.output(b.relu(old))
    b.output(b.mul(m.k_scale, z))


def a_copy_of_the_scales(m):
    b = m.b
    old = b._out("kept", (PAGES, KV))
    b._node("Identity", [m.k_scale], [old])
    m.write(m.input("x"))
    b.output(b.sub(m.k_scale, old))


def the_scales_under_another_shape(m):
    b = m.b
    old = b.reshape(m.k_scale, (PAGES * KV,))
    m.write(m.input("x"))
    b.output(b.add(old, m.input("z", (PAGES * KV,))))


def scales_joined_and_split(m):
    b = m.b
    z = m.input("z", (PAGES, KV))
    joined = b.concat([m.k_scale, z], axis=1)
    m.write(m.input("x"))
    one, two = b.split(joined, 2, axis=1)
    b.output(b.mul(one, two))


def turned_twice(m):
    b = m.b
    once = b.transpose(m.k_scale)
    m.write(m.input("x"))
    b.output(b.transpose(once))


def the_scales_into_a_norm(m):
    b = m.b
    z = m.input("z", (PAGES, KV))
    s = b.add(m.k_scale, z)
    m.write(m.input("x"))
    one, zero = b.const("one", np.ones(KV, F32)), b.const("zero", np.zeros(KV, F32))
    b.output(b.layernorm(s, one, zero))


def a_late_addend_of_the_scales(m):
    """The scales, as they are after the write, are added to a convolution from
    before it."""
    b = m.b
    img = m.input("img", (1, 1, PAGES, KV))
    w = b.const("w", np.full((1, 1, 1, 1), 0.5, F32))
    early = b.conv(img, w)
    m.write(m.input("x"))
    scales = b.reshape(m.k_scale, (1, 1, PAGES, KV))
    b.output(b.relu(b.add(early, scales)))


def two_writes(m):
    """Both attentions see what stood there when they were added, though the
    second write's rows are there first."""
    b = m.b
    late, q = m.input("x"), m.input("q")
    m.write(b.exp(b.mul(late, q)))
    one = m.attend(q)
    m.write(late)
    b.output(one)
    b.output(m.attend(q))


def a_write_of_what_the_cache_answered(m):
    b = m.b
    q = m.input("q")
    m.write(b.add(m.attend(q), m.input("x")))
    b.output(m.attend(q))


def scales_that_begin_as_a_copy(m):
    """The cache's scales start as a copy of an input, every run."""
    b = m.b
    start = b._out("start", (PAGES, KV))
    b._node("Identity", [m.input("z", (PAGES, KV))], [start])
    m.cache = (m.cache[0], m.cache[1], start, m.cache[3])
    m.write(m.input("x"))
    b.output(m.attend(m.input("q")))


GRAPHS = [keys_behind_a_fused_residual, a_read_on_either_side, a_chain_that_starts_before_the_write, a_copy_of_the_scales,
          the_scales_under_another_shape, scales_joined_and_split, turned_twice, the_scales_into_a_norm,
          a_late_addend_of_the_scales, two_writes, a_write_of_what_the_cache_answered,
          scales_that_begin_as_a_copy]


def run(make, level, as_inputs, device, lib):
    from nnc_py_amd.compiler.executor import Executor, build_program
    m = Made(as_inputs)
    make(m)
    m.feeds["lengths"] = m.feeds["lengths"].copy()
    ex = Executor(build_program(m.b.build(), level), device, lib)
    for name, a in {**m.lasting, **m.feeds}.items():
        if name in m.b.g.tensors:
            ex.set_input(name, a)
    results = []
    for i in range(2):
        ex.run()
        results += [ex.get(o).copy() for o in m.b.g.outputs + [c for c in m.cache if c != "start"]]
        ex.set_input("lengths", m.feeds["lengths"] + I32(ROWS))
        for name in ("x", "img"):
            if name in m.feeds:
                ex.set_input(name, m.feeds[name] * F32(1.5))
    return results


@pytest.mark.parametrize("as_inputs", [False, True])
@pytest.mark.parametrize("make", GRAPHS, ids=lambda f: f.__name__)
def test_every_node_sees_the_cache_of_its_place(make, as_inputs, oracle_lib, pkg):
    want = run(make, 0, as_inputs, False, oracle_lib)
    assert any(w.any() for w in want)
    for level in (1, 2, 3):
        for got, w in zip(run(make, level, as_inputs, False, oracle_lib), want):
            np.testing.assert_allclose(got, w, rtol=1e-6, atol=1e-6, err_msg=f"level {level}")


@pytest.mark.parametrize("make", GRAPHS, ids=lambda f: f.__name__)
def test_the_calls_keep_their_order(make, pkg):
    """Nodes that read or write a tensor which one of them writes run in the
    order in which they were added."""
    from nnc_py_amd.compiler.executor import build_program

    def order(level):
        m = Made()
        make(m)
        prog = build_program(m.b.build(), level)
        held = set(m.cache)
        return [n.name for n in prog.order if held & set(n.inputs)]
    want = order(0)
    for level in (1, 2, 3):
        assert order(level) == want, level


def test_fusion_beside_a_cache_goes_on(pkg):
    """What neither reads nor writes the cache is fused as ever."""
    from nnc_py_amd.compiler.executor import build_program
    m = Made()
    b = m.b
    x, q = m.input("x"), m.input("q")
    m.write(b.relu(b.add(x, q)))
    b.output(b.sigmoid(b.add(m.attend(q), x)))
    calls = [c.op for c in build_program(b.build(), 3).calls]
    assert calls == ["nnc_add_relu", "nnc_hip_kv_write", "nnc_hip_kv_attention", "nnc_add_sigmoid"]


def half_graph(pkg):
    """Rows of a fused projection in float16: written, attended, normed."""
    from nnc_py_amd.compiler.builder import GraphBuilder
    b = GraphBuilder("half")
    qkv = b.input("qkv", (ROWS, 3 * WIDTH), "float16")
    cache = b.kv_cache("cache", PAGES, KV, PAGE, DIM)
    place = [b.input("table", (1, 2), "int32"), b.input("starts", (2,), "int32"), b.input("lengths", (1,), "int32")]
    b.kv_write(qkv, qkv, cache, *place, k_col=WIDTH, v_col=2 * WIDTH)
    a = b.output(b.kv_attention(qkv, cache, *place, heads=KV))
    b.output(b.rms_norm(a, b.const("w", np.ones(WIDTH, np.float16))))
    return b.build()


def test_attention_answers_in_the_queries_type(pkg):
    g = half_graph(pkg)
    assert [g.tensors[o].dtype for o in g.outputs] == ["float16", "float16"]


@pytest.mark.gpu
@pytest.mark.parametrize("level", [0, 3])
def test_a_half_precision_graph_on_the_device(level, hip, pkg):
    import serving8 as s8
    from nnc_py_amd import runtime
    from nnc_py_amd.compiler.executor import Executor, build_program
    runtime.clear_error()
    ex = Executor(build_program(half_graph(pkg), level), True, hip)
    rng = np.random.default_rng(3)
    table, starts = np.array([[2, 0]], I32), np.array([0, ROWS], I32)
    cache = s8.Cache(rng, PAGES, KV, PAGE, DIM, table, filled=False)
    for n in range(1, 20):  # (the first call's row before the sequence has no position)
        qkv = rng.standard_normal((ROWS, 3 * WIDTH)).astype(np.float16)
        for name, a in (("qkv", qkv), ("table", table), ("starts", starts), ("lengths", np.array([n], I32))):
            ex.set_input(name, a)
        ex.run()
        q, k, v = qkv.reshape(ROWS, 3, KV, DIM).transpose(1, 0, 2, 3)
        cache.write(k, v, starts, [n])
        out, about = s8.attention(q, cache, starts, [n], F32(DIM ** -0.5), 0)
        a, y = (ex.get(o) for o in ex.prog.graph.outputs)
        assert (np.abs(a.reshape(out.shape).astype(np.float64) - out) <= s8.attention_bound(np.float16, DIM, out, *about)).all()
        want = s8.rms_norm(a, None, np.ones(WIDTH, np.float16), 1e-6)[3]
        assert (np.abs(y.astype(np.float64) - want) <= s8.U16 * 1.01 * np.abs(want) + s8.SUB16).all()
    assert runtime.last_error()[0] == 0
