"""Each kernel of the 8-bit product and of the row operators, at sizes that the
library's rule gives to it (256 CUs): the product's calls name the kernel that
has to have run, the row operators' sizes are those of the rule. Against plain
float64 forms, as in test_serving8.py."""

from __future__ import annotations

import numpy as np
import pytest

import serving8 as s8
from serving8 import F16, F32, I8
from test_serving8 import check_norm, check_product, dev, norm_inputs, run_attention  # noqa: F401 (dev: fixture)

pytestmark = pytest.mark.gpu

# rows and columns that end inside a tile, K that ends inside a slice (128) and
# inside 16, fewer slices than stages and more
KERNELS = {
    "rows16": [(5, 300, 1040), (16, 4096, 2049), (1, 33, 5000)],
    "rows32": [(17, 2050, 80), (30, 4097, 1041)],
    "rows64": [(33, 2050, 81), (48, 4097, 145), (100, 2050, 80)],
    "64x64": [(200, 300, 640), (130, 1000, 301), (512, 130, 2064), (300, 1000, 1040)],
    "64x64_split": [(200, 64, 2064), (1024, 64, 2064), (257, 130, 3000), (130, 257, 4111), (129, 300, 4112)],
    "128x128": [(512, 4099, 81), (520, 4100, 656), (1024, 2050, 401), (1000, 4000, 1040)],
    "256x128": [(777, 5000, 80), (800, 5001, 657)],
    "256x256": [(2048, 4099, 80), (2100, 4200, 529), (2304, 4096, 1040)],
}


def ran(call):
    """Kernel names, launches and work of the timing table over `call`."""
    from nnc_py_amd import runtime
    runtime.profile_reset()
    runtime.profile_enable(True)
    try:
        call()
    finally:
        runtime.profile_enable(False)
    return {r["name"]: r for r in runtime.profile_table()}


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("kernel,size", [(k, s) for k, sizes in KERNELS.items() for s in sizes])
def test_matmul_i8_kernel(kernel, size, t, dev):  # noqa: F811
    m, n, k = size
    rng = np.random.default_rng(m + 7 * n + 13 * k)
    table = ran(lambda: check_product(dev, rng, m, n, k, t, bias=(m + n) % 2 == 0, full=k % 2 == 0))
    names = {f"nnc_hip_matmul_i8_{kernel}"}
    if k % 16 and not kernel.startswith("rows"):
        names.add("nnc_hip_matmul_i8_pack")
    assert set(table) == names


@pytest.mark.parametrize("kernel,size", [("128x128", (520, 4100, 656)), ("256x128", (777, 5000, 80)), ("256x256", (2304, 4096, 272)),
                                         ("64x64_split", (200, 64, 2064))])
def test_matmul_i8_kernel_with_operands_that_start_anywhere(kernel, size, dev):  # noqa: F811
    m, n, k = size
    rng = np.random.default_rng(k)
    table = ran(lambda: check_product(dev, rng, m, n, k, F16, shift={"w": 3, "sa": 4, "sw": 8, "b": 4, "out": 2}))
    assert set(table) == {f"nnc_hip_matmul_i8_{kernel}", "nnc_hip_matmul_i8_pack"}


def test_matmul_i8_split_sums_are_joined_alike_each_time(dev):  # noqa: F811
    """Counters and partial sums of one call are left ready for the next, of
    other sizes too: twenty calls in turn, the same bits."""
    rng = np.random.default_rng(0)
    calls = []
    for m, n, k in ((200, 64, 2064), (130, 257, 4112), (257, 130, 3008)):
        a, w = rng.integers(-127, 128, (m, k)).astype(I8), rng.integers(-127, 128, (n, k)).astype(I8)
        sa, sw = rng.uniform(0.01, 0.02, m).astype(F32), rng.uniform(0.01, 0.02, n).astype(F32)
        want = (a.astype(np.float64) @ w.astype(np.float64).T).astype(F32) * (sa[:, None] * sw)
        calls.append((dev({"a": a, "sa": sa, "w": w, "sw": sw, "out": np.zeros((m, n), F32)}), want))
    for i in range(20):
        d, want = calls[i % 3]
        d.call("nnc_hip_matmul_i8", "a", "sa", "w", "sw", None, "out")
        np.testing.assert_array_equal(d.get("out"), want)  # exact sum, one rounding of each product


@pytest.mark.parametrize("size", [(8, 512, 1024), (300, 400, 512), (300, 400, 513), (1024, 2050, 401)])
def test_matmul_i8_work_in_the_timing_table(size, dev):  # noqa: F811
    """The operation's work stands beside the launch that does it, the bytes of
    laying operands out beside that launch."""
    m, n, k = size
    rng = np.random.default_rng(1)
    table = ran(lambda: check_product(dev, rng, m, n, k, F32))
    pack = table.pop("nnc_hip_matmul_i8_pack", None)
    (product,) = table.values()
    assert product["flops"] == 2.0 * m * n * k and product["bytes"] == m * k + n * k + 4.0 * m * n
    assert (pack is not None) == (k % 16 != 0)
    if pack:
        assert pack["flops"] == 0 and pack["bytes"] == (m + n) * (k + -(-k // 16) * 16)


@pytest.mark.parametrize("window,rows,reach", [(0, 1, 4000), (1, 1, 1), (700, 1, 700), (700, 5, 704), (3999, 5, 4000), (2 ** 31 - 1, 1, 4000)])
def test_kv_attention_work_in_the_timing_table(window, rows, reach, dev):  # noqa: F811
    """The cache's bytes once: as far as the longest sequence or its window reaches."""
    rng = np.random.default_rng(2)
    table = ran(lambda: run_attention(dev, rng, [4000, 4000], [rows, rows], 4, 2, 64, 16, F16, window=window, max_length=4000, pad=0))
    assert [r["bytes"] for r in table.values()] == [2.0 * 2 * 64 * reach * 2]


# rows for every wave of the GPU and short ones (a wave a row: one, two and four
# packs a lane), outputs over 8 MiB (stored past the caches), the widest rows
# that registers hold, and wider ones
ROWS = [(4100, 64), (4096, 256), (4100, 520), (4099, 1000), (4097, 1024), (5000, 2048), (700, 16384), (3, 16384), (3, 8192), (3, 16392)]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("rows,width", ROWS)
def test_rms_norm_kernels(rows, width, int8, t, dev):  # noqa: F811
    rng = np.random.default_rng(rows + width)
    x, res, w = norm_inputs(rng, rows, width, t, True)
    check_norm(dev, x, None, w, int8)
    check_norm(dev, x, res, w, int8)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("rows,width", ROWS + [(9000, 1000)])
def test_quantize_and_dequantize_kernels(rows, width, t, dev):  # noqa: F811
    rng = np.random.default_rng(width)
    x = (rng.standard_normal((rows, width)) * rng.uniform(1e-3, 1e3, (rows, 1))).astype(t)
    d = dev({"x": x, "q": np.zeros(x.shape, I8), "s": np.zeros(rows, F32), "y": np.zeros_like(x)})
    d.call("nnc_hip_quantize_rows", "x", "q", "s")
    unit = s8.unit8(s8.absmax(x.astype(F32), 1))
    q = s8.whole8(x.astype(F32), unit[:, None])
    np.testing.assert_array_equal(d.get("s"), unit)
    np.testing.assert_array_equal(d.get("q"), q)
    d.call("nnc_hip_dequantize_rows", "q", "s", "y")
    np.testing.assert_array_equal(d.get("y"), (q.astype(F32) * unit[:, None]).astype(t))


def test_captured_products_replayed(dev, hip):  # noqa: F811
    """A norm to 8 bits and products that lay operands out, split k and take the
    largest tiles, captured together (they share the workspace) and replayed
    with other inputs, eager calls in between: the same bits as eager."""
    from nnc_py_amd import runtime
    rng = np.random.default_rng(5)
    jobs = []
    for m, n, k in ((200, 64, 2064), (300, 400, 513), (2048, 4096, 144), (4, 512, 256)):
        w = rng.integers(-127, 128, (n, k)).astype(I8)
        d = dev({"x": rng.standard_normal((m, k)).astype(F16), "one": np.ones(k, F16), "a": np.zeros((m, k), I8), "sa": np.zeros(m, F32),
                 "w": w, "sw": rng.uniform(0.01, 0.02, n).astype(F32), "b": rng.standard_normal(n).astype(F32), "out": np.zeros((m, n), F16)})
        jobs.append((d, (m, k)))

    def calls(d):
        hip.nnc_hip_rms_norm(d.t("x"), None, d.t("one"), None, d.t("a"), d.t("sa"), 1e-6)
        hip.nnc_hip_matmul_i8(d.t("a"), d.t("sa"), d.t("w"), d.t("sw"), d.t("b"), d.t("out"))
    for d, _ in jobs:  # the workspace has its size before the capture
        calls(d)
    runtime.sync()
    runtime.check(hip.nnc_hip_graph_begin(), "begin")
    for d, _ in jobs:
        calls(d)
    runtime.check(hip.nnc_hip_graph_end(), "end")
    for i in range(5):
        for d, shape in jobs:
            d.set("x", (rng.standard_normal(shape) * (i + 1)).astype(F16))
        runtime.check(hip.nnc_hip_graph_launch(), "launch")
        runtime.sync()
        got = [d.get("out") for d, _ in jobs]
        for (d, _), replayed in zip(jobs, got):
            assert replayed.any()
            calls(d)
            runtime.sync()
            np.testing.assert_array_equal(d.get("out"), replayed)
    assert runtime.last_error()[0] == 0
    hip.nnc_hip_graph_destroy()
