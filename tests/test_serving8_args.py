"""The 8-bit serving operators without a GPU: which calls they refuse, and the
index arithmetic of ragged batches with any numbers in the device arrays."""

from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
EINVAL, EUNSUPP, ESTATE = 1, 4, 5
F32, F16, I32, I8, U8, I64 = 0, 1, 2, 3, 4, 6
SIZE = {F32: 4, F16: 2, I32: 4, I8: 1, U8: 1, I64: 8}


def test_index_arithmetic_of_ragged_batches(tmp_path):
    exe = tmp_path / "ragged_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'nnc-py_amd' / 'csrc'}", str(ROOT / "tests" / "native" / "ragged_check.cpp"), "-o", str(exe)],
                   check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout == "ok\n", res.stdout + res.stderr


class Lib:
    """The library in a process that has not initialised it: a call whose
    arguments are in order ends with ESTATE, before any device call."""

    def __init__(self, abi, runtime):
        self.abi, self.lib = abi, runtime.load()
        self.rt = runtime
        self.kept = []

    def t(self, dtype, *shape, data=4096, rank=None):
        n = SIZE[dtype]
        for d in shape:
            n *= max(d, 0)
        t, sh = self.abi.make_tensor(data, dtype, shape, n)
        if rank is not None:
            t.ndim = rank
        self.kept += [t, sh]
        return ctypes.pointer(t)

    def code(self, fn, *args):
        self.rt.clear_error()
        getattr(self.lib, fn)(*args)
        return self.rt.last_error()[0]


@pytest.fixture
def lib(abi, pkg):
    import torch
    from nnc_py_amd import runtime
    if torch.cuda.is_available():
        pytest.skip("a GPU is there: these calls would run")
    if not runtime.LIB_PATH.exists():
        pytest.fail("libnnc_hip.so is not built: run __graft_entry__.build()")
    return Lib(abi, runtime)


def variants(good, changes):
    """good: argument dict; changes: (what, {argument: replacement}, code)."""
    for what, change, code in changes:
        yield what, {**good, **change}, code


def check(lib, fn, good, changes):
    assert lib.code(fn, *good.values()) == ESTATE, "the call in order"
    for what, args, code in variants(good, changes):
        assert lib.code(fn, *args.values()) == code, what


def test_rms_norm_refusals(lib):
    t = lib.t
    good = {"in": t(F16, 4, 64), "res": t(F16, 4, 64), "w": t(F16, 64), "sum": t(F16, 4, 64), "out": t(I8, 4, 64),
            "scale": t(F32, 4), "eps": 1e-6}
    check(lib, "nnc_hip_rms_norm", good, [
        ("no input", {"in": None}, EINVAL), ("no weight", {"w": None}, EINVAL), ("no output", {"out": None}, EINVAL),
        ("no data", {"res": t(F16, 4, 64, data=0)}, EINVAL), ("integers", {"in": t(I32, 4, 64)}, EUNSUPP),
        ("mixed types", {"w": t(F32, 64)}, EUNSUPP), ("mixed residual", {"res": t(F32, 4, 64)}, EUNSUPP),
        ("float output of another type", {"out": t(F32, 4, 64), "scale": None}, EUNSUPP), ("uint8 output", {"out": t(U8, 4, 64)}, EUNSUPP),
        ("scale with a float output", {"out": t(F16, 4, 64)}, EINVAL), ("int8 without scale", {"scale": None}, EINVAL),
        ("scales of another count", {"scale": t(F32, 5)}, EINVAL), ("scales of another type", {"scale": t(F16, 4)}, EINVAL),
        ("weight of another width", {"w": t(F16, 32)}, EINVAL), ("output of other rows", {"out": t(I8, 2, 128)}, EINVAL),
        ("residual of another size", {"res": t(F16, 5, 64)}, EINVAL), ("sum without residual", {"res": None}, EINVAL),
        ("eps 0", {"eps": 0.0}, EINVAL), ("eps NaN", {"eps": float("nan")}, EINVAL), ("negative extent", {"in": t(F16, -4, 64)}, EINVAL),
        ("no extents", {"in": t(F16, 4, 64, rank=0)}, EINVAL)])


def test_row_refusals(lib):
    t = lib.t
    check(lib, "nnc_hip_quantize_rows", {"in": t(F32, 4, 64), "out": t(I8, 4, 64), "scale": t(F32, 4)}, [
        ("no scale", {"scale": None}, EINVAL), ("types", {"in": t(I8, 4, 64)}, EUNSUPP), ("types", {"out": t(U8, 4, 64)}, EUNSUPP),
        ("sizes", {"out": t(I8, 4, 32)}, EINVAL), ("scales", {"scale": t(F32, 64)}, EINVAL)])
    check(lib, "nnc_hip_dequantize_rows", {"in": t(I8, 4, 64), "scale": t(F32, 4), "out": t(F16, 4, 64)}, [
        ("no input", {"in": None}, EINVAL), ("types", {"out": t(I32, 4, 64)}, EUNSUPP), ("sizes", {"in": t(I8, 8, 32)}, EINVAL),
        ("scales", {"scale": t(F32, 3)}, EINVAL)])


def test_matmul_i8_refusals(lib):
    t = lib.t
    good = {"a": t(I8, 2, 3, 64), "sa": t(F32, 6), "w": t(I8, 10, 64), "sw": t(F32, 10), "bias": t(F32, 10), "out": t(F16, 2, 3, 10)}
    check(lib, "nnc_hip_matmul_i8", good, [
        ("no weights", {"w": None}, EINVAL), ("uint8", {"a": t(U8, 2, 3, 64)}, EUNSUPP), ("float16 bias", {"bias": t(F16, 10)}, EUNSUPP),
        ("integer output", {"out": t(I32, 2, 3, 10)}, EUNSUPP), ("rows of w", {"w": t(I8, 10, 32)}, EINVAL),
        ("w of three extents", {"w": t(I8, 1, 10, 64)}, EINVAL), ("output width", {"out": t(F16, 2, 3, 11)}, EINVAL),
        ("output rows", {"out": t(F16, 5, 10)}, EINVAL), ("scales", {"sa": t(F32, 5)}, EINVAL), ("scales", {"sw": t(F32, 6)}, EINVAL),
        ("bias", {"bias": t(F32, 6)}, EINVAL), ("no k", {"a": t(I8, 2, 3, 0), "w": t(I8, 10, 0)}, EUNSUPP),
        ("too long", {"a": t(I8, 6, 131072), "w": t(I8, 10, 131072), "out": t(F16, 6, 10)}, EUNSUPP)])
    assert lib.code("nnc_hip_matmul_i8", t(I8, 0, 64), t(F32, 0), t(I8, 10, 64), t(F32, 10), None, t(F32, 0, 10)) == 0


def cache(lib, **change):
    t = lib.t
    good = {"k_cache": t(I8, 9, 2, 16, 64), "v_cache": t(I8, 9, 2, 64, 16), "k_scale": t(F32, 9, 2), "v_scale": t(F32, 9, 2),
            "table": t(I32, 3, 4), "starts": t(I32, 4), "lengths": t(I32, 3)}
    return {**good, **change}


def cache_changes(t):
    return [("no cache", {"k_cache": None}, EINVAL), ("no lengths", {"lengths": None}, EINVAL), ("no data", {"table": t(I32, 3, 4, data=0)}, EINVAL),
            ("uint8 cache", {"v_cache": t(U8, 9, 2, 64, 16)}, EUNSUPP), ("float16 scales", {"k_scale": t(F16, 9, 2)}, EUNSUPP),
            ("int64 table", {"table": t(I64, 3, 4)}, EUNSUPP), ("int64 lengths", {"lengths": t(I64, 3)}, EUNSUPP),
            ("V like K", {"v_cache": t(I8, 9, 2, 16, 64)}, EINVAL), ("other pages", {"v_cache": t(I8, 8, 2, 64, 16)}, EINVAL),
            ("rank", {"k_cache": t(I8, 18, 16, 64)}, EINVAL), ("scales", {"v_scale": t(F32, 9)}, EINVAL),
            ("page of 8", {"k_cache": t(I8, 9, 2, 8, 64), "v_cache": t(I8, 9, 2, 64, 8)}, EUNSUPP),
            ("page of 24", {"k_cache": t(I8, 9, 2, 24, 64), "v_cache": t(I8, 9, 2, 64, 24)}, EUNSUPP),
            ("page of 272", {"k_cache": t(I8, 9, 2, 272, 64), "v_cache": t(I8, 9, 2, 64, 272)}, EUNSUPP),
            ("dim of 96", {"k_cache": t(I8, 9, 2, 16, 96), "v_cache": t(I8, 9, 2, 96, 16)}, EUNSUPP),
            ("no pages", {"k_cache": t(I8, 0, 2, 16, 64), "v_cache": t(I8, 0, 2, 64, 16), "k_scale": t(F32, 0, 2), "v_scale": t(F32, 0, 2)}, EINVAL),
            ("starts", {"starts": t(I32, 3)}, EINVAL), ("lengths", {"lengths": t(I32, 4)}, EINVAL), ("flat table", {"table": t(I32, 12)}, EINVAL),
            ("unaligned", {"k_cache": t(I8, 9, 2, 16, 64, data=4104)}, EUNSUPP)]


def test_kv_write_and_read_refusals(lib):
    t = lib.t
    rows = [("columns", {"k_col": 65}, EINVAL), ("columns", {"v_col": -1}, EINVAL), ("types", {"k": t(I8, 7, 192)}, EUNSUPP),
            ("mixed types", {"v": t(F32, 7, 192)}, EINVAL), ("mixed rows", {"v": t(F16, 6, 192)}, EINVAL), ("no rows' data", {"k": None}, EINVAL)]
    good = {"k": t(F16, 7, 192), "v": t(F16, 7, 192), **cache(lib), "k_col": 0, "v_col": 64}
    check(lib, "nnc_hip_kv_write", good, cache_changes(t) + rows)
    good = {**cache(lib), "k": t(F16, 7, 192), "v": t(F16, 7, 192), "k_col": 0, "v_col": 64}
    check(lib, "nnc_hip_kv_read", good, cache_changes(t) + rows)


def test_kv_attention_refusals(lib):
    t = lib.t
    good = {"q": t(F32, 7, 300), **cache(lib), "out": t(F32, 7, 256), "q_col": 44, "heads": 4, "scale": 0.125, "window": 0, "max_length": 0}
    check(lib, "nnc_hip_kv_attention", good, cache_changes(t) + [
        ("columns", {"q_col": 45}, EINVAL), ("heads", {"heads": 3}, EINVAL), ("heads", {"heads": 0}, EINVAL), ("no q", {"q": None}, EINVAL),
        ("integers", {"q": t(I32, 7, 300)}, EUNSUPP), ("output type", {"out": t(F16, 7, 256)}, EINVAL), ("no output", {"out": None}, EINVAL),
        ("output rows", {"out": t(F32, 8, 256)}, EINVAL), ("output shape", {"out": t(F32, 7 * 256)}, EINVAL), ("window", {"window": -1}, EINVAL),
        ("max_length", {"max_length": -1}, EINVAL), ("scale", {"scale": 0.0}, EINVAL), ("scale", {"scale": float("inf")}, EINVAL),
        ("scale", {"scale": float("nan")}, EINVAL), ("unaligned", {"out": t(F32, 7, 256, data=4100)}, EUNSUPP)])


def test_as_many_cached_heads_as_a_grid_has_rows_for(lib):
    """K and V of a page and head are rows of a grid: 32767 heads at most."""
    t = lib.t
    for heads, code in ((32767, ESTATE), (32768, EINVAL)):
        args = {**cache(lib, k_cache=t(I8, 1, heads, 256, 256), v_cache=t(I8, 1, heads, 256, 256), k_scale=t(F32, 1, heads),
                        v_scale=t(F32, 1, heads))}
        x = t(F16, 7, heads * 256)
        assert lib.code("nnc_hip_kv_write", x, x, *args.values(), 0, 0) == code
        assert lib.code("nnc_hip_kv_read", *args.values(), x, x, 0, 0) == code
        assert lib.code("nnc_hip_kv_attention", x, *args.values(), x, 0, heads, 1.0, 0, 0) == code


def test_every_kernel_with_large_lds_raises_its_own_limit(pkg):
    """The limit of dynamic LDS belongs to a kernel: each one that is launched
    with more than 64 KB (pages of 256 positions by 256) has a flag of its own
    for having raised it."""
    from nnc_py_amd import runtime
    names = subprocess.run(["nm", str(runtime.LIB_PATH)], check=True, capture_output=True, text=True).stdout.split()
    kernels = {n.removeprefix("_ZN3nnc") for n in names if re.fullmatch(r"_ZN3nnc\d+kv_\w+_quads_k\w+Li1024E\w+", n)}
    assert len(kernels) == 5
    flags = [n for n in names if n.startswith("_ZGV") and "launch_quads" in n]
    for k in kernels:
        assert any(k in f for f in flags), k
