"""Rotary positions, tree attention and token log probabilities without a GPU:
which calls they refuse, the index arithmetic of masks, tables of angles."""

from __future__ import annotations

import subprocess
from pathlib import Path

import numpy as np
import pytest

from test_serving8_args import EINVAL, ESTATE, EUNSUPP, F16, F32, I8, I32, I64, Lib, cache, cache_changes, check

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def lib(abi, pkg):
    # the calls in order name memory that is not there: none may run where the
    # library could have been initialised, whatever another runtime says
    if Path("/dev/kfd").exists():
        pytest.skip("a GPU is there: these calls would run")
    from nnc_py_amd import runtime
    return Lib(abi, runtime)


def test_index_arithmetic_of_masks(tmp_path):
    exe = tmp_path / "tree_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'nnc-py_amd' / 'csrc'}", str(ROOT / "tests" / "native" / "tree_check.cpp"), "-o", str(exe)],
                   check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout == "ok\n", res.stdout + res.stderr


def test_rope_refusals(lib):
    t = lib.t
    far = 1 << 20
    good = {"in": t(F16, 7, 300), "weight": t(F16, 64), "angles": t(F32, 50, 32), "positions": t(I32, 7), "out": t(F16, 7, 256, data=far),
            "col": 44, "out_col": 0, "heads": 4, "dim": 64, "interleaved": 0, "eps": 1e-6}
    check(lib, "nnc_hip_rope", good, [
        ("no input", {"in": None}, EINVAL), ("no output", {"out": None}, EINVAL), ("integers", {"in": t(I32, 7, 300)}, EUNSUPP),
        ("columns", {"col": 45}, EINVAL), ("columns", {"out_col": 1}, EINVAL), ("columns", {"col": -1}, EINVAL),
        ("heads", {"heads": 0}, EINVAL), ("heads", {"heads": 65536}, EINVAL), ("dim", {"dim": 0}, EINVAL), ("dim", {"dim": -64}, EINVAL),
        ("output type", {"out": t(F32, 7, 256, data=far)}, EINVAL), ("output rows", {"out": t(F16, 8, 256, data=far)}, EINVAL),
        ("weight type", {"weight": t(F32, 64)}, EUNSUPP), ("weight size", {"weight": t(F16, 128)}, EINVAL), ("no weights", {"weight": t(F16, 64, data=0)}, EINVAL),
        ("float16 angles", {"angles": t(F16, 50, 32)}, EUNSUPP), ("odd rot", {"angles": t(F32, 50, 31)}, EINVAL),
        ("rot 0", {"angles": t(F32, 50, 0)}, EINVAL), ("rot above dim", {"angles": t(F32, 50, 66)}, EINVAL), ("no places", {"angles": t(F32, 0, 32)}, EINVAL),
        ("flat angles", {"angles": t(F32, 1600)}, EINVAL), ("angles without positions", {"positions": None}, EINVAL),
        ("positions without angles", {"angles": None}, EINVAL), ("int64 positions", {"positions": t(I64, 7)}, EUNSUPP),
        ("positions", {"positions": t(I32, 6)}, EINVAL), ("eps", {"eps": -1.0}, EINVAL), ("eps", {"eps": float("nan")}, EINVAL),
        ("eps", {"eps": float("inf")}, EINVAL),
        ("shifted by a column", {"out": t(F16, 7, 300), "out_col": 43}, EINVAL), ("over other rows", {"out": t(F16, 7, 300, data=4096 + 600), "out_col": 0}, EINVAL),
        ("other row length", {"out": t(F16, 7, 256)}, EINVAL)])
    fine = [{"out": t(F16, 7, 300), "out_col": 44}, {"weight": None, "eps": -1.0}, {"weight": t(F16, 4, 64)}, {"angles": None, "positions": None},
            {"in": t(F16, 7, 600), "out": t(F16, 7, 600), "out_col": 300}, {"eps": 0.0}, {"angles": t(F32, 1, 2)},
            {"in": t(F16, 7, 600), "out": t(F16, 7, 600, data=4096 + 600), "out_col": 0}, {"dim": 32, "heads": 8, "weight": t(F16, 8, 32)}]
    for change in fine:
        assert lib.code("nnc_hip_rope", *{**good, **change}.values()) == ESTATE, change
    assert lib.code("nnc_hip_rope", t(F16, 0, 300), None, None, None, t(F16, 0, 256), 0, 0, 4, 64, 0, 1e-6) == 0


def rope_kv_write(lib, **change):
    t = lib.t
    x = t(F16, 7, 512)
    good = {"q": x, "k": x, "v": x, "q_weight": t(F16, 64), "k_weight": t(F16, 64), "angles": t(F32, 50, 32), "positions": t(I32, 7),
            "q_out": t(F16, 7, 256, data=1 << 20), **cache(lib), "q_col": 0, "heads": 4, "k_col": 256, "v_col": 384, "interleaved": 1, "eps": 1e-6}
    return {**good, **change}


def test_rope_kv_write_refusals(lib):
    t = lib.t
    check(lib, "nnc_hip_rope_kv_write", rope_kv_write(lib), cache_changes(t) + [
        ("no keys", {"k": None}, EINVAL), ("no values", {"v": None}, EINVAL), ("integers", {"k": t(I8, 7, 512)}, EUNSUPP),
        ("queries of another type", {"q": t(F32, 7, 512)}, EINVAL), ("queries of other rows", {"q": t(F16, 6, 512)}, EINVAL),
        ("columns", {"q_col": 257}, EINVAL), ("columns", {"k_col": 385}, EINVAL), ("columns", {"v_col": -1}, EINVAL),
        ("heads", {"heads": 0}, EINVAL), ("weight without queries", {"q": None, "q_out": None}, EINVAL),
        ("output without queries", {"q": None, "q_weight": None}, EINVAL), ("weights", {"k_weight": t(F16, 3, 64)}, EINVAL),
        ("weights", {"q_weight": t(F32, 64)}, EUNSUPP), ("angles", {"angles": t(F32, 50, 128)}, EINVAL),
        ("positions without angles", {"angles": None}, EINVAL), ("positions", {"positions": t(I32, 9)}, EINVAL),
        ("output", {"q_out": t(F16, 7, 128, data=1 << 20)}, EINVAL), ("output", {"q_out": t(F32, 7, 256, data=1 << 20)}, EINVAL),
        ("queries over keys", {"q_out": None, "k_col": 192}, EINVAL), ("queries over values", {"q_out": None, "v_col": 250}, EINVAL),
        ("output over the rows", {"q_out": t(F16, 7, 256)}, EINVAL), ("eps", {"eps": float("nan")}, EINVAL)])
    fine = [{"q_out": None}, {"positions": None}, {"angles": None, "positions": None}, {"q_weight": None, "k_weight": None},
            {"q": None, "q_weight": None, "q_out": None}, {"q_weight": t(F16, 4, 64), "k_weight": t(F16, 2, 64)}]
    for change in fine:
        assert lib.code("nnc_hip_rope_kv_write", *rope_kv_write(lib, **change).values()) == ESTATE, change


def test_kv_tree_attention_refusals(lib):
    t = lib.t
    good = {"q": t(F32, 7, 300), **cache(lib), "tree": t(I32, 7, 2), "out": t(F32, 7, 256), "q_col": 44, "heads": 4, "scale": 0.125, "window": 0,
            "max_length": 0}
    check(lib, "nnc_hip_kv_tree_attention", good, cache_changes(t) + [
        ("columns", {"q_col": 45}, EINVAL), ("heads", {"heads": 3}, EINVAL), ("heads", {"heads": 0}, EINVAL), ("no q", {"q": None}, EINVAL),
        ("integers", {"q": t(I32, 7, 300)}, EUNSUPP), ("output type", {"out": t(F16, 7, 256)}, EINVAL), ("no output", {"out": None}, EINVAL),
        ("output rows", {"out": t(F32, 8, 256)}, EINVAL), ("window", {"window": -1}, EINVAL), ("max_length", {"max_length": -1}, EINVAL),
        ("scale", {"scale": 0.0}, EINVAL), ("scale", {"scale": float("nan")}, EINVAL), ("unaligned", {"out": t(F32, 7, 256, data=4100)}, EUNSUPP),
        ("no tree", {"tree": None}, EINVAL), ("tree rows", {"tree": t(I32, 6, 2)}, EINVAL), ("no words", {"tree": t(I32, 7, 0)}, EINVAL),
        ("flat tree", {"tree": t(I32, 14)}, EINVAL), ("int64 tree", {"tree": t(I64, 7, 1)}, EUNSUPP)])


def test_token_logprobs_refusals(lib):
    t = lib.t
    good = {"logits": t(F16, 2, 3, 1000), "tokens": t(I32, 6), "logprob": t(F32, 6), "entropy": t(F32, 2, 3), "top_index": t(I32, 2, 3, 5),
            "top_logprob": t(F32, 6, 5), "scale": 1.0}
    check(lib, "nnc_hip_token_logprobs", good, [
        ("no logits", {"logits": None}, EINVAL), ("integers", {"logits": t(I32, 6, 1000)}, EUNSUPP), ("no vocabulary", {"logits": t(F16, 6, 0)}, EINVAL),
        ("logprob without tokens", {"tokens": None}, EINVAL), ("tokens without logprob", {"logprob": None}, EINVAL), ("int64 tokens", {"tokens": t(I64, 6)}, EUNSUPP),
        ("tokens", {"tokens": t(I32, 5)}, EINVAL), ("logprob", {"logprob": t(F32, 7)}, EINVAL), ("types", {"entropy": t(F16, 6)}, EUNSUPP),
        ("entropy", {"entropy": t(F32, 5)}, EINVAL), ("index without values", {"top_logprob": None}, EINVAL), ("values without index", {"top_index": None}, EINVAL),
        ("alternatives", {"top_index": t(I32, 6, 65), "top_logprob": t(F32, 6, 65)}, EUNSUPP), ("alternatives", {"top_logprob": t(F32, 6, 4)}, EINVAL),
        ("alternatives", {"top_logprob": t(F32, 5, 6)}, EINVAL), ("alternatives", {"top_index": t(I32, 6, 0), "top_logprob": t(F32, 6, 0)}, EUNSUPP),
        ("rows", {"top_index": t(I32, 5, 5), "top_logprob": t(F32, 5, 5)}, EINVAL), ("types", {"top_index": t(I64, 6, 5)}, EUNSUPP),
        ("scale", {"scale": 0.0}, EINVAL), ("scale", {"scale": float("inf")}, EINVAL), ("scale", {"scale": float("nan")}, EINVAL)])
    assert lib.code("nnc_hip_token_logprobs", t(F16, 6, 1000), None, None, None, None, None, 1.0) == 0
    assert lib.code("nnc_hip_token_logprobs", t(F16, 0, 1000), t(I32, 0), t(F32, 0), None, None, None, 1.0) == 0


def test_angles(pkg):
    from nnc_py_amd import rotary
    a = rotary.angles(5000, 64)
    assert a.shape == (5000, 64) and a.dtype == np.float32
    at, i = 4999, 17
    want = at * 10000.0 ** (-2 * i / 64)
    assert abs(a[at, i] - np.cos(want)) <= 2.0 ** -24 and abs(a[at, 32 + i] - np.sin(want)) <= 2.0 ** -24
    # positions stretched: place 4 p of a table with factor 4 is place p of one without
    np.testing.assert_allclose(rotary.angles(400, 64, factor=4.0)[::4], a[:100], rtol=0, atol=2.0 ** -23)
    np.testing.assert_array_equal(rotary.angles(np.array([7, 3]), 64), a[[7, 3]])
    np.testing.assert_allclose(rotary.angles(10, 64, amplitude=1.25), 1.25 * a[:10].astype(np.float64), rtol=0, atol=1.25 * 2.0 ** -23)
    # by wavelength: short waves stay, long ones are divided, between them a line
    f, g = rotary.frequencies(64), rotary.frequencies(64, factor=8.0, original=1024, low=1.0, high=4.0)
    fits = 1024 * f / (2 * np.pi)
    np.testing.assert_array_equal(g[fits >= 4], f[fits >= 4])
    np.testing.assert_allclose(g[fits <= 1], f[fits <= 1] / 8, rtol=1e-15)
    mid = (fits > 1) & (fits < 4)
    assert mid.any() and (g[mid] < f[mid]).all() and (g[mid] > f[mid] / 8).all()
    for bad in ({"rot": 7}, {"rot": 0}, {"rot": 8, "factor": 0.0}, {"rot": 8, "original": 100, "low": 4.0, "high": 4.0}):
        with pytest.raises(ValueError):
            rotary.frequencies(**bad)
