"""The serving ops on the GPU against the oracle in float64 (``oracle.serving_eval``).

Tolerances follow from the kernels' roundings (u = 2^-24, half a step of fp32):

* rms_norm: h is one fp32 addition (exact match), y one rounding of a float64 value
  (1.01 u of itself); 8-bit values and scales match the oracle's exactly (both sides
  round a float64 quotient; the inputs are no ties).
* cache: exact, bytes and scales.
* matmul_int4: see ``_int4_bound``.
* paged_attention: see ``_attention_bound``.
"""

from __future__ import annotations

import threading

import numpy as np
import pytest

from metellus_amd.api import compile_program, run, run_batch
from metellus_amd.orchestrator import KVCache, Operations
from metellus_amd.runtime import Buffer, Dispatch, Runtime, hip_backend
from oracle import serving_eval
from oracle.ir_eval import evaluate

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = ["float32", "int8", "float8_e4m3"]


def _put(ops: Operations, name: str, a: np.ndarray) -> None:
    ops.input(name, a.shape, dtype=str(a.dtype))
    ops.from_numpy(a, name)


def _close(got, want, bound):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    flat = np.isfinite(want)
    np.testing.assert_array_equal(got[~flat & ~np.isnan(want)], want[~flat & ~np.isnan(want)])
    bound = np.broadcast_to(bound, want.shape)
    off = np.abs(got - want)[flat]
    assert np.all(off <= bound[flat]), f"off by {np.max(off / np.maximum(bound[flat], 1e-300)):.3g} times the bound"


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------


def _norm_check(ops, eight: bool, summed: bool):
    env, ref = run(ops).env, evaluate(ops)
    if summed:
        np.testing.assert_array_equal(env["h"], ref["h"])
    if eight:
        np.testing.assert_array_equal(env["s"], ref["s"])
        np.testing.assert_array_equal(env["y"], ref["y"])
        with np.errstate(invalid="ignore"):
            want = env["y"].astype(np.float32) * env["s"][:, None]
        np.testing.assert_array_equal(env["z"], want)
    else:
        _close(env["y"], ref["y"], 1.01 * U * np.abs(ref["y"]) + 1e-45)


@pytest.mark.parametrize("rows, cols", [
    (1, 1), (1, 3), (5, 64), (3, 255), (300, 256), (1, 4096), (70, 4096), (37, 1023), (2, 8191), (9, 16384), (2, 40001),
    (1100, 130),
])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("eight", [False, True])
def test_rms_norm(rows, cols, residual, eight):
    rng = np.random.default_rng(rows * 100003 + cols)
    ops = Operations()
    _put(ops, "x", rng.standard_normal((rows, cols)).astype(np.float32))
    _put(ops, "w", (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32))
    kwargs = {}
    if residual:
        _put(ops, "r", (3 * rng.standard_normal((rows, cols))).astype(np.float32))
        kwargs = {"residual": "r", "sum_out": "h"}
    ops.rms_norm("x", out="y", weight="w", scales="s" if eight else None, **kwargs)
    if eight:
        ops.dequantize("y", scales="s", out="z")
    _norm_check(ops, eight, residual)


@pytest.mark.parametrize("eight", [False, True])
def test_rms_norm_of_strided_rows(eight):
    """x a transposed view, the residual rows with gaps, no weight."""
    rng = np.random.default_rng(5)
    ops = Operations()
    _put(ops, "x_", rng.standard_normal((130, 33)).astype(np.float32))
    ops.transpose("x_", out="x")
    ops.input("r", (33, 130), row_stride=130, col_stride=1)
    ops.from_numpy(rng.standard_normal((33, 130)).astype(np.float32), "r")
    ops.rms_norm("x", out="y", residual="r", sum_out="h", scales="s" if eight else None)
    if eight:
        ops.dequantize("y", scales="s", out="z")
    _norm_check(ops, eight, True)


def test_rms_norm_special_rows():
    """Zeros (eps keeps them), the largest and the smallest values, infinities and NaN."""
    x = np.random.default_rng(6).standard_normal((7, 300)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e38)
    x[2] *= np.float32(1e-38)
    x[3, 17] = np.inf
    x[4, 200] = np.nan
    x[5, :] = 0
    x[5, 7] = 1e-45
    for eight in (False, True):
        ops = Operations()
        _put(ops, "x", x)
        ops.rms_norm("x", out="y", scales="s" if eight else None)
        if eight:
            ops.dequantize("y", scales="s", out="z")
        env = run(ops).env
        if eight:
            ref = evaluate(ops)
            np.testing.assert_array_equal(env["s"], ref["s"])
            np.testing.assert_array_equal(env["y"], ref["y"])
            assert np.all(np.isnan(env["z"][3:5])) and np.all(env["z"][0] == 0)
        else:
            ref = evaluate(ops)["y"]
            # a row with an infinity: inf / inf at it, 0 elsewhere
            _close(env["y"], ref, 1.01 * U * np.abs(ref) + 1e-45)


@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 5), (4, 16), (7, 1023), (1, 4097)])
def test_dequantize(rows, cols):
    rng = np.random.default_rng(rows + cols)
    ops = Operations()
    _put(ops, "q", rng.integers(-128, 128, (rows, cols)).astype(np.int8))
    s = rng.standard_normal(rows).astype(np.float32)
    s[-1] = np.nan
    _put(ops, "s", s)
    ops.dequantize("q", scales="s", out="y")
    np.testing.assert_array_equal(run(ops).env["y"], ops.uploads["q"].astype(np.float32) * s[:, None])


# ---------------------------------------------------------------------------
# 4-bit products
# ---------------------------------------------------------------------------


def _int4_bound(ops: Operations) -> np.ndarray:
    """Per block of 128 k and row n, with s the group's scale:

    * x in fp32 becomes multiples of 2^-30 of a power of two P, max < P <= 2 max:
      128 * (8 + |8 - z|) * 2 max * 2^-30 * |s| (truncation, so a whole step);
    * the product's digits are exact integers; hi and lo each round once (lo < 2^30
      steps, 2^6 steps of 2^-30 P / 16), their fma once, with zeros another fma of
      that on both terms, times s, the addition: under 8 u of sum |x| (8 + |8 - z|) |s|,
      and 2^6 * 2 max * 2^-30 |s|;
    * adding up: a running sum of a wave's groups, then of at most 16 waves that have a
      block each at the least: under groups + 8 terms, u each of the magnitude so far.
    """
    (op,) = ops.build()
    x = np.abs(ops.uploads["x"].astype(np.float64))
    s = np.abs(ops.uploads["s"].astype(np.float64))
    z = ops.uploads["z"].astype(np.float64) if op.zeros is not None else np.full(s.shape, 8.0)
    weight = (8 + np.abs(8 - z)) * s
    k, group = x.shape[1], op.group
    total, steps = 0.0, 0.0
    for g in range(k // group):
        xs = x[:, g * group : (g + 1) * group]
        total = total + xs.sum(axis=1)[:, None] * weight[None, :, g]
        blk = g * group // 128
        top = x[:, blk * 128 : blk * 128 + 128].max(axis=1)
        steps = steps + top[:, None] * 2.0**-29 * (group * weight[:, g] + 64 * s[:, g])[None]
    bound = (8 + k // group + 8) * U * total
    if op.x_scales is None:
        return bound + steps
    return (bound + 2 * U * total) * np.abs(ops.uploads["xs"].astype(np.float64))[:, None]


def _int4(rows, k, n, group, eight, zeros, seed, strides=False):
    rng = np.random.default_rng(seed)
    ops = Operations()
    if eight:
        _put(ops, "x", rng.integers(-127, 128, (rows, k)).astype(np.int8))
        _put(ops, "xs", rng.uniform(0.01, 0.02, rows).astype(np.float32))
    elif strides:
        ops.input("x_", (k, rows))
        ops.from_numpy(rng.standard_normal((k, rows)).astype(np.float32), "x_")
        ops.transpose("x_", out="x")
    else:
        _put(ops, "x", rng.standard_normal((rows, k)).astype(np.float32))
    _put(ops, "w", rng.integers(0, 256, (n, k // 2)).astype(np.uint8))
    _put(ops, "s", rng.uniform(-0.02, 0.02, (n, k // group)).astype(np.float32))
    if zeros:
        _put(ops, "z", rng.uniform(0, 15, (n, k // group)).astype(np.float32))
    ops.matmul_int4("x", weights="w", scales="s", out="y", zeros="z" if zeros else None, x_scales="xs" if eight else None)
    return ops


@pytest.mark.parametrize("rows, k, n", [
    (1, 32, 1), (1, 128, 16), (2, 160, 17), (1, 4096, 100), (3, 1024, 64), (4, 416, 33), (5, 5024, 99), (8, 768, 1000),
    (13, 256, 31), (16, 2048, 48), (17, 128, 16), (50, 320, 70), (1, 128, 16500), (6, 128, 33000),
])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
def test_matmul_int4(rows, k, n, group, eight, zeros):
    group = group if k % group == 0 else 32
    ops = _int4(rows, k, n, group, eight, zeros, rows * 1000 + k + n)
    got, want = run(ops).env["y"], evaluate(ops)["y"]
    assert got.shape == (rows, n) and got.dtype == np.float32
    _close(got, want, _int4_bound(ops))


@pytest.mark.parametrize("rows, k, n, group, eight, zeros", [
    # enough weight rows that the waves share x: one, two and more rows, k in phases,
    # ragged, weight rows that end inside a tile, more rows than one pass takes
    (1, 1056, 24590, 32, False, True), (2, 1152, 24577, 64, False, False), (3, 640, 33000, 128, False, True),
    (16, 1632, 24600, 32, False, False), (16, 1664, 24576, 128, False, True), (7, 1024, 24579, 64, False, True),
    (20, 416, 24601, 32, False, True), (16, 1632, 24600, 32, True, True), (5, 7744, 24577, 64, True, False),
    (6, 416, 16400, 32, False, True), (4, 416, 20479, 32, False, True), (16, 384, 16385, 128, True, False),
    # sixteen waves to a making of digits, k in phases and not
    (16, 1728, 65540, 64, False, True), (7, 384, 65536, 128, False, False), (11, 352, 70001, 32, False, False),
    # two tiles of weight rows a wave, with an odd number of tiles and without
    (5, 416, 4099, 32, False, True), (16, 1056, 4128, 32, False, True), (9, 512, 8200, 128, False, False),
    (16, 704, 4100, 64, True, True), (6, 384, 5000, 128, True, False), (33, 288, 4097, 32, True, True),
    # four tiles
    (5, 416, 8205, 32, False, True), (16, 704, 16384, 64, False, True), (8, 1152, 11008, 128, False, False),
    (12, 640, 9000, 128, False, True), (20, 288, 8193, 32, False, False),
    # sixteen waves, shares of k that differ by one, k shorter than the waves
    (1, 5024, 2000, 32, False, True), (2, 4416, 300, 64, False, False), (4, 2592, 4096, 32, False, True),
    (8, 3200, 500, 128, False, True), (16, 11008, 40, 64, True, False), (1, 2080, 33, 32, True, True),
])
def test_matmul_int4_however_it_is_cut(rows, k, n, group, eight, zeros):
    ops = _int4(rows, k, n, group, eight, zeros, rows + k + n)
    _close(run(ops).env["y"], evaluate(ops)["y"], _int4_bound(ops))


@pytest.mark.parametrize("rows, n", [(1, 24577), (6, 24577), (6, 4100), (1, 100)])
def test_matmul_int4_values_that_are_not_finite_however_it_is_cut(rows, n):
    """Blocks at the ends and inside a wave's share of k; the row's other blocks hold
    finite values, the row after it stays finite."""
    ops = _int4(rows, 1696, n, 32, False, False, n)
    x = ops.uploads["x"]
    x[0, 3] = np.inf
    if rows > 5:
        x[2, 1695], x[4, 800], x[4, 1000] = np.nan, np.inf, -np.inf
    got, want = run(ops).env["y"], evaluate(ops)["y"]
    with np.errstate(invalid="ignore"):
        _close(got, want, np.nan_to_num(_int4_bound(ops), nan=0.0, posinf=0.0))
    if rows > 5:
        assert np.all(np.isfinite(got[[1, 3, 5]])) and np.all(np.isnan(got[2]))


def test_matmul_int4_of_a_transposed_x():
    ops = _int4(7, 288, 40, 32, False, True, 3, strides=True)
    want = evaluate(ops)["y"]
    x = ops.uploads["x_"].T
    ops._uploads["x"] = np.ascontiguousarray(x)  # (for the bound alone)
    bound = _int4_bound(ops)
    del ops._uploads["x"]
    _close(run(ops).env["y"], want, bound)


def test_matmul_int4_ranges_and_special_values():
    """Blocks of very different size in a row, subnormal and huge x, zero rows, and rows
    with infinities and NaN, whose other blocks and neighbours are as ever."""
    ops = _int4(9, 512, 37, 64, False, True, 4)
    x = ops.uploads["x"]
    x[0, :128] *= np.float32(1e30)
    x[1, 128:256] *= np.float32(1e-30)
    x[2] = (x[2].astype(np.float64) * 1e-40).astype(np.float32)
    x[3] = 0
    x[4, 5] = 3e38
    x[5, 130] = np.inf
    x[6, 300] = np.nan
    x[7, 10], x[7, 400] = np.inf, -np.inf
    x[8, 64:70] = -np.inf
    got, want = run(ops).env["y"], evaluate(ops)["y"]
    with np.errstate(invalid="ignore", over="ignore"):
        bound = np.nan_to_num(_int4_bound(ops), nan=0.0, posinf=0.0) + 2e-45
        want = np.where(np.abs(want) > np.finfo(np.float32).max, np.copysign(np.inf, want), want)
    _close(got, want, bound)


def test_matmul_int4_nibble_order_and_zero():
    """q = 8 with no zeros is nothing; one q of 9 takes one x out, exactly."""
    k = 256
    x = np.arange(1, k + 1, dtype=np.float32)[None]
    for at in (0, 1, 31, 32, 127, 128, 255):
        w = np.full((3, k // 2), 0x88, np.uint8)
        w[1, at // 2] += 16 if at % 2 else 1
        ops = Operations()
        _put(ops, "x", x)
        _put(ops, "w", w)
        _put(ops, "s", np.ones((3, k // 128), np.float32))
        ops.matmul_int4("x", weights="w", scales="s", out="y")
        np.testing.assert_array_equal(run(ops).env["y"], [[0, at + 1, 0]])


# ---------------------------------------------------------------------------
# cache
# ---------------------------------------------------------------------------


def _state(spec: KVCache, data: np.ndarray):
    """Values as bytes and scales of all pages (the padding apart)."""
    parts = [serving_eval._page_parts(spec, np.ascontiguousarray(data), p) for p in range(spec.pages)]
    return np.stack([p[0] for p in parts]), None if parts[0][1] is None else np.stack([p[1] for p in parts])


def _same_state(spec, got, want):
    for a, b in zip(_state(spec, got), _state(spec, want)):
        if a is not None:
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pages, page_size, kv_heads, dim, tokens", [
    (1, 1, 1, 16, 1), (5, 4, 2, 48, 7), (9, 16, 8, 128, 40), (3, 20, 3, 80, 33), (40, 64, 1, 256, 2100), (7, 3, 33, 16, 5),
    (90, 64, 4, 32, 5001), (150, 128, 2, 16, 18005),
])
def test_cache_write_and_read(dtype, pages, page_size, kv_heads, dim, tokens):
    spec = KVCache(pages=pages, page_size=page_size, kv_heads=kv_heads, dim=dim, dtype=dtype)
    rng = np.random.default_rng(pages * 7 + dim)
    ops = Operations()
    ops.kv_cache("cache", pages=pages, page_size=page_size, kv_heads=kv_heads, dim=dim, dtype=dtype)
    old = rng.standard_normal((2, spec.slots, kv_heads, dim)).astype(np.float32)
    ops.from_numpy(spec.pack(old[0], old[1]), "cache")
    for name in ("k", "v"):
        _put(ops, name, (10 ** rng.uniform(-3, 3, (tokens, 1)) * rng.standard_normal((tokens, spec.row))).astype(np.float32))
    slots = rng.permutation(max(tokens, spec.slots))[:tokens].astype(np.int32)  # those past the cache are passed over
    if tokens > 4:
        slots[1], slots[2], slots[4] = -1, np.int32(2**31 - 1), slots[0]  # padding, and the same slot twice
    _put(ops, "slots", slots)
    back = np.concatenate([rng.permutation(spec.slots), [-5, spec.slots]]).astype(np.int32)
    _put(ops, "back", back)
    ops.cache_write("cache", k="k", v="v", slots="slots", out="written")
    ops.cache_read("written", slots="back", k_out="kb", v_out="vb")
    env, ref = run(ops).env, evaluate(ops)
    _same_state(spec, env["written"], ref["written"])
    for name in ("kb", "vb"):
        np.testing.assert_array_equal(env[name], ref[name].astype(np.float32))
        assert np.all(env[name][-2:] == 0)


@pytest.mark.parametrize("dtype", ["int8", "float8_e4m3"])
def test_cache_write_rounds_to_the_nearest_step(dtype):
    """Values on and next to every border between two steps, at scales from the
    smallest to the largest: the exact quotient decides."""
    rng = np.random.default_rng(8)
    steps = np.arange(-127, 127) + 0.5 if dtype == "int8" else np.concatenate(
        [(serving_eval.E4M3[:126] + serving_eval.E4M3[1:127]) / 2, -serving_eval.E4M3[:127]])
    peak = 127.0 if dtype == "int8" else 448.0
    spec = KVCache(pages=64, page_size=1, kv_heads=1, dim=256, dtype=dtype)
    rows = []
    for i in range(spec.slots):
        scale = np.float32(2.0 ** rng.uniform(-149 + 9, 118) if i % 4 else 2.0 ** rng.integers(-130, 118))
        row = (np.resize(steps, 256) * np.float64(scale)).astype(np.float32)
        row[1::3] = np.nextafter(row[1::3], np.float32(np.inf))
        row[2::3] = np.nextafter(row[2::3], np.float32(-np.inf))
        row[0] = np.float32(np.float64(scale) * peak)
        rows.append(row)
    k = np.stack(rows)
    k[-1], k[-2], k[-3, 5], k[-4, 6] = 0, 1e-45, np.nan, -np.inf
    ops = Operations()
    ops.kv_cache("cache", pages=64, page_size=1, kv_heads=1, dim=256, dtype=dtype)
    ops.from_numpy(spec.empty(), "cache")
    _put(ops, "k", k)
    _put(ops, "v", -k)
    _put(ops, "slots", rng.permutation(64).astype(np.int32))
    ops.cache_write("cache", k="k", v="v", slots="slots", out="written")
    _same_state(spec, run(ops).env["written"], evaluate(ops)["written"])


@pytest.mark.parametrize("tokens, kv_heads", [(100, 1), (300, 8), (3000, 2)])
def test_of_rows_that_name_one_slot_the_last_is_stored(tokens, kv_heads):
    spec = KVCache(pages=4, page_size=4, kv_heads=kv_heads, dim=16, dtype="int8")
    rng = np.random.default_rng(tokens)
    ops = Operations()
    ops.kv_cache("cache", pages=4, page_size=4, kv_heads=kv_heads, dim=16, dtype="int8")
    ops.from_numpy(spec.empty(), "cache")
    for name in ("k", "v"):
        _put(ops, name, rng.standard_normal((tokens, spec.row)).astype(np.float32))
    _put(ops, "slots", rng.integers(-2, 18, tokens).astype(np.int32))
    ops.cache_write("cache", k="k", v="v", slots="slots", out="written")
    want = evaluate(ops)["written"]
    for _ in range(3):
        _same_state(spec, run(ops).env["written"], want)


def test_cache_write_of_strided_rows():
    spec = KVCache(pages=3, page_size=8, kv_heads=2, dim=32, dtype="float8_e4m3")
    rng = np.random.default_rng(11)
    ops = Operations()
    ops.kv_cache("cache", pages=3, page_size=8, kv_heads=2, dim=32, dtype="float8_e4m3")
    ops.from_numpy(spec.empty(), "cache")
    _put(ops, "k_", rng.standard_normal((64, 9)).astype(np.float32))
    ops.transpose("k_", out="k")
    _put(ops, "v_", rng.standard_normal((18, 32)).astype(np.float32))
    ops.reshape("v_", (9, 64), out="v")
    _put(ops, "slots", rng.permutation(24)[:9].astype(np.int32))
    ops.cache_write("cache", k="k", v="v", slots="slots", out="written")
    _same_state(spec, run(ops).env["written"], evaluate(ops)["written"])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def _attention(dtype, heads, kv_heads, dim, page_size, width, lengths, seed=0, holes=(), scale=None):
    """A program over pages in no order; rows that no position reaches hold NaN."""
    rng = np.random.default_rng(seed)
    b = len(lengths)
    used = [min(width, max(0, -(-n // page_size))) for n in lengths]
    pages = sum(used) + 2
    spec = KVCache(pages=pages, page_size=page_size, kv_heads=kv_heads, dim=dim, dtype=dtype)
    k, v = rng.standard_normal((2, spec.slots, kv_heads, dim)).astype(np.float32)
    order, at = rng.permutation(pages), 0
    table = np.full((b, width), -1, np.int32)
    live = np.zeros(spec.slots, bool)
    for i, u in enumerate(used):
        table[i, :u] = order[at : at + u]
        at += u
        for p in range(min(lengths[i], width * page_size)):
            live[table[i, p // page_size] * page_size + p % page_size] = True
    for i, page, bad in holes:
        table[i, page] = bad
    k[~live], v[~live] = np.nan, np.nan
    ops = Operations()
    ops.kv_cache("cache", pages=pages, page_size=page_size, kv_heads=kv_heads, dim=dim, dtype=dtype)
    ops.from_numpy(spec.pack(k, v), "cache")
    _put(ops, "q", rng.standard_normal((b, heads * dim)).astype(np.float32))
    _put(ops, "pages", table)
    _put(ops, "lengths", np.array(lengths, np.int32))
    ops.paged_attention("q", cache="cache", pages="pages", lengths="lengths", out="o", heads=heads, scale=scale)
    return ops


def _attention_bound(ops: Operations) -> np.ndarray:
    """A score q . k * scale * log2(e): the factor rounds once, q times it once, the
    products' fma chain dim times, the two halves' sum and a key's scale once more (8 bits:
    hi's chain, mid's and lo's at 2^-8 of its size, their sum), so (dim + 5) u of sum
    |q||k| scale, in both numerator and denominator: twice that in
    the exponent.  2^x of the device and the difference x - m add 2^-22 and u of the
    largest |score| log2(e).  Weights and sums are added in chains no longer than the
    positions, with at most 3 more roundings for each joining step and a value's scale.
    (8 bits: a wave's sum rounds 3 times for each position of its own, for the parts of its
    weight, and of n positions the first wave of at least two has 32 or (n + 32) / 2 at the
    most, its weights' sum a few: under 2 (n + 16).)"""
    (op,) = ops.build()
    found = []
    get = lambda t: ops.uploads[t.buffer_key]  # noqa: E731
    share = op.heads // op.spec.kv_heads
    for q, k, v in serving_eval.attention_rows(op, get):
        o = np.zeros(q.shape)
        for h in range(op.heads if k.shape[1] else 0):
            kk, vv = np.nan_to_num(np.abs(k[h // share])), np.nan_to_num(np.abs(v[h // share]))
            mag = (kk @ np.abs(q[h])) * abs(op.scale)
            s = k[h // share] @ q[h] * op.scale
            e = np.exp(s - s.max())
            p = e / e.sum()
            chain = kk.shape[0]
            rel = 2 * (op.spec.dim + 5) * U * mag.max() + 4 * U * mag.max() + 2 * 2.0**-22 + 2 * (chain + 16) * U
            o[h] = 1.1 * rel * (p @ vv)
        found.append(o.reshape(-1))
    return np.stack(found) + 1e-30


CASES = [
    # heads, kv_heads, dim, page_size, width, lengths
    (1, 1, 16, 1, 3, [1, 2, 3]),
    (4, 4, 64, 16, 4, [0, 1, 15, 16, 17, 64]),
    (8, 2, 128, 16, 40, [640, 5, 0, 333]),
    (6, 2, 96, 20, 9, [180, 41, 1]),
    (16, 1, 128, 64, 5, [320, 257]),
    (40, 2, 80, 48, 7, [336, 47, 49]),
    (17, 1, 32, 7, 30, [210, 100]),
    (8, 8, 256, 32, 12, [384, 31]),
    (3, 3, 48, 5, 13, [65, 64, 1]),
    (12, 4, 112, 16, 20, [77, 320]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads, dim, page_size, width, lengths", CASES)
def test_paged_attention(dtype, heads, kv_heads, dim, page_size, width, lengths):
    ops = _attention(dtype, heads, kv_heads, dim, page_size, width, lengths, seed=dim + heads)
    _close(run(ops).env["o"], evaluate(ops)["o"], _attention_bound(ops))


MANY = [
    # more sequences than a wave has lanes; a key head's query heads taken in parts;
    # 16 of them with long rows; pages that end anywhere
    (4, 2, 32, 16, 6, [(37 * i) % 97 for i in range(130)]),
    (2, 1, 64, 8, 70, [0] * 63 + [500, 0, 3] + [1] * 62 + [560, 0]),
    (32, 2, 256, 16, 40, [640, 100]),
    (36, 1, 256, 9, 30, [270]),
    (16, 1, 128, 5, 60, [300, 298, 7]),
    (33, 1, 128, 16, 20, [320, 1]),
    # dims of which 32 is no divisor, with as many heads as are held at once and one more
    (16, 1, 240, 16, 30, [480, 33]), (17, 1, 208, 7, 40, [280, 5]), (32, 2, 144, 16, 20, [300]), (5, 1, 176, 32, 9, [288, 100]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads, dim, page_size, width, lengths", MANY)
def test_paged_attention_of_many_sequences_and_heads(dtype, heads, kv_heads, dim, page_size, width, lengths):
    ops = _attention(dtype, heads, kv_heads, dim, page_size, width, lengths, seed=dim + heads)
    _close(run(ops).env["o"], evaluate(ops)["o"], _attention_bound(ops))


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_attention_of_long_split_sequences(dtype):
    """Lengths that end inside a part, at its border and in the first of many, joined
    by the last workgroup; the same bits every time."""
    ops = _attention(dtype, 8, 2, 64, 16, 256, [4096, 4095, 1, 1023, 0, 2049], seed=3)
    (g,) = compile_program(ops)
    assert g.kernel.workspace_bytes > 0
    first = run(ops).env["o"]
    _close(first, evaluate(ops)["o"], _attention_bound(ops))
    for _ in range(4):
        np.testing.assert_array_equal(run(ops).env["o"], first)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page_size", [16, 12])
def test_paged_attention_bad_pages_and_lengths(dtype, page_size):
    """Holes in the table (negative numbers, numbers past the cache), lengths below
    zero and beyond the table."""
    holes = [(0, 1, -1), (0, 2, 10**6), (1, 0, -(2**31)), (1, 1, 2**31 - 1), (1, 2, -7), (3, 0, -1)]
    ops = _attention(dtype, 4, 2, 64, page_size, 6, [6 * page_size, 3 * page_size, 5, 2 * page_size + 1], seed=9, holes=holes)
    lengths = ops.uploads["lengths"]
    lengths[0] = 2**31 - 1
    lengths[2] = -3
    env = run(ops).env["o"]
    _close(env, evaluate(ops)["o"], _attention_bound(ops))
    assert np.all(env[1] == 0) and np.all(env[2] == 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_attention_of_a_transposed_q(dtype):
    plain = _attention(dtype, 8, 2, 64, 16, 40, [640, 3, 77, 0, 600], seed=31)
    ops = Operations()
    ops.kv_cache("cache", **{k: getattr(plain.build()[0].spec, k) for k in ("pages", "page_size", "kv_heads", "dim", "dtype")})
    for name in ("cache", "pages", "lengths"):
        if name != "cache":
            ops.input(name, plain.uploads[name].shape, dtype="int32")
        ops.from_numpy(plain.uploads[name], name)
    _put(ops, "q_", np.ascontiguousarray(plain.uploads["q"].T))
    ops.transpose("q_", out="q")
    ops.paged_attention("q", cache="cache", pages="pages", lengths="lengths", out="o", heads=8)
    np.testing.assert_array_equal(run(ops).env["o"], run(plain).env["o"])


def test_paged_attention_values_that_are_not_finite():
    """Scores of -inf weigh nothing beside others and give NaN alone, as softmax does;
    an infinite value reaches its own dim."""
    spec = KVCache(pages=3, page_size=16, kv_heads=1, dim=16)
    rng = np.random.default_rng(12)
    k, v = rng.standard_normal((2, spec.slots, 1, 16)).astype(np.float32)
    k[:, 0, 0] = np.abs(k[:, 0, 0]) + 1
    k[3, 0, 0] = k[20, 0, 0] = -np.inf  # one among others
    k[32:, 0, 0] = -np.inf  # a sequence of nothing else
    v[5, 0, 2], v[7, 0, 3] = np.inf, np.nan
    ops = Operations()
    ops.kv_cache("cache", pages=3, page_size=16, kv_heads=1, dim=16)
    ops.from_numpy(spec.pack(k, v), "cache")
    _put(ops, "q", np.abs(rng.standard_normal((2, 32))).astype(np.float32))
    _put(ops, "pages", np.array([[0, 1], [2, -1]], np.int32))
    _put(ops, "lengths", np.array([32, 16], np.int32))
    ops.paged_attention("q", cache="cache", pages="pages", lengths="lengths", out="o", heads=2)
    got, want = run(ops).env["o"], evaluate(ops)["o"]
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.isinf(got), np.isinf(want))
    assert np.all(np.isnan(got[1])) and np.isinf(got[0, 2]) and np.isnan(got[0, 3])
    fine = np.isfinite(want)
    np.testing.assert_allclose(got[fine], want[fine], rtol=1e-5, atol=1e-6)


def test_paged_attention_large_and_small_scores():
    """Scores of hundreds (one position takes all), and a scale of 0 (the mean)."""
    ops = _attention("float32", 4, 2, 64, 16, 8, [100, 128], seed=4, scale=20.0)
    got, want = run(ops).env["o"], evaluate(ops)["o"]
    _close(got, want, _attention_bound(ops))
    ops = _attention("int8", 4, 2, 64, 16, 8, [100, 128], seed=4, scale=0.0)
    _close(run(ops).env["o"], evaluate(ops)["o"], _attention_bound(ops))


# ---------------------------------------------------------------------------
# together, and the ways a program runs
# ---------------------------------------------------------------------------

B, DIM, HEADS, KV, WIDTH_FF = 3, 64, 4, 2, 384


def _step_program(dtype: str, seed: int, weights_seed: int = 1) -> Operations:
    """One decode step: norm in 8 bits -> q, k, v -> cache -> attention -> output
    projection -> residual norm -> gated block, in the framework's other ops too."""
    hidden = HEADS * DIM
    rng, wrng = np.random.default_rng(seed), np.random.default_rng(weights_seed)
    ops = Operations()
    _put(ops, "h0", rng.standard_normal((B, hidden)).astype(np.float32))
    _put(ops, "norm1", (1 + 0.1 * wrng.standard_normal(hidden)).astype(np.float32))
    _put(ops, "norm2", (1 + 0.1 * wrng.standard_normal(hidden)).astype(np.float32))

    def weight(name, n, k, group=64):
        _put(ops, name, wrng.integers(0, 256, (n, k // 2)).astype(np.uint8))
        _put(ops, name + "_s", (wrng.uniform(0.5, 1.5, (n, k // group)) / (4.6 * np.sqrt(k))).astype(np.float32))

    weight("wq", hidden, hidden)
    weight("wk", KV * DIM, hidden)
    weight("wv", KV * DIM, hidden)
    weight("wo", hidden, hidden)
    weight("w1", WIDTH_FF, hidden)
    weight("w2", WIDTH_FF, hidden)
    weight("w3", hidden, WIDTH_FF, 128)
    spec = ops.kv_cache("cache", pages=8, page_size=4, kv_heads=KV, dim=DIM, dtype=dtype)
    old = rng.standard_normal((2, spec.slots, KV, DIM)).astype(np.float32)
    ops.from_numpy(spec.pack(old[0], old[1]), "cache")
    table = rng.permutation(8)[: 2 * B].reshape(B, 2).astype(np.int32)
    lengths = np.array([1, 4, 7], np.int32)  # with the new token
    _put(ops, "pages", table)
    _put(ops, "lengths", lengths)
    _put(ops, "slots", np.array([table[i, (n - 1) // 4] * 4 + (n - 1) % 4 for i, n in enumerate(lengths)], np.int32))

    ops.rms_norm("h0", weight="norm1", out="x8", scales="xs")
    for p in "qkv":
        ops.matmul_int4("x8", weights=f"w{p}", scales=f"w{p}_s", x_scales="xs", out=p)
    ops.cache_write("cache", k="k", v="v", slots="slots", out="cache1")
    ops.paged_attention("q", cache="cache1", pages="pages", lengths="lengths", heads=HEADS, out="a")
    ops.matmul_int4("a", weights="wo", scales="wo_s", out="attn")
    ops.rms_norm("attn", residual="h0", sum_out="h1", weight="norm2", out="x2")
    ops.matmul_int4("x2", weights="w1", scales="w1_s", out="g1")
    ops.matmul_int4("x2", weights="w2", scales="w2_s", out="g2")
    ops.elementwise("negate", out="n", operands=("g1",))
    ops.elementwise("exp", out="e", operands=("n",))
    ops.elementwise("add", out="p", operands=("e", 1.0))
    ops.elementwise("recip", out="sig", operands=("p",))
    ops.elementwise("mul", out="g", operands=("g1", "sig"))
    ops.elementwise("mul", out="z", operands=("g", "g2"))
    ops.matmul_int4("z", weights="w3", scales="w3_s", out="mlp")
    ops.elementwise("add", out="h2", operands=("mlp", "h1"))
    return ops


@pytest.mark.parametrize("dtype", TYPES)
def test_a_decode_step(dtype):
    """Stages round to 8 bits between exact ones, so a last bit before a border moves a
    value by a step (1/127 of its row's largest, 2^-4 of itself in e4m3); a step moves a
    few values in hundreds, each weighed by about 1/sqrt(256)."""
    ops = _step_program(dtype, 2)
    env, ref = run(ops).env, evaluate(ops)
    np.testing.assert_array_equal(env["x8"], ref["x8"])
    for name in ("q", "k", "v"):
        np.testing.assert_allclose(env[name], ref[name], rtol=0, atol=256 * 40 * U)
    step = 2.0**-4 if dtype == "float8_e4m3" else 2.0**-7
    assert np.all(np.isfinite(env["h2"]))
    rms = np.sqrt(np.mean(ref["h2"] ** 2))
    assert np.sqrt(np.mean((env["h2"] - ref["h2"]) ** 2)) <= (step if dtype != "float32" else 1e-5) * rms


def _resident(ops: Operations, groups):
    env = {name: Buffer.from_numpy(a) for name, a in ops.uploads.items()}
    for t in ops.tensors.values():
        if t.buffer_key not in env:
            env[t.buffer_key] = Buffer(t.nbytes)
            env[t.buffer_key].fill(0xFF)
    return env


def test_a_resident_program_runs_again_and_again():
    """Device buffers, one launch sequence: the same results each time, and two programs
    in turn (they share the workspace) do not disturb each other."""
    programs = [_attention("int8", 8, 2, 64, 16, 256, [4096, 700], seed=s) for s in (1, 2)]
    want = [run(ops).env["o"] for ops in programs]
    made = []
    for ops in programs:
        groups = compile_program(ops)
        made.append((Runtime(tuple(Dispatch(g.kernel, g.bindings, g.dims, g.grid, g.threads) for g in groups)), _resident(ops, groups)))
    for _ in range(3):
        for (runtime, env), o in zip(made, want):
            runtime.run(env)
        for (runtime, env), o in zip(made, want):
            np.testing.assert_array_equal(env["o"].numpy(o.shape, np.float32), o)


def test_attention_next_to_products_that_use_the_same_workspace():
    """A product of few tiles (summed in parts), a split attention and the product of its
    output: again and again, with the workspace's flags left zero by each."""
    ops = _attention("int8", 8, 2, 64, 16, 256, [4096, 700], seed=40)
    rng = np.random.default_rng(40)
    _put(ops, "wv", rng.standard_normal((512, 64)).astype(np.float32))
    _put(ops, "a", rng.standard_normal((64, 8192)).astype(np.float32))
    _put(ops, "b", rng.standard_normal((8192, 64)).astype(np.float32))
    ops.matmul("a", "b", out="c")
    ops.matmul("o", "wv", out="p")
    groups = compile_program(ops)
    assert sum(g.kernel.workspace_bytes > 0 for g in groups) >= 2
    first = run(ops).env
    want = evaluate(ops)
    _close(first["c"], want["c"], 1e-4 * np.sqrt(8192) * np.abs(want["c"]) + 8192 * U * (np.abs(ops.uploads["a"]) @ np.abs(ops.uploads["b"])))
    for _ in range(3):
        env = run(ops).env
        for name in ("o", "c", "p"):
            if name in first:
                np.testing.assert_array_equal(env[name], first[name])
    hip_backend.check_workspace()


def test_two_threads_at_once():
    """Each thread runs programs of its own over and over; they share the stream and the
    workspace."""
    programs = [[_attention("int8", 8, 2, 64, 16, 256, [4096, 700 + s], seed=s), _int4(5, 1056, 500, 32, False, True, s)] for s in (1, 2)]
    want = [[run(ops).env for ops in each] for each in programs]
    wrong = []

    def work(each, env):
        try:
            for _ in range(10):
                for ops, ref, name in zip(each, env, ("o", "y")):
                    if not np.array_equal(run(ops).env[name], ref[name]):
                        wrong.append(name)
        except Exception as e:  # (an assertion in a thread would be lost)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=pair) for pair in zip(programs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_decoding_token_after_token():
    """The cache lives in a device buffer over several steps, each writing a slot and
    attending over what is there: as a whole recomputation gives it."""
    spec = KVCache(pages=4, page_size=4, kv_heads=2, dim=32, dtype="int8")
    rng = np.random.default_rng(21)
    ops = Operations()
    ops.kv_cache("cache", pages=4, page_size=4, kv_heads=2, dim=32, dtype="int8")
    ops.from_numpy(spec.empty(), "cache")
    for name in ("k", "v"):
        _put(ops, name, np.zeros((1, 64), np.float32))
    _put(ops, "q", np.zeros((1, 128), np.float32))
    _put(ops, "slots", np.zeros(1, np.int32))
    _put(ops, "pages", np.array([[2, 0, 3, 1]], np.int32))
    _put(ops, "lengths", np.zeros(1, np.int32))
    ops.cache_write("cache", k="k", v="v", slots="slots", out="c1")
    ops.paged_attention("q", cache="c1", pages="pages", lengths="lengths", heads=4, out="o")
    groups = compile_program(ops)
    env = _resident(ops, groups)
    runtime = Runtime(tuple(Dispatch(g.kernel, g.bindings, g.dims, g.grid, g.threads) for g in groups))
    state = spec.empty()
    for t in range(16):
        step = {n: rng.standard_normal(ops.tensors[n].shape).astype(np.float32) for n in ("k", "v", "q")}
        step["slots"] = np.array([[2, 0, 3, 1][t // 4] * 4 + t % 4], np.int32)
        step["lengths"] = np.array([t + 1], np.int32)
        for name, a in step.items():
            env[name].write(a)
        runtime.run(env)
        inputs = {**ops.uploads, **step, "cache": state}
        ref = evaluate(ops, inputs)
        state = ref["c1"]
        np.testing.assert_allclose(env["o"].numpy((1, 128), np.float32), ref["o"], rtol=0, atol=2e-5)
    _same_state(spec, env["cache"].numpy(spec.shape, np.uint8), state)


def test_batched_programs_give_the_same_as_each_alone():
    programs = [_step_program("int8", s) for s in (1, 2, 3)]
    alone = [run(ops).env for ops in programs]
    together = run_batch(programs)
    for a, b in zip(alone, together):
        for name in ("x8", "k", "cache1", "a", "h2"):
            np.testing.assert_array_equal(a[name], b.env[name])


def test_a_batch_of_split_attentions():
    programs = [_attention("float32", 4, 2, 64, 16, 128, [2048, 1000 + s], seed=s) for s in range(3)]
    for ops, got in zip(programs, run_batch(programs)):
        _close(got.env["o"], evaluate(ops)["o"], _attention_bound(ops))


def test_a_batch_that_the_kernel_was_not_made_for():
    """The kernel of one program launched for four: its workspace has room for one, so
    each runs in one workgroup."""
    programs = [_attention("int8", 4, 2, 64, 16, 128, [2048, 1000 + s], seed=s) for s in range(4)]
    (g,) = compile_program(programs[0])
    assert g.grid[0] > 1 and g.kernel.workspace_bytes > 0
    envs = [_resident(ops, (g,)) for ops in programs]
    kernel = g.kernel.batched()
    tables = [Buffer.from_numpy(np.array([env[key].device_address for env in envs], np.uint64)) for key in g.bindings]
    hip_backend.launch(kernel.handle, tables, g.dims, kernel.dims_slot_index, (*g.grid[:2], 4), g.threads,
                       workspace=kernel.workspace_bytes)
    for ops, env in zip(programs, envs):
        _close(env["o"].numpy(ops.tensors["o"].shape, np.float32), evaluate(ops)["o"], _attention_bound(ops))


def test_launches_that_allocate_nothing():
    """``launch_noalloc`` with its static scratch: the join's counters are left zero."""
    ops = _attention("float8_e4m3", 8, 2, 64, 16, 256, [4096, 513], seed=6)
    want = run(ops).env["o"]
    (g,) = compile_program(ops)
    env = _resident(ops, (g,))
    for _ in range(3):
        env["o"].fill(0xFF)
        err = hip_backend.launch_noalloc(g.kernel.handle, [env[k] for k in g.bindings], g.dims, g.kernel.dims_slot_index, g.grid,
                                         g.threads, scratch=g.kernel.workspace_bytes)
        assert err == 0
        np.testing.assert_array_equal(env["o"].numpy(want.shape, np.float32), want)


def test_a_cache_beyond_4_gib():
    """Pages whose bytes lie past 32 bits."""
    pages, page_size = 5000, 16
    spec = KVCache(pages=pages, page_size=page_size, kv_heads=32, dim=256)
    assert spec.pages * spec.page_bytes > 2**32 + 2**28
    ops = Operations()
    ops.kv_cache("cache", pages=pages, page_size=page_size, kv_heads=32, dim=256)
    rng = np.random.default_rng(30)
    t = 20
    slots = np.concatenate([[(pages - 1) * page_size + i for i in range(10)], 4 * page_size + np.arange(10)]).astype(np.int32)
    for name in ("k", "v"):
        _put(ops, name, rng.standard_normal((t, spec.row)).astype(np.float32))
    _put(ops, "slots", slots)
    _put(ops, "q", rng.standard_normal((1, 32 * 256)).astype(np.float32))
    _put(ops, "pages", np.array([[pages - 1, 4]], np.int32))
    _put(ops, "lengths", np.array([10], np.int32))
    ops.cache_write("cache", k="k", v="v", slots="slots", out="c1")
    ops.cache_read("c1", slots="slots", k_out="kb", v_out="vb")
    ops.paged_attention("q", cache="c1", pages="pages", lengths="lengths", heads=32, out="o")
    groups = compile_program(ops)
    env = _resident(ops, groups)  # 0xFF everywhere: NaN
    env["cache"] = env["cache"] if "cache" in env else Buffer(spec.pages * spec.page_bytes)
    Runtime(tuple(Dispatch(g.kernel, g.bindings, g.dims, g.grid, g.threads) for g in groups)).run(env)
    for name, src in (("kb", "k"), ("vb", "v")):
        np.testing.assert_array_equal(env[name].numpy((t, spec.row), np.float32), ops.uploads[src])
    k, v = (ops.uploads[n][:10].reshape(10, 32, 256).astype(np.float64) for n in "kv")
    q = ops.uploads["q"].reshape(32, 256).astype(np.float64)
    s = np.einsum("hd,phd->hp", q, k) / 16
    p = np.exp(s - s.max(1, keepdims=True))
    want = np.einsum("hp,phd->hd", p / p.sum(1, keepdims=True), v)
    np.testing.assert_allclose(env["o"].numpy((32, 256), np.float32), want, rtol=0, atol=1e-4)
    for b in env.values():
        b.release()
    hip_backend.trim()


# ---------------------------------------------------------------------------
# keys that are NaN
# ---------------------------------------------------------------------------


def _with_nan_keys(ops: Operations, at) -> Operations:
    """NaN in the key of head ``h`` at position ``p`` of sequence ``b``, for each (b, p, h) of ``at``."""
    (op,) = ops.build()
    spec, table = op.spec, ops.uploads["pages"]
    k, v = (np.array(a) for a in spec.unpack(ops.uploads["cache"]))
    for b, p, h in at:
        k[table[b, p // spec.page_size] * spec.page_size + p % spec.page_size, h, 1] = np.nan
    ops.from_numpy(spec.pack(k, v), "cache")
    return ops


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page_size", [16, 12])
def test_paged_attention_of_a_nan_key_alone_in_a_tile(dtype, page_size):
    """The newest position, the only one of its tile, is NaN: so is the softmax, of its key
    head alone.  Lengths of one more than any number of tiles of 16 and 32, and others."""
    lengths = [1, 2, 17, 33, 49, 65, 97, 129, 161, 193, 257, 34, 40]
    ops = _attention(dtype, 4, 2, 64, page_size, 24, lengths, seed=51)
    _with_nan_keys(ops, [(b, n - 1, b % 2) for b, n in enumerate(lengths[:-2])] + [(11, 32, 0), (12, 5, 1)])
    got, want = run(ops).env["o"], evaluate(ops)["o"]
    with np.errstate(invalid="ignore"):
        _close(got, want, _attention_bound(ops))
    nan = np.isnan(got).reshape(len(lengths), 2, -1)
    for b in range(len(lengths)):
        bad = b % 2 if b < 11 else b - 11
        assert np.all(nan[b, bad]) and not np.any(nan[b, 1 - bad])


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_attention_of_a_nan_key_alone_in_a_workgroups_part(dtype):
    """Sequences split over workgroups, a last part of one position."""
    for dim in (64, 256):
        ops = _attention(dtype, 4, 2, dim, 16, 257, [4097], seed=52)
        (g,) = compile_program(ops)
        assert g.kernel.workspace_bytes > 0
        _with_nan_keys(ops, [(0, 4096, 1)])
        got, want = run(ops).env["o"], evaluate(ops)["o"]
        with np.errstate(invalid="ignore"):
            _close(got, want, _attention_bound(ops))
        assert np.all(np.isnan(got.reshape(2, -1)[1])) and np.all(np.isfinite(got.reshape(2, -1)[0]))


def test_paged_attention_of_a_nan_key_beside_scores_of_minus_infinity():
    """A tile of one NaN score and others of -inf, next to tiles of finite scores and next
    to tiles of -inf alone."""
    ops = _attention("float32", 2, 1, 16, 16, 3, [48, 48, 48], seed=53)
    (op,) = ops.build()
    k, v = (np.array(a) for a in op.spec.unpack(ops.uploads["cache"]))
    ops.uploads["q"][:] = np.abs(ops.uploads["q"])
    for b in range(3):
        at = ops.uploads["pages"][b][:, None] * 16 + np.arange(16)
        k[at[1], 0, 0] = -np.inf
        if b > 0:
            k[at[1, 7], 0] = np.nan
        if b > 1:
            k[at[0], 0, 0] = k[at[2], 0, 0] = -np.inf
    ops.from_numpy(op.spec.pack(k, v), "cache")
    got, want = run(ops).env["o"], evaluate(ops)["o"]
    assert np.all(np.isfinite(want[0])) and np.all(np.isnan(want[1:]))
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ops.uploads["pages"][0, 1] = -1  # scores of -inf weigh what positions that are not there do
    np.testing.assert_array_equal(got[0], run(ops).env["o"][0])


# ---------------------------------------------------------------------------
# 4-bit products of x with outliers
# ---------------------------------------------------------------------------


def _outlier_bound(ops: Operations, blocks) -> np.ndarray:
    """As ``_int4_bound``, but a block of x in which a few values stand far above all
    others (``blocks[m]`` names those of row m) is held to what products in fp32 are: a
    weight rounds twice (q - z, times s), 32 terms of a lane's chain round once each, two
    additions join the four lanes: 36 u of sum |x| |q - z| |s|, and no step of the largest."""
    (op,) = ops.build()
    x = np.abs(ops.uploads["x"].astype(np.float64))
    s = ops.uploads["s"].astype(np.float64)
    z = ops.uploads["z"].astype(np.float64) if op.zeros is not None else np.full(s.shape, 8.0)
    raw, (rows, k), group = ops.uploads["w"], x.shape, op.group
    q = np.empty((raw.shape[0], k))
    q[:, 0::2], q[:, 1::2] = raw & 15, raw >> 4
    own = np.abs(q - np.repeat(z, group, axis=1)) * np.abs(np.repeat(s, group, axis=1))
    most = np.repeat((8 + np.abs(8 - z)) * np.abs(s), group, axis=1)
    total, steps = np.zeros((rows, len(raw))), np.zeros((rows, len(raw)))
    for m in range(rows):
        for b in range(-(-k // 128)):
            at = slice(128 * b, min(k, 128 * b + 128))
            if b in blocks[m]:
                total[m] += own[:, at] @ x[m, at] * (1 + 36 / (8 + k // group))
            else:
                total[m] += most[:, at] @ x[m, at]
                steps[m] += x[m, at].max() * 2.0**-29 * (most[:, at].sum(axis=1) + 64 * np.abs(s[:, 128 * b // group : -(-at.stop // group)]).sum(axis=1))
    return (8 + k // group + 8) * U * total + steps


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows, n, group, size", [
    # splitting k (one, two and four tiles), sharing x's digits (one phase and several, 8 and 16 waves)
    (1, 100, 32, 1e6), (1, 100, 64, 1e9), (2, 700, 32, 1e4), (3, 4100, 32, 3e5), (6, 4100, 64, 1e12), (16, 4100, 32, 1e6), (8, 9000, 32, 1e5),
    (1, 24577, 32, 1e6), (2, 24577, 64, 1e7), (4, 24577, 32, 2e3), (6, 24577, 64, 1e6), (16, 16500, 32, 1e30), (9, 65540, 64, 1e6),
])
def test_matmul_int4_of_x_with_outliers(rows, n, group, size, zeros):
    """Channels of x ``size`` times the others, whose weights are zero: the others' products
    are as right as they are alone."""
    k = 1696 if group == 32 else 1728
    ops = _int4(rows, k, n, group, False, zeros, n + rows)
    x, w = ops.uploads["x"], ops.uploads["w"]
    channels = [(0, 5), (0, 130), (rows - 1, 700), (rows - 1, 701), (rows // 2, k - 1)]
    blocks = [set() for _ in range(rows)]
    if zeros:
        z = ops.uploads["z"]
        z[:] = np.round(z)
    for m, at in channels:
        x[m, at] = size * (1 + abs(x[m, at])) * (-1) ** at
        blocks[m].add(at // 128)
        q = z[:, at // group].astype(np.uint8) if zeros else np.full(n, 8, np.uint8)
        w[:, at // 2] = (w[:, at // 2] & 0x0F) | (q << 4) if at % 2 else (w[:, at // 2] & 0xF0) | q
    _close(run(ops).env["y"], evaluate(ops)["y"], _outlier_bound(ops, blocks))


def test_matmul_int4_of_values_over_many_magnitudes():
    """Values log-uniform over 2^-60 to 2^60, weights zero but for the smallest halves of
    each block: what is left is held to its own size.  And subnormal values beside 1."""
    rng = np.random.default_rng(60)
    k, n = 512, 40
    x = (2.0 ** rng.uniform(-60, 60, (3, k)) * rng.choice([-1, 1], (3, k))).astype(np.float32)
    x[2] = (rng.integers(-2000, 2000, k) * 2.0**-149).astype(np.float32)
    x[2, 7::128] = 1
    ops = _int4(3, k, n, 128, False, False, 61)
    ops.uploads["x"][:] = x
    ops.uploads["s"][:] = 1.0
    for m in range(3):
        big = np.zeros(k, bool)
        for b in range(0, k, 128):
            a = np.abs(x[m, b : b + 128])
            big[b : b + 128] = a > (np.median(a) if m < 2 else 0.5)
        w = np.random.default_rng(m).integers(0, 16, (n, k)).astype(np.uint8)
        w[:, big] = 8
        ops.uploads["w"][:] = w[:, 0::2] | (w[:, 1::2] << 4)
        got, want = run(ops).env["y"][m], evaluate(ops)["y"][m]
        # every block is one of fp32 products: 36 u, and a wave's and the waves' sums
        bound = (36 + k // 128 + 8) * U * (np.abs(w - 8.0) @ np.abs(x[m].astype(np.float64))) + 2.0**-149
        _close(got, want, bound)


def test_matmul_int4_of_subnormal_row_scales():
    """x in 8 bits of rows so small that their scales are subnormal: y is their product
    rounded, not one of a scale that lost bits."""
    ops = _int4(5, 4096, 70, 64, True, False, 62)
    ops.uploads["x"][:] = 127
    ops.uploads["s"][:] = np.abs(ops.uploads["s"])
    w = ops.uploads["w"]
    w[:] = (w & 0x77) | 0x88  # q of 8 to 15
    ops.uploads["xs"][:] = np.array([2.0**-149, 3 * 2.0**-149, 1000 * 2.0**-149, 1e-39, 0.01], np.float32)
    _close(run(ops).env["y"], evaluate(ops)["y"], _int4_bound(ops) + 2.0**-149)


def test_what_shares_the_workspace_is_right_as_well_as_repeatable():
    """A split attention between a product summed in parts and the product of its output.
    A product of k terms rounds at most k + 16 times on the way (its chain, 16 parts); the
    attention's error goes through the second product."""
    alone, ops = (_attention("int8", 8, 2, 64, 16, 256, [4096, 700], seed=40) for _ in range(2))
    rng = np.random.default_rng(41)
    _put(ops, "wv", rng.standard_normal((512, 64)).astype(np.float32))
    _put(ops, "a", rng.standard_normal((64, 8192)).astype(np.float32))
    _put(ops, "b", rng.standard_normal((8192, 64)).astype(np.float32))
    ops.matmul("a", "b", out="c")
    ops.matmul("o", "wv", out="p")
    ops.elementwise("exp", out="e", operands=("o",))  # (o is read twice, so it stays a buffer)
    assert sum(g.kernel.workspace_bytes > 0 for g in compile_program(ops)) >= 2
    want, off, wv = evaluate(ops), _attention_bound(alone), np.abs(ops.uploads["wv"].astype(np.float64))
    a, b = (np.abs(ops.uploads[n].astype(np.float64)) for n in "ab")
    bounds = {"o": off, "c": (8192 + 16) * U * (a @ b), "p": off @ wv + (512 + 17) * U * (np.abs(want["o"]) @ wv)}
    for _ in range(3):
        env = run(ops).env
        for name, bound in bounds.items():
            _close(env[name], want[name], bound)
    hip_backend.check_workspace()


@pytest.mark.parametrize("dtype", ["int8", "float8_e4m3"])
def test_cache_write_by_the_definition(dtype):
    """2048 rows of N(0, 1), some of them very small or large, apart from the oracle: a scale is
    the largest over the peak but for two roundings (2^-24 of it each, and half of the smallest
    subnormal), a value the nearest multiple of it: half a step of x / scale off."""
    spec = KVCache(pages=16, page_size=64, kv_heads=2, dim=64, dtype=dtype)
    rng = np.random.default_rng(71)
    ops = Operations()
    ops.kv_cache("cache", pages=16, page_size=64, kv_heads=2, dim=64, dtype=dtype)
    ops.from_numpy(spec.empty(), "cache")
    kv = rng.standard_normal((2, spec.slots, spec.row))
    kv[:, :200] *= 2.0 ** rng.integers(-140, 120, (2, 200, 1))
    kv = kv.astype(np.float32)
    for name, a in zip("kv", kv):
        _put(ops, name, a)
    _put(ops, "slots", np.arange(spec.slots, dtype=np.int32))
    ops.cache_write("cache", k="k", v="v", slots="slots", out="written")
    got = run(ops).env["written"]
    peak = 127.0 if dtype == "int8" else 448.0
    rows = kv.reshape(2, 16, 64, 2, 64).transpose(1, 0, 3, 2, 4).astype(np.float64)  # page, part, head, slot
    parts = [serving_eval._page_parts(spec, got, p) for p in range(spec.pages)]
    s, want = np.stack([p[1] for p in parts]).astype(np.float64), np.abs(rows).max(axis=-1) / peak
    assert np.all(np.abs(s - want) <= want * 2.01 * 2.0**-24 + 2.0**-150)
    raw = np.ascontiguousarray(np.stack([p[0] for p in parts]))
    held = raw.view(np.int8).astype(np.float64) if dtype == "int8" else serving_eval.E4M3[raw]
    v = np.clip(np.divide(rows, s[..., None], out=np.zeros_like(rows), where=s[..., None] > 0), -peak, peak)
    half = 0.5 if dtype == "int8" else np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(v), 2.0**-6))), -6) - 4)
    assert np.all(np.abs(held - v) <= half)


@pytest.mark.parametrize("n, zeros", [(70, True), (70, False), (16400, True)])
def test_matmul_int4_with_outliers_of_a_transposed_x_of_more_rows_than_one_pass(n, zeros):
    """20 rows, the outliers in the first and the second pass's rows; alone, again, and in a batch."""
    rows, k, group = 20, 416, 32
    programs, bounds = [], []
    for seed in (81, 82):
        ops = _int4(rows, k, n, group, False, zeros, seed, strides=True)
        x, w = ops.uploads["x_"], ops.uploads["w"]  # (columns of x_ are rows of x)
        blocks = [set() for _ in range(rows)]
        if zeros:
            ops.uploads["z"][:] = np.round(ops.uploads["z"])
        for m, at in ((0, 7), (3, 131), (16, 260), (19, k - 2)):
            x[at, m] = 1e6
            blocks[m].add(at // 128)
            q = ops.uploads["z"][:, at // group].astype(np.uint8) if zeros else np.full(n, 8, np.uint8)
            w[:, at // 2] = (w[:, at // 2] & 0x0F) | (q << 4) if at % 2 else (w[:, at // 2] & 0xF0) | q
        programs.append(ops)
        ops._uploads["x"] = np.ascontiguousarray(x.T)  # (for the bound alone)
        bounds.append(_outlier_bound(ops, blocks))
        del ops._uploads["x"]
    for ops, got, bound in zip(programs, run_batch(programs), bounds):
        want = evaluate(ops)["y"]
        first = run(ops).env["y"]
        _close(first, want, bound)
        np.testing.assert_array_equal(got.env["y"], first)
        np.testing.assert_array_equal(run(ops).env["y"], first)
