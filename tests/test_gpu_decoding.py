"""The decoding ops on the GPU against the oracle in float64 (``oracle.decoding_eval``).

Tolerances follow from the kernels' roundings (u = 2^-24, half a step of fp32):

* page_tables: exact.
* rotary: see ``_rotary_bound``.
* adapters: see ``_adapter_bound``.
* sample: tokens exact; a logprob is rounded once, and the sum of n weights held in
  2^-s is off by n 2^-s of a sum that is 1 at the least (s = 62 - log2 n, 44 at the most).
"""

from __future__ import annotations

import threading

import numpy as np
import pytest

from metellus_amd.api import compile_program, run, run_batch
from metellus_amd.orchestrator import KVCache, Operations, Rotary
from metellus_amd.orchestrator.decoding import ADAPTER_DOWN_WAVES, AdapterDownOp, AdapterUpOp
from metellus_amd.runtime import Buffer, Dispatch, Runtime
from oracle import decoding_eval
from oracle.ir_eval import evaluate

pytestmark = pytest.mark.gpu

U = 2.0**-24


def _put(ops: Operations, name: str, a: np.ndarray) -> None:
    ops.input(name, a.shape, dtype=str(a.dtype))
    ops.from_numpy(a, name)


def _close(got, want, bound):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    flat = np.isfinite(want)
    np.testing.assert_array_equal(got[~flat & ~np.isnan(want)], want[~flat & ~np.isnan(want)])
    bound = np.broadcast_to(bound, want.shape)
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)[flat]
    assert np.all(off <= bound[flat]), f"off by {np.max(off / np.maximum(bound[flat], 1e-300)):.3g} times the bound"


# ---------------------------------------------------------------------------
# block tables
# ---------------------------------------------------------------------------

PAGE_OUTPUTS = ("slots", "positions", "ends", "used", "table")


def _page_ops(table, free, lengths, counts, page_size, tokens):
    ops = Operations()
    for name, v in (("pages", table), ("free", free), ("lengths", lengths), ("counts", counts)):
        _put(ops, name, np.asarray(v, np.int32))
    ops.page_tables("pages", free="free", lengths="lengths", counts="counts", page_size=page_size, tokens=tokens, out="table",
                    slots="slots", positions="positions", ends="ends", used="used")
    return ops


def _page_check(ops):
    env, ref = run(ops).env, evaluate(ops)
    for name in PAGE_OUTPUTS:
        np.testing.assert_array_equal(env[name], ref[name], err_msg=name)
        assert env[name].dtype == np.int32


@pytest.mark.parametrize("sequences, width, page_size, most, tokens", [
    (1, 1, 1, 1, 1), (1, 4, 16, 1, 3), (3, 7, 5, 4, 9), (64, 9, 16, 1, 64), (65, 3, 20, 30, 500), (255, 4, 8, 2, 300),
    (256, 4, 8, 2, 256), (257, 4, 8, 2, 250), (512, 5, 16, 2, 600), (513, 5, 16, 2, 600), (1023, 6, 3, 9, 4000), (1025, 6, 16, 3, 1000), (5000, 3, 7, 2, 9000),
    (2, 9000, 16, 30000, 70000),
])
def test_page_tables(sequences, width, page_size, most, tokens):
    rng = np.random.default_rng(sequences * 1009 + tokens)
    lengths = rng.integers(0, width * page_size + 1, sequences)
    counts = rng.integers(0, most + 1, sequences)
    table = np.full((sequences, width), -1)
    used = -(-lengths // page_size)
    numbers = rng.permutation(2 * sequences * width).astype(np.int32)
    live = np.arange(width)[None] < used[:, None]
    table[live] = numbers[: live.sum()]
    _page_check(_page_ops(table, numbers[live.sum() :], lengths, counts, page_size, tokens))


def test_page_tables_of_lengths_out_of_range():
    """Lengths and counts below 0, beyond the table, and as large as they get; numbers below 0
    and pages whose slots are past int32."""
    big = 2**31 - 1
    lengths = [-5, big, 30, 31, 32, 0, -(2**31), 7, 16]
    counts = [3, 2, 5, 1, 1, -4, 1, big, big]
    table = np.tile(np.arange(4, dtype=np.int32), (9, 1)) + 10 * np.arange(9, dtype=np.int32)[:, None]
    table[2, 3], table[7, 0] = -9, 2**29
    _page_check(_page_ops(table, [100, 101, -7, 2**28, 103, 104, 105, 106], lengths, counts, 8, 60))


def test_page_tables_out_of_pages():
    """More pages needed than there are: the rest of the entries is -1, and their tokens
    have no slots."""
    lengths, counts = [0, 16, 3], [40, 1, 60]
    ops = _page_ops(np.full((3, 8), 77), [5, 6, 7], lengths, counts, 16, 128)
    _page_check(ops)
    env = run(ops).env
    assert env["used"][0] == 3 + 1 + 3
    np.testing.assert_array_equal(env["table"][1], [77, -1, 77, 77, 77, 77, 77, 77])  # others as they were


def test_page_tables_of_few_rows():
    """Sequences whose tokens the rows do not hold still grow."""
    _page_check(_page_ops(np.zeros((5, 6), np.int32), np.arange(20, 40), [0, 3, 8, 9, 2], [6, 0, 9, 4, 5], 4, 8))


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------


def _rotary_bound(spec, x, positions):
    """y1 = c x1 - s x2: c and s are rounded once (u of themselves), s x2 once more (u),
    and the sum once; so |c x1| u + 2 |s x2| u + |y1| u, 1 % more for what is u^2 and for
    the 64 bits before, and the smallest step for products that have few bits.  y2 alike."""
    angles = decoding_eval.rotary_angles(spec, positions)
    heads = np.abs(x.astype(np.float64)).reshape(x.shape[0], -1, spec.dim)
    bound = np.zeros(heads.shape)
    for j, (a, b) in enumerate(decoding_eval.rotary_pairs(spec)):
        c, s = np.abs(np.cos(angles[:, j, None])) * spec.magnitude, np.abs(np.sin(angles[:, j, None])) * spec.magnitude
        for one, two in ((a, b), (b, a)):
            bound[:, :, one] = 1.01 * U * (2 * heads[:, :, one] * c + 3 * heads[:, :, two] * s) + 2.0**-148
    return bound.reshape(x.shape)


def _rotary_check(ops, spec, **names):
    env, ref = run(ops).env, evaluate(ops)
    at = ops.uploads["at"]
    for name, out in names.items():
        x = ops.uploads[name] if name in ops.uploads else ops.uploads[name + "_"].T
        _close(env[out], ref[out], _rotary_bound(spec, x, at))


SPECS = [
    Rotary(dim=128), Rotary(dim=64, layout="interleaved"), Rotary(dim=96, part=40, layout="interleaved", factor=4.0),
    Rotary(dim=80, part=20), Rotary(dim=10, part=6, layout="interleaved"), Rotary(dim=3, part=2),
    Rotary(dim=256, base=500000.0, factor=8.0, original=8192, low=1.0, high=4.0),
    Rotary(dim=128, part=64, factor=16.0, original=4096, magnitude=1.2772588722239782),
    Rotary(dim=8, frequencies=(1.0, -0.5, 0.0, 1048576.0)), Rotary(dim=160, part=96),
]


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("rows", [1, 3, 17, 1025])
def test_rotary(spec, rows):
    rng = np.random.default_rng(rows + spec.dim)
    ops = Operations()
    _put(ops, "q", rng.standard_normal((rows, 3 * spec.dim)).astype(np.float32))
    _put(ops, "k", rng.standard_normal((rows, 2 * spec.dim)).astype(np.float32))
    _put(ops, "at", rng.integers(0, 200000, rows).astype(np.int32))
    ops.rotary("q", positions="at", out="q1", rotary=spec, k="k", k_out="k1")
    _rotary_check(ops, spec, q="q1", k="k1")


@pytest.mark.parametrize("spec", [Rotary(dim=32), Rotary(dim=32, layout="interleaved"), Rotary(dim=64, frequencies=(2.0**20, -0.3) * 16)])
def test_rotary_far_positions(spec):
    """The farthest positions of int32, below 0 too, and the largest frequencies; q alone."""
    at = np.array([0, 1, -1, 2**31 - 1, -(2**31), 2**24 + 1, 1000003], np.int32)
    rng = np.random.default_rng(2)
    ops = Operations()
    _put(ops, "q", rng.standard_normal((7, 64)).astype(np.float32))
    _put(ops, "at", at)
    ops.rotary("q", positions="at", out="q1", rotary=spec)
    _rotary_check(ops, spec, q="q1")


@pytest.mark.parametrize("spec", [SPECS[0], SPECS[2], SPECS[4]])
def test_rotary_of_strided_rows(spec):
    """q a transposed view, k rows with gaps; infinities and NaN stay with their pairs."""
    rng = np.random.default_rng(5)
    d = spec.dim
    ops = Operations()
    q = rng.standard_normal((2 * d, 5)).astype(np.float32)
    q[d, 2], q[d + 1, 3] = np.inf, np.nan
    _put(ops, "q_", q)
    ops.transpose("q_", out="q")
    ops.input("k", (5, d), row_stride=d, col_stride=1)
    ops.from_numpy(rng.standard_normal((5, d)).astype(np.float32), "k")
    _put(ops, "at", np.arange(5, dtype=np.int32))
    ops.rotary("q", positions="at", out="q1", rotary=spec, k="k", k_out="k1")
    _rotary_check(ops, spec, q="q1", k="k1")


def test_rotary_keeps_what_is_not_turned():
    """Elements behind ``part`` are the same bits, and so is a head at position 0."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((4, 192)).astype(np.float32)
    ops = Operations()
    _put(ops, "q", x)
    _put(ops, "at", np.array([0, 5, 6, 0], np.int32))
    ops.rotary("q", positions="at", out="y", rotary=Rotary(dim=96, part=64))
    y = run(ops).env["y"]
    np.testing.assert_array_equal(y.reshape(4, 2, 96)[:, :, 64:], x.reshape(4, 2, 96)[:, :, 64:])
    np.testing.assert_array_equal(y[[0, 3]], x[[0, 3]])


# ---------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------


def _adapter_bound(ops):
    """``down`` is a wave's fp32 sum over its blocks of 64 columns (each term at most two
    roundings, its product's and the sum's), then sums over waves and splits; ``up`` a sum
    over the rank, rounded up to 16, of what is off by that; scaled and added to base with
    one rounding.  u of the magnitudes for each."""
    down, up = [next(o for o in ops.build() if isinstance(o, kind)) for kind in (AdapterDownOp, AdapterUpOp)]
    value = {n: a.astype(np.float64) for n, a in ops.uploads.items()}
    x = value["x"] if "x" in value else value["x_"].T
    base = evaluate(ops)["y"]
    inner, rank, n = x.shape[1], down.rank, up.y.shape[1]
    waves = ADAPTER_DOWN_WAVES
    terms = 2 * 64 * -(-inner // (64 * down.splits * waves)) + waves + down.splits
    bound = np.abs(base) * U
    for m, i in enumerate(ops.uploads["ids"]):
        if 0 <= i < down.held:
            t = np.abs(value["a"][i * rank : (i + 1) * rank]) @ np.abs(x[m])
            each = np.abs(value["b"][i * n : (i + 1) * n]) @ t
            scale = abs(value["s"][i]) if up.scales is not None else 1.0
            bound[m] += 1.01 * U * (terms + 2 * (rank + 15)) * each * scale
    return bound + 2.0**-149


def _adapters(rows, inner, cols, rank, held, ids, scales=True, seed=1, strides=False):
    rng = np.random.default_rng(seed)
    ops = Operations()
    x, base = rng.standard_normal((rows, inner)).astype(np.float32), rng.standard_normal((rows, cols)).astype(np.float32)
    if strides:
        for name, v in (("x", x), ("base", base)):
            _put(ops, name + "_", np.ascontiguousarray(v.T))
            ops.transpose(name + "_", out=name)
    else:
        _put(ops, "x", x)
        _put(ops, "base", base)
    _put(ops, "a", rng.standard_normal((held * rank, inner)).astype(np.float32))
    _put(ops, "b", rng.standard_normal((held * cols, rank)).astype(np.float32))
    _put(ops, "ids", np.asarray(ids, np.int32))
    if scales:
        _put(ops, "s", rng.uniform(-2, 2, held).astype(np.float32))
    ops.adapters("x", base="base", a="a", b="b", ids="ids", scales="s" if scales else None, out="y")
    return ops


def _adapter_check(ops):
    env, ref = run(ops).env, evaluate(ops)
    _close(env["y"], ref["y"], _adapter_bound(ops))
    assert set(env) & set(ops.scratch) == set()
    return env["y"]


@pytest.mark.parametrize("rows, inner, cols, rank, held", [
    (1, 1, 1, 1, 1), (1, 64, 16, 4, 2), (1, 4096, 300, 16, 3), (2, 100, 17, 8, 5), (7, 333, 129, 23, 4), (16, 512, 256, 16, 16),
    (17, 1000, 1003, 64, 3), (33, 257, 65, 5, 40), (100, 640, 1024, 65, 7), (3, 129, 260, 256, 2), (600, 96, 48, 12, 9),
    (1024, 1500, 100, 16, 5), (1100, 70, 33, 64, 3), (1061, 600, 70, 70, 200),
    (5, 11008, 50, 20, 3), (40, 7003, 90, 33, 3), (1100, 6001, 500, 33, 2), (2050, 2048, 64, 100, 4), (3, 3, 3, 2, 2),
])
@pytest.mark.parametrize("scales", [False, True])
def test_adapters(rows, inner, cols, rank, held, scales):
    rng = np.random.default_rng(rows + inner)
    ids = rng.integers(-1, held, rows)
    _adapter_check(_adapters(rows, inner, cols, rank, held, ids, scales, seed=rows * 31 + rank))


@pytest.mark.parametrize("ids", [
    [0] * 40, list(range(40)), [i // 7 for i in range(40)], [-1] * 40, [-1, 3] * 20, [39 - i for i in range(40)],
    [2**31 - 1, -(2**31), 40, 39, 0] * 8,
])
def test_adapters_by_group(ids):
    """Rows that share one, that have one each, in runs, in turn; ids that are no adapter's."""
    ops = _adapters(40, 300, 70, 8, 40, ids)
    y = _adapter_check(ops)
    none = [m for m, i in enumerate(ids) if not 0 <= i < 40]
    np.testing.assert_array_equal(y[none], ops.uploads["base"][none])


@pytest.mark.parametrize("rows, inner, cols, rank, held", [
    (2100, 2501, 2500, 64, 3), (4100, 2560, 2499, 33, 8), (2100, 2500, 2503, 100, 40), (80000, 70, 67, 64, 9), (82000, 66, 71, 256, 5),
    (2048, 2600, 2561, 64, 900),
])
def test_adapters_of_many_rows(rows, inner, cols, rank, held):
    """Tiles whose groups one workgroup does all: of 64 rows, and of 16 for ranks above 64."""
    rng = np.random.default_rng(rows + inner)
    runs = np.sort(rng.integers(-1, held, rows // 2))
    ops = _adapters(rows, inner, cols, rank, held, np.concatenate([runs, rng.integers(-1, held, rows - len(runs))]))
    assert next(o for o in ops.build() if isinstance(o, AdapterUpOp)).many
    _adapter_check(ops)


@pytest.mark.parametrize("rows, rank", [(19, 6), (140, 6), (1030, 6), (80000, 64)])
def test_adapters_of_strided_rows(rows, rank):
    _adapter_check(_adapters(rows, 130, 70, rank, 3, [i % 4 - 1 for i in range(rows)], strides=True))


@pytest.mark.parametrize("rows, rank, held", [(128, 5, 3), (130, 16, 300), (700, 8, 1), (1025, 7, 64), (4099, 4, 600), (8300, 6, 40)])
@pytest.mark.parametrize("kind", ["random", "turns", "runs", "few"])
def test_adapters_by_any_order_of_rows(rows, rank, held, kind):
    """Rows of many adapters, also more than are put in order at once: against the formula,
    and another order of the same rows gives the same bits."""
    rng = np.random.default_rng(rows)
    ids = {"random": rng.integers(-1, held + 1, rows), "turns": np.arange(rows) % held, "runs": np.arange(rows) // 33 % held,
           "few": np.where(rng.random(rows) < 0.01, held - 1, -1)}[kind]
    ops = _adapters(rows, 70, 37, rank, held, ids)
    y = _adapter_check(ops)
    other = rng.permutation(rows)
    again = _adapters(rows, 70, 37, rank, held, ids[other])
    for name in ("x", "base"):
        again.uploads[name][:] = ops.uploads[name][other]
    np.testing.assert_array_equal(run(again).env["y"], y[other])


def test_adapters_rows_do_not_mix():
    """Infinities and NaN of a row, and of an adapter, stay with the rows that have them."""
    ops = _adapters(18, 200, 40, 9, 4, [0, 1, 2, 3, -1, 0] * 3, scales=False)
    ops.uploads["x"][1, 7], ops.uploads["x"][3, 100] = np.inf, np.nan
    ops.uploads["a"][2 * 9 + 1, 5] = np.nan
    clean = _adapters(18, 200, 40, 9, 4, [0, 1, 2, 3, -1, 0] * 3, scales=False)
    got, want = run(ops).env["y"], run(clean).env["y"]
    for m in range(18):
        if m in (1, 3) or m % 6 == 2:
            assert not np.any(np.isfinite(got[m]))
        else:
            np.testing.assert_array_equal(got[m], want[m])


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------


def _sample_ops(x, u, **asked):
    ops = Operations()
    _put(ops, "x", np.asarray(x, np.float32))
    _put(ops, "u", np.asarray(u, np.float32))
    rows = ops.uploads["x"].shape[0]
    for name, v in asked.items():
        _put(ops, name, np.broadcast_to(np.asarray(v, np.int32 if name == "top_k" else np.float32), (rows,)).copy())
    ops.sample("x", uniforms="u", out="t", logprobs="lp", **{n: n for n in asked})
    return ops


def _sample_check(ops):
    env, ref = run(ops).env, evaluate(ops)
    np.testing.assert_array_equal(env["t"], ref["t"])
    n = ops.tensors["x"].shape[1]
    _close(env["lp"], ref["lp"], 1.01 * U * np.abs(ref["lp"]) + n * 2.0 ** -min(44, 62 - (n - 1).bit_length()) + 2.0**-149)
    return env["t"]


FILTERS = [
    {}, {"temperatures": 0.7}, {"top_k": 1}, {"top_k": 40, "temperatures": 1.3}, {"top_p": 0.9}, {"min_p": 0.05},
    {"top_k": 50, "top_p": 0.8, "min_p": 0.02, "temperatures": 0.6}, {"top_p": 0.999, "temperatures": 2.0},
    {"top_k": 1000, "top_p": 0.95}, {"temperatures": 0.0}, {"temperatures": 0.01, "top_k": 7}, {"temperatures": 1e30, "top_p": 0.5},
]


@pytest.mark.parametrize("rows, cols", [(1, 1), (2, 2), (5, 63), (7, 1000), (3, 4096), (4, 4097), (3, 8191), (2, 32003), (2, 131072)])
@pytest.mark.parametrize("asked", FILTERS)
def test_sample(rows, cols, asked):
    rng = np.random.default_rng(rows * 7 + cols)
    x = 2 * rng.standard_normal((rows, cols)).astype(np.float32)
    x[:, rng.integers(0, cols, 5)] += 6
    _sample_check(_sample_ops(x, rng.random(rows), **asked))


def test_sample_rows_ask_for_different_things():
    rng = np.random.default_rng(3)
    rows = 64
    _sample_check(_sample_ops(
        3 * rng.standard_normal((rows, 5003)), rng.random(rows), temperatures=rng.choice([0.0, 0.5, 1.0, -1.0, np.nan, 3.0], rows),
        top_k=rng.choice([0, 1, 5, 100, 5003, 10**6, -3], rows), top_p=rng.choice([0.0, 0.3, 0.9, 1.0, 2.0, -1.0, np.nan], rows),
        min_p=rng.choice([0.0, 0.1, 1.0, 5.0, -1.0, np.nan], rows)))


@pytest.mark.parametrize("cols", [8, 1000, 20000])
def test_sample_equal_logits(cols):
    """Ties: every index of a row of equals, cut by k and by p in the middle of them."""
    u = (np.arange(16) + 0.5) / 16
    x = np.zeros((16, cols), np.float32)
    x[:, ::2] = -0.0  # (no other value than 0)
    assert len(set(_sample_check(_sample_ops(x, u)).tolist())) == min(16, cols)
    for asked in ({"top_k": cols // 4}, {"top_p": 0.5}, {"top_k": cols // 2, "top_p": 0.5}, {"min_p": 1.0}):
        t = _sample_check(_sample_ops(x, u, **asked))
        assert t.max() < cols // (4 if "top_k" in asked else 2) or "min_p" in asked
    x[:, 5:] = -1.0
    x[:, cols - 1] = 2.0
    for asked in ({"top_k": 3}, {"top_k": 7, "top_p": 0.75}, {"top_p": 0.9, "temperatures": 0.25}, {"top_k": cols - 1}):
        _sample_check(_sample_ops(x, u, **asked))


@pytest.mark.parametrize("cols", [30, 9000])
def test_sample_uniforms_at_their_ends(cols):
    """u of 0, next to 1, and outside: the first and the last that stayed."""
    rng = np.random.default_rng(8)
    u = np.array([0.0, 1 - 2.0**-24, 1.0, 7.0, -1.0, np.nan, np.inf, -np.inf, 1e-45], np.float32)
    x = np.tile(rng.standard_normal(cols).astype(np.float32), (9, 1))
    x[:, 0] = x[:, -1] = -np.inf
    for asked in ({}, {"top_k": 9}, {"top_p": 0.4}, {"min_p": 0.3}):
        t = _sample_check(_sample_ops(x, u, **asked))
        assert t[0] == t[4] == t[5] == t[7] > 0 and t[2] == t[3] == t[6] < cols - 1


@pytest.mark.parametrize("cols", [5, 700, 12345])
def test_sample_masked_rows(cols):
    """Rows of -inf, of the type's lowest value, with infinities and NaN, one that is left."""
    low = np.finfo(np.float32).min
    x = np.zeros((9, cols), np.float32)
    x[0] = -np.inf
    x[1] = low
    x[2, 3] = np.nan
    x[3], x[3, 4] = -np.inf, -3.0
    x[4, 1] = x[4, 3] = np.inf
    x[5], x[5, 2] = -np.inf, low
    x[6, 0] = -np.nan
    x[7], x[7, 1], x[7, 2] = low, 3e38, np.inf
    x[8] = 1e-45
    u = np.full(9, 0.6)
    for asked in ({}, {"top_k": 2}, {"top_p": 0.7}, {"min_p": 0.5}, {"temperatures": 0.0}, {"top_k": 4, "top_p": 0.5},
                  {"temperatures": np.inf}, {"temperatures": 1e-45}):
        t = _sample_check(_sample_ops(x, u, **asked))
        assert t[0] == t[2] == t[6] == -1 and t[3] == 4 and t[5] == 2


@pytest.mark.parametrize("cols", [300, 30000])
def test_sample_cut_between_weights(cols):
    """p next to where a third of the logits, all equal, weigh as much as the rest: 32 bits
    do not see on which side it is, 64 do."""
    p = np.float32(0.5) + np.arange(-8, 9).astype(np.float32) * np.float32(2.0**-24)
    x = np.full((17, cols), -np.log(2.0), np.float32)
    x[:, : cols // 3] = 0.0
    t = _sample_check(_sample_ops(x, np.full(17, 1 - 2.0**-24), top_p=p))
    assert (t < cols // 3).any() and (t >= cols // 3).any()


@pytest.mark.parametrize("rows, cols", [(1, 40000), (3, 70001), (2, 262144)])
@pytest.mark.parametrize("scale", [0.1, 1.0, 30.0, 1e6])
def test_sample_spreads_of_logits(rows, cols, scale):
    """From rows that are next to even -- more in a bin than are listed -- to ones in which a
    few logits have all the weight, or are past the bins' grid."""
    rng = np.random.default_rng(cols)
    x = scale * rng.standard_normal((rows, cols))
    for asked in ({}, {"top_p": 0.6}, {"top_k": 30}, {"top_k": 20000}, {"top_k": 20000, "top_p": 0.3}, {"min_p": 0.4},
                  {"top_k": 300, "top_p": 0.7, "min_p": 0.01}):
        _sample_check(_sample_ops(x, rng.random(rows), **asked))


@pytest.mark.parametrize("rows, cols", [(3, 600), (2, 50000), (1, 300000)])
def test_sample_logits_of_few_bits(rows, cols):
    """Logits of eight bits, as of a product in bfloat16: hundreds are equal at every cut."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x = (x.view(np.uint32) & 0xFFFF0000).view(np.float32)
    for asked in ({}, {"top_p": 0.6}, {"top_k": 300}, {"top_k": 2000, "top_p": 0.5}, {"top_k": 150, "top_p": 0.7},
                  {"top_k": 37, "top_p": 0.01, "temperatures": 0.3}, {"top_p": 0.97, "min_p": 0.02, "temperatures": 1.7}):
        _sample_check(_sample_ops(x, rng.random(rows), **asked))


@pytest.mark.parametrize("rows, cols", [(520, 9000), (1, 1048576), (700, 70), (65, 33000)])
def test_sample_many_rows_and_columns(rows, cols):
    rng = np.random.default_rng(rows)
    x = 2 * rng.standard_normal((rows, cols)).astype(np.float32)
    _sample_check(_sample_ops(x, rng.random(rows), top_k=rng.choice([0, 40, 3000], rows), top_p=rng.choice([0.5, 0.95, 1.0], rows),
                              temperatures=rng.choice([0.0, 0.5, 1.0], rows)))


def test_sample_a_bin_of_many():
    """Rows of one chunk, all of whose logits are in one bin: more than 16 bits count."""
    rows, cols = 260, 131072
    u = (np.arange(rows) + 0.5) / rows
    ops = _sample_ops(np.zeros((rows, cols), np.float32), u, top_k=70000)
    assert len(ops.build()) == 1
    t = run(ops).env["t"]
    np.testing.assert_array_equal(t, np.floor(u.astype(np.float32).astype(np.float64) * 70000).astype(np.int32))


@pytest.mark.parametrize("cols", [301, 30001])
def test_sample_of_strided_logits(cols):
    rng = np.random.default_rng(9)
    ops = Operations()
    _put(ops, "x_", rng.standard_normal((cols, 4)).astype(np.float32))
    ops.transpose("x_", out="x")
    _put(ops, "u", rng.random(4).astype(np.float32))
    _put(ops, "k", np.array([3, 0, 50, 1], np.int32))
    ops.sample("x", uniforms="u", out="t", top_k="k")
    np.testing.assert_array_equal(run(ops).env["t"], evaluate(ops)["t"])


def test_sample_draws_what_it_says():
    """Over an even grid of numbers, each token comes as often as its probability says (a
    token's share of the grid is off by one point at the most)."""
    x = np.array([1.0, 0.0, 2.0, -1.0, 0.5], np.float32)
    n = 4000
    t = _sample_check(_sample_ops(np.tile(x, (n, 1)), (np.arange(n) + 0.5) / n, temperatures=0.8))
    p = np.exp(x.astype(np.float64) / np.float32(0.8))
    assert np.all(np.abs(np.bincount(t, minlength=5) - n * p / p.sum()) <= 1)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

HEADS, KV_HEADS, DIM, COLS = 4, 2, 32, 100


def _step(seed, sequences=5):
    """A decode step: slots and positions, adapters beside a shared product, rotation, the
    cache written, attention over it, logits and tokens."""
    rng = np.random.default_rng(seed)
    ops = Operations()
    spec = KVCache(pages=40, page_size=8, kv_heads=KV_HEADS, dim=DIM)
    lengths = rng.integers(0, 30, sequences).astype(np.int32)
    lengths[0], lengths[1] = 0, 16
    table = np.full((sequences, 5), -1, np.int32)
    order = rng.permutation(40).astype(np.int32)
    at = 0
    for b, n in enumerate(-(-lengths // 8)):
        table[b, :n] = order[at : at + n]
        at += n
    counts = np.ones(sequences, np.int32)
    counts[-1] = 0
    for name, v in (("pages", table), ("free", order[at:]), ("lengths", lengths), ("counts", counts)):
        _put(ops, name, v)
    kv = rng.standard_normal((2, spec.slots, KV_HEADS, DIM)).astype(np.float32)
    ops.kv_cache("cache", pages=40, page_size=8, kv_heads=KV_HEADS, dim=DIM)
    ops.from_numpy(spec.pack(kv[0], kv[1]), "cache")
    for name, shape in (("x", (sequences, 64)), ("wq", (64, HEADS * DIM)), ("k", (sequences, KV_HEADS * DIM)),
                        ("v", (sequences, KV_HEADS * DIM)), ("a", (3 * 4, 64)), ("b", (3 * HEADS * DIM, 4)),
                        ("wo", (HEADS * DIM, COLS))):
        _put(ops, name, (rng.standard_normal(shape) / 8).astype(np.float32))
    _put(ops, "ids", rng.integers(-1, 3, sequences).astype(np.int32))
    _put(ops, "u", rng.random(sequences).astype(np.float32))
    _put(ops, "topk", np.full(sequences, 5, np.int32))
    ops.page_tables("pages", free="free", lengths="lengths", counts="counts", page_size=8, tokens=sequences, out="table",
                    slots="slots", positions="at", ends="ends", used="used")
    ops.matmul("x", "wq", out="q0")
    ops.adapters("x", base="q0", a="a", b="b", ids="ids", out="q1")
    ops.rotary("q1", positions="at", out="q", rotary=Rotary(dim=DIM), k="k", k_out="kr")
    ops.cache_write("cache", k="kr", v="v", slots="slots", out="cache1")
    ops.paged_attention("q", cache="cache1", pages="table", lengths="ends", heads=HEADS, out="o")
    ops.matmul("o", "wo", out="logits")
    ops.sample("logits", uniforms="u", out="tokens", top_k="topk")
    return ops


NAMES = ["table", "slots", "at", "ends", "used", "q1", "q", "kr", "o", "logits", "tokens"]


def test_a_decode_step():
    """Each op's result from what it was given on the GPU, so that no rounding before it
    decides a cut: whole numbers exactly, the rest by the fp32 bars of their sizes (a few
    dozen terms around 1: 2^-14 of the largest)."""
    ops = _step(1)
    env, ref = run(ops, outputs=NAMES).env, evaluate(ops)
    for name in ("table", "slots", "at", "ends", "used"):
        np.testing.assert_array_equal(env[name], ref[name], err_msg=name)
    for name in ("q1", "q", "kr", "o", "logits"):
        assert np.abs(env[name] - ref[name]).max() <= 2.0**-14 * np.abs(ref[name]).max(), name
    u, k = ops.uploads["u"], ops.uploads["topk"]
    want = [decoding_eval.sample_row(env["logits"][b], u[b], top_k=k[b])[0] for b in range(5)]
    np.testing.assert_array_equal(env["tokens"], want)


def test_a_batch_of_decode_steps():
    programs = [_step(s) for s in range(1, 5)]
    for ops, got in zip(programs, run_batch(programs, outputs=NAMES)):
        alone = run(ops, outputs=NAMES).env
        for name in NAMES:
            np.testing.assert_array_equal(got.env[name], alone[name], err_msg=name)


def test_a_loop_of_steps_keeps_its_buffers():
    """The program compiled once and run again and again over one dict of buffers, as a
    serving loop does; every run gives what the first gave."""
    ops = _step(2)
    groups = compile_program(ops)
    env = {}
    for name, v in ops.uploads.items():
        env[name] = Buffer.from_numpy(v)
    for t in ops.tensors.values():
        if t.buffer_key not in env:
            env[t.buffer_key] = Buffer(t.nbytes)
    runtime = Runtime(tuple(Dispatch(g.kernel, g.bindings, g.dims, g.grid, g.threads) for g in groups))
    want = run(ops, outputs=NAMES).env
    for _ in range(3):
        runtime.run(env)
        for name in NAMES:
            t = ops.tensors[name]
            np.testing.assert_array_equal(env[t.buffer_key].numpy(t.shape, np.dtype(t.stored)), want[name], err_msg=name)


def test_steps_of_two_threads():
    programs = [_step(7), _step(8)]
    want = [run(p, outputs=NAMES).env for p in programs]
    got: list = [None, None]

    def work(i):
        for _ in range(4):
            got[i] = run(programs[i], outputs=NAMES).env

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        for name in NAMES:
            np.testing.assert_array_equal(a[name], b[name], err_msg=name)


def test_one_tensor_for_several_arguments():
    rng = np.random.default_rng(77)
    ops = Operations()
    spec = Rotary(dim=16)
    _put(ops, "x", rng.standard_normal((6, 32)).astype(np.float32))
    _put(ops, "n", np.array([3, 0, 5, 1, 2, 4], np.int32))
    ops.rotary("x", positions="n", out="y", rotary=spec, k="x", k_out="z")
    _put(ops, "ab", rng.standard_normal((64, 32)).astype(np.float32))
    ops.adapters("x", base="x", a="ab", b="ab", ids="n", out="w")
    _put(ops, "u", rng.random(6).astype(np.float32))
    ops.sample("x", uniforms="u", temperatures="u", top_k="n", top_p="u", min_p="u", out="t")
    _put(ops, "table", np.full((6, 9), -1, np.int32))
    ops.page_tables("table", free="n", lengths="n", counts="n", page_size=4, tokens=20, out="table1", slots="s", positions="p",
                    ends="e", used="used")
    env, ref = run(ops).env, evaluate(ops)
    bound = _rotary_bound(spec, ops.uploads["x"], ops.uploads["n"])
    _close(env["y"], ref["y"], bound)
    _close(env["z"], ref["z"], bound)
    held = np.abs(ops.uploads["ab"].astype(np.float64)).reshape(2, 32, 32)  # two adapters' A, and their B
    each = np.zeros((6, 32))
    for m, i in enumerate(ops.uploads["n"]):
        if i < 2:
            each[m] = held[i] @ (held[i] @ np.abs(ops.uploads["x"][m].astype(np.float64)))
    # (_adapter_bound's terms: one block of 64 columns, the waves, one share; rank 32)
    _close(env["w"], ref["w"], np.abs(ref["w"]) * U + 1.01 * U * (2 * 64 + ADAPTER_DOWN_WAVES + 1 + 2 * (32 + 15)) * each + 2.0**-149)
    for name in ("t", "table1", "s", "p", "e", "used"):
        np.testing.assert_array_equal(env[name], ref[name], err_msg=name)


@pytest.mark.parametrize("rows, cols", [(4, 50), (4, 300), (2, 40000)])
def test_sample_weights_just_below_the_largest(rows, cols):
    """min_p = 1 keeps the largest and its equals, however close the others come; all that are
    finite at an infinite temperature."""
    x = np.full((rows, cols), -1e-20, np.float32)
    x[:, [1, cols - 2]] = 0.0
    x[:, 3] = -1e-25
    x[:, 4] = -np.inf
    for asked in ({"min_p": 1.0}, {"min_p": 1.0, "top_k": 100}, {"min_p": 1.0, "top_p": 0.9, "temperatures": 1e30},
                  {"min_p": 0.5, "temperatures": np.inf}, {"min_p": 1.0, "temperatures": np.inf}):
        ops = _sample_ops(x, (np.arange(rows) + 0.5) / rows, **asked)
        t = _sample_check(ops)
        if asked.get("temperatures") != np.inf:
            assert set(t) == {1, cols - 2}


@pytest.mark.parametrize("rows, cols", [(3, 50), (3, 40000)])
def test_run_again_with_other_inputs(rows, cols):
    """Nothing is kept from a call for the next: a program run over and over, other logits,
    numbers and ids each time, scratch as the run before left it."""
    rng = np.random.default_rng(cols)
    for _ in range(3):
        x = (3 * rng.standard_normal((rows, cols))).astype(np.float32)
        ops = _sample_ops(x, rng.random(rows), top_k=rng.integers(0, 60, rows), top_p=rng.uniform(0.2, 1.1, rows))
        _sample_check(ops)


class _Kept:
    """A program compiled once, and its buffers, which start full of 0xF9 bytes: what no
    kernel writes is no token (-101058055), and no scratch is clear."""

    def __init__(self, ops):
        groups = compile_program(ops)
        self.ops, self.env = ops, {name: Buffer.from_numpy(v) for name, v in ops.uploads.items()}
        for t in ops.tensors.values():
            if t.buffer_key not in self.env:
                self.env[t.buffer_key] = Buffer(t.nbytes)
                self.env[t.buffer_key].fill(0xF9)
        self.runtime = Runtime(tuple(Dispatch(g.kernel, g.bindings, g.dims, g.grid, g.threads) for g in groups))

    def run(self, **inputs):
        """With other inputs, where given; all that the program has made."""
        for name, v in inputs.items():
            self.ops.uploads[name][...] = v
            self.env[name].write(self.ops.uploads[name])
        self.runtime.run(self.env)
        return {n: self.env[t.buffer_key].numpy(t.shape, np.dtype(t.stored)) for n, t in self.ops.tensors.items()}


def _sample_compare(ops, env):
    ref = evaluate(ops)
    np.testing.assert_array_equal(env["t"], ref["t"])
    n = ops.tensors["x"].shape[1]
    _close(env["lp"], ref["lp"], 1.01 * U * np.abs(ref["lp"]) + n * 2.0 ** -min(44, 62 - (n - 1).bit_length()) + 2.0**-149)


OFF = {"top_k": (0, -3, 10**6), "top_p": (1.0, 2.0, np.nan)}  # what cuts nothing


@pytest.mark.parametrize("cols", [5, 700, 12345, 40000])
@pytest.mark.parametrize("temperature", [1.0, 1e-36, 1e-37, 1e-38, 1e-45, 3e38, np.inf])
def test_sample_rows_off_the_grid_that_nothing_cuts(cols, temperature):
    """Rows that k and p leave whole in programs that have k or p: with infinities one in four
    neighbours and four, and logits that fp32 does not hold divided by the temperature."""
    rng = np.random.default_rng(cols)
    low, x = np.finfo(np.float32).min, rng.standard_normal((9, cols)).astype(np.float32)
    x[0, 3] = np.inf
    x[1, 1] = x[1, cols - 1] = np.inf
    x[2, :4] = np.inf
    x[3], x[3, 2] = low, 30.0
    x[4], x[4, 4] = -np.inf, np.inf
    x[5], x[5, 0] = -30.0, low
    x[6] = np.inf
    x[7, 2], x[7, 4] = 3e38, -np.inf
    for name, values in OFF.items():
        for off in values:
            ops = _sample_ops(x, rng.random(9), temperatures=temperature, **{name: off})
            _sample_compare(ops, _Kept(ops).run())


@pytest.mark.parametrize("cols", [700, 12345, 40000])
def test_sample_rows_cut_and_whole_with_infinities(cols):
    """The same rows beside each other cut by k, by p, by both and by neither, at ordinary and
    at tiny temperatures."""
    rng = np.random.default_rng(cols + 1)
    low, rows = np.finfo(np.float32).min, 256
    x = 3 * rng.standard_normal((rows, cols)).astype(np.float32)
    x[0::8, 3] = np.inf
    x[1::8, 1] = x[1::8, cols - 1] = np.inf
    x[2::8, 8:12] = np.inf
    x[3::8] = -np.inf
    x[3::8, 6] = 1.0
    x[4::8, 9:] = low
    x[5::8], x[5::8, 7] = low, np.inf
    ops = _sample_ops(
        x, rng.random(rows), temperatures=rng.choice([1.0, 0.7, 1e-36, 1e-38, 1e-45, 0.0, np.inf], rows),
        top_k=rng.choice([0, 2, 50, 10**6], rows), top_p=rng.choice([1.0, 0.7, np.nan], rows), min_p=rng.choice([0.0, 0.5], rows))
    _sample_compare(ops, _Kept(ops).run())


def _grow(ops, i, pages, lengths, free="free", **call):
    ops.page_tables(pages, free=free, lengths=lengths, counts=f"counts{i}", page_size=call.pop("page_size"), tokens=call.pop("tokens"),
                    out=f"table{i}", slots=f"slots{i}", positions=f"positions{i}", ends=f"ends{i}", used=f"used{i}", **call)


@pytest.mark.parametrize("sequences, width, page_size, tokens", [(1, 40, 1, 9), (5, 9, 4, 30), (300, 12, 16, 700), (1030, 8, 3, 4000)])
def test_a_table_grows_by_several_steps(sequences, width, page_size, tokens):
    """Three steps in a program, from one list: each goes on where the one before ended, so
    every page has one owner."""
    rng = np.random.default_rng(sequences)
    ops = Operations()
    _put(ops, "table0", np.full((sequences, width), -1, np.int32))
    _put(ops, "free", rng.permutation(sequences * width).astype(np.int32))
    _put(ops, "ends0", np.zeros(sequences, np.int32))
    for i in (1, 2, 3):
        _put(ops, f"counts{i}", rng.integers(0, width * page_size // 4 + 2, sequences).astype(np.int32))
        _grow(ops, i, f"table{i - 1}", f"ends{i - 1}", page_size=page_size, tokens=tokens)
    names = [f"{n}{i}" for i in (1, 2, 3) for n in ("slots", "positions", "ends", "used")] + ["table3"]
    env, ref = run(ops, outputs=names).env, evaluate(ops)
    for name in names:
        np.testing.assert_array_equal(env[name], ref[name], err_msg=name)
    held = env["table3"][env["table3"] >= 0]
    assert len(held) == len(set(held.tolist())) == env["used3"][0]


@pytest.mark.parametrize("taken", [0, 3, 7, 8, 100, 2**31 - 1, -1, -(2**31)])
def test_page_tables_behind_what_is_taken(taken):
    """From the middle of the list, its end and behind it; numbers below 0 are 0."""
    ops = Operations()
    _put(ops, "table0", np.full((3, 5), -1, np.int32))
    _put(ops, "free", np.arange(10, 18, dtype=np.int32))
    for name, v in (("ends0", [0, 4, 9]), ("counts1", [9, 1, 6]), ("gone", [taken])):
        _put(ops, name, np.array(v, np.int32))
    _grow(ops, 1, "table0", "ends0", page_size=4, tokens=20, taken="gone")
    env, ref = run(ops).env, evaluate(ops)
    for name in ("table1", "slots1", "positions1", "ends1", "used1"):
        np.testing.assert_array_equal(env[name], ref[name], err_msg=name)


def test_a_loop_of_steps_that_grow():
    """A program run again and again over its buffers, each step's lengths and what is gone of
    the list from the step before: a table that fills up page by page, and attention over it
    that reads what each step wrote."""
    rng = np.random.default_rng(21)
    sequences, page_size, width, heads, dim = 6, 4, 5, 2, 32
    spec = KVCache(pages=sequences * width, page_size=page_size, kv_heads=heads, dim=dim)
    ops = Operations()
    _put(ops, "table0", np.full((sequences, width), -1, np.int32))
    _put(ops, "free", rng.permutation(sequences * width).astype(np.int32))
    _put(ops, "ends0", np.zeros(sequences, np.int32))
    _put(ops, "gone", np.zeros(1, np.int32))
    _put(ops, "counts1", np.ones(sequences, np.int32))
    for name in ("q", "k", "v"):
        _put(ops, name, np.zeros((sequences, heads * dim), np.float32))
    ops.kv_cache("cache", pages=spec.pages, page_size=page_size, kv_heads=heads, dim=dim)
    ops.from_numpy(spec.empty(), "cache")
    _grow(ops, 1, "table0", "ends0", page_size=page_size, tokens=sequences, taken="gone")
    ops.cache_write("cache", k="k", v="v", slots="slots1", out="cache1")
    ops.paged_attention("q", cache="cache1", pages="table1", lengths="ends1", heads=heads, out="o")
    kept, more = _Kept(ops), {}
    for step in range(width * page_size + 2):
        data = {n: rng.standard_normal((sequences, heads * dim)).astype(np.float32) for n in ("q", "k", "v")}
        counts = (np.arange(sequences) % 3 <= step % 3).astype(np.int32)  # (not all go on in each)
        got = kept.run(**data, counts1=counts, **more)
        ref = evaluate(ops)
        for name in ("table1", "slots1", "positions1", "ends1", "used1"):
            np.testing.assert_array_equal(got[name], ref[name], err_msg=f"{name}, step {step}")
        # (attention's sum of up to 20 products of terms around 1: 2^-14 of the largest)
        assert np.abs(got["o"] - ref["o"]).max() <= 2.0**-14 * max(1.0, np.abs(ref["o"]).max())
        ops.uploads["table0"][...], ops.uploads["cache"][...] = got["table1"], got["cache1"]  # (the oracle's next state)
        more = {"ends0": got["ends1"], "gone": got["used1"]}
    held = got["table1"][got["table1"] >= 0]
    assert len(held) == len(set(held.tolist())) == got["used1"][0] and (got["ends1"] == width * page_size).any()


def _sample_inputs(rng, rows, cols):
    """Logits and what rows ask of them: cut or whole, greedy, masked, and drawn from by one
    workgroup (a bin of more logits than are listed)."""
    x = (3 * rng.standard_normal((rows, cols))).astype(np.float32)
    kind = rng.integers(0, 7, rows)
    x[kind == 0] = rng.standard_normal((int((kind == 0).sum()), cols)) / 100  # (one bin of all)
    x[kind == 1, rng.integers(0, cols)] = np.nan
    x[kind == 2] = -np.inf
    x[kind == 2, rng.integers(0, cols)] = 5
    x[kind == 3, rng.integers(0, cols)] = np.inf
    return {
        "x": x, "u": rng.random(rows), "temperatures": rng.choice([0.0, 0.7, 1.0, 1.5, 1e-38], rows),
        "top_k": np.where(kind == 0, cols // 3, rng.choice([0, 1, 30, 400, 10**6], rows)),
        "top_p": rng.choice([0.3, 0.9, 0.99, 1.0, np.nan], rows), "min_p": rng.choice([0.0, 0.05], rows),
    }


@pytest.mark.parametrize("rows, cols", [(24, 300), (24, 40000), (3, 131072), (24, 9001)])
def test_sample_again_in_its_buffers(rows, cols):
    """Nothing is kept from a call for the next: one program over one set of buffers, other
    logits and numbers in each run, so that rows change between the paths, over scratch as
    the run before left it.  Answers are cleared to what is no token before each run."""
    rng = np.random.default_rng(rows * cols)
    first = _sample_inputs(rng, rows, cols)
    kept = _Kept(_sample_ops(first.pop("x"), first.pop("u"), **first))
    for _ in range(6):
        for name in ("t", "lp"):
            kept.env[name].fill(0xF9)
        _sample_compare(kept.ops, kept.run(**_sample_inputs(rng, rows, cols)))


@pytest.mark.parametrize("rows, inner, cols, rank, held", [
    (9, 300, 70, 8, 4), (128, 300, 70, 8, 4), (200, 257, 65, 16, 90), (700, 130, 37, 5, 300), (4200, 70, 37, 4, 50),
    (2048, 2600, 2561, 64, 40),
])
def test_adapters_again_in_their_buffers(rows, inner, cols, rank, held):
    """The same for adapters: other rows, ids in another order -- in runs, at random, of few,
    none, all alike -- and other weights each time."""
    rng = np.random.default_rng(rows + rank)
    kept = _Kept(_adapters(rows, inner, cols, rank, held, rng.integers(-1, held, rows)))
    kinds = (np.arange(rows) * held // rows, rng.integers(-1, held + 1, rows), np.where(rng.random(rows) < 0.03, held - 1, -1),
             np.full(rows, -1), np.full(rows, held // 2), np.arange(rows)[::-1] % held)
    for ids in kinds:
        kept.env["y"].fill(0xF9)
        env = kept.run(x=rng.standard_normal((rows, inner)), base=rng.standard_normal((rows, cols)), ids=ids,
                       a=rng.standard_normal((held * rank, inner)), s=rng.uniform(-2, 2, held))
        _close(env["y"], evaluate(kept.ops)["y"], _adapter_bound(kept.ops))


def test_rotary_again_in_its_buffers():
    rng = np.random.default_rng(31)
    spec = Rotary(dim=64, part=48, layout="interleaved")
    ops = Operations()
    _put(ops, "q", np.zeros((70, 192), np.float32))
    _put(ops, "k", np.zeros((70, 64), np.float32))
    _put(ops, "at", np.zeros(70, np.int32))
    ops.rotary("q", positions="at", out="q1", rotary=spec, k="k", k_out="k1")
    kept = _Kept(ops)
    for far in (100, 2**20, 2**31 - 1):
        env = kept.run(q=rng.standard_normal((70, 192)), k=rng.standard_normal((70, 64)), at=rng.integers(-far, far, 70))
        ref = evaluate(ops)
        for name, out in (("q", "q1"), ("k", "k1")):
            _close(env[out], ref[out], _rotary_bound(spec, ops.uploads[name], ops.uploads["at"]))


@pytest.mark.parametrize("rows, cols", [(513, 12345), (600, 4097), (300, 66000)])
def test_sample_long_rows_of_one_chunk(rows, cols):
    """So many rows that one workgroup has each: one kernel, without scratch."""
    rng = np.random.default_rng(rows)
    first = _sample_inputs(rng, rows, cols)
    kept = _Kept(_sample_ops(first.pop("x"), first.pop("u"), **first))
    assert len(kept.ops.build()) == 1
    _sample_compare(kept.ops, kept.run())


def _grown(seed, pages, sequences=5, width=6, page_size=4, heads=2, dim=16):
    """Two steps of prompts in a program, from a list of ``pages``; attention behind each."""
    rng = np.random.default_rng(seed)
    ops = Operations()
    spec = KVCache(pages=sequences * width, page_size=page_size, kv_heads=heads, dim=dim)
    _put(ops, "table0", np.full((sequences, width), -1, np.int32))
    _put(ops, "free", rng.permutation(spec.pages)[:pages].astype(np.int32))
    _put(ops, "ends0", np.zeros(sequences, np.int32))
    ops.kv_cache("cache0", pages=spec.pages, page_size=page_size, kv_heads=heads, dim=dim)
    ops.from_numpy(spec.empty(), "cache0")
    _put(ops, "q", rng.standard_normal((sequences, heads * dim)).astype(np.float32))
    for i in (1, 2):
        _put(ops, f"counts{i}", rng.integers(0, 11, sequences).astype(np.int32))
        for name in ("k", "v"):
            _put(ops, f"{name}{i}", rng.standard_normal((55, heads * dim)).astype(np.float32))
        _grow(ops, i, f"table{i - 1}", f"ends{i - 1}", page_size=page_size, tokens=55)
        ops.cache_write(f"cache{i - 1}", k=f"k{i}", v=f"v{i}", slots=f"slots{i}", out=f"cache{i}")
        ops.paged_attention("q", cache=f"cache{i}", pages=f"table{i}", lengths=f"ends{i}", heads=heads, out=f"o{i}")
    return ops


GROWN = [f"{n}{i}" for i in (1, 2) for n in ("slots", "positions", "ends", "used", "o")] + ["table2"]


@pytest.mark.parametrize("pages", [30, 7, 1])
def test_two_steps_with_attention(pages):
    """With pages enough, and with too few: what has no page is a hole, then and later."""
    ops = _grown(pages, pages)
    env, ref = run(ops, outputs=GROWN).env, evaluate(ops)
    for name in GROWN:
        if name.startswith("o"):  # (sums of up to 20 products of terms around 1: 2^-14 of the largest)
            assert np.abs(env[name] - ref[name]).max() <= 2.0**-14 * max(1.0, np.abs(ref[name]).max()), name
        else:
            np.testing.assert_array_equal(env[name], ref[name], err_msg=name)
    assert (env["used2"][0] > pages) == (pages < 30)


def test_a_batch_of_two_steps():
    programs = [_grown(s, 14) for s in range(3)]
    for ops, got in zip(programs, run_batch(programs, outputs=GROWN)):
        alone = run(ops, outputs=GROWN).env
        for name in GROWN:
            np.testing.assert_array_equal(got.env[name], alone[name], err_msg=name)
