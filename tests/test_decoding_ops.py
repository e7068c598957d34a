"""The decoding ops without a GPU: what the builder and the scheduler accept and refuse,
the order around a table written in place, a rotation's frequencies, the oracle on cases
worked out by hand, and that every kernel variant compiles for gfx950."""

from __future__ import annotations

import functools
import math

import numpy as np
import pytest

from metellus_amd.api import compile_program
from metellus_amd.orchestrator import Operations, Rotary
from metellus_amd.orchestrator.decoding import ADAPTER_ORDER_ROWS, adapter_many, adapter_splits, sample_chunks
from metellus_amd.orchestrator.fusion import fuse
from metellus_amd.orchestrator.scheduler import schedule
from metellus_amd.runtime import hip_backend
from metellus_amd.runtime.program import Dispatch, Download, Free
from oracle import decoding_eval
from oracle.ir_eval import evaluate


def _ops(**inputs) -> Operations:
    """Inputs by name: a shape, or (shape, dtype)."""
    ops = Operations()
    for name, what in inputs.items():
        if isinstance(what[0], tuple):
            ops.input(name, what[0], dtype=what[1])
        else:
            ops.input(name, what)
    return ops


PAGES = dict(pages=((4, 6), "int32"), free=((9,), "int32"), lengths=((4,), "int32"), counts=((4,), "int32"))
PAGE_CALL = dict(pages="pages", free="free", lengths="lengths", counts="counts", page_size=8, tokens=10, out="table",
                 slots="slots", positions="positions", ends="ends", used="used")
ROTARY = dict(q=(3, 64), k=(3, 32), at=((3,), "int32"))
ADAPTERS = dict(x=(5, 12), y=(5, 20), a=(3 * 4, 12), b=(3 * 20, 4), ids=((5,), "int32"), s=(3,))
ADAPTER_CALL = dict(x="x", base="y", a="a", b="b", ids="ids", out="z")
SAMPLE = dict(x=(3, 50), u=(3,), k=((3,), "int32"), p=(3,))


# -- refusals -------------------------------------------------------------------


@pytest.mark.parametrize("inputs, call, match", [
    (dict(pages=((24,), "int32")), {}, "must be 2D"),
    (dict(pages=(4, 6)), {}, "must be int32"),
    (dict(free=((3, 3), "int32")), {}, "free must be 1D"),
    (dict(free=(9,)), {}, "free must be int32"),
    (dict(lengths=((5,), "int32")), {}, "lengths must have shape"),
    (dict(counts=((3,), "int32")), {}, "counts must have shape"),
    ({}, dict(page_size=0), "page_size must be a positive int"),
    ({}, dict(page_size=True), "page_size must be a positive int"),
    ({}, dict(page_size=2**29), "positions and entries are int32"),
    ({}, dict(tokens=0), "tokens must be a positive int32"),
    ({}, dict(tokens=2**31), "tokens must be a positive int32"),
    ({}, dict(slots="table"), "output names must differ"),
    ({}, dict(ends="free"), "already defined"),
    ({}, dict(pages="nothing"), "is not declared"),
])
def test_page_tables_refusals(inputs, call, match):
    ops = _ops(**{**PAGES, **inputs})
    with pytest.raises(ValueError, match=match):
        ops.page_tables(**{**PAGE_CALL, **call})
    assert not ops.build() and "table" not in ops.tensors and "slots" not in ops.tensors


def test_a_written_table_has_one_name():
    ops = _ops(**PAGES, q=(4, 32))
    ops.kv_cache("cache", pages=20, page_size=8, kv_heads=1, dim=32)
    ops.page_tables(**PAGE_CALL)
    for call in (
        lambda: ops.paged_attention("q", cache="cache", pages="pages", lengths="ends", heads=1, out="o"),
        lambda: ops.transpose("pages", out="t"),
        lambda: ops.reshape("pages", (24,), out="t"),
        lambda: ops.page_tables(**{**PAGE_CALL, **{n: n + "2" for n in ("out", "slots", "positions", "ends", "used")}}),
    ):
        with pytest.raises(ValueError, match="its buffer now holds 'table' — read that"):
            call()
    ops.paged_attention("q", cache="cache", pages="table", lengths="ends", heads=1, out="o")
    more = {**PAGE_CALL, "pages": "table", "lengths": "ends", **{n: n + "2" for n in ("out", "slots", "positions", "ends", "used")}}
    assert ops.page_tables(**more).buffer_key == "pages"  # a step after the step


def test_a_table_with_views_is_not_written():
    ops = _ops(**PAGES)
    ops.reshape("pages", (24,), out="flat")
    with pytest.raises(ValueError, match="can be no view and have none"):
        ops.page_tables(**PAGE_CALL)
    ops = _ops(**PAGES)
    ops.input("wide", (6, 4), dtype="int32")
    ops.reshape("wide", (4, 6), out="view")
    with pytest.raises(ValueError, match="can be no view and have none"):
        ops.page_tables(**{**PAGE_CALL, "pages": "view"})


@pytest.mark.parametrize("inputs, call, match", [
    (dict(q=(3, 60)), {}, "whole heads of 32"),
    (dict(k=(4, 32)), {}, "k must have 3 rows"),
    (dict(at=((4,), "int32")), {}, "positions must have shape"),
    (dict(at=(3,)), {}, "positions must be int32"),
    (dict(q=(96,)), {}, "must be 2D"),
    ({}, dict(k_out=None), "go together"),
    ({}, dict(rotary=128), "must be a Rotary"),
    ({}, dict(out="k"), "already defined"),
    ({}, dict(k_out="q1"), "output names must differ"),
])
def test_rotary_refusals(inputs, call, match):
    ops = _ops(**{**ROTARY, **inputs})
    with pytest.raises(ValueError, match=match):
        ops.rotary(**{**dict(x="q", positions="at", out="q1", rotary=Rotary(dim=32), k="k", k_out="k1"), **call})
    assert not ops.build()


@pytest.mark.parametrize("wrong, match", [
    (dict(dim=0), "dim must be a positive int"),
    (dict(dim=258), "at most 256"),
    (dict(dim=64, part=33), "part must be even"),
    (dict(dim=64, part=66), "part must be even and at most"),
    (dict(dim=63), "part must be even"),
    (dict(dim=64, layout="both"), "layout must be one of"),
    (dict(dim=64, base=0.5), "base must be"),
    (dict(dim=64, base=math.inf), "base must be"),
    (dict(dim=64, factor=0.0), "factor must be"),
    (dict(dim=64, factor=math.nan), "factor must be"),
    (dict(dim=64, original=0), "original must be"),
    (dict(dim=64, original=4096, low=4.0, high=4.0), "low < high"),
    (dict(dim=64, magnitude=math.nan), "magnitude must be"),
    (dict(dim=64, frequencies=(1.0,)), "need as many frequencies"),
    (dict(dim=2, frequencies=(math.nan,)), "finite and within"),
])
def test_rotation_refusals(wrong, match):
    with pytest.raises(ValueError, match=match):
        Rotary(**wrong)


@pytest.mark.parametrize("inputs, call, match", [
    (dict(a=(3 * 4, 13)), {}, "must have shape"),
    (dict(a=(3 * 4 + 1, 12)), {}, "must have shape"),
    (dict(a=(4 * 4, 12)), {}, "must have shape"),
    (dict(b=(3 * 20 + 1, 4)), {}, "must have shape"),
    (dict(b=(60 * 4,)), {}, "b must be 2D"),
    (dict(y=(4, 20)), {}, "as many rows"),
    (dict(ids=((4,), "int32")), {}, "ids must have shape"),
    (dict(ids=(5,)), {}, "ids must be int32"),
    (dict(x=((5, 12), "int8")), {}, "x must be float32"),
    (dict(a=((12, 12), "int8")), {}, "a must be float32"),
    (dict(a=(3 * 257, 12), b=(60, 257)), {}, "ranks up to 256"),
    (dict(s=(4,)), dict(scales="s"), "scales must have shape"),
    ({}, dict(out="x"), "already defined"),
    ({}, dict(a="at"), "a must be dense"),
])
def test_adapters_refusals(inputs, call, match):
    ops = _ops(**{**ADAPTERS, "turned": (12, 12), **inputs})
    ops.transpose("turned", out="at")
    with pytest.raises(ValueError, match=match):
        ops.adapters(**{**ADAPTER_CALL, **call})
    assert not ops.build() and not ops.scratch and "z.down" not in ops.tensors


@pytest.mark.parametrize("inputs, call, match", [
    (dict(x=(50,)), {}, "must be 2D"),
    (dict(x=((3, 50), "int8")), {}, "logits must be float32"),
    (dict(x=(3, 2**20 + 1)), {}, "columns"),
    (dict(u=(4,)), {}, "uniforms must have shape"),
    ({}, dict(top_k="p"), "top_k must be int32"),
    ({}, dict(top_p="k"), "top_p must be float32"),
    (dict(p=(2,)), dict(min_p="p"), "min_p must have shape"),
    (dict(p=(3, 1)), dict(temperatures="p"), "temperatures must be 1D"),
    ({}, dict(out="u"), "already defined"),
    ({}, dict(logprobs="t"), "output names must differ"),
])
def test_sample_refusals(inputs, call, match):
    ops = _ops(**{**SAMPLE, **inputs})
    with pytest.raises(ValueError, match=match):
        ops.sample(**{**dict(logits="x", uniforms="u", out="t"), **call})
    assert not ops.build()


# -- programs ----------------------------------------------------------------------


def test_who_read_the_older_table_comes_first():
    """Attention over the table as it was is before the op that writes it, whatever else it
    waits for."""
    ops = _ops(**PAGES, x=(4, 8), w=(8, 32))
    ops.kv_cache("cache", pages=20, page_size=8, kv_heads=1, dim=32)
    ops.matmul("x", "w", out="q")
    ops.paged_attention("q", cache="cache", pages="pages", lengths="lengths", heads=1, out="o")
    ops.page_tables(**PAGE_CALL)
    ops.paged_attention("q", cache="cache", pages="table", lengths="ends", heads=1, out="o2")
    kinds = [v.ops[0].out.name for v in fuse(ops.build())]
    assert kinds.index("o") < kinds.index("table") < kinds.index("o2")


def test_scheduling_a_table():
    """The new state is downloaded from the input's buffer; the old one is no output."""
    ops = _ops(**PAGES)
    for name, (shape, _) in PAGES.items():
        ops.from_numpy(np.zeros(shape, np.int32), name)
    ops.page_tables(**PAGE_CALL)
    groups = compile_program(ops)
    steps = schedule(ops, groups).fragments
    assert {s.into for s in steps if isinstance(s, Download)} == {"table", "slots", "positions", "ends", "used"}
    some = schedule(ops, groups, outputs=["slots"]).fragments
    assert [s.into for s in some if isinstance(s, Download)] == ["slots"]
    with pytest.raises(ValueError, match="program inputs"):
        schedule(ops, groups, outputs=["pages"])


def test_scheduling_adapters():
    """What lies between the two products is no output, and nothing reads it."""
    ops = _ops(**ADAPTERS)
    ops.adapters(**ADAPTER_CALL, scales="s")
    for name, shape in ADAPTERS.items():
        shape, dtype = shape if isinstance(shape[0], tuple) else (shape, "float32")
        ops.from_numpy(np.zeros(shape, dtype), name)
    groups = compile_program(ops)
    steps = schedule(ops, groups).fragments
    assert [s.into for s in steps if isinstance(s, Download)] == ["z"]
    assert "z.down" in [s.name for s in steps if isinstance(s, Free)]
    assert len([s for s in steps if isinstance(s, Dispatch)]) == 2
    with pytest.raises(ValueError, match="not materialised"):
        schedule(ops, groups, outputs=["z.down"])
    with pytest.raises(ValueError, match="operator's own"):
        ops.reduction("sum", out="r", x="z.down")


def test_scheduling_adapters_of_many_rows():
    """The rows in the order that they are taken in are no output either; fewer rows have none."""
    for rows, own in ((ADAPTER_ORDER_ROWS, {"z.down", "z.order"}), (ADAPTER_ORDER_ROWS - 1, {"z.down"})):
        ops = _ops(x=(rows, 8), y=(rows, 20), a=(12, 8), b=(60, 4), s=(3,), ids=((rows,), "int32"))
        for t in list(ops.tensors.values()):
            ops.from_numpy(np.zeros(t.shape, t.stored), t.name)
        ops.adapters(**ADAPTER_CALL, scales="s")
        steps = schedule(ops, compile_program(ops)).fragments
        assert ops.scratch == own and [s.into for s in steps if isinstance(s, Download)] == ["z"]
        assert set(evaluate(ops)) == own | {"z"}


def test_shares_of_columns():
    few, many = [functools.partial(adapter_splits, many=m) for m in (False, True)]
    assert few(1, 4096) == 8 and few(1, 100) == 1 and few(8, 11008) == 12 and few(32, 4096) == 8 and few(600, 4096) == 5
    assert many(4096, 4096) == 4 and many(3000, 4096) == 5 and many(16384, 4096) == 1
    for rows in (1, 3, 50, 700, 1024, 5000, 20000):
        for inner in (1, 511, 513, 5003, 16384):
            for shares in (few, many):
                assert 1 <= shares(rows, inner) <= -(-inner // 512)
    assert adapter_many(2048, 4096, 4096, 64) and not adapter_many(2048, 4096, 2048, 64) and not adapter_many(2048, 1024, 4096, 64)
    assert not adapter_many(2048, 4096, 4096, 16) and not adapter_many(4096, 1024, 1024, 256)


def test_scheduling_a_draw():
    """Rows of several chunks take two kernels, whose own tensors are no outputs; short ones one."""
    for cols, kernels in ((50, 1), (40000, 2)):
        ops = _ops(**{**SAMPLE, "x": (3, cols)})
        ops.sample("x", uniforms="u", out="t", top_k="k", top_p="p", logprobs="lp")
        for name in SAMPLE:
            t = ops.tensors[name]
            ops.from_numpy(np.zeros(t.shape, t.stored), name)
        steps = schedule(ops, compile_program(ops)).fragments
        assert len([s for s in steps if isinstance(s, Dispatch)]) == kernels
        assert sorted(s.into for s in steps if isinstance(s, Download)) == ["lp", "t"]


def test_chunks_of_a_row():
    assert sample_chunks(1, 131072) == (8192, 16) and sample_chunks(64, 131072) == (16384, 8) and sample_chunks(1, 70) == (4096, 1)
    for rows in (1, 7, 300, 5000):
        for cols in (1, 4096, 4097, 100003, 2**20):
            chunk, chunks = sample_chunks(rows, cols)
            assert chunks * chunk >= cols > (chunks - 1) * chunk and chunks <= 16 and (chunks == 1 or rows * chunks <= 512)


# -- a rotation's frequencies --------------------------------------------------------


@pytest.mark.parametrize("spec", [
    Rotary(dim=128), Rotary(dim=64, factor=4.0), Rotary(dim=128, base=500000.0, factor=8.0, original=8192, low=1.0, high=4.0),
    Rotary(dim=96, part=40, factor=32.0, original=4096), Rotary(dim=4, frequencies=(0.5, -3.0)),
])
def test_frequencies(spec):
    """As the definition says (two ways of the mix: 2^-50 of a value), and in turns: the
    two doubles together are the frequency over 2 pi to 2^-100."""
    np.testing.assert_allclose(spec.angles, decoding_eval.rotary_frequencies(spec), rtol=2.0**-50)
    two_pi = 2 * 31415926535897932384626433832795028841971693993751
    for f, (head, tail) in zip(spec.angles, spec.turns):
        n, d = float(f).as_integer_ratio()
        (hn, hd), (tn, td) = head.as_integer_ratio(), tail.as_integer_ratio()
        # (head + tail) * 2 pi - f, in units of 10^-49 / (hd td d)
        off = abs((hn * td + tn * hd) * two_pi * d - n * 10**49 * hd * td)
        assert off * 2**100 <= abs(n) * 10**49 * hd * td
        assert abs(tail) <= abs(head) * 2.0**-53


# -- the oracle ----------------------------------------------------------------------


def test_oracle_of_a_table():
    ops = _ops(pages=((3, 3), "int32"), free=((4,), "int32"), lengths=((3,), "int32"), counts=((3,), "int32"))
    for name, v in (("pages", [[7, -1, -1], [-1, -1, -1], [1, 2, 3]]), ("free", [9, 8, 6, 5]), ("lengths", [3, 0, 11]), ("counts", [2, 5, 3])):
        ops.from_numpy(np.array(v, np.int32), name)
    ops.page_tables(**{**PAGE_CALL, "page_size": 4, "tokens": 12})
    ref = evaluate(ops)
    np.testing.assert_array_equal(ref["table"], [[7, 9, -1], [8, 6, -1], [1, 2, 3]])
    np.testing.assert_array_equal(ref["positions"], [3, 4, 0, 1, 2, 3, 4, 11, -1, -1, -1, -1])
    np.testing.assert_array_equal(ref["slots"], [31, 36, 32, 33, 34, 35, 24, 15, -1, -1, -1, -1])
    np.testing.assert_array_equal(ref["ends"], [5, 5, 12])
    assert ref["used"] == [3]


def test_oracle_of_a_rotation():
    """A quarter turn takes (1, 0) to (0, 1); the whole rotation is a complex product."""
    ops = _ops(q=(2, 4), at=((2,), "int32"))
    ops.from_numpy(np.array([[1, 2, 0, 5], [1, 2, 0, 5]], np.float32), "q")
    ops.from_numpy(np.array([1, 3], np.int32), "at")
    ops.rotary("q", positions="at", out="y", rotary=Rotary(dim=4, frequencies=(math.pi / 2, 0.0)))
    np.testing.assert_allclose(evaluate(ops)["y"], [[0, 2, 1, 5], [0, 2, -1, 5]], atol=1e-15)


def test_oracle_of_adapters():
    ops = _ops(**ADAPTERS)
    rng = np.random.default_rng(0)
    made = {n: rng.standard_normal(ADAPTERS[n]).astype(np.float32) for n in ("x", "y", "a", "b", "s")}
    made["ids"] = np.array([2, -1, 0, 3, 2], np.int32)
    for n, v in made.items():
        ops.from_numpy(v, n)
    ops.adapters(**ADAPTER_CALL, scales="s")
    got = evaluate(ops)["z"]
    for m, i in enumerate(made["ids"]):
        want = made["y"][m].astype(np.float64)
        if 0 <= i < 3:
            want = want + made["s"][i] * (made["b"][20 * i : 20 * i + 20].astype(np.float64) @ (made["a"][4 * i : 4 * i + 4].astype(np.float64) @ made["x"][m]))
        np.testing.assert_allclose(got[m], want, rtol=1e-6, atol=1e-6)  # (down is rounded to fp32 in between)


def test_oracle_of_a_draw():
    x = np.log(np.array([1, 4, 2, 4, 5], np.float32))
    draw = decoding_eval.sample_row
    assert [draw(x, u)[0] for u in (0.0, 0.05, 0.07, 0.31, 0.35, 0.43, 0.44, 0.68, 0.7, 0.99)] == [0, 0, 1, 1, 2, 2, 3, 3, 4, 4]
    assert draw(x, 0.0, top_k=2)[0] == 1 and draw(x, 0.99, top_k=2)[0] == 4  # 5, and the first of the 4s
    assert draw(x, 0.3, top_p=0.5)[0] == 1 and draw(x, 0.5, top_p=0.5)[0] == 4  # 5 of 16 is less than 8: the first 4 too
    assert draw(x, 0.0, min_p=0.5)[0] == 1 and draw(x, 0.3, min_p=0.9)[0] == 4
    assert draw(x, 0.9, temperature=0.0) == (4, 0.0)
    close = np.array([-1e-20, 0, 0, -1e-25], np.float32)  # all of weight 1 as numbers of 64 bits
    assert draw(close, 0.9, min_p=1.0) == (2, pytest.approx(math.log(1 / 2))) and draw(close, 0.9)[0] == 3
    assert draw(close, 0.9, min_p=1.0, temperature=math.inf)[0] == 3
    assert draw(x, 1.0)[0] == 4 and draw(x, 0.2)[1] == pytest.approx(math.log(4 / 16))
    assert draw(np.array([-np.inf, np.nan]), 0.5)[0] == -1 and draw(np.array([-np.inf] * 2), 0.5)[0] == -1


# -- kernels compile --------------------------------------------------------------------


def _compile(ops: Operations) -> None:
    for g in compile_program(ops):
        hip_backend.compile_only(g.kernel.source)
        hip_backend.compile_only(g.kernel.batched().source)


@pytest.mark.parametrize("sequences", [4, 300])
def test_page_tables_compile(sequences):
    ops = _ops(pages=((sequences, 6), "int32"), free=((9,), "int32"), lengths=((sequences,), "int32"), counts=((sequences,), "int32"))
    ops.page_tables(**PAGE_CALL)
    _compile(ops)


@pytest.mark.parametrize("spec", [Rotary(dim=32), Rotary(dim=32, layout="interleaved"), Rotary(dim=16, part=6),
                                  Rotary(dim=16, part=6, layout="interleaved")])
def test_rotary_compiles(spec):
    ops = _ops(**ROTARY)
    ops.rotary("q", positions="at", out="q1", rotary=spec, k="k", k_out="k1")
    _compile(ops)


@pytest.mark.parametrize("rows", [5, 2000])
@pytest.mark.parametrize("rank", [3, 16, 100])
def test_adapters_compile(rank, rows):
    ops = _ops(**{**ADAPTERS, "x": (rows, 12), "y": (rows, 20), "ids": ((rows,), "int32"), "a": (3 * rank, 12), "b": (60, rank)})
    ops.adapters(**ADAPTER_CALL, scales="s" if rank == 16 else None)
    _compile(ops)


@pytest.mark.parametrize("asked", [{}, dict(top_k="k"), dict(top_k="k", top_p="p", min_p="p", temperatures="p", logprobs="lp")])
@pytest.mark.parametrize("cols", [50, 40000])
def test_sample_compiles(asked, cols):
    ops = _ops(**{**SAMPLE, "x": (3, cols)})
    ops.sample("x", uniforms="u", out="t", **asked)
    _compile(ops)


# -- calls at the border of what is allowed -----------------------------------------------


@pytest.mark.parametrize("taken", ["t", "t.best", "t.counts", "t.bins", "t.sums", "t.list"])
def test_sample_names_differ_from_its_own_tensors(taken):
    """Also from those of the first of the two kernels that rows of several chunks take; a
    refused call leaves no name behind."""
    ops = _ops(**{**SAMPLE, "x": (3, 40000)})
    before = set(ops.tensors)
    with pytest.raises(ValueError, match="output names must differ"):
        ops.sample("x", uniforms="u", out="t", top_k="k", logprobs=taken)
    assert not ops.build() and not ops.scratch and set(ops.tensors) == before
    ops.sample("x", uniforms="u", out="t", top_k="k", logprobs="lp")
    assert len(compile_program(ops)) == 2


@pytest.mark.parametrize("page_size", [np.int32(2**29), np.int64(2**29), np.uint32(2**29), np.int32(2**30)])
def test_page_sizes_of_numpy_are_checked_as_others(page_size):
    """A table's positions are counted in Python's whole numbers, which do not wrap."""
    ops = _ops(**PAGES)
    with pytest.raises(ValueError, match="positions and entries are int32"):
        ops.page_tables(**{**PAGE_CALL, "page_size": page_size})
    wide = _ops(**{**PAGES, "pages": ((4, 9000), "int32")})
    for i, small in enumerate((np.int8(16), np.uint8(16), np.int16(16))):
        call = {**PAGE_CALL, "page_size": small, **{n: f"{n}{i}" for n in ("out", "slots", "positions", "ends", "used")}}
        wide.page_tables(**{**call, "pages": "pages" if i == 0 else f"out{i - 1}"})
    assert [type(op.page_size) for op in wide.build()] == [int] * 3


def test_rotations_by_numbers_of_numpy():
    """Numbers of numpy's types count as the Python numbers that they are equal to: the same
    spec, with the same turns, in the same kernel."""
    f32 = np.float32
    spec = Rotary(dim=np.int64(64), base=f32(500000), factor=f32(8), original=np.int32(8192), low=f32(1), high=f32(4),
                  magnitude=f32(1.25))
    plain = Rotary(dim=64, base=500000.0, factor=8.0, original=8192, low=1.0, high=4.0, magnitude=1.25)
    assert spec == plain and spec.turns == plain.turns and all(type(f) is float for f in spec.angles)
    assert Rotary(dim=64, base=f32(10000), factor=f32(4)).turns == Rotary(dim=64, factor=4.0).turns
    ops = _ops(**{**ROTARY, "k": (3, 64)})
    ops.rotary("q", positions="at", out="q1", rotary=spec, k="k", k_out="k1")
    (one,) = compile_program(ops)
    ops = _ops(**{**ROTARY, "k": (3, 64)})
    ops.rotary("q", positions="at", out="q1", rotary=plain, k="k", k_out="k1")
    (two,) = compile_program(ops)
    assert one.kernel.source == two.kernel.source


@pytest.mark.parametrize("name", ["base", "factor", "low", "high", "magnitude"])
@pytest.mark.parametrize("value", ["1", None, 1j, 10**400, [2.0]])
def test_rotations_by_what_is_no_number(name, value):
    with pytest.raises(ValueError, match=f"rotary: {name} must be"):
        Rotary(dim=64, original=4096, **{name: value})


def _more(i: int, **call) -> dict:
    """The i-th step on the same table."""
    before = "table" if i == 2 else f"out{i - 1}"
    return {**PAGE_CALL, "pages": before, "lengths": "ends" if i == 2 else f"ends{i - 1}",
            **{n: f"{n}{i}" for n in ("out", "slots", "positions", "ends", "used")}, **call}


def test_steps_of_a_table_take_other_pages():
    """A program that makes room in a table again goes on in ``free`` where it was; another
    list begins at its first, and so does another table."""
    ops = _ops(**PAGES, others=((9,), "int32"), pages2=((4, 6), "int32"), gone=((1,), "int32"))
    ops.page_tables(**PAGE_CALL)
    ops.page_tables(**_more(2))
    ops.page_tables(**_more(3, free="others"))
    ops.page_tables(**_more(4))
    ops.page_tables(**_more(5, taken="gone"))
    ops.page_tables(**{**_more(6), "pages": "pages2"})
    assert [o.taken and o.taken.name for o in ops.build()] == [None, "used", None, "used2", "gone", None]


def test_oracle_of_steps_of_a_table():
    ops = _ops(pages=((2, 4), "int32"), free=((5,), "int32"), lengths=((2,), "int32"), counts=((2,), "int32"))
    for name, v in (("pages", np.full((2, 4), -1)), ("free", [9, 8, 6, 5, 4]), ("lengths", [0, 0]), ("counts", [3, 2])):
        ops.from_numpy(np.array(v, np.int32), name)
    ops.page_tables(**{**PAGE_CALL, "page_size": 2, "tokens": 5})
    ops.page_tables(**_more(2, page_size=2, tokens=5))
    ref = evaluate(ops)
    np.testing.assert_array_equal(ref["table"], [[9, 8, -1, -1], [6, -1, -1, -1]])
    np.testing.assert_array_equal(ref["out2"], [[9, 8, 5, -1], [6, 4, -1, -1]])
    np.testing.assert_array_equal(ref["slots2"], [17, 10, 11, 8, 9])
    assert ref["used"] == [3] and ref["used2"] == [5]


@pytest.mark.parametrize("inputs, call, match", [
    (dict(gone=((2,), "int32")), {}, "taken must have shape"),
    (dict(gone=(1,)), {}, "taken must be int32"),
    (dict(gone=((1, 1), "int32")), {}, "taken must be 1D"),
    ({}, dict(taken="nothing"), "is not declared"),
])
def test_page_tables_refusals_of_taken(inputs, call, match):
    ops = _ops(**{**PAGES, "gone": ((1,), "int32"), **inputs})
    with pytest.raises(ValueError, match=match):
        ops.page_tables(**{**PAGE_CALL, "taken": "gone", **call})
    assert not ops.build() and "table" not in ops.tensors


def test_page_tables_of_taken_compile():
    ops = _ops(**PAGES, gone=((1,), "int32"))
    ops.page_tables(**PAGE_CALL, taken="gone")
    ops.page_tables(**_more(2))
    _compile(ops)
    kinds = [v.ops[0].out.name for v in fuse(ops.build())]
    assert kinds == ["table", "out2"]
