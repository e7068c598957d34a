"""The serving ops without a GPU: what the builder and the scheduler accept and
refuse, the order of a cache's readers and writers, the cache's packing on the
host against the oracle's, and that every kernel variant compiles for gfx950."""

from __future__ import annotations

import numpy as np
import pytest

from metellus_amd.api import compile_program
from metellus_amd.compute.fragments import CodegenEngine
from metellus_amd.orchestrator import KVCache, Operations
from metellus_amd.orchestrator.assembly.serving import (
    attention_workgroups,
    cache_write_tokens,
    int4_shape,
    norm_lanes,
)
from metellus_amd.orchestrator.fusion import fuse
from metellus_amd.orchestrator.scheduler import schedule
from metellus_amd.runtime import hip_backend
from metellus_amd.runtime.program import Dispatch, Download, Free
from oracle import serving_eval

CACHE = dict(pages=6, page_size=4, kv_heads=2, dim=16)


def _ops(**inputs) -> Operations:
    """Inputs by name: a shape, or (shape, dtype)."""
    ops = Operations()
    for name, what in inputs.items():
        if isinstance(what[0], tuple):
            ops.input(name, what[0], dtype=what[1])
        else:
            ops.input(name, what)
    return ops


def _cache_ops(dtype: str = "float32") -> Operations:
    ops = _ops(k=(3, 32), v=(3, 32), slots=((3,), "int32"), q=(2, 64), pages=((2, 3), "int32"), lengths=((2,), "int32"))
    ops.kv_cache("cache", dtype=dtype, **CACHE)
    return ops


# -- refusals -------------------------------------------------------------------


def test_inputs_of_other_types():
    ops = _ops(i=((3,), "int32"), b=((2, 4), "uint8"))
    assert ops.tensors["i"].nbytes == 12 and ops.tensors["b"].nbytes == 8
    ops.from_numpy(np.zeros(3, np.int32), "i")
    with pytest.raises(ValueError, match="dtype must be int32; got float32"):
        ops.from_numpy(np.zeros(3, np.float32), "i")
    with pytest.raises(ValueError, match="dtype must be one of"):
        ops.input("h", (2, 2), dtype="float16")
    with pytest.raises(ValueError, match="already declared as int32"):
        ops.input("i", (3,), dtype="float32")


@pytest.mark.parametrize("call", [
    lambda ops: ops.matmul(a="b", b="x", out="o"),
    lambda ops: ops.elementwise("add", out="o", operands=("b", 1.0)),
    lambda ops: ops.elementwise("add", out="o", operands=("x", "b")),
    lambda ops: ops.reduction("sum", out="o", x="b"),
])
def test_primitive_ops_take_fp32_only(call):
    ops = _ops(x=(4, 4), b=((4, 4), "int8"))
    with pytest.raises(ValueError, match="takes fp32 tensors"):
        call(ops)
    ops.transpose("b", out="bt")
    with pytest.raises(ValueError, match="takes fp32 tensors"):
        ops.reshape("bt", (16,), out="o")
    assert not ops.build()


@pytest.mark.parametrize("kwargs, message", [
    (dict(weight="w3"), "weight must have shape"),
    (dict(weight="wi"), "weight must be float32"),
    (dict(residual="r3"), "residual must have shape"),
    (dict(sum_out="h"), "needs a residual"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(x="wi"), "must be 2D"),
    (dict(x="xi"), "must be float32"),
    (dict(residual="r", sum_out="y"), "output names must differ"),
    (dict(out="x"), "already defined"),
    (dict(weight="w2"), "must be dense"),
])
def test_rms_norm_refuses(kwargs, message):
    ops = _ops(x=(4, 8), r=(4, 8), r3=(4, 4), w3=(4,), wi=((8,), "int32"), xi=((4, 8), "int32"))
    ops.input("w2", (8,), row_stride=2, col_stride=0)
    with pytest.raises(ValueError, match=message):
        ops.rms_norm(**{"x": "x", "out": "y", **kwargs})
    assert not ops.build() and "y" not in ops.tensors


@pytest.mark.parametrize("kwargs, message", [
    (dict(weights="w2"), "hold 128 columns; x has 64"),
    (dict(scales="s3"), "groups dividing 64"),
    (dict(scales="s16"), "groups of"),
    (dict(scales="sn"), "scales must have shape"),
    (dict(zeros="s1"), "zeros must have shape"),
    (dict(x="x8"), "must be float32"),
    (dict(x_scales="xs"), "must be int8"),
    (dict(x="x8", x_scales="s2"), "x_scales must have shape"),
    (dict(weights="x"), "must be uint8"),
    (dict(weights="wt"), "must be dense"),
    (dict(x="x8t", x_scales="xs"), "must be dense"),
    (dict(weights="cache"), "is a kv cache"),
    (dict(weights="none"), "is not declared"),
])
def test_matmul_int4_refuses(kwargs, message):
    ops = _ops(x=(3, 64), x8=((3, 64), "int8"), w=((5, 32), "uint8"), w2=((5, 64), "uint8"), s2=(5, 2), s1=(5, 1), s3=(5, 3),
               s16=(5, 4), sn=(4, 2), xs=(3,), w_=((32, 5), "uint8"), x8_=((64, 3), "int8"))
    ops.transpose("w_", out="wt")
    ops.transpose("x8_", out="x8t")
    ops.kv_cache("cache", **CACHE)
    with pytest.raises(ValueError, match=message):
        ops.matmul_int4(**{"x": "x", "weights": "w", "scales": "s2", "out": "y", **kwargs})
    assert not ops.build()


def test_dequantize_refuses():
    ops = _ops(x=(3, 8), q=((3, 8), "int8"), s=(3,), s2=(4,), q_=((8, 3), "int8"))
    ops.transpose("q_", out="qt")
    for kwargs, message in ((dict(x="x"), "must be int8"), (dict(scales="s2"), "shape"), (dict(x="qt"), "must be dense")):
        with pytest.raises(ValueError, match=message):
            ops.dequantize(**{"x": "q", "scales": "s", "out": "y", **kwargs})


@pytest.mark.parametrize("change, message", [
    (dict(pages=0), "pages must be a positive int"),
    (dict(page_size=True), "page_size must be a positive int"),
    (dict(kv_heads=1.5), "kv_heads must be a positive int"),
    (dict(dim=24), "multiple of 16"),
    (dict(dim=272), "multiple of 16 up to 256"),
    (dict(dtype="float16"), "dtype must be one of"),
    (dict(page_size=2**27), "too large"),
    (dict(pages=2**31), "page numbers are int32"),
])
def test_kv_cache_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        Operations().kv_cache("c", **{**CACHE, **change})


def test_kv_cache_is_only_for_its_ops():
    ops = _cache_ops()
    for call in (lambda: ops.reshape("cache", (4, 8), out="o"), lambda: ops.transpose("cache", out="o")):
        with pytest.raises(ValueError, match="is a kv cache"):
            call()
    with pytest.raises(ValueError, match="is not a kv cache"):
        ops.cache_read("q", slots="slots", k_out="a", v_out="b")
    with pytest.raises(ValueError, match="already declared"):
        ops.kv_cache("cache", **{**CACHE, "dim": 32})
    with pytest.raises(ValueError, match="already declared"):
        ops.kv_cache("q", **CACHE)
    assert ops.kv_cache("cache", **CACHE) == KVCache(**CACHE)


def test_cache_ops_refuse():
    ops = _cache_ops()
    ops.input("f", (3,))
    ops.input("k4", (4, 32))
    with pytest.raises(ValueError, match="slots must be int32"):
        ops.cache_write("cache", k="k", v="v", slots="f", out="o")
    with pytest.raises(ValueError, match="v must have shape"):
        ops.cache_write("cache", k="k", v="k4", slots="slots", out="o")
    with pytest.raises(ValueError, match="k must have shape"):
        ops.cache_write("cache", k="q", v="v", slots="slots", out="o")
    with pytest.raises(ValueError, match="slots must be int32"):
        ops.cache_read("cache", slots="f", k_out="a", v_out="b")
    with pytest.raises(ValueError, match="slots must be 1D"):
        ops.cache_read("cache", slots="pages", k_out="a", v_out="b")
    with pytest.raises(ValueError, match="output names must differ"):
        ops.cache_read("cache", slots="slots", k_out="a", v_out="a")
    assert not ops.build()


@pytest.mark.parametrize("change, message", [
    (dict(heads=3), "do not divide over 2"),
    (dict(heads=0), "positive int"),
    (dict(heads=8), r"q must have shape \(2, 128\)"),
    (dict(pages="slots"), "pages must have shape"),
    (dict(pages="pf"), "pages must be int32"),
    (dict(lengths="slots"), "lengths must have shape"),
    (dict(scale=float("inf")), "scale must be finite"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(scale=-3e38), "within 2e38"),
    (dict(pages="pt"), "must be dense"),
    (dict(cache="q"), "is not a kv cache"),
])
def test_paged_attention_refuses(change, message):
    ops = _cache_ops()
    ops.input("pf", (2, 3))
    ops.input("p_", (3, 2), dtype="int32")
    ops.transpose("p_", out="pt")
    with pytest.raises(ValueError, match=message):
        ops.paged_attention(**{"q": "q", "cache": "cache", "pages": "pages", "lengths": "lengths", "out": "o", "heads": 4, **change})
    assert not ops.build()


# -- a cache's states -----------------------------------------------------------


def test_a_written_cache_is_read_by_its_new_name():
    ops = _cache_ops()
    t = ops.cache_write("cache", k="k", v="v", slots="slots", out="c1")
    assert t.buffer_key == "cache" and t.dtype == "uint8"
    for call in (
        lambda: ops.cache_read("cache", slots="slots", k_out="a", v_out="b"),
        lambda: ops.cache_write("cache", k="k", v="v", slots="slots", out="c2"),
        lambda: ops.paged_attention("q", cache="cache", pages="pages", lengths="lengths", heads=4, out="o"),
    ):
        with pytest.raises(ValueError, match="its buffer now holds 'c1'"):
            call()
    with pytest.raises(ValueError, match="view"):
        ops.from_numpy(np.zeros(t.shape, np.uint8), "c1")


def test_a_write_comes_after_the_readers_of_the_older_state():
    """A reader delayed by the values it waits for (its query comes out of a fused
    chain that ends late) still precedes the write."""
    ops = _cache_ops()
    ops.input("other", (2, 64))
    ops.paged_attention("q", cache="cache", pages="pages", lengths="lengths", heads=4, out="before")
    ops.cache_read("cache", slots="slots", k_out="ka", v_out="va")
    ops.cache_write("cache", k="k", v="v", slots="slots", out="c1")
    ops.paged_attention("q", cache="c1", pages="pages", lengths="lengths", heads=4, out="after")
    ops.cache_write("c1", k="v", v="k", slots="slots", out="c2")
    order = [v.ops[0].out.name for v in fuse(ops.build())]
    assert order.index("before") < order.index("c1") < order.index("after") < order.index("c2")
    assert order.index("ka") < order.index("c1")
    write = next(op for op in ops.build() if op.out.name == "c1")
    assert {"before", "ka"} <= {t.name for t in write.inputs}


def test_only_the_last_state_is_downloaded():
    ops = _cache_ops()
    rng = np.random.default_rng(0)
    for name in ("k", "v"):
        ops.from_numpy(rng.standard_normal((3, 32)).astype(np.float32), name)
    ops.from_numpy(np.arange(3, dtype=np.int32), "slots")
    ops.from_numpy(KVCache(**CACHE).empty(), "cache")
    ops.cache_write("cache", k="k", v="v", slots="slots", out="c1")
    ops.cache_write("c1", k="v", v="k", slots="slots", out="c2")
    steps = schedule(ops, compile_program(ops)).fragments
    assert [(s.name, s.into, s.dtype) for s in steps if isinstance(s, Download)] == [("cache", "c2", np.uint8)]
    assert {s.name for s in steps if isinstance(s, Free)} == {"cache", "k", "v", "slots"}
    with pytest.raises(ValueError, match="a later write overwrites"):
        schedule(ops, compile_program(ops), outputs=["c1"])


def test_an_op_on_a_view_comes_after_its_owner_and_keeps_it():
    """The view's owner is written although another op could have swallowed it."""
    ops = _ops(a=(4, 8), b=(8, 16), w=(8,))
    ops.matmul(a="a", b="b", out="c")
    ops.reshape("c", (8, 8), out="cv")
    ops.elementwise("exp", out="e", operands=("c",))
    ops.rms_norm("cv", weight="w", out="y")
    groups = compile_program(ops)
    assert any("c" in g.outputs for g in groups)
    order = [out for g in groups for out in g.outputs]
    assert order.index("c") < order.index("y")


def test_outputs_of_an_op_all_get_buffers():
    ops = _ops(x=(4, 8), r=(4, 8))
    ops.from_numpy(np.ones((4, 8), np.float32), "x")
    ops.from_numpy(np.ones((4, 8), np.float32), "r")
    ops.rms_norm("x", residual="r", sum_out="h", out="y", scales="s")
    ops.elementwise("exp", out="e", operands=("h",))
    (norm, chain) = compile_program(ops)
    assert set(norm.outputs) == {"y", "s", "h"} and chain.bindings == ("h", "e")
    steps = schedule(ops, (norm, chain)).fragments
    got = {s.into: (s.shape, s.dtype) for s in steps if isinstance(s, Download)}
    assert got == {"y": ((4, 8), np.int8), "s": ((4,), np.float32), "h": ((4, 8), np.float32), "e": ((4, 8), np.float32)}
    assert sum(isinstance(s, Dispatch) for s in steps) == 2


# -- packing --------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["float32", "int8", "float8_e4m3"])
@pytest.mark.parametrize("page_size, kv_heads, dim", [(4, 2, 16), (1, 3, 48), (5, 1, 128)])
def test_packing_matches_the_oracle(dtype, page_size, kv_heads, dim):
    spec = KVCache(pages=3, page_size=page_size, kv_heads=kv_heads, dim=dim, dtype=dtype)
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, spec.slots, kv_heads, dim)).astype(np.float32)
    k[0, 0] = 0
    v[-1, -1, 3] = np.inf
    k[-1, 0, :] = -np.arange(dim)  # ties
    data = spec.pack(k, v)
    assert data.shape == spec.shape and spec.page_bytes % 16 == 0
    gk, gv = spec.unpack(data)
    for slot in range(spec.slots):
        want = serving_eval.slot_rows(spec, data, slot).astype(np.float32)
        np.testing.assert_array_equal(gk[slot], want[0])
        np.testing.assert_array_equal(gv[slot], want[1])
        for got, src in ((gk[slot], k[slot]), (gv[slot], v[slot])):
            for h in range(kv_heads):
                if dtype == "float32":
                    np.testing.assert_array_equal(got[h], src[h])
                    continue
                raw, scale = serving_eval.quantize(src[h], dtype)
                held = raw.view(np.int8).astype(np.float32) if dtype == "int8" else serving_eval.E4M3[raw].astype(np.float32)
                np.testing.assert_array_equal(got[h], held * scale)


def test_e4m3_rounding_is_to_the_nearest():
    """Every value and every midpoint of e4m3, and its neighbours in float64."""
    table = serving_eval.E4M3[:127]
    mid = (table[:-1] + table[1:]) / 2
    v = np.concatenate([table, mid, np.nextafter(mid, 0), np.nextafter(mid, 1e9)])
    got = serving_eval.E4M3[serving_eval.nearest_e4m3(v)]
    assert np.all(np.abs(got - v) <= np.abs(table[None] - v[:, None]).min(axis=1))
    at = serving_eval.nearest_e4m3(mid)
    assert np.all(at % 2 == 0)


# -- kernels --------------------------------------------------------------------


@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 4096), (777, 5003), (4096, 64), (3, 40001)])
@pytest.mark.parametrize("eight", [False, True])
def test_norm_kernels_compile(rows, cols, eight):
    ops = _ops(x=(rows, cols), r=(cols, rows), w=(cols,))
    ops.transpose("r", out="rt")
    ops.rms_norm("x", weight="w", residual="rt", sum_out="h", out="y", scales="s" if eight else None)
    if eight:
        ops.dequantize("y", scales="s", out="z")
    for g in compile_program(ops):
        assert hip_backend.compile_only(g.kernel.source) > 0


@pytest.mark.parametrize("dtype", ["float32", "int8", "float8_e4m3"])
@pytest.mark.parametrize("heads, kv_heads, dim, page_size, width", [
    (4, 4, 128, 16, 128), (40, 2, 96, 20, 4), (6, 2, 16, 1, 7), (8, 1, 256, 64, 2048), (3, 3, 80, 48, 3),
])
def test_cache_kernels_compile(dtype, heads, kv_heads, dim, page_size, width):
    ops = _ops(q=(2, heads * dim), k=(3, kv_heads * dim), v=(3, kv_heads * dim), slots=((3,), "int32"),
               pages=((2, width), "int32"), lengths=((2,), "int32"))
    ops.kv_cache("c", pages=9, page_size=page_size, kv_heads=kv_heads, dim=dim, dtype=dtype)
    ops.cache_write("c", k="k", v="v", slots="slots", out="c1")
    ops.cache_read("c1", slots="slots", k_out="kb", v_out="vb")
    ops.paged_attention("q", cache="c1", pages="pages", lengths="lengths", heads=heads, out="o")
    for g in compile_program(ops):
        assert hip_backend.compile_only(g.kernel.source) > 0
        batched = g.kernel.batched()
        assert hip_backend.compile_only(CodegenEngine().render(list(batched.fragments), batched.ctx)) > 0


@pytest.mark.parametrize("rows, k, n", [(1, 32, 1), (5, 5024, 99), (16, 1024, 40000), (33, 256, 64)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("eight", [False, True])
def test_int4_kernels_compile(rows, k, n, group, eight):
    group = group if k % group == 0 else 32
    ops = _ops(x=((rows, k), "int8" if eight else "float32"), w=((n, k // 2), "uint8"), s=(n, k // group), z=(n, k // group),
               xs=(rows,))
    ops.matmul_int4("x", weights="w", scales="s", zeros="z", x_scales="xs" if eight else None, out="y")
    (g,) = compile_program(ops)
    assert hip_backend.compile_only(g.kernel.source) > 0


def test_launch_rules_stay_within_what_the_kernels_take():
    for cols in (1, 63, 64, 255, 1024, 4096, 16384, 100000):
        assert norm_lanes(cols) in (64, 256, 1024)
    for pairs in (1, 8, 256, 1022, 1023, 5000):
        for capacity in (1, 16, 100, 2048, 131072, 2**31 - 2048):
            for batch in (1, 3, 32, 1023, 5000):
                groups = attention_workgroups(pairs, capacity, 128, batch)
                assert 1 <= groups <= pairs * -(-capacity // 128) and (groups == 1 or groups * batch <= 1023)
    for tokens in (1, 5, 1024, 100000):
        for heads in (1, 8, 64):
            assert 1 <= cache_write_tokens(tokens, heads) <= 32
    for rows in (1, 4, 16, 100):
        for k in (32, 128, 4096, 16384):
            for n in (1, 100, 4096, 131072):
                for eight in (False, True):
                    shape = int4_shape(rows, k, n, 32, eight, True)
                    assert 1 <= shape["waves"] <= 16 and shape["tiles"] in (1, 2, 4) and shape["together"] in (1, 2, 4)


@pytest.mark.parametrize("view", ["transpose", "reshape"])
@pytest.mark.parametrize("first", ["norm", "matmul", "reduction"])
def test_a_chain_that_begins_before_a_view_of_another_kernels_output_runs_after_it(first, view):
    ops = _ops(x=(64, 64), w=(64, 64))
    ops.elementwise("exp", out="e", operands=("x",))
    if first == "norm":
        ops.rms_norm("x", out="h")
    elif first == "matmul":
        ops.matmul("x", "w", out="h")
    else:
        ops.reduction("max", out="h", x="x")
    if first == "reduction":
        ops.reshape("h", (64, 1), out="v")
    elif view == "transpose":
        ops.transpose("h", out="v")
    else:
        ops.reshape("h", (64, 64), out="v")
    ops.elementwise("add", out="z", operands=("e", "v"), **({"y_broadcast": "col"} if first == "reduction" else {}))
    groups = compile_program(ops)
    assert [g.bindings[1] if "e" in g.outputs or "z" in g.outputs else "h" for g in groups] == ["h", "z"]


@pytest.mark.parametrize("dtype", ["float32", "int8", "float8_e4m3"])
def test_attention_of_every_dim_fits_in_lds(dtype):
    for dim in range(16, 257, 16):
        for share in (1, 3, 8, 16, 17):
            for width in (1, 20, 1000):
                ops = _ops(q=(2, share * dim), pages=((2, width), "int32"), lengths=((2,), "int32"))
                ops.kv_cache("c", pages=9, page_size=16, kv_heads=1, dim=dim, dtype=dtype)
                ops.paged_attention("q", cache="c", pages="pages", lengths="lengths", heads=share, out="o")
                (g,) = compile_program(ops)
                assert sum(a.shape[0] * 4 for f in g.kernel.fragments for a in f.tgmem_accesses) <= 163840


@pytest.mark.parametrize("label", ["int8", "int32", "uint8", "float16", "anything"])
def test_a_programs_dtype_is_a_label(label):
    """Every op takes a program's tensors whatever its label says: they are fp32."""
    ops = Operations(dtype=label)
    for name in ("x", "y"):
        assert ops.from_numpy(np.ones((4, 4), np.float32), name).dtype == label
    ops.input("x", (4, 4), dtype="float32")
    with pytest.raises(ValueError, match="already declared as float32"):
        ops.input("x", (4, 4), dtype="int8" if label == "int8" else "int32")
    ops.transpose("y", out="yt")
    ops.matmul("x", "yt", out="m")
    ops.elementwise("add", out="e", operands=("m", "yt"))
    ops.reduction("sum", out="r", x="e")
    ops.reshape("yt", (16,), out="f")  # a copy
    ops.rms_norm("e", out="n")
    ops.rms_norm("n", out="n8", scales="s")
    ops.dequantize("n8", scales="s", out="d")
    ops.elementwise("add", out="z", operands=("d", "x"))
    assert all(t.dtype == label and t.nbytes == 4 * t.element_count for n, t in ops.tensors.items() if n != "n8")
    assert ops.tensors["n8"].nbytes == 16
    with pytest.raises(ValueError, match="x must be int8; got float32"):
        ops.dequantize("x", scales="s", out="q")
    with pytest.raises(ValueError, match="takes fp32 tensors"):
        ops.elementwise("exp", out="q", operands=("n8",))
    steps = schedule(ops, compile_program(ops)).fragments
    assert {s.into: s.dtype for s in steps if isinstance(s, Download) and s.into in ("r", "z", "n8")} == {
        "r": np.float32, "z": np.float32, "n8": np.int8}


def test_attention_has_no_runtime_rows():
    """Its number of sequences is compiled in: no dim could name another."""
    ops = _cache_ops()
    ops.paged_attention("q", cache="cache", pages="pages", lengths="lengths", heads=4, out="o")
    (g,) = compile_program(ops)
    assert g.dims == () and g.kernel.dim_names == ()
    assert hip_backend.compile_only(g.kernel.source) > 0


@pytest.mark.parametrize("dtype, peak", [("int8", 127.0), ("float8_e4m3", 448.0)])
def test_packing_by_the_definition(dtype, peak):
    """A scale is the largest over the peak but for two roundings (2^-24 of it each, and half of
    the smallest subnormal); a value is the nearest multiple: half a step of x / scale off."""
    spec = KVCache(pages=8, page_size=16, kv_heads=4, dim=32, dtype=dtype)
    kv = np.random.default_rng(3).standard_normal((2, spec.slots, 4, 32)).astype(np.float32)
    kv[0, :20] *= np.float32(1e-38)
    data = spec.pack(kv[0], kv[1])
    want = np.abs(kv).max(axis=-1).astype(np.float64) / peak
    for slot in range(spec.slots):
        values, scales = serving_eval._page_parts(spec, data, slot // 16)
        s = scales[:, :, slot % 16].astype(np.float64)
        assert np.all(np.abs(s - want[:, slot]) <= want[:, slot] * 2.01 * 2.0**-24 + 2.0**-150)
        raw = np.ascontiguousarray(values[:, :, slot % 16])
        held = raw.view(np.int8).astype(np.float64) if dtype == "int8" else serving_eval.E4M3[raw]
        v = np.clip(kv[:, slot].astype(np.float64) / s[..., None], -peak, peak)
        half = 0.5 if dtype == "int8" else np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(v), 2.0**-6))), -6) - 4)
        assert np.all(np.abs(held - v) <= half)
