"""Serving strategies: one kernel per op, a call of a device function of
``csrc/mt_serving.h`` specialised for the op's sizes and strides.

Bindings are the op's tensors in the order of the device function's
parameters.  The rows (or tokens) of norms, cache ops and products are a runtime
dim: a 4-bit product takes at most as many in a launch as it was cut for (the
sets of rows are compiled in).  Attention has none: it is compiled for its number
of sequences and the width of its table.  How a kernel splits its work is chosen
here, by sizes and types alone.
"""

from __future__ import annotations

from metellus_amd.compute.fragments import CodegenContext, serving_header
from metellus_amd.compute.serving import ServingFragment
from metellus_amd.orchestrator.assembly.decision import DecisionView
from metellus_amd.orchestrator.ir import Tensor
from metellus_amd.orchestrator.kernel_group import FusionStrategy, KernelGroup
from metellus_amd.orchestrator.serving import (
    CacheReadOp,
    CacheWriteOp,
    DequantizeOp,
    Int4MatmulOp,
    KVCache,
    PagedAttentionOp,
    RmsNormOp,
)
from metellus_amd.runtime.program import Kernel

SERVING = frozenset(
    {
        FusionStrategy.RMS_NORM,
        FusionStrategy.DEQUANTIZE,
        FusionStrategy.INT4_MATMUL,
        FusionStrategy.CACHE_WRITE,
        FusionStrategy.CACHE_READ,
        FusionStrategy.PAGED_ATTENTION,
    }
)

_KIND = {"float32": 0, "int8": 1, "float8_e4m3": 2}
_CTYPE = {"float32": "float", "int32": "int", "int8": "signed char", "uint8": "unsigned char"}
WS_HEAD_BYTES = 4096  # the workspace's flag words


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


class _Signature:
    """Kernel parameters in order; a parameter is named by its role, since two may
    be bound to the same buffer."""

    def __init__(self) -> None:
        self.buffers: list[str] = []
        self.bindings: list[str] = []

    def add(self, role: str, t: Tensor | None, *, out: bool = False) -> str:
        """The argument for ``t`` (``nullptr`` for a tensor that is not there)."""
        if t is None:
            return "nullptr"
        self.buffers.append(f"{'' if out else 'const '}{_CTYPE[t.stored]}* __restrict__ p_{role}")
        self.bindings.append(t.buffer_key)
        return f"p_{role}"


def _group(decision: DecisionView, sig: _Signature, fragment: ServingFragment, function_name: str, dims: dict[str, int],
           grid: tuple[int, int, int], lanes: int, **context) -> KernelGroup:
    ctx = CodegenContext(
        function_name=function_name,
        buffers=tuple(sig.buffers),
        dims=tuple(dims),
        tg_x=lanes,
        tg_y=1,
        helpers=(serving_header(),),
        **context,
    )
    return KernelGroup(
        kernel=Kernel(fragments=(fragment,), ctx=ctx),
        bindings=tuple(sig.bindings),
        dims=tuple(dims.values()),
        grid=grid,
        threads=(lanes, 1, 1),
        ops=decision.ops,
        strategy=decision.strategy,
    )


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------

NORM_KEEP = 8  # float4s a lane keeps of a row at most; longer rows are read again for each pass


def norm_lanes(cols: int) -> int:
    """Lanes that share a row: a wave, 256 or 1024 lanes where they keep it in registers
    (777 rows of 5003: 256 lanes 7.3 us, 1024 9.3; one row of 4096 is the same with any)."""
    return 64 if cols <= 1024 else 256 if cols <= 1024 * NORM_KEEP else 1024


def _assemble_norm(decision: DecisionView, op: RmsNormOp, function_name: str | None) -> KernelGroup:
    rows, cols = op.x.shape
    T = norm_lanes(cols)
    per = _ceil(cols, 4 * T)
    eight = op.scales is not None
    res = op.residual
    sig = _Signature()
    args = (
        sig.add("x", op.x),
        sig.add("residual", res),
        sig.add("weight", op.weight),
        repr(float(op.eps)),
        sig.add("sum", op.sum_out, out=True),
        "nullptr" if eight else sig.add("y", op.y, out=True),
        sig.add("y", op.y, out=True) if eight else "nullptr",
        sig.add("scales", op.scales, out=True),
        "M",
        "(double*)mt_lds" if T > 64 else "nullptr",
    )
    frag = ServingFragment(
        "mt_rms_norm",
        (cols, T, per if per <= NORM_KEEP else 0, op.x.row_stride, op.x.col_stride,
         res.row_stride if res else 0, res.col_stride if res else 0, res is not None, op.sum_out is not None,
         op.weight is not None, eight),
        args,
        lds_bytes=8 * T // 64 if T > 64 else 0,
        name="rms_norm",
    )
    grid = (_ceil(rows, 4) if T == 64 else rows, 1, 1)
    return _group(decision, sig, frag, function_name or f"rms_norm_{op.y.name}", {"M": rows}, grid, max(T, 256))


def _assemble_dequantize(decision: DecisionView, op: DequantizeOp, function_name: str | None) -> KernelGroup:
    rows, cols = op.x.shape
    sig = _Signature()
    args = (sig.add("x", op.x), sig.add("scales", op.scales), sig.add("y", op.y, out=True), f"(size_t)M * {cols}u")
    frag = ServingFragment("mt_dequantize", (cols,), args, name="dequantize")
    grid = (_ceil(rows * cols, 16 * 256), 1, 1)
    return _group(decision, sig, frag, function_name or f"dequantize_{op.y.name}", {"M": rows}, grid, 256)


# ---------------------------------------------------------------------------
# cache
# ---------------------------------------------------------------------------


def _cache_template(spec: KVCache) -> tuple[int, ...]:
    return (_KIND[spec.dtype], spec.kv_heads, spec.page_size, spec.dim)


def cache_write_tokens(tokens: int, kv_heads: int) -> int:
    """Tokens of a workgroup: its 16 row slots full, and up to 16 while more than
    1024 workgroups remain, for each of them looks through the slots behind its own."""
    few = max(1, 8 // kv_heads)
    return max(few, min(16, tokens // 1024))


def _assemble_cache_write(decision: DecisionView, op: CacheWriteOp, function_name: str | None) -> KernelGroup:
    spec, tokens = op.spec, op.k.shape[0]
    tb = cache_write_tokens(tokens, spec.kv_heads)
    sig = _Signature()
    args = (sig.add("k", op.k), sig.add("v", op.v), sig.add("slots", op.slots),
            sig.add("cache", op.cache, out=True), "M", "(unsigned*)mt_lds")
    frag = ServingFragment(
        "mt_cache_write",
        (*_cache_template(spec), spec.pages, tb, op.k.row_stride, op.k.col_stride, op.v.row_stride, op.v.col_stride),
        args,
        lds_bytes=16,
        name="cache_write",
    )
    return _group(decision, sig, frag, function_name or f"cache_write_{op.written.name}", {"M": tokens},
                  (_ceil(tokens, tb), 1, 1), 256)


def _assemble_cache_read(decision: DecisionView, op: CacheReadOp, function_name: str | None) -> KernelGroup:
    spec, rows = op.spec, op.slots.shape[0]
    sig = _Signature()
    args = (sig.add("cache", op.cache), sig.add("slots", op.slots), sig.add("k", op.k, out=True),
            sig.add("v", op.v, out=True), "M")
    frag = ServingFragment("mt_cache_read", (*_cache_template(spec), spec.pages), args, name="cache_read")
    grid = (_ceil(rows * 2 * spec.kv_heads, 64), 1, 1)
    return _group(decision, sig, frag, function_name or f"cache_read_{op.k.name}", {"M": rows}, grid, 256)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

ATTENTION_WAVES = 8
ATTENTION_WORKGROUPS = 256  # one to a compute unit; the device cuts the work into as many equal ranges


def attention_workgroups(pairs: int, capacity: int, step: int, batch: int, most: int = ATTENTION_WORKGROUPS) -> int:
    """Workgroups of a launch: one for each unit of ``step`` positions of a sequence
    (``pairs`` of them, times key heads) that there is room for, ``most`` at most, and a
    counter each in the workspace's head for all of a batch."""
    return max(1, min(most, pairs * _ceil(capacity, step), (WS_HEAD_BYTES // 4 - 1) // batch))


def _assemble_attention(decision: DecisionView, op: PagedAttentionOp, function_name: str | None, batch: int) -> KernelGroup:
    spec, rows = op.spec, op.q.shape[0]
    share = op.heads // spec.kv_heads  # query heads of a key head
    # At most 16 query heads at once, an MFMA's columns; 8 of long fp32 rows.  Eight waves to
    # a compute unit; four, with twice the registers each, for long rows.
    heavy = spec.dim > 128
    held = min(share, 8 if heavy and spec.dtype == "float32" else 16)
    parts = _ceil(share, held)
    pairs = rows * spec.kv_heads * parts
    waves, most = 4 if heavy else ATTENTION_WAVES, ATTENTION_WORKGROUPS
    if spec.dtype != "float32" and not heavy and op.capacity <= 512:
        # Short sequences in 8 bits: their ends are most of the time, and overlap where smaller
        # workgroups share a compute unit (8 key heads of 128 in int8, evenly ragged lengths, four
        # or two waves for eight: 1024 sequences of up to 256 keys 130, 110 and 175 us, 64 of 64
        # 9.1, 8.2 and 13; 256 of 512 55 and 62, 64 of 300 17.9 and 18.8; 64 of 1024 27 and 27;
        # fp32 no faster).
        waves, most = (2, 4 * ATTENTION_WORKGROUPS) if op.capacity <= 256 else (4, 2 * ATTENTION_WORKGROUPS)
    step = (16 if spec.dtype == "float32" else 32) * waves
    groups = attention_workgroups(pairs, op.capacity, step, batch, most)
    floats = _ceil(held * (spec.dim + 2), 4) * 4
    # q's operands in LDS: 16 bytes a lane for 16 dims of fp32, or for 32 (16) of three bf16 parts
    if spec.dtype == "float32":
        q_bytes = 1024 * (spec.dim // 16)
    else:
        q_bytes = 1024 * 3 * (spec.dim // (32 if spec.dim % 32 == 0 else 16))
    ws = WS_HEAD_BYTES + 4 * batch * groups * 2 * floats if groups > 1 else 0
    sig = _Signature()
    args = (sig.add("q", op.q), sig.add("cache", op.cache), sig.add("pages", op.pages), sig.add("lengths", op.lengths),
            sig.add("o", op.o, out=True), repr(float(op.scale)), "mt_ws" if ws else "nullptr", "mt_lds")
    frag = ServingFragment(
        "mt_paged_attention",
        (*_cache_template(spec), spec.pages, op.pages.shape[1], share, held, waves, groups, batch, rows,
         op.q.row_stride, op.q.col_stride),
        args,
        lds_bytes=2 * q_bytes + 4 * waves * floats + 16,
        name="paged_attention",
    )
    return _group(decision, sig, frag, function_name or f"paged_attention_{op.o.name}", {},
                  (groups, 1, 1), 64 * waves, workspace_bytes=ws, workspace_batched=True,
                  workspace_waits=False)


# ---------------------------------------------------------------------------
# 4-bit products
# ---------------------------------------------------------------------------


INT4_WORKGROUPS = 256  # one for each compute unit
INT4_LDS = 131072  # bytes of digits at a time, where the waves share them


def int4_shape(rows: int, k: int, n: int, group: int, eight: bool, zeros: bool) -> dict:
    """How a product is cut: ``shared`` (digits of x in LDS, waves on tiles of their
    own) or waves that split k; ``waves`` of a workgroup, ``tiles`` of 16 weight rows
    that a wave takes together, blocks of 128 k that it loads ``together``; ``each`` row
    of x in a set of MFMA rows, ``sets`` of them; ``phase``, blocks of k whose digits
    are in LDS at once.

    Figures below: us a pass over three input sets in turn, sizes as weight rows x columns
    (n x k), groups of 128 unless said."""
    held = min(rows, 16)
    sets = 1 if eight else _ceil(held, 4)
    each = 4 if eight or held > 2 else held
    # Enough weight rows for a tile to most waves of the GPU: the waves share x's digits
    # (4 rows, 131072 x 4096: 62, splitting k 109; 8 rows, 20480 x 4096 18 and 26; 16400 x
    # 4096, the next tile after four a workgroup, 18 and 24; one row, 24000 x 4096 13.5 and
    # 13.6).  Fewer rows: splitting k (8 rows, 16384 x 4096: 15, shared 18; 11008 x 4096 14, 17).
    shared = _ceil(n, 16) > 4 * INT4_WORKGROUPS if rows > 4 else _ceil(n, 16) >= 5 * INT4_WORKGROUPS
    blocks = _ceil(k, 128)
    made = 1 if eight else 4 // each  # blocks of x made into digits at once
    tiles, waves, together = 1, 8, 4
    if shared:
        # Sixteen waves to a making of digits, each making some, where they still leave a
        # workgroup to each compute unit (fp32, 131072 x 4096: 8 rows 80, eight waves 84; 16
        # rows 102 and 118; 4 rows 69 and 61; 8 rows, groups of 32 with zeros, 65536 x 2048: 43, 43).
        if sets > 1 and group > 32 and _ceil(n, 16) >= 16 * INT4_WORKGROUPS:
            waves, together = 16, 2
    else:
        # Two tiles a wave halve the work on x, once one is more than a workgroup to each
        # compute unit (4099 x 5024, groups of 32 with zeros: 5 rows 16, one tile 18; 16 rows 24
        # and 35; 8 bits, 16 rows, 8192 x 11008: 16 and 19; fp32, 4 rows 18, the one tile taken 20).
        # Sixteen waves where it is not (1 row, 4096 x 11008: 7.9, eight waves 8.9).
        many = _ceil(n, 16) > INT4_WORKGROUPS
        tiles = 2 if rows > 4 and many else 1
        # Four for fp32 where two are more than that and four are not (11008 x 8192: 8 rows 24,
        # two tiles 30; 16 rows 35 and 47, of groups of 64 39 and 52; in 8 bits 19, the two taken
        # 22), as long as a block's sums and scales stay few (of groups of 32 two, 61; four, a
        # block at once, 47).
        if tiles == 2 and 2 * INT4_WORKGROUPS < _ceil(n, 16) <= 4 * INT4_WORKGROUPS and not eight and sets * 128 // group < 16:
            tiles = 4
        waves = 16 if not many and sets <= 2 else 8
        if eight:  # (1 row, 11008 x 8192: groups of 128 one block 17.4, two 15.3; of 32, 20.9 and 24.3)
            together = 1 if group == 32 else 2
        elif rows <= 2:  # (2 rows, 11008 x 8192: two blocks 16.2, four 16.7)
            together = made
        else:
            # As many as leave the waves' shares even (5 rows, 4099 x 5024, 40 blocks: one 16,
            # two 18, four 29), and whose scales fit in registers.
            share = {u: _ceil(_ceil(blocks, u), waves) * u for u in (1, 2, 4)
                     if u == 1 or u * tiles * max(1, sets // 2) * (1 + zeros) <= group // 16}
            together = max(u for u in share if share[u] <= 1.1 * min(share.values()))
        waves = min(waves, _ceil(blocks, together))
    block = (512 * each + 16) * sets
    return {"shared": shared, "waves": waves, "tiles": tiles, "together": together, "each": each, "sets": sets,
            "phase": min(_ceil(blocks, 4) * 4, INT4_LDS // block // 4 * 4), "block": block}


def _assemble_int4(decision: DecisionView, op: Int4MatmulOp, function_name: str | None) -> KernelGroup:
    (rows, k), n = op.x.shape, op.weights.shape[0]
    eight = op.x_scales is not None
    shape = int4_shape(rows, k, n, op.group, eight, op.zeros is not None)
    waves, tiles, shared, sets = shape["waves"], shape["tiles"], shape["shared"], shape["sets"]
    sig = _Signature()
    args = (
        "nullptr" if eight else sig.add("x", op.x),
        sig.add("x", op.x) if eight else "nullptr",
        sig.add("x_scales", op.x_scales),
        sig.add("weights", op.weights),
        sig.add("scales", op.scales),
        sig.add("zeros", op.zeros),
        sig.add("y", op.y, out=True),
        "M",
        "mt_lds",
    )
    if shared:
        lds = shape["phase"] * shape["block"]
    else:
        lds = max(0 if eight else 2048 * sets * waves, waves * tiles * 256 * (4 if eight else sets))
    frag = ServingFragment(
        "mt_matmul_int4",
        (eight, shared, shape["phase"], shape["each"], sets, k, n, op.group, op.zeros is not None, tiles, shape["together"],
         waves, op.x.row_stride, op.x.col_stride),
        args,
        lds_bytes=lds,
        name="int4_matmul",
    )
    groups = _ceil(n, 16 * tiles)
    if shared:
        groups = min(_ceil(groups, waves), INT4_WORKGROUPS)
    return _group(decision, sig, frag, function_name or f"int4_matmul_{op.y.name}", {"M": rows}, (groups, _ceil(rows, 16), 1),
                  64 * waves)


_ASSEMBLE = {
    RmsNormOp: _assemble_norm,
    DequantizeOp: _assemble_dequantize,
    CacheWriteOp: _assemble_cache_write,
    CacheReadOp: _assemble_cache_read,
    Int4MatmulOp: _assemble_int4,
}


def assemble_serving(decision: DecisionView, function_name: str | None, *, batch: int = 1) -> KernelGroup:
    op = decision.serving_op
    if isinstance(op, PagedAttentionOp):
        return _assemble_attention(decision, op, function_name, batch)
    return _ASSEMBLE[type(op)](decision, op, function_name)
