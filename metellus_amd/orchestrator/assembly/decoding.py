"""Decoding strategies: one kernel per op, a call of a device function of
``csrc/mt_decoding.h`` specialised for the op's sizes and strides, as the serving
strategies are.  How a kernel splits its work is chosen here, by sizes and types
alone.
"""

from __future__ import annotations

from metellus_amd.compute.fragments import decoding_header
from metellus_amd.compute.serving import ServingFragment
from metellus_amd.orchestrator.assembly.decision import DecisionView
from metellus_amd.orchestrator.assembly.serving import _ceil, _group, _Signature
from metellus_amd.orchestrator.decoding import (
    ADAPTER_DOWN_WAVES,
    SAMPLE_LIST,
    AdapterDownOp,
    AdapterUpOp,
    PageTablesOp,
    Rotary,
    RotaryOp,
    SampleOp,
    SampleScanOp,
    sample_bins,
    sample_chunks,
)
from metellus_amd.orchestrator.ir import Tensor
from metellus_amd.orchestrator.kernel_group import FusionStrategy, KernelGroup

DECODING = frozenset(
    {
        FusionStrategy.PAGE_TABLES,
        FusionStrategy.ROTARY,
        FusionStrategy.ADAPTER_DOWN,
        FusionStrategy.ADAPTER_UP,
        FusionStrategy.SAMPLE_SCAN,
        FusionStrategy.SAMPLE,
    }
)


def _strides(t: Tensor | None) -> tuple[int, int]:
    return (t.row_stride, t.col_stride) if t is not None else (0, 0)


# ---------------------------------------------------------------------------
# block tables
# ---------------------------------------------------------------------------


def page_table_lanes(sequences: int) -> int:
    """Lanes that add up the sequences.  (us, 256, 512 and 1024: 32 sequences 5.4, 5.4, 5.9; 1021
    with 16384 tokens 6.2, 5.9, 6.8; 2048 6.7, 5.9, 6.0.)"""
    return 256 if sequences <= 256 else 512


def _assemble_page_tables(decision: DecisionView, op: PageTablesOp, function_name: str | None) -> KernelGroup:
    (sequences, width), tokens = op.pages.shape, op.slots.shape[0]
    lanes = page_table_lanes(sequences)
    sig = _Signature()
    args = (
        sig.add("pages", op.pages, out=True),
        sig.add("free", op.free),
        sig.add("taken", op.taken),
        sig.add("lengths", op.lengths),
        sig.add("counts", op.counts),
        sig.add("slots", op.slots, out=True),
        sig.add("positions", op.positions, out=True),
        sig.add("ends", op.ends, out=True),
        sig.add("used", op.used, out=True),
        "M", "S", "W", "F", "(unsigned*)mt_lds",
    )
    frag = ServingFragment(
        "mt_page_tables",
        (op.page_size, lanes),
        args,
        lds_bytes=4 * (2 * (lanes + 1) + 2 * (lanes // 64)),
        name="page_tables",
    )
    dims = {"M": tokens, "S": sequences, "W": width, "F": op.free.shape[0]}
    return _group(decision, sig, frag, function_name or f"page_tables_{op.written.name}", dims,
                  (min(256, _ceil(tokens, lanes)), 1, 1), lanes, headers=(decoding_header(),))


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------


def rotary_vector(spec: Rotary, *tensors: Tensor | None) -> int:
    """Elements that a lane takes at once: four where pairs and what is left of a head
    divide by it and elements are neighbours."""
    dense = all(t is None or t.col_stride == 1 for t in tensors)
    quads = spec.part % (8 if spec.layout == "half" else 4) == 0 and spec.dim % 4 == 0
    return 4 if dense and quads else 1


def rotary_rows(rows: int, elements: int) -> int:
    """Rows of a workgroup, by what a row has: as many as make 2048, up to 4.  (us, 1, 2 and 4 rows,
    16384 of 2 heads of 64 7.2, 5.7, 5.4; of 16 24.3, 21.0, 21.3; 8192 of 40 heads of 128 58, 61,
    64; 512 of them 5.8, 6.0, 6.5.)"""
    return max(1, min(4, 2048 // elements)) if rows >= 1024 else 1


def _turns(spec: Rotary) -> str:
    rows = ", ".join(f"{{{a.hex()}, {b.hex()}}}" for a, b in spec.turns)
    return f"static __device__ const double mt_turns[{spec.part // 2}][2] = {{{rows}}};"


def _assemble_rotary(decision: DecisionView, op: RotaryOp, function_name: str | None) -> KernelGroup:
    spec, rows = op.spec, op.x.shape[0]
    heads = op.x.shape[1] // spec.dim
    kv_heads = op.k.shape[1] // spec.dim if op.k is not None else 0
    together = rotary_rows(rows, (heads + kv_heads) * spec.dim)
    sig = _Signature()
    args = (
        sig.add("x", op.x),
        sig.add("k", op.k),
        sig.add("positions", op.positions),
        "mt_turns",
        repr(spec.magnitude),
        sig.add("y", op.y, out=True),
        sig.add("k_out", op.k_out, out=True),
        "M",
        "(mt_f32x2*)mt_lds",
    )
    frag = ServingFragment(
        "mt_rotary",
        (spec.dim, spec.part, spec.layout == "interleaved", rotary_vector(spec, op.x, op.k), heads, *_strides(op.x),
         kv_heads, *_strides(op.k), together),
        args,
        lds_bytes=together * spec.part // 2 * 8,
        name="rotary",
    )
    return _group(decision, sig, frag, function_name or f"rotary_{op.y.name}", {"M": rows}, (_ceil(rows, together), 1, 1), 256,
                  headers=(decoding_header(), _turns(spec)))


# ---------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------

ADAPTER_TURNS = 256, 2  # rows, from which on as many workgroups take a tile's groups in turn
ADAPTER_BLOCKS = 4  # of 16 ranks, that a wave multiplies x by at once


def adapter_tile(rank: int, many: bool) -> int:
    """Blocks of 16 rows in a tile: one where the rank leaves no registers for more."""
    return 4 if many and rank <= 64 else 1


def adapter_turns(rows: int, many: bool) -> int:
    """Workgroups that take a tile's groups in turn; 0: one for each row that may lead one, which
    has nothing to do where it does not.  (us, 0, 1, 2, 4 and 8, ids drawn from 64, rank 64 of
    4096 x 4096: 150 rows 48, 100, 68, 72, 69; 300 59, 72, 61, 62, 69; 600 74, 70, 63, 66, 71;
    1000 102, 78, 72, 75, 86; 8 prompts: 600 43, 38, 39, 40, 43; 2000 of 1024 x 1024 39, 39, 28,
    29, 34.)"""
    least, turns = ADAPTER_TURNS
    return 1 if many else turns if rows >= least else 0


def _adapter_grid(rows: int, tile: int, turns: int, shares: int) -> tuple[int, int, int]:
    tiles = _ceil(rows, 16 * tile)
    return (8 * _ceil(tiles, 8) * shares, turns, 1) if turns else (tiles * shares, 16 * tile, 1)


def _assemble_adapter_down(decision: DecisionView, op: AdapterDownOp, function_name: str | None) -> KernelGroup:
    rows, inner = op.x.shape
    blocks = min(ADAPTER_BLOCKS, _ceil(op.rank, 16))
    tile, turns = adapter_tile(op.rank, op.many), adapter_turns(rows, op.many)
    waves = ADAPTER_DOWN_WAVES
    order, lds_bytes = op.order is not None, waves * tile * blocks * 1024
    if order:  # sums, numbers of 256 bins a wave, a byte for each of 4096 rows; a tile's rows
        lds_bytes = 4 * 64 + max(lds_bytes, waves * (8 + 4 * 256) + 4096)
    sig = _Signature()
    args = (sig.add("x", op.x), sig.add("a", op.a), sig.add("ids", op.ids), sig.add("down", op.down, out=True),
            sig.add("order", op.order, out=True), "M", "(mt_f32x4*)mt_lds")
    frag = ServingFragment(
        "mt_adapter_down",
        (inner, op.rank, blocks, tile, turns, order, op.splits, op.held, waves, *_strides(op.x)),
        args,
        lds_bytes=lds_bytes,
        name="adapter_down",
    )
    grid = _adapter_grid(rows, tile, turns, op.splits * _ceil(op.rank, 16 * blocks))
    return _group(decision, sig, frag, function_name or f"adapter_down_{op.name}", {"M": rows}, grid, 64 * waves,
                  headers=(decoding_header(),))


def adapter_up_shape(rank: int, many: bool) -> tuple[int, int, int]:
    """Waves of a workgroup, how often each takes a set of columns, and the blocks of 16 in a
    set.  (us, 1, 2 and 4 blocks: 77 rows, rank 23, 12.8, 12.9, 14.3; 32 rows of 11008 12.6, 11.5,
    11.7; 600 of 4096, rank 64, 62, 61, 63; 4096 86, 73, 74, and 80 with 2 taken once; 16 rows, rank
    128, 16.9 and 17.6.)"""
    return 4, 2 if many else 1, 2 if rank <= 64 else 1


def _assemble_adapter_up(decision: DecisionView, op: AdapterUpOp, function_name: str | None) -> KernelGroup:
    rows, cols = op.base.shape
    tile, turns = adapter_tile(op.rank, op.many), adapter_turns(rows, op.many)
    waves, per, blocks = adapter_up_shape(op.rank, op.many)
    lds_bytes = 64 * (tile * (16 * _ceil(op.rank, 16) + 4) + waves * (16 * blocks + 4))
    order = op.order is not None
    lds_bytes += 4 * 64 if order else 0
    sig = _Signature()
    args = (sig.add("base", op.base), sig.add("down", op.down), sig.add("b", op.b), sig.add("ids", op.ids),
            sig.add("order", op.order), sig.add("scales", op.scales), sig.add("out", op.y, out=True), "M", "(float*)mt_lds")
    frag = ServingFragment(
        "mt_adapter_up",
        (cols, op.rank, tile, turns, order, op.splits, op.held, waves, per, blocks, *_strides(op.base)),
        args,
        lds_bytes=lds_bytes,
        name="adapter_up",
    )
    grid = _adapter_grid(rows, tile, turns, _ceil(cols, 16 * waves * per * blocks))
    return _group(decision, sig, frag, function_name or f"adapter_up_{op.y.name}", {"M": rows}, grid, 64 * waves,
                  headers=(decoding_header(),))


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------

SAMPLE_WAVES = 8
SAMPLE_CUT_WORDS = SAMPLE_WAVES + 8 + 1024 + 2 * 256  # of LDS, that finding a cut in a list takes


def _words(sig: _Signature, role: str, t: Tensor | None, *, out: bool = False) -> str:
    """A buffer of 64-bit words."""
    arg = sig.add(role, t, out=out)
    return arg if t is None else f"({'' if out else 'const '}mt_u64*){arg}"


def _assemble_sample_scan(decision: DecisionView, op: SampleScanOp, function_name: str | None) -> KernelGroup:
    rows, cols = op.logits.shape
    chunk, chunks = sample_chunks(rows, cols)
    cuts = op.bins is not None
    sig = _Signature()
    args = (
        sig.add("logits", op.logits),
        sig.add("temperatures", op.temperatures),
        sig.add("top_k", op.top_k),
        sig.add("top_p", op.top_p),
        _words(sig, "best", op.best, out=True),
        _words(sig, "bins", op.bins, out=True),
        f"(unsigned*){sig.add('counts', op.counts, out=True)}",
        "(mt_u64*)mt_lds",
    )
    frag = ServingFragment(
        "mt_sample_scan",
        (cols, chunk, chunks, sample_bins(cols), *_strides(op.logits), cuts),
        args,
        lds_bytes=8 * (SAMPLE_WAVES + (sample_bins(cols) if cuts else 0)),
        name="sample_scan",
    )
    return _group(decision, sig, frag, function_name or f"sample_scan_{op.name}", {}, (rows * chunks, 1, 1), 64 * SAMPLE_WAVES,
                  headers=(decoding_header(),))


def _assemble_sample(decision: DecisionView, op: SampleOp, function_name: str | None) -> KernelGroup:
    rows, cols = op.logits.shape
    chunk, chunks = sample_chunks(rows, cols)
    cuts = op.top_k is not None or op.top_p is not None
    sig = _Signature()
    args = (
        sig.add("logits", op.logits),
        sig.add("uniforms", op.uniforms),
        sig.add("temperatures", op.temperatures),
        sig.add("top_k", op.top_k),
        sig.add("top_p", op.top_p),
        sig.add("min_p", op.min_p),
        _words(sig, "best", op.best),
        _words(sig, "bins", op.bins),
        "nullptr" if op.counts is None else f"(unsigned*){sig.add('counts', op.counts, out=True)}",
        _words(sig, "sums", op.sums, out=True),
        _words(sig, "list", op.listed, out=True),
        sig.add("tokens", op.tokens, out=True),
        sig.add("logprobs", op.logprobs, out=True),
        "(mt_u64*)mt_lds",
    )
    # A row of ones adds up in 63 bits, and what lies below the bins weighs nothing.
    shift = min(44, 62 - (cols - 1).bit_length())
    frag = ServingFragment(
        "mt_sample_pick",
        (cols, chunk, chunks, sample_bins(cols), shift, *_strides(op.logits), cuts),
        args,
        # (64 powers; one workgroup for a whole row takes two words a wave and 256)
        lds_bytes=8 * (64 + max(SAMPLE_WAVES + 8 + chunk * chunks // 256 + (SAMPLE_CUT_WORDS + SAMPLE_LIST if cuts else 0), 2 * SAMPLE_WAVES + 256)),
        name="sample",
    )
    return _group(decision, sig, frag, function_name or f"sample_{op.tokens.name}", {}, (rows * chunks, 1, 1), 64 * SAMPLE_WAVES,
                  headers=(decoding_header(),))


_ASSEMBLE = {
    PageTablesOp: _assemble_page_tables,
    RotaryOp: _assemble_rotary,
    AdapterDownOp: _assemble_adapter_down,
    AdapterUpOp: _assemble_adapter_up,
    SampleScanOp: _assemble_sample_scan,
    SampleOp: _assemble_sample,
}


def assemble_decoding(decision: DecisionView, function_name: str | None) -> KernelGroup:
    op = decision.serving_op
    return _ASSEMBLE[type(op)](decision, op, function_name)
