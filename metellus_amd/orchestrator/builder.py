"""``Operations``: name-keyed builder for the primitive IR.

Same surface as the reference builder (reference:
src/orchestrator/builder.py:50-342): ``input``, ``from_numpy``, ``matmul``,
``elementwise``, ``transpose``, ``reshape``, ``reduction``, ``build``,
``tensors``, ``uploads``; beyond it the serving ops (``rms_norm``,
``dequantize``, ``matmul_int4``, ``kv_cache``, ``cache_write``, ``cache_read``,
``paged_attention``), the decoding ops (``page_tables``, ``rotary``, ``adapters``,
``sample``) and inputs of their types.  Validation is delegated to the op dataclasses;
the builder resolves names, keeps SSA freshness and records host payloads.

    ops = Operations()
    ops.from_numpy(a, "a"); ops.from_numpy(b, "b")
    ops.matmul(a="a", b="b", out="c")
    ops.elementwise("max", out="y", operands=("c", 0.0))   # relu
    program = ops.build()
"""

from __future__ import annotations

import numpy as np

from metellus_amd.compute.elementwise.elementwise import BroadcastSpec
from metellus_amd.orchestrator.decoding import (
    ADAPTER_ORDER_ROWS,
    ADAPTER_RANK_MAX,
    SAMPLE_LIST,
    AdapterDownOp,
    AdapterUpOp,
    PageTablesOp,
    Rotary,
    RotaryOp,
    SampleOp,
    SampleScanOp,
    adapter_many,
    adapter_splits,
    sample_bins,
    sample_chunks,
)
from metellus_amd.orchestrator.ir import (
    ITEM_BYTES,
    ElementwiseOp,
    Layout,
    MatmulOp,
    OperandValue,
    Program,
    ReductionOp,
    Scalar,
    ShapeOp,
    Tensor,
)
from metellus_amd.orchestrator.serving import (
    CacheReadOp,
    CacheWriteOp,
    DequantizeOp,
    Int4MatmulOp,
    KVCache,
    PagedAttentionOp,
    RmsNormOp,
)


def _addressable_elements(t: Tensor) -> int:
    """Elements a strided tensor can touch: (rows-1)*rs + (cols-1)*cs + 1
    (reference: builder.py:335-342)."""
    rank = len(t.shape)
    if rank == 0:
        return 1
    if rank == 1:
        return (t.shape[0] - 1) * t.row_stride + 1
    rows, cols = t.shape
    return (rows - 1) * t.row_stride + (cols - 1) * t.col_stride + 1


class Operations:
    """Mutable program builder; ``build()`` returns a snapshot list."""

    def __init__(self, dtype: str = "float32") -> None:
        self._dtype = dtype
        self._tensors: dict[str, Tensor] = {}
        self._ops: Program = []
        self._uploads: dict[str, np.ndarray] = {}
        self._caches: dict[str, KVCache] = {}
        self._written: dict[str, str] = {}  # a cache's older state -> the state after the write
        self._cache_readers: dict[str, list[Tensor]] = {}
        self._tables: dict[str, str] = {}  # a block table's older state -> the state after it
        self._used: dict[tuple[str, str], str] = {}  # (table, free)'s buffers -> how many of free are gone
        self._scratch: set[str] = set()  # what one kernel of an operator leaves for the next

    # -- registry ------------------------------------------------------------

    def input(
        self,
        name: str,
        shape: tuple[int, ...],
        layout: Layout = Layout.ROW_MAJOR,
        row_stride: int | None = None,
        col_stride: int | None = None,
        dtype: str | None = None,
    ) -> Tensor:
        """Declare a caller-supplied tensor.  Redeclaring with the same shape
        returns the existing tensor.  ``dtype`` is what its elements are stored
        as, one of ``float32`` (the default, whatever the program's label),
        ``int32``, ``int8``, ``uint8``; the serving ops say which of their
        operands take the others."""
        if dtype is not None and dtype not in ITEM_BYTES:
            raise ValueError(f"input: dtype must be one of {tuple(ITEM_BYTES)}; got {dtype!r}")
        return self._declare(name, shape, layout=layout, row_stride=row_stride, col_stride=col_stride, dtype=dtype)

    def from_numpy(self, arr: np.ndarray, name: str) -> Tensor:
        """Declare ``name`` as an input and record ``arr`` for upload.  Only
        float32 arrays -- arrays of its type for a name declared as an input of
        another type -- and storage owners (not views) are accepted
        (reference: builder.py:80-118)."""
        known = self._tensors.get(name)
        want = known.stored if known is not None else "float32"
        if arr.dtype != np.dtype(want):
            raise ValueError(f"from_numpy: array dtype must be {want}; got {arr.dtype}")
        t = self._declare(name, tuple(arr.shape))
        if t.buffer_key != name:
            raise ValueError(
                f"from_numpy: {name!r} is a view of {t.buffer_key!r}; only storage owners can be uploaded"
            )
        if tuple(arr.shape) != t.shape:
            raise ValueError(
                f"from_numpy: array shape {tuple(arr.shape)} does not match declared tensor shape {t.shape}"
            )
        need = _addressable_elements(t)
        if arr.size < need:
            raise ValueError(
                f"from_numpy: array with shape {tuple(arr.shape)} provides {arr.size} elements, "
                f"but tensor {name!r} with strides (row_stride={t.row_stride}, "
                f"col_stride={t.col_stride}) can address {need} elements"
            )
        self._uploads[name] = arr
        return t

    def _declare(
        self,
        name: str,
        shape: tuple[int, ...],
        *,
        layout: Layout = Layout.ROW_MAJOR,
        row_stride: int | None = None,
        col_stride: int | None = None,
        dtype: str | None = None,
    ) -> Tensor:
        shape = tuple(shape)
        known = self._tensors.get(name)
        if known is not None:
            if known.shape != shape:
                raise ValueError(
                    f"tensor {name!r} already declared with shape {known.shape}, "
                    f"cannot redeclare as {shape}"
                )
            if dtype is not None and known.stored != dtype:
                raise ValueError(f"tensor {name!r} already declared as {known.stored}, cannot redeclare as {dtype}")
            return known
        t = Tensor(
            name=name,
            shape=shape,
            dtype=self._label(dtype),
            stored=dtype or "float32",
            layout=layout,
            row_stride=-1 if row_stride is None else row_stride,
            col_stride=-1 if col_stride is None else col_stride,
        )
        self._tensors[name] = t
        return t

    def _lookup(self, name: str) -> Tensor:
        t = self._tensors.get(name)
        if t is None:
            raise ValueError(
                f"tensor {name!r} is not declared — call ops.input(...) first or use an op that produces it"
            )
        if name in self._tables:
            raise ValueError(
                f"block table {name!r} has been written since; its buffer now holds {self._tables[name]!r} — read that"
            )
        if name in self._scratch:
            raise ValueError(f"tensor {name!r} is an operator's own; no op reads it")
        return t

    def _lookup_float(self, name: str) -> Tensor:
        """An operand of the primitive ops, whose kernels read fp32."""
        t = self._lookup(name)
        if t.stored != "float32":
            raise ValueError(f"tensor {name!r} is {t.stored}; this op takes fp32 tensors")
        return t

    def _fresh(self, name: str, shape: tuple[int, ...], dtype: str | None = None) -> Tensor:
        """Output tensor for a new op; registered only after the op
        validates, so a rejected op leaves no stray name."""
        if name in self._tensors:
            raise ValueError(f"output tensor {name!r} already defined; IR is SSA — pick a fresh name")
        return Tensor(name=name, shape=tuple(shape), dtype=self._label(dtype), stored=dtype or "float32")

    def _label(self, dtype: str | None) -> str:
        """fp32 tensors carry the program's label, whatever it is; others their type."""
        return self._dtype if dtype in (None, "float32") else dtype

    def _emit(self, out: Tensor, op) -> Tensor:
        self._tensors[out.name] = out
        self._ops.append(op)
        return out

    # -- ops -----------------------------------------------------------------

    def matmul(self, a: str, b: str, out: str) -> Tensor:
        ta, tb = self._lookup_float(a), self._lookup_float(b)
        t_out = self._fresh(out, (ta.shape[0], tb.shape[-1]))
        return self._emit(t_out, MatmulOp(out=t_out, a=ta, b=tb))

    def elementwise(
        self,
        op: str,
        out: str,
        operands: tuple[str | int | float, ...],
        y_broadcast: BroadcastSpec | str = BroadcastSpec.NONE,
        cond_broadcast: BroadcastSpec | str = BroadcastSpec.NONE,
    ) -> Tensor:
        """Tensor names resolve to declared tensors; int/float literals
        become ``Scalar`` operands (``bool`` is rejected)."""
        y_bc = BroadcastSpec(y_broadcast)
        c_bc = BroadcastSpec(cond_broadcast)
        resolved: list[OperandValue] = []
        for o in operands:
            if isinstance(o, str):
                resolved.append(self._lookup_float(o))
            elif isinstance(o, (int, float)) and not isinstance(o, bool):
                resolved.append(Scalar(value=float(o)))
            else:
                raise ValueError(f"operand {o!r} must be a tensor name (str) or numeric literal (int/float)")
        if not resolved or not isinstance(resolved[0], Tensor):
            first = operands[0] if operands else None
            raise ValueError(
                f"elementwise {op!r}: operand[0] must be a tensor name; got {first!r}. "
                "Scalars are only allowed as secondary operands."
            )
        t_out = self._fresh(out, resolved[0].shape)
        node = ElementwiseOp(
            out=t_out, op=op, operands=tuple(resolved), y_broadcast=y_bc, cond_broadcast=c_bc
        )
        return self._emit(t_out, node)

    def transpose(self, name: str, out: str) -> Tensor:
        """Metadata-only transpose: a view sharing ``name``'s buffer."""
        src = self._lookup(name)
        self._no_cache("transpose", name)
        if out in self._tensors:
            raise ValueError(f"view tensor {out!r} already declared; pick a fresh name")
        view = src.transpose(out)
        self._tensors[out] = view
        return view

    def reshape(self, name: str, new_shape: tuple[int, ...], out: str) -> Tensor:
        """View when the source iterates linearly (or the shape is
        unchanged); otherwise a ``ShapeOp`` copy into a fresh buffer
        (reference: builder.py:259-305)."""
        src = self._lookup(name)
        self._no_cache("reshape", name)
        if out in self._tensors:
            raise ValueError(f"reshape output {out!r} already declared; pick a fresh name")
        target = tuple(new_shape)
        if src.can_reshape_as_view(target):
            view = src.reshape_view(target, out)
            self._tensors[out] = view
            return view
        if not 1 <= len(target) <= 2:
            raise ValueError(f"reshape target rank must be 1D or 2D in v0; got {target}")
        count = 1
        for d in target:
            count *= d
        if count != src.element_count:
            raise ValueError(
                f"reshape element-count mismatch: {src.shape} ({src.element_count}) → {target} ({count})"
            )
        t_out = self._fresh(out, target)
        return self._emit(t_out, ShapeOp(out=t_out, input=self._lookup_float(name)))

    def reduction(self, op: str, out: str, x: str, axis: int = -1) -> Tensor:
        from metellus_amd.compute.reduction.reduction import REDUCTION_OPS

        if op not in REDUCTION_OPS:
            raise ValueError(f"reduction op {op!r} not in {REDUCTION_OPS}")
        tx = self._lookup_float(x)
        ax = axis if axis >= 0 else len(tx.shape) + axis
        if 0 <= ax < len(tx.shape):
            shape = tx.shape[:ax] + tx.shape[ax + 1 :]
        else:
            shape = tx.shape[:-1] or (1,)
        t_out = self._fresh(out, shape)
        return self._emit(t_out, ReductionOp(out=t_out, op=op, input=tx, axis=axis))

    # -- serving ops (no counterpart in the reference) -------------------------

    def _owners(self, *tensors: Tensor | None) -> tuple[Tensor, ...]:
        """The owners of the views among ``tensors``, whose writers an op that
        reads the views comes after."""
        found = {t.buffer_key: self._tensors[t.buffer_key] for t in tensors if t is not None and t.buffer_key != t.name}
        return tuple(found.values())

    def _emit_all(self, op) -> None:
        names = [t.name for t in op.outs]
        if len(set(names)) < len(names):
            raise ValueError(f"output names must differ; got {names}")
        for t in op.outs:
            self._tensors[t.name] = t
        self._ops.append(op)

    def _no_cache(self, what: str, name: str) -> None:
        if name in self._caches:
            raise ValueError(f"{what}: {name!r} is a kv cache; only cache_write, cache_read and paged_attention take one")

    def _cache(self, name: str) -> tuple[Tensor, KVCache]:
        t = self._lookup(name)
        if name not in self._caches:
            raise ValueError(f"tensor {name!r} is not a kv cache — declare it with ops.kv_cache(...)")
        if name in self._written:
            raise ValueError(
                f"kv cache {name!r} has been written since; its buffer now holds {self._written[name]!r} — read that"
            )
        return t, self._caches[name]

    def _optional(self, name: str | None) -> Tensor | None:
        return None if name is None else self._lookup(name)

    def rms_norm(
        self,
        x: str,
        out: str,
        weight: str | None = None,
        residual: str | None = None,
        sum_out: str | None = None,
        scales: str | None = None,
        eps: float = 1e-5,
    ) -> Tensor:
        """``out`` = h / sqrt(mean(h^2) + eps) * weight by rows, h = x + residual
        (``sum_out`` keeps it).  ``scales`` names a further output: ``out`` is then
        int8, rounded to the nearest multiple of its row's scale, max / 127."""
        tx, tw, tr = self._lookup(x), self._optional(weight), self._optional(residual)
        op = RmsNormOp(
            y=self._fresh(out, tx.shape, "float32" if scales is None else "int8"),
            x=tx,
            weight=tw,
            residual=tr,
            sum_out=None if sum_out is None else self._fresh(sum_out, tx.shape, "float32"),
            scales=None if scales is None else self._fresh(scales, tx.shape[:1], "float32"),
            eps=float(eps),
            after=self._owners(tx, tw, tr),
        )
        self._emit_all(op)
        return op.y

    def dequantize(self, x: str, scales: str, out: str) -> Tensor:
        """``out`` = ``x`` (int8) times its row's scale, fp32."""
        tx, ts = self._lookup(x), self._lookup(scales)
        op = DequantizeOp(y=self._fresh(out, tx.shape, "float32"), x=tx, scales=ts, after=self._owners(tx, ts))
        self._emit_all(op)
        return op.y

    def matmul_int4(
        self,
        x: str,
        weights: str,
        scales: str,
        out: str,
        zeros: str | None = None,
        x_scales: str | None = None,
    ) -> Tensor:
        """``out`` = x @ W^T for a W held in 4 bits: W[n, k] = scales[n, k / group] *
        (q[n, k] - zeros[n, k / group]), zeros 8 where not given.  ``weights``
        (uint8, N x K/2): two of a row's q to a byte, the even one in the low bits.
        Groups of 32, 64 or 128, by the width of ``scales``.  ``x_scales``: x is
        int8 with a scale per row.  Made for few rows; any number is right, 16 at a
        time."""
        tx, tw, ts = self._lookup(x), self._lookup(weights), self._lookup(scales)
        self._no_cache("matmul_int4", weights)
        tz, txs = self._optional(zeros), self._optional(x_scales)
        op = Int4MatmulOp(
            y=self._fresh(out, (tx.shape[0], tw.shape[0]), "float32"),
            x=tx,
            weights=tw,
            scales=ts,
            zeros=tz,
            x_scales=txs,
            after=self._owners(tx, tw, ts, tz, txs),
        )
        self._emit_all(op)
        return op.y

    def kv_cache(
        self, name: str, pages: int, page_size: int, kv_heads: int, dim: int, dtype: str = "float32"
    ) -> KVCache:
        """Declare a paged key-value cache as an input (uint8, one row per page;
        see ``KVCache`` for its layout and for packing on the host)."""
        spec = KVCache(pages=pages, page_size=page_size, kv_heads=kv_heads, dim=dim, dtype=dtype)
        if name in self._tensors and self._caches.get(name) != spec:
            raise ValueError(f"tensor {name!r} already declared, cannot redeclare as {spec}")
        self._declare(name, spec.shape, dtype="uint8")
        self._caches[name] = spec
        return spec

    def cache_write(self, cache: str, k: str, v: str, slots: str, out: str) -> Tensor:
        """Store row t of ``k`` and ``v`` (fp32, kv_heads * dim) in slot
        ``slots[t]`` (int32), quantised to the cache's type.  In place: ``out`` is
        the cache's state after it, on the same buffer, and ``cache`` may not be
        read any more.  A slot outside the cache is passed over (-1 for a padded
        row); of rows that name one slot the last is stored."""
        tc, spec = self._cache(cache)
        tk, tv, ts = self._lookup(k), self._lookup(v), self._lookup(slots)
        fresh = self._fresh(out, tc.shape, "uint8")
        op = CacheWriteOp(
            written=Tensor(name=fresh.name, shape=tc.shape, dtype="uint8", stored="uint8", buffer_key=tc.buffer_key),
            cache=tc,
            spec=spec,
            k=tk,
            v=tv,
            slots=ts,
            after=(*self._owners(tk, tv, ts), *self._cache_readers.get(cache, ())),
        )
        self._emit_all(op)
        self._caches[out] = spec
        self._written[cache] = out
        return op.written

    def cache_read(self, cache: str, slots: str, k_out: str, v_out: str) -> tuple[Tensor, Tensor]:
        """Keys and values of the slots ``slots`` (int32) as fp32 rows of
        kv_heads * dim; zeros for a slot outside the cache."""
        tc, spec = self._cache(cache)
        ts = self._lookup(slots)
        shape = (ts.shape[0], spec.row) if len(ts.shape) == 1 else (1, spec.row)
        op = CacheReadOp(
            k=self._fresh(k_out, shape, "float32"),
            v=self._fresh(v_out, shape, "float32"),
            cache=tc,
            spec=spec,
            slots=ts,
            after=self._owners(ts),
        )
        self._emit_all(op)
        self._cache_readers.setdefault(cache, []).append(op.out)
        return op.k, op.v

    def paged_attention(
        self, q: str, cache: str, pages: str, lengths: str, out: str, heads: int, scale: float | None = None
    ) -> Tensor:
        """Attention of one new token per sequence: row b of ``q`` (heads * dim)
        against the first ``lengths[b]`` positions of its pages ``pages[b]`` (both
        int32), ``scale`` 1 / sqrt(dim) unless given.  Heads may share key heads.
        Positions in pages outside the cache (-1) hold no keys; a sequence without
        keys gives zeros."""
        tc, spec = self._cache(cache)
        tq, tp, tl = self._lookup(q), self._lookup(pages), self._lookup(lengths)
        op = PagedAttentionOp(
            o=self._fresh(out, tq.shape, "float32"),
            q=tq,
            cache=tc,
            spec=spec,
            pages=tp,
            lengths=tl,
            heads=heads,
            scale=float(spec.dim**-0.5 if scale is None else scale),
            after=self._owners(tq, tp, tl),
        )
        self._emit_all(op)
        self._cache_readers.setdefault(cache, []).append(op.out)
        return op.o

    # -- decoding ops (no counterpart in the reference) -------------------------

    def page_tables(
        self,
        pages: str,
        free: str,
        lengths: str,
        counts: str,
        page_size: int,
        tokens: int,
        out: str,
        slots: str,
        positions: str,
        ends: str,
        used: str,
        taken: str | None = None,
    ) -> Tensor:
        """Make room for a step's tokens: sequence b goes on from ``lengths[b]`` by
        ``counts[b]`` positions, and the pages that it lacks are taken from ``free`` in
        turn.  In place: ``out`` is the table after it, on the buffer of ``pages``, which
        may not be read any more; entries that no new page goes to are left as they were.
        Further outputs, int32 all: ``slots`` and ``positions`` of ``tokens`` rows (each
        sequence's after the other's; -1 behind the last, which ``cache_write`` passes
        over), the lengths after the step in ``ends``, and in ``used`` how many of ``free`` are
        gone after it (more than it has: the rest of the entries is -1, and their tokens
        have no slots).  A sequence grows to the end of its table and no further.

        ``taken`` (int32, one number) is how many of ``free`` are gone before the step, so the
        ``used`` of the step before; without it none are, but in a program that has made
        room in this table from this ``free`` before, what is gone since.  A ``free`` that
        begins with pages that an earlier step gave out gives them out again."""
        tp, tf, tl, tc = self._lookup(pages), self._lookup(free), self._lookup(lengths), self._lookup(counts)
        tt = self._optional(taken if taken is not None else self._used.get((tp.buffer_key, tf.buffer_key)))
        if isinstance(tokens, bool) or not isinstance(tokens, (int, np.integer)) or not 0 < tokens < 2**31:
            raise ValueError(f"page_tables tokens must be a positive int32; got {tokens!r}")
        states = {pages, *self._tables}
        views = sorted(n for n, t in self._tensors.items() if t.buffer_key == tp.buffer_key and n not in states)
        if views or (tp.buffer_key != pages and pages not in self._tables.values()):
            raise ValueError(f"page_tables writes {pages!r} in place: it can be no view and have none; got {views or [tp.buffer_key]}")
        fresh = self._fresh(out, tp.shape, "int32")
        op = PageTablesOp(
            written=Tensor(name=fresh.name, shape=tp.shape, dtype="int32", stored="int32", buffer_key=tp.buffer_key),
            slots=self._fresh(slots, (int(tokens),), "int32"),
            positions=self._fresh(positions, (int(tokens),), "int32"),
            ends=self._fresh(ends, tl.shape, "int32"),
            used=self._fresh(used, (1,), "int32"),
            pages=tp,
            free=tf,
            lengths=tl,
            counts=tc,
            page_size=page_size,
            taken=tt,
            after=(
                *self._owners(tf, tl, tc, tt),
                *(o.out for o in self._ops if any(t.name == pages for t in o.inputs)),  # who read the older state
            ),
        )
        self._emit_all(op)
        self._tables[pages] = out
        self._used[tp.buffer_key, tf.buffer_key] = used
        return op.written

    def rotary(
        self, x: str, positions: str, out: str, rotary: Rotary, k: str | None = None, k_out: str | None = None
    ) -> Tensor:
        """``out`` is ``x`` with the heads of row t turned to ``positions[t]`` (int32, any),
        as ``rotary`` says; ``k_out`` is ``k`` turned alike, in the same launch."""
        if not isinstance(rotary, Rotary):
            raise ValueError(f"rotary must be a Rotary; got {rotary!r}")
        tx, tp, tk = self._lookup(x), self._lookup(positions), self._optional(k)
        if (k is None) != (k_out is None):
            raise ValueError("rotary: k and k_out go together")
        op = RotaryOp(
            y=self._fresh(out, tx.shape, "float32"),
            x=tx,
            positions=tp,
            spec=rotary,
            k=tk,
            k_out=None if tk is None else self._fresh(k_out, tk.shape, "float32"),
            after=self._owners(tx, tp, tk),
        )
        self._emit_all(op)
        return op.y

    def adapters(
        self, x: str, base: str, a: str, b: str, ids: str, out: str, scales: str | None = None
    ) -> Tensor:
        """``out`` = ``base`` + scales[i] * B_i (A_i x) by rows, i = ``ids`` of the row
        (int32): low-rank adapters, each row's own, beside a product that all share
        (``base``).  ``a`` (adapters * rank, columns of x) and ``b`` (adapters * columns of
        base, rank) hold every adapter's A and B, one after the other (all of one rank: a
        smaller one has zeros behind its own, which are read and multiplied as others are);
        ``scales`` are 1 unless given.  A row whose id is none of theirs (-1) is its row of ``base``."""
        tx, ty, ta, tb = self._lookup(x), self._lookup_float(base), self._lookup(a), self._lookup(b)
        ti, ts = self._lookup(ids), self._optional(scales)
        for label, t in (("x", tx), ("base", ty), ("a", ta), ("b", tb)):
            if len(t.shape) != 2:
                raise ValueError(f"adapters {label} must be 2D; got shape {t.shape} ({t.name!r})")
        cols, rank = ty.shape[1], tb.shape[1]
        if rank > ADAPTER_RANK_MAX:
            raise ValueError(f"adapters: ranks up to {ADAPTER_RANK_MAX}; {b!r} has {rank}")
        if tb.shape[0] % cols or ta.shape[0] != tb.shape[0] // cols * rank:
            raise ValueError(
                f"adapters a must have shape (adapters * rank, {tx.shape[1]}) and b (adapters * {cols}, rank); "
                f"got {ta.shape} and {tb.shape}"
            )
        if tx.shape[0] != ty.shape[0]:
            raise ValueError(f"adapters x and base must have as many rows; got {tx.shape} and {ty.shape}")
        many = adapter_many(*tx.shape, cols, rank)
        splits = adapter_splits(*tx.shape, many)
        down = AdapterDownOp(
            down=self._fresh(f"{out}.down", (splits * tx.shape[0], -(-rank // 4) * 4), "float32"),
            x=tx,
            a=ta,
            ids=ti,
            rank=rank,
            splits=splits,
            many=many,
            name=out,
            order=self._fresh(f"{out}.order", (tx.shape[0], 2), "int32") if tx.shape[0] >= ADAPTER_ORDER_ROWS else None,
            after=self._owners(tx, ta, ti),
        )
        up = AdapterUpOp(
            y=self._fresh(out, ty.shape, "float32"),
            base=ty,
            down=down.down,
            b=tb,
            ids=ti,
            rank=rank,
            splits=splits,
            many=many,
            scales=ts,
            order=down.order,
            after=self._owners(ty, tb, ti, ts),
        )
        self._emit_all(down)
        self._emit_all(up)
        self._scratch.update(t.name for t in down.outs)
        return up.y

    def sample(
        self,
        logits: str,
        uniforms: str,
        out: str,
        temperatures: str | None = None,
        top_k: str | None = None,
        top_p: str | None = None,
        min_p: str | None = None,
        logprobs: str | None = None,
    ) -> Tensor:
        """``out`` (int32) is a token for each row of ``logits``, drawn by the row's number
        in ``uniforms``, 0 <= u < 1 (others count as the nearer end).  With w_i =
        exp((x_i - max) / temperature): the ``top_k`` largest logits (int32; none or below
        1: all; the lower index first among equals), of those the fewest of the largest
        that weigh ``top_p`` of them (1 and above: all), of those the ones with
        w_i >= ``min_p``; then the first index up to which more than u of the weight that
        is left has come by.  All four are a number for each row.  A temperature of 0 (or
        below, or NaN) takes the largest, 1 where not given.  ``logprobs``: the logarithm
        of the probability that the token was drawn with.  Logits of +inf share
        all the weight.  A row of -inf alone, or with a NaN, gives -1, its logprob NaN.
        Weights are held to 2^-44 of the largest (2^-42 for the longest rows): what weighs
        less than half of that weighs nothing, at the ends of u too."""
        tl, tu = self._lookup(logits), self._lookup(uniforms)
        given = {n: self._optional(v) for n, v in
                 (("temperatures", temperatures), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p))}
        if len(tl.shape) != 2:
            raise ValueError(f"sample logits must be 2D; got shape {tl.shape} ({tl.name!r})")
        rows, cols = tl.shape
        chunk, chunks = sample_chunks(rows, cols)
        apart, cuts = chunks > 1, top_k is not None or top_p is not None

        def made(part: str, rows: int, words: int, wanted: bool = True) -> Tensor | None:
            return self._fresh(f"{out}.{part}", (rows, 2 * words), "int32") if wanted else None

        pick = SampleOp(
            tokens=self._fresh(out, (rows,), "int32"),
            logits=tl,
            uniforms=tu,
            best=made("best", rows * chunks, 1, apart),
            counts=made("counts", rows, 1, apart),
            bins=made("bins", rows * chunks, sample_bins(cols), apart and cuts),
            sums=made("sums", rows, (2 + chunk // 256) * chunks, apart),
            listed=made("list", rows, SAMPLE_LIST, apart and cuts),
            logprobs=None if logprobs is None else self._fresh(logprobs, (rows,), "float32"),
            after=self._owners(tl, tu, *given.values()),
            **given,
        )
        if apart:
            scan = SampleScanOp(
                best=pick.best,
                counts=pick.counts,
                logits=tl,
                name=out,
                bins=pick.bins,
                **{n: t if cuts else None for n, t in given.items() if n != "min_p"},
                after=self._owners(tl, *given.values()),
            )
        names = [t.name for t in (*(scan.outs if apart else ()), *pick.outs)]
        if len(set(names)) < len(names):
            raise ValueError(f"output names must differ; got {names}")
        if apart:
            self._emit_all(scan)
        self._emit_all(pick)
        own = (pick.best, pick.counts, pick.bins, pick.sums, pick.listed)
        self._scratch.update(t.name for t in own if t is not None)
        return pick.tokens

    # -- results -------------------------------------------------------------

    def build(self) -> Program:
        return list(self._ops)

    @property
    def tensors(self) -> dict[str, Tensor]:
        return dict(self._tensors)

    @property
    def uploads(self) -> dict[str, np.ndarray]:
        return dict(self._uploads)

    @property
    def scratch(self) -> frozenset[str]:
        """Tensors that one kernel of an operator leaves for the next: no outputs."""
        return frozenset(self._scratch)
