"""``Operations``: name-keyed builder for the primitive IR.

Same surface as the reference builder (reference:
src/orchestrator/builder.py:50-342): ``input``, ``from_numpy``, ``matmul``,
``elementwise``, ``transpose``, ``reshape``, ``reduction``, ``build``,
``tensors``, ``uploads``; beyond it the serving ops (``rms_norm``,
``dequantize``, ``matmul_int4``, ``kv_cache``, ``cache_write``, ``cache_read``,
``paged_attention``) and inputs of their types.  Validation is delegated to the op dataclasses;
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

    # -- results -------------------------------------------------------------

    def build(self) -> Program:
        return list(self._ops)

    @property
    def tensors(self) -> dict[str, Tensor]:
        return dict(self._tensors)

    @property
    def uploads(self) -> dict[str, np.ndarray]:
        return dict(self._uploads)
