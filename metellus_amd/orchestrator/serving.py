"""The serving ops: one decode step of a model with a paged key-value cache.

No counterpart in the reference.  They stand in a program next to the four
primitive ops: names, SSA and validation are the same, but they are written as
whole operators (each becomes one kernel, never fused with its neighbours),
may write several tensors (``outs``) and take tensors of other types than fp32:

* ``RmsNormOp``        h = x + residual, y = h / rms(h) * weight, y fp32 or int8 + row scales
* ``DequantizeOp``     int8 rows and their scales back to fp32
* ``Int4MatmulOp``     few rows against 4-bit weights with group scales
* ``CacheWriteOp``     keys and values into the slots of a paged cache, in place
* ``CacheReadOp``      slots of the cache back to fp32
* ``PagedAttentionOp`` one new token per sequence over the cache

``KVCache`` describes a cache: its types, its layout, and packing on the host.

A ``CacheWriteOp`` writes into its cache's own buffer, so its output is a new
SSA name on that buffer (as a view is), and the old name may not be read after
it.  ``after`` orders ops beyond the tensors they read: a write comes after
every op that reads the older state, and an op that reads a view comes after
the op that writes the view's owner.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from metellus_amd.orchestrator.ir import Tensor

HEAD_DIM_MAX = 256
CACHE_TYPES = ("float32", "int8", "float8_e4m3")
_PEAK = {"int8": 127.0, "float8_e4m3": 448.0}
INT4_GROUPS = (32, 64, 128)
_INT32_MAX = 2**31 - 1


def _e4m3_table() -> np.ndarray:
    """The value of each e4m3 byte (OCP: bias 7, no infinities, 0x7F is NaN)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0**-9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v).astype(np.float32)


@dataclass(frozen=True)
class KVCache:
    """A paged key-value cache: ``pages`` pages of ``page_size`` slots, each slot
    a key and a value row of ``dim`` per head.

    ``dtype`` is ``float32``, ``int8`` (a row is whole numbers in +-127 times its
    scale) or ``float8_e4m3`` (OCP e4m3 in +-448 times its scale).  A page is one
    row of ``page_bytes``: [keys | values], each [kv_heads][page_size][dim], then
    for the 8-bit types one fp32 scale for each of those rows, keys first, padded
    to 16 bytes.  Slot ``s`` is row ``s % page_size`` of page ``s // page_size``.
    """

    pages: int
    page_size: int
    kv_heads: int
    dim: int
    dtype: str = "float32"

    def __post_init__(self) -> None:
        for name in ("pages", "page_size", "kv_heads", "dim"):
            v = getattr(self, name)
            if isinstance(v, bool) or not isinstance(v, (int, np.integer)) or v <= 0:
                raise ValueError(f"kv cache: {name} must be a positive int; got {v!r}")
            object.__setattr__(self, name, int(v))
        if self.dtype not in CACHE_TYPES:
            raise ValueError(f"kv cache: dtype must be one of {CACHE_TYPES}; got {self.dtype!r}")
        if self.dim % 16 or self.dim > HEAD_DIM_MAX:
            raise ValueError(f"kv cache: dim must be a multiple of 16 up to {HEAD_DIM_MAX}; got {self.dim}")
        if self.page_bytes > _INT32_MAX:
            raise ValueError(f"kv cache: a page of {self.page_bytes} bytes is too large (2 GiB at most)")
        if self.pages > _INT32_MAX:
            raise ValueError(f"kv cache: {self.pages} pages; page numbers are int32")

    @property
    def item_bytes(self) -> int:
        return 4 if self.dtype == "float32" else 1

    @property
    def _value_bytes(self) -> int:
        return 2 * self.kv_heads * self.page_size * self.dim * self.item_bytes

    @property
    def page_bytes(self) -> int:
        n = self._value_bytes
        if self.dtype != "float32":
            n += 8 * self.kv_heads * self.page_size
        return -(-n // 16) * 16

    @property
    def row(self) -> int:
        """Elements of one slot's keys (or values)."""
        return self.kv_heads * self.dim

    @property
    def slots(self) -> int:
        return self.pages * self.page_size

    @property
    def shape(self) -> tuple[int, int]:
        """Shape of the cache's tensor (uint8)."""
        return (self.pages, self.page_bytes)

    def empty(self) -> np.ndarray:
        """The bytes of a cache whose slots all hold zeros."""
        return np.zeros(self.shape, dtype=np.uint8)

    def unpack(self, data: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
        """Keys and values of every slot, ``(slots, kv_heads, dim)`` fp32 each."""
        data = np.ascontiguousarray(data, dtype=np.uint8).reshape(self.shape)
        inner = (2, self.kv_heads, self.page_size)
        raw = np.ascontiguousarray(data[:, : self._value_bytes])
        if self.dtype == "float32":
            v = raw.view(np.float32).reshape(self.pages, *inner, self.dim)
        else:
            at = slice(self._value_bytes, self._value_bytes + 8 * self.kv_heads * self.page_size)
            scales = np.ascontiguousarray(data[:, at]).view(np.float32).reshape(self.pages, *inner, 1)
            if self.dtype == "int8":
                held = raw.view(np.int8).astype(np.float32)
            else:
                held = _e4m3_table()[raw]
            with np.errstate(invalid="ignore"):
                v = held.reshape(self.pages, *inner, self.dim) * scales
        v = v.transpose(1, 0, 3, 2, 4).reshape(2, self.slots, self.kv_heads, self.dim)
        return v[0], v[1]

    def pack(self, keys: np.ndarray, values: np.ndarray) -> np.ndarray:
        """The cache's bytes from the keys and values of every slot (the layouts of
        ``unpack``), quantised as ``CacheWriteOp`` does."""
        kv = np.stack([np.asarray(keys, dtype=np.float32), np.asarray(values, dtype=np.float32)])
        kv = kv.reshape(2, self.pages, self.page_size, self.kv_heads, self.dim).transpose(1, 0, 3, 2, 4)
        data = self.empty()
        if self.dtype == "float32":
            data[:, : self._value_bytes] = np.ascontiguousarray(kv).reshape(self.pages, -1).view(np.uint8)
            return data
        held, scales = quantize_rows(kv, self.dtype)
        data[:, : self._value_bytes] = held.reshape(self.pages, -1)
        at = slice(self._value_bytes, self._value_bytes + 8 * self.kv_heads * self.page_size)
        data[:, at] = np.ascontiguousarray(scales).reshape(self.pages, -1).view(np.uint8)
        return data


def quantize_rows(x: np.ndarray, dtype: str) -> tuple[np.ndarray, np.ndarray]:
    """Last-axis rows of fp32 in 8 bits (as bytes) and a fp32 scale each: the
    largest magnitude times fp32's 1/127 (``int8``) or 1/448 (``float8_e4m3``), which is
    within 2^-23 of the quotient, the values ``x / scale`` rounded to the nearest, ties to even.  A row of zeros has the
    scale 0; a row with a value that is not finite is zeros with the scale NaN."""
    x = np.asarray(x, dtype=np.float32)
    peak = _PEAK[dtype]
    top = np.abs(x).max(axis=-1)
    fine = np.isfinite(top)
    scale = np.where(fine, np.where(fine, top, 0) * (np.float32(1) / np.float32(peak)), np.float32(np.nan)).astype(np.float32)
    div = np.where(fine & (scale > 0), scale, 1).astype(np.float64)[..., None]
    v = np.where((fine & (scale > 0))[..., None], x, 0).astype(np.float64) / div  # 64 bits: borders fall as they should
    if dtype == "int8":
        return np.clip(np.rint(v), -peak, peak).astype(np.int8).view(np.uint8), scale
    a = np.abs(v)
    step = np.exp2(np.maximum(np.frexp(a)[1] - 1, -6) - 3.0)
    a = np.minimum(np.rint(a / step) * step, peak)
    table = _e4m3_table()[:127].astype(np.float64)  # 0 .. 448, ascending
    code = np.searchsorted(table, a).astype(np.uint8)
    return np.where(np.signbit(v), code | 128, code).astype(np.uint8), scale


# ---------------------------------------------------------------------------
# ops
# ---------------------------------------------------------------------------


def _want(label: str, t: Tensor, dtype: str, shape: tuple[int, ...]) -> None:
    if t.stored != dtype:
        raise ValueError(f"{label} must be {dtype}; got {t.stored} ({t.name!r})")
    if t.shape != shape:
        raise ValueError(f"{label} must have shape {shape}; got {t.shape} ({t.name!r})")


def _dense(label: str, t: Tensor) -> None:
    if not t.is_contiguous():
        raise ValueError(f"{label} must be dense, row after row; got strides ({t.row_stride}, {t.col_stride}) ({t.name!r})")


def _rows(label: str, t: Tensor, dtype: str) -> tuple[int, int]:
    """A 2-D tensor of ``dtype`` (fp32 ones may have any strides)."""
    if len(t.shape) != 2:
        raise ValueError(f"{label} must be 2D; got shape {t.shape} ({t.name!r})")
    _want(label, t, dtype, t.shape)
    if t.row_stride < 0 or t.col_stride < 0 or max(t.row_stride, t.col_stride) > _INT32_MAX:
        raise ValueError(f"{label}: strides ({t.row_stride}, {t.col_stride}) are out of range ({t.name!r})")
    return t.shape


class ServingOp:
    """An op that is one kernel of its own; ``out`` is its first output."""

    after: tuple[Tensor, ...]

    @property
    def outs(self) -> tuple[Tensor, ...]:
        raise NotImplementedError

    @property
    def out(self) -> Tensor:
        return self.outs[0]

    @property
    def reads(self) -> tuple[Tensor, ...]:
        """The tensors the kernel reads."""
        raise NotImplementedError

    @property
    def overwrites(self) -> Tensor | None:
        """The older name of a buffer that the op writes in place (its new one is among
        ``outs``)."""
        return None

    @property
    def inputs(self) -> tuple[Tensor, ...]:
        known = {t.name for t in self.reads}
        return (*self.reads, *(t for t in self.after if t.name not in known))


@dataclass(frozen=True)
class RmsNormOp(ServingOp):
    """``scales`` set: ``y`` is int8 and ``scales`` its row scales."""

    y: Tensor
    x: Tensor
    weight: Tensor | None = None
    residual: Tensor | None = None
    sum_out: Tensor | None = None
    scales: Tensor | None = None
    eps: float = 1e-5
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows, cols = _rows("rms_norm x", self.x, "float32")
        if self.residual is not None:
            _rows("rms_norm residual", self.residual, "float32")
            _want("rms_norm residual", self.residual, "float32", (rows, cols))
        if self.sum_out is not None and self.residual is None:
            raise ValueError("rms_norm sum_out needs a residual: without one the sum is x itself")
        if self.weight is not None:
            _want("rms_norm weight", self.weight, "float32", (cols,))
            _dense("rms_norm weight", self.weight)
        if not 0.0 <= self.eps < float("inf"):
            raise ValueError(f"rms_norm eps must be finite and not negative; got {self.eps}")

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.y, self.scales, self.sum_out) if t is not None)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.x, self.residual, self.weight) if t is not None)


@dataclass(frozen=True)
class DequantizeOp(ServingOp):
    y: Tensor
    x: Tensor
    scales: Tensor
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows, _ = _rows("dequantize x", self.x, "int8")
        _dense("dequantize x", self.x)
        _want("dequantize scales", self.scales, "float32", (rows,))
        _dense("dequantize scales", self.scales)

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return (self.y,)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return (self.x, self.scales)


@dataclass(frozen=True)
class Int4MatmulOp(ServingOp):
    """y[m, n] = sum over the groups g of scales[n, g] * sum over g's k of
    x[m, k] * (q[n, k] - zeros[n, g]), zeros 8 where none are given.  Byte j of
    row n of ``weights`` holds q[n, 2 j] in its low and q[n, 2 j + 1] in its high
    four bits.  x is fp32, or int8 with a scale per row (``x_scales``)."""

    y: Tensor
    x: Tensor
    weights: Tensor
    scales: Tensor
    zeros: Tensor | None = None
    x_scales: Tensor | None = None
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows, k = _rows("matmul_int4 x", self.x, "float32" if self.x_scales is None else "int8")
        n, half = _rows("matmul_int4 weights", self.weights, "uint8")
        if 2 * half != k:
            raise ValueError(f"matmul_int4: weights {self.weights.shape} hold {2 * half} columns; x has {k}")
        if len(self.scales.shape) != 2 or self.scales.shape[0] != n or k % self.scales.shape[1]:
            raise ValueError(f"matmul_int4 scales must have shape ({n}, groups) with groups dividing {k}; got {self.scales.shape}")
        if self.group not in INT4_GROUPS:
            raise ValueError(f"matmul_int4: groups of {INT4_GROUPS} columns only; scales {self.scales.shape} give {self.group}")
        _want("matmul_int4 scales", self.scales, "float32", self.scales.shape)
        for label, t in (("weights", self.weights), ("scales", self.scales), ("zeros", self.zeros)):
            if t is not None:
                _dense(f"matmul_int4 {label}", t)
        if self.zeros is not None:
            _want("matmul_int4 zeros", self.zeros, "float32", self.scales.shape)
        if self.x_scales is not None:
            _dense("matmul_int4 x", self.x)
            _want("matmul_int4 x_scales", self.x_scales, "float32", (rows,))
            _dense("matmul_int4 x_scales", self.x_scales)

    @property
    def group(self) -> int:
        return self.x.shape[1] // self.scales.shape[1]

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return (self.y,)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.x, self.weights, self.scales, self.zeros, self.x_scales) if t is not None)


@dataclass(frozen=True)
class CacheWriteOp(ServingOp):
    """Row t of ``k`` and ``v`` goes to slot ``slots[t]``; slots outside the cache
    are passed over, and of rows that name one slot the last is stored."""

    written: Tensor
    cache: Tensor
    spec: KVCache
    k: Tensor
    v: Tensor
    slots: Tensor
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows, _ = _rows("cache_write k", self.k, "float32")
        _want("cache_write k", self.k, "float32", (rows, self.spec.row))
        _rows("cache_write v", self.v, "float32")
        _want("cache_write v", self.v, "float32", (rows, self.spec.row))
        _want("cache_write slots", self.slots, "int32", (rows,))
        _dense("cache_write slots", self.slots)

    @property
    def overwrites(self) -> Tensor:
        return self.cache

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return (self.written,)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return (self.k, self.v, self.slots, self.cache)


@dataclass(frozen=True)
class CacheReadOp(ServingOp):
    """Row r of ``k`` and ``v`` is slot ``slots[r]``, zeros for one outside the cache."""

    k: Tensor
    v: Tensor
    cache: Tensor
    spec: KVCache
    slots: Tensor
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        if len(self.slots.shape) != 1:
            raise ValueError(f"cache_read slots must be 1D; got shape {self.slots.shape}")
        _want("cache_read slots", self.slots, "int32", self.slots.shape)
        _dense("cache_read slots", self.slots)

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return (self.k, self.v)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return (self.cache, self.slots)


@dataclass(frozen=True)
class PagedAttentionOp(ServingOp):
    """o[b, h] = softmax(scale * q[b, h] . keys) @ values over the first
    ``lengths[b]`` positions of sequence b, position p in row p % page_size of page
    ``pages[b, p // page_size]``.  Query head h reads key head
    h // (heads / kv_heads).  Lengths below 0 count as 0, lengths beyond the table
    as its end; a page number outside the cache is a hole whose positions hold no
    keys.  A sequence without keys gives zeros."""

    o: Tensor
    q: Tensor
    cache: Tensor
    spec: KVCache
    pages: Tensor
    lengths: Tensor
    heads: int
    scale: float
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        if isinstance(self.heads, bool) or not isinstance(self.heads, (int, np.integer)) or self.heads <= 0:
            raise ValueError(f"paged_attention heads must be a positive int; got {self.heads!r}")
        if self.heads % self.spec.kv_heads:
            raise ValueError(f"paged_attention: {self.heads} heads do not divide over {self.spec.kv_heads} key heads")
        rows, _ = _rows("paged_attention q", self.q, "float32")
        _want("paged_attention q", self.q, "float32", (rows, self.heads * self.spec.dim))
        if len(self.pages.shape) != 2 or self.pages.shape[0] != rows:
            raise ValueError(f"paged_attention pages must have shape ({rows}, pages per sequence); got {self.pages.shape}")
        _want("paged_attention pages", self.pages, "int32", self.pages.shape)
        _dense("paged_attention pages", self.pages)
        _want("paged_attention lengths", self.lengths, "int32", (rows,))
        _dense("paged_attention lengths", self.lengths)
        if self.capacity > _INT32_MAX - 1024:
            raise ValueError(f"paged_attention: a table of {self.capacity} positions; lengths are int32")
        if not abs(self.scale) <= 2e38:  # (times log2(e) it is fp32 on the device)
            raise ValueError(f"paged_attention scale must be finite and within 2e38; got {self.scale}")

    @property
    def capacity(self) -> int:
        """Positions that a row of the table has room for."""
        return self.pages.shape[1] * self.spec.page_size

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return (self.o,)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return (self.q, self.cache, self.pages, self.lengths)
