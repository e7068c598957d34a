"""The serving ops in float64 (test infrastructure only; see ``ir_eval``).

Written from the ops' definitions, one row at a time, apart from the product's
packing and kernels.  fp32 results come back as float64 (before their one
rounding), 8-bit ones in their type.
"""

from __future__ import annotations

import numpy as np

from oracle.decoding_eval import evaluate_decoding

F32, F64 = np.float32, np.float64


def e4m3(code: int) -> float:
    """The value of an e4m3 byte (OCP: bias 7, no infinities, 0x7F NaN)."""
    sign = -1.0 if code & 128 else 1.0
    e, m = (code >> 3) & 15, code & 7
    if e == 15 and m == 7:
        return float("nan")
    return sign * (m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))


E4M3 = np.array([e4m3(c) for c in range(256)])


def nearest_e4m3(v: np.ndarray) -> np.ndarray:
    """Bytes of the nearest e4m3 values, ties to the even byte."""
    a = np.abs(v)
    table = E4M3[:127]
    hi = np.clip(np.searchsorted(table, a), 1, 126)
    below, above = a - table[hi - 1], table[hi] - a
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return (np.where(up, hi, hi - 1) | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def quantize(row: np.ndarray, held: str):
    """(bytes, scale) of one row.  float32 rows: scale = max times float32's 1/127 or
    1/448; float64 rows (a norm's): max / 127 rounded to float32."""
    row = np.asarray(row)
    if not np.all(np.isfinite(row)):
        return np.zeros(row.shape, np.uint8), F32(np.nan)
    peak = 127.0 if held == "int8" else 448.0
    top = np.abs(row).max()
    scale = F32(top * (F32(1) / F32(peak))) if row.dtype == F32 else F32(top / peak)
    if scale == 0:
        return np.zeros(row.shape, np.uint8), scale
    v = row.astype(F64) / F64(scale)
    if held == "int8":
        return np.clip(np.rint(v), -127, 127).astype(np.int8).view(np.uint8), scale
    return nearest_e4m3(np.clip(v, -448, 448)), scale


def _page_parts(spec, data: np.ndarray, page: int):
    """(values as bytes [2][heads][page_size][dim * item], scales [2][heads][page_size] or None) of a page,
    views into ``data``."""
    item = 4 if spec.dtype == "float32" else 1
    rows = 2 * spec.kv_heads * spec.page_size
    n = rows * spec.dim * item
    values = data[page, :n].reshape(2, spec.kv_heads, spec.page_size, spec.dim * item)
    if item == 4:
        return values, None
    return values, data[page, n : n + 4 * rows].view(F32).reshape(2, spec.kv_heads, spec.page_size)


def slot_rows(spec, data: np.ndarray, slot: int) -> np.ndarray:
    """Keys and values of a slot, float64 (2, kv_heads, dim)."""
    values, scales = _page_parts(spec, data, slot // spec.page_size)
    raw = np.ascontiguousarray(values[:, :, slot % spec.page_size])
    if scales is None:
        return raw.view(F32).astype(F64)
    held = raw.view(np.int8).astype(F64) if spec.dtype == "int8" else E4M3[raw]
    with np.errstate(invalid="ignore"):
        return held * scales[:, :, slot % spec.page_size, None].astype(F64)


def _norm(op, get):
    x = np.ascontiguousarray(get(op.x))
    h = x if op.residual is None else x + get(op.residual)  # float32, rounded once
    wide = h.astype(F64)
    with np.errstate(all="ignore"):
        y = wide / np.sqrt((wide * wide).mean(axis=1, keepdims=True) + op.eps)
        if op.weight is not None:
            y = y * get(op.weight).astype(F64)
    found = {} if op.sum_out is None else {op.sum_out.name: h}
    if op.scales is None:
        return {**found, op.y.name: y}
    rows = [quantize(r, "int8") for r in y]
    q = np.stack([r[0] for r in rows]).view(np.int8)
    return {**found, op.y.name: q, op.scales.name: np.array([r[1] for r in rows], F32)}


def _int4(op, get):
    raw = np.ascontiguousarray(get(op.weights))
    q = np.empty((raw.shape[0], 2 * raw.shape[1]))
    q[:, 0::2], q[:, 1::2] = raw & 15, raw >> 4
    x = get(op.x).astype(F64)
    scales = get(op.scales).astype(F64)
    zeros = np.full(scales.shape, 8.0) if op.zeros is None else get(op.zeros).astype(F64)
    y = np.zeros((x.shape[0], raw.shape[0]))
    with np.errstate(all="ignore"):
        for g in range(scales.shape[1]):
            at = slice(g * op.group, (g + 1) * op.group)
            y += (x[:, at] @ (q[:, at] - zeros[:, g : g + 1]).T) * scales[:, g]
        if op.x_scales is not None:
            y *= get(op.x_scales).astype(F64)[:, None]
    return {op.y.name: y}


def _write(op, get):
    spec, data = op.spec, np.array(get(op.cache))
    kv = np.stack([get(op.k), get(op.v)], axis=1).reshape(-1, 2, spec.kv_heads, spec.dim)
    for t, slot in enumerate(get(op.slots)):
        if not 0 <= slot < spec.slots:
            continue
        values, scales = _page_parts(spec, data, slot // spec.page_size)
        for part in range(2):
            for h in range(spec.kv_heads):
                row = np.ascontiguousarray(kv[t, part, h])
                at = (part, h, slot % spec.page_size)
                if scales is None:
                    values[at] = row.view(np.uint8)
                else:
                    values[at], scales[at] = quantize(row, spec.dtype)
    return {op.written.name: data}


def _read(op, get):
    spec, data, slots = op.spec, np.ascontiguousarray(get(op.cache)), get(op.slots)
    found = np.zeros((len(slots), 2, spec.kv_heads, spec.dim))
    for r, slot in enumerate(slots):
        if 0 <= slot < spec.slots:
            found[r] = slot_rows(spec, data, slot)
    return {op.k.name: found[:, 0].reshape(len(slots), -1), op.v.name: found[:, 1].reshape(len(slots), -1)}


def attention_rows(op, get):
    """(q, keys, values) of each sequence: (heads, dim) and (kv_heads, positions, dim)."""
    spec, data, table = op.spec, np.ascontiguousarray(get(op.cache)), get(op.pages)
    for b, length in enumerate(get(op.lengths)):
        held = []
        for at in range(max(0, min(int(length), op.capacity))):
            page = table[b, at // spec.page_size]
            if 0 <= page < spec.pages:
                held.append(slot_rows(spec, data, int(page) * spec.page_size + at % spec.page_size))
        kv = np.stack(held, axis=2) if held else np.zeros((2, spec.kv_heads, 0, spec.dim))
        yield get(op.q)[b].astype(F64).reshape(op.heads, spec.dim), kv[0], kv[1]


def _attention(op, get):
    found = []
    for q, k, v in attention_rows(op, get):
        o = np.zeros(q.shape)
        share = op.heads // op.spec.kv_heads
        for h in range(op.heads if k.shape[1] else 0):
            with np.errstate(all="ignore"):
                s = k[h // share] @ q[h] * op.scale
                e = np.exp(s - s.max())
                o[h] = e @ v[h // share] / e.sum()
        found.append(o.reshape(-1))
    return {op.o.name: np.stack(found)}


def evaluate_serving(op, get) -> dict:
    """``{output name: array}`` of one op; ``get(tensor)`` reads an input."""
    kind = type(op).__name__
    if kind == "DequantizeOp":
        with np.errstate(invalid="ignore"):
            return {op.y.name: get(op.x).astype(F64) * get(op.scales).astype(F64)[:, None]}
    known = {"RmsNormOp": _norm, "Int4MatmulOp": _int4, "CacheWriteOp": _write, "CacheReadOp": _read,
             "PagedAttentionOp": _attention}
    return known[kind](op, get) if kind in known else evaluate_decoding(op, get)
