"""The decoding ops in float64 (test infrastructure only; see ``ir_eval``).

Written from the ops' definitions, one sequence, row or head at a time, apart from the
product's kernels.  fp32 results come back as float64 (before their one rounding).
"""

from __future__ import annotations

import math

import numpy as np

F64 = np.float64


def _page_tables(op, get):
    p, table, free = op.page_size, np.array(get(op.pages)), list(get(op.free))
    width, rows = table.shape[1], op.slots.shape[0]
    slots, positions, ends = [], [], []
    used = 0 if op.taken is None else max(0, int(get(op.taken)[0]))
    for b, (length, count) in enumerate(zip(get(op.lengths).tolist(), get(op.counts).tolist())):
        begin = min(max(length, 0), width * p)
        have = -(-begin // p)
        end = min(begin + max(count, 0), width * p)
        for entry in range(have, -(-end // p)):
            table[b, entry] = free[used] if used < len(free) else -1
            used += 1
        for i in range(min(max(count, 0), rows - len(slots))):
            at = begin + i
            positions.append(at if at < end else -1)
            page = int(table[b, at // p]) if at < end else -1
            slot = page * p + at % p
            slots.append(slot if page >= 0 and slot < 2**31 else -1)
        ends.append(end)
    pad = [-1] * (rows - len(slots))
    made = {op.slots: slots + pad, op.positions: positions + pad, op.ends: ends, op.used: [min(used, 2**31 - 1)]}
    return {op.written.name: table, **{t.name: np.array(v, np.int32) for t, v in made.items()}}


def rotary_frequencies(spec):
    """Radians a pair turns for a step, by the definition."""
    if spec.frequencies is not None:
        return list(spec.frequencies)
    found = []
    for i in range(spec.part // 2):
        f = spec.base ** (-2 * i / spec.part)
        if spec.original is None:
            found.append(f / spec.factor)
            continue
        turns = spec.original * f / (2 * math.pi)
        if turns >= spec.high:
            found.append(f)
        elif turns <= spec.low:
            found.append(f / spec.factor)
        else:
            g = (turns - spec.low) / (spec.high - spec.low)
            found.append(f * g + f / spec.factor * (1 - g))
    return found


def rotary_pairs(spec):
    """The elements of a head that are pairs."""
    h = spec.part // 2
    return [(i, i + h) if spec.layout == "half" else (2 * i, 2 * i + 1) for i in range(h)]


def rotary_angles(spec, positions):
    """Angles of [row, pair] within one turn.  Products of a position and a frequency are
    taken as whole numbers, so that far positions lose nothing."""
    two_pi = 31415926535897932384626433832795028841971693993751 * 2  # times 10^-49
    found = np.empty((len(positions), spec.part // 2))
    for j, f in enumerate(rotary_frequencies(spec)):
        n, d = float(f).as_integer_ratio()
        for r, at in enumerate(positions):
            # at * n / d radians, in units of 10^-49
            found[r, j] = (int(at) * n * 10**49 // d) % two_pi / 10**49
    return found


def _rotary(op, get):
    spec = op.spec
    angles = rotary_angles(spec, get(op.positions))
    found = {}
    for x, out in ((op.x, op.y), (op.k, op.k_out)):
        if x is None:
            continue
        heads = get(x).astype(F64).reshape(x.shape[0], -1, spec.dim)
        y = heads.copy()
        for j, (a, b) in enumerate(rotary_pairs(spec)):
            c, s = np.cos(angles[:, j, None]) * spec.magnitude, np.sin(angles[:, j, None]) * spec.magnitude
            with np.errstate(all="ignore"):
                y[:, :, a] = heads[:, :, a] * c - heads[:, :, b] * s
                y[:, :, b] = heads[:, :, b] * c + heads[:, :, a] * s
        found[out.name] = y.reshape(x.shape)
    return found


def _adapter_down(op, get):
    x, a = get(op.x).astype(F64), np.ascontiguousarray(get(op.a)).astype(F64)
    down = np.zeros(op.down.shape)
    for m, i in enumerate(get(op.ids)):
        if 0 <= i < op.held:
            with np.errstate(all="ignore"):
                down[m, : op.rank] = a[i * op.rank : (i + 1) * op.rank] @ x[m]  # (the first part has it all)
    found = {op.down.name: down}
    if op.order is not None:  # (in which order rows are taken is the kernel's choice)
        ids = np.asarray(get(op.ids))
        found[op.order.name] = np.stack([np.arange(len(ids)), np.where((ids < 0) | (ids >= op.held), -1, ids)], axis=1).astype(np.int32)
    return found


def _adapter_up(op, get):
    y, b = get(op.base).astype(F64), np.ascontiguousarray(get(op.b)).astype(F64)
    n = y.shape[1]
    down = get(op.down).astype(F64).reshape(op.splits, -1, op.down.shape[1]).sum(axis=0)[:, : op.rank]
    for m, i in enumerate(get(op.ids)):
        if 0 <= i < op.held:
            with np.errstate(all="ignore"):
                scale = 1.0 if op.scales is None else float(get(op.scales)[i])
                y[m] = y[m] + scale * (b[i * n : (i + 1) * n] @ down[m])
    return {op.y.name: y}


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logarithm of its probability) of one row; sums in more than 64 bits."""
    x = np.asarray(x).astype(F64)
    if np.isnan(x).any() or x.max() == -math.inf:
        return -1, math.nan
    top = x.max()
    if not temperature > 0:
        return int(np.nonzero(x == top)[0][0]), 0.0
    with np.errstate(all="ignore"):
        scaled = np.where(x == top, 0.0, np.where((x == -math.inf) | (top == math.inf), -math.inf, (x - top) / F64(temperature)))
    weight = np.exp(scaled.astype(np.longdouble))
    order = np.lexsort((np.arange(len(x)), -x))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        upto = np.cumsum(weight[order])
        before = upto - weight[order]
        order = order[: max(1, int((before < np.longdouble(top_p) * upto[-1]).sum()))]
    if min_p > 0:
        order = order[scaled[order] >= math.log(min(1.0, float(min_p)))]  # (of weights, not of what they are rounded to)
    order = np.sort(order)
    upto = np.cumsum(weight[order])
    behind = np.nonzero(upto > (np.longdouble(u) if u > 0 else 0) * upto[-1])[0]
    at = order[behind[0]] if len(behind) else order[np.nonzero(weight[order])[0][-1]]
    return int(at), float(scaled[at] - np.log(upto[-1]))


def _sample_scan(op, get):
    return {t.name: np.zeros(t.shape, np.int32) for t in op.outs}  # the kernels' own


def _sample(op, get):
    x = get(op.logits)
    asked = {}
    for name in ("temperatures", "top_k", "top_p", "min_p"):
        t = getattr(op, name)
        if t is not None:
            asked[name.rstrip("s") if name == "temperatures" else name] = get(t)
    found = [sample_row(x[r], get(op.uniforms)[r], **{n: v[r] for n, v in asked.items()}) for r in range(x.shape[0])]
    made = {t.name: np.zeros(t.shape, np.int32) for t in (op.sums, op.listed) if t is not None}  # the kernels' own
    made[op.tokens.name] = np.array([f[0] for f in found], np.int32)
    if op.logprobs is not None:
        made[op.logprobs.name] = np.array([f[1] for f in found])
    return made


def evaluate_decoding(op, get) -> dict:
    """``{output name: array}`` of one op; ``get(tensor)`` reads an input."""
    return {"PageTablesOp": _page_tables, "RotaryOp": _rotary, "AdapterDownOp": _adapter_down,
            "AdapterUpOp": _adapter_up, "SampleScanOp": _sample_scan, "SampleOp": _sample}[type(op).__name__](op, get)
