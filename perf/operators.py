"""Performance cases of the serving operators: one decode step of a model with a paged cache.

Four operators: ``norm`` (residual addition and RMS norm, in 32 or 8 bits), ``matvec`` (few rows
against 4-bit weights with group scales), ``cache`` (new keys and values quantised into a paged
cache, and slots read back) and ``attention`` (one new token a sequence over that cache).  A case
names its operator under ``op`` and gives its sizes.

``run`` computes a case in its plain form, from elementary torch operations, or, where ``own`` is
set, by the framework: the program is written with ``Operations``, compiled, and kept with its
device buffers, as a program that serves does; a pass is one ``Runtime.run``.

The cache's bytes: a row of ``page_bytes`` per page holds [keys | values], each
[kv_heads][page_size][dim]; 8-bit types follow them with one fp32 scale per row of ``dim``, keys
first.  Rows are padded to 16 bytes.  Slot s is row s % page_size of page s // page_size.
"""

import math
import random

import torch

own = False  # the framework's operators instead of the plain forms

EPS = 1e-5
PEAK = {"int8": 127.0, "float8_e4m3": 448.0}  # what a row's largest magnitude is scaled to
ITEM = {"float32": 4, "int8": 1, "float8_e4m3": 1}
HELD = {"float32": torch.float32, "int8": torch.int8, "float8_e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # One token between two layers: latency is all there is.
        {"name": "norm-token", "op": "norm", "rows": 1, "cols": 4096, "residual": True, "out": "float32"},
        # A prompt's rows, given on in 8 bits.
        {"name": "norm-prompt", "op": "norm", "rows": 4096, "cols": 4096, "residual": True, "out": "int8"},
        # Odd sizes, and no residual (a model's first norm).
        {"name": "norm-ragged", "op": "norm", "rows": 777, "cols": 5003, "residual": False, "out": "float32"},
        # One token against a gated block's first weight.
        {"name": "matvec-token", "op": "matvec", "rows": 1, "inner": 4096, "cols": 11008, "group": 128,
         "x": "float32", "zeros": False},
        # A batch of tokens in 8 bits against its last weight.
        {"name": "matvec-batch", "op": "matvec", "rows": 16, "inner": 11008, "cols": 4096, "group": 64,
         "x": "int8", "zeros": False},
        # Odd sizes, small groups with zero points.
        {"name": "matvec-ragged", "op": "matvec", "rows": 5, "inner": 5024, "cols": 4099, "group": 32,
         "x": "float32", "zeros": True},
        # The logits of a few sequences over a large vocabulary.
        {"name": "matvec-logits", "op": "matvec", "rows": 4, "inner": 4096, "cols": 131072, "group": 128,
         "x": "float32", "zeros": False},
        # One new token for each of 32 short sequences; the whole cache is read back.
        {"name": "cache-token", "op": "cache", "tokens": 32, "pages": 32, "page_size": 16, "kv_heads": 8,
         "dim": 128, "held": "int8"},
        # A long prompt's keys and values into pages in no order.
        {"name": "cache-prompt", "op": "cache", "tokens": 8192, "pages": 1024, "page_size": 16, "kv_heads": 8,
         "dim": 128, "held": "float8_e4m3"},
        # One sequence, as many key heads as query heads, nothing quantised.
        {"name": "attention-token", "op": "attention", "sequences": 1, "keys": 2048, "heads": 32, "kv_heads": 32,
         "dim": 128, "page_size": 16, "held": "float32"},
        # A serving batch of ragged lengths, four query heads to a key head.
        {"name": "attention-batch", "op": "attention", "sequences": 32, "keys": 8192, "heads": 32, "kv_heads": 8,
         "dim": 128, "page_size": 16, "held": "int8"},
        # One very long context, its length odd.
        {"name": "attention-long", "op": "attention", "sequences": 1, "keys": 131071, "heads": 32, "kv_heads": 8,
         "dim": 128, "page_size": 64, "held": "float8_e4m3"},
    ]


def _log(rng, low, high, step=1):
    """A size spread over the logarithm of [low, high], a multiple of ``step``."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(("norm", "matvec", "matvec", "cache", "attention", "attention"))
    if op == "norm":
        cols = _log(rng, 64, 16384, rng.choice((1, 64)))
        return {"op": op, "rows": _log(rng, 1, min(8192, 2**24 // cols)), "cols": cols,
                "residual": rng.random() < 0.7, "out": rng.choice(("float32", "int8"))}
    if op == "matvec":
        group = rng.choice((32, 64, 128))
        inner = _log(rng, 256, 16384, group)
        rows = _log(rng, 1, 16)
        return {"op": op, "rows": rows, "inner": inner,
                "cols": _log(rng, 64, min(65536, 2**28 // inner, 2**31 // (inner * rows)), rng.choice((1, 64))), "group": group,
                "x": rng.choice(("float32", "float32", "int8")), "zeros": rng.random() < 0.3}
    if op == "cache":
        kv_heads, dim, page_size = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 96, 128, 256)), rng.choice((8, 16, 20, 64))
        tokens = _log(rng, 1, min(8192, 2**22 // (kv_heads * dim)))
        return {"op": op, "tokens": tokens, "pages": -(-tokens // page_size) + _log(rng, 1, 32), "page_size": page_size,
                "kv_heads": kv_heads, "dim": dim, "held": rng.choice(("float32", "int8", "float8_e4m3"))}
    kv_heads, dim, page_size = rng.choice((1, 2, 4, 8, 16, 32)), rng.choice((64, 96, 128, 256)), rng.choice((8, 16, 20, 64))
    sequences, held = _log(rng, 1, 64), rng.choice(("float32", "int8", "float8_e4m3"))
    most = 2**27 // (sequences * kv_heads * dim * ITEM[held])
    return {"op": op, "sequences": sequences, "keys": _log(rng, 1, max(1, min(131072, most))),
            "heads": kv_heads * rng.choice((1, 2, 4, 8)), "kv_heads": kv_heads, "dim": dim, "page_size": page_size,
            "held": held}


# ---------------------------------------------------------------------------
# the cache's layout
# ---------------------------------------------------------------------------


def _page_bytes(case):
    rows = 2 * case["kv_heads"] * case["page_size"]
    held = case["held"]
    return -(-(rows * case["dim"] * ITEM[held] + (0 if held == "float32" else 4 * rows)) // 16) * 16


def _views(case, cache):
    """The values ([pages, 2, kv_heads, page_size, dim]) and scales ([pages, 2, kv_heads,
    page_size], or None) in the cache's bytes."""
    h, p, d = case["kv_heads"], case["page_size"], case["dim"]
    n = 2 * h * p * d * ITEM[case["held"]]
    values = cache[:, :n].view(HELD[case["held"]]).unflatten(1, (2, h, p, d))
    if case["held"] == "float32":
        return values, None
    return values, cache[:, n : n + 8 * h * p].view(torch.float32).unflatten(1, (2, h, p))


def _lengths(case):
    """The lengths of a ragged batch, their sum the same for every seed: even steps up to
    ``keys``, and one sequence that has no key yet where there are many."""
    b, n = case["sequences"], case["keys"]
    made = [max(1, n * (i + 1) // b) for i in range(b)]
    if b >= 8:
        made[0] = 0
    return made


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _filled_cache(case, pages, gen):
    """Pages full of keys and values of about N(0, 1)."""
    shape = (pages, 2, case["kv_heads"], case["page_size"], case["dim"])
    cache = torch.zeros(pages, _page_bytes(case), dtype=torch.uint8, device="cuda")
    values, scales = _views(case, cache)
    x = torch.randn(shape, generator=gen, device="cuda")
    if scales is None:
        values.copy_(x)
        return cache
    x *= PEAK[case["held"]] / 4
    x.clamp_(-PEAK[case["held"]], PEAK[case["held"]])
    if case["held"] == "int8":
        x.round_()
    values.copy_(x.to(values.dtype))
    scales.copy_((0.75 + 0.5 * torch.rand(shape[:-1], generator=gen, device="cuda")) * (4 / PEAK[case["held"]]))
    return cache


def _inputs(case, seed):
    """Every input of the case from the seed alone, on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "norm":
        made = {"x": normal(case["rows"], case["cols"]), "weight": 1 + 0.1 * normal(case["cols"])}
        if case["residual"]:
            made["residual"] = 4 * normal(case["rows"], case["cols"])
        return made
    if case["op"] == "matvec":
        m, k, n, groups = case["rows"], case["inner"], case["cols"], case["inner"] // case["group"]
        made = {
            "weights": torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8),
            "scales": (0.5 + torch.rand((n, groups), generator=gen, device="cuda")) / (4.6 * math.sqrt(k)),
        }
        if case["zeros"]:
            made["zeros"] = torch.randint(5, 11, (n, groups), generator=gen, device="cuda").float()
        if case["x"] == "int8":
            made["x"] = (40 * normal(m, k)).round_().clamp_(-127, 127).to(torch.int8)
            made["x_scales"] = (0.5 + torch.rand((m,), generator=gen, device="cuda")) / 40
        else:
            made["x"] = normal(m, k)
        return made
    if case["op"] == "cache":
        slots, row = case["pages"] * case["page_size"], case["kv_heads"] * case["dim"]
        at = torch.randperm(slots, generator=gen, device="cuda")[: case["tokens"]].int()
        return {
            "cache": _filled_cache(case, case["pages"], gen),
            "k": normal(case["tokens"], row), "v": normal(case["tokens"], row),
            "slots": at, "back": torch.randperm(slots, generator=gen, device="cuda").int(),
        }
    lengths = _lengths(case)
    host.shuffle(lengths)
    p, table_width = case["page_size"], -(-case["keys"] // case["page_size"])
    used = [-(-n // p) for n in lengths]
    order = list(range(sum(used) + 1))  # a page that is nobody's
    host.shuffle(order)
    table, at = [], 0
    for u in used:
        table.append(order[at : at + u] + [-1] * (table_width - u))
        at += u
    return {
        "cache": _filled_cache(case, len(order), gen), "q": normal(case["sequences"], case["heads"] * case["dim"]),
        "pages": torch.tensor(table, dtype=torch.int32).cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(),
    }


class _View:
    """A device buffer of the framework for torch (no copy); keeps the buffer alive."""

    def __init__(self, buffer, shape, typestr):
        self.buffer = buffer
        self.__cuda_array_interface__ = {
            "shape": tuple(shape), "typestr": typestr, "data": (buffer.device_address, False), "version": 2,
        }


def _tensor(buffer, shape, dtype):
    typestr = {"float32": "<f4", "int32": "<i4", "int8": "|i1", "uint8": "|u1"}[dtype]
    return torch.as_tensor(_View(buffer, shape, typestr), device="cuda")


class _Program:
    """The case's operators as a compiled program of the framework, its buffers on the GPU."""

    def __init__(self, case, inputs):
        from metellus_amd.api import compile_program
        from metellus_amd.orchestrator import Operations
        from metellus_amd.runtime import Buffer, Dispatch, Runtime

        ops = Operations()
        for name, t in inputs.items():
            if name == "cache":
                ops.kv_cache(name, pages=t.shape[0], page_size=case["page_size"], kv_heads=case["kv_heads"],
                             dim=case["dim"], dtype=case["held"])
            else:
                ops.input(name, tuple(t.shape), dtype=str(t.dtype).removeprefix("torch."))
        outputs = self._write(ops, case)
        groups = compile_program(ops)
        self.env = {}
        for name, t in inputs.items():
            self.env[name] = Buffer(t.numel() * t.element_size())
            _tensor(self.env[name], t.shape, ops.tensors[name].dtype).copy_(t)
        for name, t in ops.tensors.items():
            if t.buffer_key not in self.env:
                self.env[t.buffer_key] = Buffer(t.nbytes)
        self.outputs = {n: _tensor(self.env[ops.tensors[n].buffer_key], ops.tensors[n].shape, "float32") for n in outputs}
        steps = [Dispatch(g.kernel, g.bindings, g.dims, g.grid, g.threads) for g in groups]
        for step in steps:
            _ = step.kernel.handle  # compiled here, as a program that runs it again and again has it
        self.runtime = Runtime(tuple(steps))
        torch.cuda.synchronize()  # the inputs were written on torch's stream

    @staticmethod
    def _write(ops, case):
        if case["op"] == "norm":
            sums = {"residual": "residual", "sum_out": "h"} if case["residual"] else {}
            if case["out"] == "int8":  # held in 8 bits, and brought back for whoever wants 32
                ops.rms_norm("x", out="y8", weight="weight", eps=EPS, scales="s", **sums)
                ops.dequantize("y8", scales="s", out="y")
            else:
                ops.rms_norm("x", out="y", weight="weight", eps=EPS, **sums)
            return ["h", "y"] if case["residual"] else ["y"]
        if case["op"] == "matvec":
            ops.matmul_int4("x", weights="weights", scales="scales", out="y",
                            zeros="zeros" if case["zeros"] else None,
                            x_scales="x_scales" if case["x"] == "int8" else None)
            return ["y"]
        if case["op"] == "cache":
            ops.cache_write("cache", k="k", v="v", slots="slots", out="written")
            ops.cache_read("written", slots="back", k_out="k_back", v_out="v_back")
            return ["k_back", "v_back"]
        ops.paged_attention("q", cache="cache", pages="pages", lengths="lengths", heads=case["heads"], out="o")
        return ["o"]

    def run(self):
        self.runtime.run(self.env)
        return self.outputs


def prepare(case, seed):
    """The inputs; for the framework in its own buffers (the one memory its programs run on),
    with the compiled program."""
    inputs = _inputs(case, seed)
    if own:
        return _Program(case, inputs)
    return case, inputs


def run(state):
    if own:
        return state.run()
    case, t = state
    return {"norm": _norm, "matvec": _matvec, "cache": _cache, "attention": _attention}[case["op"]](case, **t)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _norm(case, x, weight, residual=None):
    h = x if residual is None else x + residual
    if case["out"] == "float32":
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * weight
    else:  # in 64 bits: values next to the border between two steps
        w = h.double()
        w = w / torch.sqrt((w * w).mean(1, keepdim=True) + EPS) * weight
        scale = (w.abs().amax(1, keepdim=True) / 127).float()
        y = (torch.where(scale > 0, torch.round(w / scale), 0) * scale).float()
    return {"y": y} if residual is None else {"h": h, "y": y}


def _matvec(case, x, weights, scales, zeros=None, x_scales=None):
    n, k = case["cols"], case["inner"]
    q = torch.stack((weights & 15, weights >> 4), dim=2).view(n, -1, case["group"]).float()
    w = (q - (8.0 if zeros is None else zeros[:, :, None])) * scales[:, :, None]
    x = x.float()
    if x_scales is not None:
        x = x * x_scales[:, None]
    return {"y": x @ w.view(n, k).T}


def _eight_bits(held, x):
    """Rows of fp32 as values of the held type and a scale each; quotients in 64 bits, where a
    value next to the border between two steps is seen on its side."""
    scale = x.abs().amax(-1) / PEAK[held]
    v = x.double() / torch.where(scale > 0, scale, 1)[..., None].double()
    if held == "float8_e4m3":  # three bits behind the leading one, down to 2^-9
        step = torch.exp2(torch.clamp(torch.frexp(v)[1] - 1, min=-6).double() - 3)
        v = torch.round(v / step) * step
    else:
        v = torch.round(v)
    return torch.clamp(v, -PEAK[held], PEAK[held]).float().to(HELD[held]), scale


def _cache(case, cache, k, v, slots, back):
    h, d, p = case["kv_heads"], case["dim"], case["page_size"]
    values, scales = _views(case, cache)
    new = torch.stack((k, v), dim=1).unflatten(2, (h, d))
    page, row = slots.long() // p, slots.long() % p
    if scales is None:
        values[page, :, :, row] = new
    else:
        held, scale = _eight_bits(case["held"], new)
        values.view(torch.uint8)[page, :, :, row] = held.view(torch.uint8)  # (no 8-bit float is assigned by index)
        scales[page, :, :, row] = scale
    page, row = back.long() // p, back.long() % p
    if scales is None:
        found = values[page, :, :, row]
    else:
        found = values.view(torch.uint8)[page, :, :, row].view(values.dtype).float() * scales[page, :, :, row][..., None]
    found = found.flatten(2)
    return {"k_back": found[:, 0], "v_back": found[:, 1]}


def _attention(case, cache, q, pages, lengths):
    b, h, d, p = case["sequences"], case["kv_heads"], case["dim"], case["page_size"]
    values, scales = _views(case, cache)
    at = torch.arange(case["keys"], device=q.device)
    page, row = pages[:, at // p].long(), (at % p).expand(b, -1)
    live = (at < lengths[:, None]) & (page >= 0)
    page = page.clamp(min=0)
    if scales is None:
        kv = values[page, :, :, row]  # [sequences, keys, 2, kv_heads, dim]
    else:
        kv = values.view(torch.uint8)[page, :, :, row].view(values.dtype).float() * scales[page, :, :, row][..., None]
    k, v = kv[:, :, 0].permute(0, 2, 3, 1), kv[:, :, 1].transpose(1, 2)
    scores = torch.matmul(q.view(b, h, -1, d), k.contiguous()) / math.sqrt(d)
    scores = torch.where(live[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v.contiguous()) / torch.where(total > 0, total, 1)
    return {"o": o.reshape(b, -1)}


# ---------------------------------------------------------------------------
# what a pass needs, and what it should give
# ---------------------------------------------------------------------------


def work(case):
    """Inputs read once, outputs written once; 2 flops a multiply-add, one an elementwise
    operation."""
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        moved = 4 * (2 + 2 * case["residual"]) * n + 4 * case["cols"]
        return {"bytes": moved, "flops": (4 + case["residual"]) * n}
    if case["op"] == "matvec":
        m, k, n, groups = case["rows"], case["inner"], case["cols"], case["inner"] // case["group"]
        x = m * (k + 4) if case["x"] == "int8" else 4 * m * k
        return {"bytes": n * k // 2 + 4 * n * groups * (1 + case["zeros"]) + x + 4 * m * n, "flops": 2 * m * k * n}
    row = case["kv_heads"] * case["dim"]
    held = row * ITEM[case["held"]] + (0 if case["held"] == "float32" else 4 * case["kv_heads"])
    if case["op"] == "cache":
        slots, t = case["pages"] * case["page_size"], case["tokens"]
        return {"bytes": 2 * t * (4 * row + held) + 2 * slots * (4 * row + held) + 4 * (t + slots),
                "flops": 2 * (3 * t + slots) * row}
    keys, out = sum(_lengths(case)), case["sequences"] * case["heads"] * case["dim"]
    return {"bytes": 2 * keys * held + 8 * out + 4 * keys // case["page_size"],
            "flops": 4 * keys * case["heads"] * case["dim"]}


def exact(case, seed):
    """The outputs of ``run`` in 64 bits, from the definitions."""
    t = _inputs(case, seed)
    if case["op"] == "norm":
        h = t["x"] + t["residual"] if case["residual"] else t["x"]
        h64 = h.double()
        y = h64 * torch.rsqrt(h64.pow(2).sum(1) / case["cols"] + EPS)[:, None] * t["weight"].double()
        if case["out"] == "int8":
            s = (y.abs().max(1).values / 127).float().double()[:, None]
            y = torch.round(y / s).nan_to_num_(0.0) * s
        return {"h": h64, "y": y} if case["residual"] else {"y": y}
    if case["op"] == "matvec":
        x = t["x"].double() * (t["x_scales"].double()[:, None] if case["x"] == "int8" else 1)
        y = torch.empty(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
        zeros = t.get("zeros", torch.full_like(t["scales"], 8.0))
        for n in range(0, case["cols"], 16384):
            rows = slice(n, n + 16384)
            w = torch.empty(t["weights"][rows].shape[0], case["inner"], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = t["weights"][rows] % 16, t["weights"][rows] // 16
            w -= zeros[rows].double().repeat_interleave(case["group"], 1)
            w *= t["scales"][rows].double().repeat_interleave(case["group"], 1)
            y[:, rows] = x @ w.T
        return {"y": y}
    values, scales = _views(case, t["cache"])
    h, d, p = case["kv_heads"], case["dim"], case["page_size"]
    if case["op"] == "cache":
        state = values.double() if scales is None else values.double() * scales.double()[..., None]
        state = state.permute(0, 3, 1, 2, 4).reshape(-1, 2, h, d)  # by slot
        new = torch.stack((t["k"], t["v"]), dim=1).view(-1, 2, h, d).double()
        if scales is not None:
            s = (new.abs().max(3, keepdim=True).values / PEAK[case["held"]]).float().double()
            new = new / s
            if case["held"] == "float8_e4m3":
                e = torch.floor(torch.log2(new.abs().clamp(min=2.0**-6)))
                new = torch.round(new * 2.0 ** (3 - e)) * 2.0 ** (e - 3)
            else:
                new = torch.round(new)
            new = new.clamp(-PEAK[case["held"]], PEAK[case["held"]]) * s
        state[t["slots"].long()] = new
        found = state[t["back"].long()]
        return {"k_back": found[:, 0].reshape(-1, h * d), "v_back": found[:, 1].reshape(-1, h * d)}
    o = torch.zeros(case["sequences"], h, case["heads"] // h, d, dtype=torch.float64, device="cuda")
    q = t["q"].view(o.shape).double()
    for i, n in enumerate(t["lengths"].tolist()):
        if n:
            page = t["pages"][i, : -(-n // p)].long()
            kv = values[page] if scales is None else values.view(torch.uint8)[page].view(values.dtype)
            kv = kv.double() if scales is None else kv.double() * scales[page].double()[..., None]
            kv = kv.permute(1, 2, 0, 3, 4).reshape(2, h, -1, d)[:, :, :n]
            o[i] = torch.softmax(q[i] @ kv[0].mT.contiguous() / math.sqrt(d), -1) @ kv[1]
    return {"o": o.view(case["sequences"], -1)}
