"""Performance cases of the operators around a decode step's products and attention.

Four operators: ``pages`` (block tables, slots and positions of a step's tokens from the lengths of
its sequences), ``rotary`` (queries and keys turned by their positions), ``adapters`` (low-rank
adapters of many requests beside a shared product) and ``sample`` (tokens from logits and given
random numbers).  A case names its operator under ``op`` and gives its sizes.

``run`` computes a case in its plain form, from elementary torch operations, or, where ``own`` is
set, by the framework: the program is written with ``Operations``, compiled, and kept with its
device buffers, as a program that serves does; a pass is one ``Runtime.run``.
"""

import math
import random

import torch

own = False  # the framework's operators instead of the plain forms


def listed():
    return [
        # One new token for each of 32 sequences: latency is all there is.
        {"name": "pages-step", "op": "pages", "sequences": 32, "keys": 8192, "page_size": 16, "tokens": 32},
        # Ragged prompts and sequences that only go on, odd pages, a few padded rows.
        {"name": "pages-prompts", "op": "pages", "sequences": 1021, "keys": 65536, "page_size": 20, "tokens": 16384},
        # One token's heads between the products and the cache.
        {"name": "rotary-token", "op": "rotary", "rows": 1, "heads": 32, "kv_heads": 8, "dim": 128, "part": 128,
         "layout": "half", "long": False, "far": 8192},
        # A long prompt.
        {"name": "rotary-prompt", "op": "rotary", "rows": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "part": 128,
         "layout": "half", "long": True, "far": 131072},
        # Neighbouring pairs in part of odd heads, positions far beyond the first context.
        {"name": "rotary-ragged", "op": "rotary", "rows": 777, "heads": 12, "kv_heads": 3, "dim": 96, "part": 40,
         "layout": "interleaved", "long": True, "far": 1048576},
        # One request's adapter beside a square product.
        {"name": "adapters-token", "op": "adapters", "rows": 1, "requests": 1, "held": 8, "rank": 16, "inner": 4096,
         "cols": 4096},
        # A batch of tokens, nearly each with an adapter of its own.
        {"name": "adapters-batch", "op": "adapters", "rows": 32, "requests": 32, "held": 64, "rank": 16, "inner": 4096,
         "cols": 11008},
        # Odd sizes and an odd rank; some requests have no adapter.
        {"name": "adapters-ragged", "op": "adapters", "rows": 77, "requests": 11, "held": 5, "rank": 23, "inner": 5003,
         "cols": 4099},
        # The prompts of eight requests.
        {"name": "adapters-prompt", "op": "adapters", "rows": 4096, "requests": 8, "held": 16, "rank": 64, "inner": 4096,
         "cols": 4096},
        # One sequence's next token from a large vocabulary, every filter on.
        {"name": "sample-token", "op": "sample", "rows": 1, "cols": 131072, "filters": "all"},
        # A batch whose requests ask for different things.
        {"name": "sample-batch", "op": "sample", "rows": 64, "cols": 131072, "filters": "mixed"},
        # An odd vocabulary, cut by its probabilities alone.
        {"name": "sample-ragged", "op": "sample", "rows": 17, "cols": 32003, "filters": "top_p"},
    ]


def _log(rng, low, high, step=1):
    """A size spread over the logarithm of [low, high], a multiple of ``step``."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(("pages", "rotary", "adapters", "adapters", "sample", "sample"))
    if op == "pages":
        sequences = _log(rng, 1, 2048)
        keys = _log(rng, 64, min(131072, 2**26 // sequences))
        tokens = sequences if rng.random() < 0.5 else _log(rng, 1, min(32768, sequences * keys))
        return {"op": op, "sequences": sequences, "keys": keys, "page_size": rng.choice((8, 16, 20, 64)), "tokens": tokens}
    if op == "rotary":
        kv_heads, dim = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 80, 96, 128, 256))
        heads = kv_heads * rng.choice((1, 2, 4, 8))
        return {"op": op, "rows": _log(rng, 1, min(16384, 2**25 // ((heads + kv_heads) * dim))), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "part": rng.choice((dim, dim, dim // 2, 2 * rng.randint(1, dim // 2))),
                "layout": rng.choice(("half", "interleaved")), "long": rng.random() < 0.5, "far": _log(rng, 64, 1048576)}
    if op == "adapters":
        inner, cols = _log(rng, 64, 16384, rng.choice((1, 64))), _log(rng, 64, 16384, rng.choice((1, 64)))
        rows, rank = _log(rng, 1, min(4096, 13 * 10**6 // max(inner, cols))), rng.choice((4, 8, 16, 32, 64, rng.randint(1, 64)))
        requests = rows if rng.random() < 0.5 else _log(rng, 1, rows)
        return {"op": op, "rows": rows, "requests": requests, "held": _log(rng, 1, max(1, min(64, 2**25 // (rank * (inner + cols))))),
                "rank": rank, "inner": inner, "cols": cols}
    cols = _log(rng, 500, 262144)
    return {"op": op, "rows": _log(rng, 1, min(128, 2**23 // cols)), "cols": cols,
            "filters": rng.choice(("all", "mixed", "mixed", "top_k", "top_p", "min_p", "none"))}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _counts(case):
    """New tokens and earlier lengths of the sequences, their sums the same for every seed.  A
    sixteenth of the rows is padding."""
    n, rows = case["sequences"], case["tokens"] - case["tokens"] // 16
    if rows <= n:
        counts = [1] * rows + [0] * (n - rows)
    else:
        counts = [min(case["keys"], max(1, 2 * rows * i // (n * n))) for i in range(n)]
        while sum(counts) > rows:
            top = max(range(n), key=lambda i: counts[i])
            counts[top] -= min(counts[top], sum(counts) - rows)
    lengths = [(case["keys"] - c) * ((i * 7) % n + 1) // n for i, c in enumerate(counts)]
    return lengths, counts


def _pages_needed(case):
    p = case["page_size"]
    return [-(-(a + c) // p) - -(-a // p) for a, c in zip(*_counts(case))]


def _frequencies(case):
    """Angles for one step of position: base 10000, and for long contexts those that turn seldom
    within 8192 positions slowed down eight times, those in between by parts."""
    f = [10000.0 ** (-2 * i / case["part"]) for i in range(case["part"] // 2)]
    if not case["long"]:
        return f
    kept = [min(1.0, max(0.0, (8192 * v / (2 * math.pi) - 1) / (4 - 1))) for v in f]
    return [(1 - g) * v / 8 + g * v for g, v in zip(kept, f)]


def _ids(case):
    """The adapter of each request; every eighth has none."""
    return [-1 if i % 8 == 7 else i % case["held"] for i in range(case["requests"])]


def _row_request(case):
    return [r * case["requests"] // case["rows"] for r in range(case["rows"])]


def _has(case):
    f = case["filters"]
    return {"top_k": f in ("all", "mixed", "top_k"), "top_p": f in ("all", "mixed", "top_p"), "min_p": f in ("all", "mixed", "min_p")}


def _inputs(case, seed):
    """Every input of the case from the seed alone, on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def ints(values):
        return torch.tensor(values, dtype=torch.int32).cuda()

    if case["op"] == "pages":
        pairs = list(zip(*_counts(case)))
        host.shuffle(pairs)
        p, width = case["page_size"], -(-case["keys"] // case["page_size"])
        used = torch.tensor([-(-a // p) for a, _ in pairs])
        held, need = int(used.sum()), sum(_pages_needed(case))
        order = torch.randperm(held + need + 8, generator=torch.Generator().manual_seed(seed)).int()
        table = torch.full((case["sequences"], width), -1, dtype=torch.int32)
        table[torch.arange(width)[None] < used[:, None]] = order[:held]
        return {"pages": table.cuda(), "free": order[held:].cuda(), "lengths": ints([a for a, _ in pairs]),
                "counts": ints([c for _, c in pairs])}
    if case["op"] == "rotary":
        first = host.randint(0, max(0, case["far"] - case["rows"]))  # a prompt's rows follow each other
        return {"q": normal(case["rows"], case["heads"] * case["dim"]), "k": normal(case["rows"], case["kv_heads"] * case["dim"]),
                "positions": ints(range(first, first + case["rows"]))}
    if case["op"] == "adapters":
        m, n, k, r, s = case["rows"], case["cols"], case["inner"], case["rank"], case["held"]
        ids, names = _ids(case), list(range(s))
        host.shuffle(ids)
        host.shuffle(names)
        return {"x": normal(m, k), "base": normal(m, n), "a": normal(s * r, k) / math.sqrt(k), "b": normal(s * n, r) / math.sqrt(r),
                "scales": 0.5 + torch.rand((s,), generator=gen, device="cuda"),
                "ids": ints([-1 if ids[q] < 0 else names[ids[q]] for q in _row_request(case)])}
    rows, cols, has = case["rows"], case["cols"], _has(case)
    # A broad row with a few likely tokens far above it, as a model's are.
    logits = normal(rows, cols) * (1 + torch.rand((rows, 1), generator=gen, device="cuda"))
    likely = torch.randint(0, cols, (rows, 1), generator=gen, device="cuda")
    likely = (likely + torch.arange(40, device="cuda") * (cols // 40)) % cols
    logits.scatter_(1, likely, 6 + 6 * torch.rand((rows, 40), generator=gen, device="cuda"))
    made = {"logits": logits, "uniforms": torch.rand((rows,), generator=gen, device="cuda")}
    mixed = case["filters"] == "mixed"

    def asked(values, off):
        return [host.choice((*values, off)) if mixed else host.choice(values) for _ in range(rows)]

    made["temperatures"] = torch.tensor(asked((0.6, 0.8, 1.0, 1.3), 0.0)).cuda()
    if has["top_k"]:
        made["top_k"] = ints(asked((20, 40, 50, 200), 0))
    if has["top_p"]:
        made["top_p"] = torch.tensor(asked((0.8, 0.9, 0.95), 1.0)).cuda()
    if has["min_p"]:
        made["min_p"] = torch.tensor(asked((0.02, 0.05, 0.1), 0.0)).cuda()
    return made


class _View:
    """A device buffer of the framework for torch (no copy); keeps the buffer alive."""

    def __init__(self, buffer, shape, typestr):
        self.buffer = buffer
        self.__cuda_array_interface__ = {
            "shape": tuple(shape), "typestr": typestr, "data": (buffer.device_address, False), "version": 2,
        }


def _tensor(buffer, shape, dtype):
    return torch.as_tensor(_View(buffer, shape, {"float32": "<f4", "int32": "<i4"}[dtype]), device="cuda")


class _Program:
    """The case's operators as a compiled program of the framework, its buffers on the GPU."""

    def __init__(self, case, inputs):
        from metellus_amd.api import compile_program
        from metellus_amd.orchestrator import Operations
        from metellus_amd.runtime import Buffer, Dispatch, Runtime

        ops = Operations()
        for name, t in inputs.items():
            ops.input(name, tuple(t.shape), dtype=str(t.dtype).removeprefix("torch."))
        outputs = self._write(ops, case, inputs)
        groups = compile_program(ops)
        self.env = {}
        for name, t in inputs.items():
            self.env[name] = Buffer(t.numel() * t.element_size())
            _tensor(self.env[name], t.shape, ops.tensors[name].stored).copy_(t)
        for t in ops.tensors.values():
            if t.buffer_key not in self.env:
                self.env[t.buffer_key] = Buffer(t.nbytes)
        self.outputs = {label: _tensor(self.env[ops.tensors[n].buffer_key], ops.tensors[n].shape, ops.tensors[n].stored)
                        for label, n in outputs.items()}
        steps = [Dispatch(g.kernel, g.bindings, g.dims, g.grid, g.threads) for g in groups]
        for step in steps:
            _ = step.kernel.handle  # compiled here, as a program that runs it again and again has it
        self.runtime = Runtime(tuple(steps))
        torch.cuda.synchronize()  # the inputs were written on torch's stream

    @staticmethod
    def _write(ops, case, inputs):
        """Writes the program; its outputs by label."""
        if case["op"] == "pages":
            ops.page_tables("pages", free="free", lengths="lengths", counts="counts", page_size=case["page_size"],
                            tokens=case["tokens"], out="table", slots="slots", positions="positions", ends="ends", used="used")
            return {n: n for n in ("table", "slots", "positions", "ends", "used")}
        if case["op"] == "rotary":
            from metellus_amd.orchestrator import Rotary

            more = {"factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0} if case["long"] else {}
            ops.rotary("q", positions="positions", out="q_out", k="k", k_out="k_out",
                       rotary=Rotary(dim=case["dim"], part=case["part"], layout=case["layout"], **more))
            return {"q": "q_out", "k": "k_out"}
        if case["op"] == "adapters":
            ops.adapters("x", base="base", a="a", b="b", ids="ids", scales="scales", out="y")
            return {"y": "y"}
        ops.sample("logits", uniforms="uniforms", out="tokens", logprobs="logprobs",
                   **{n: n for n in ("temperatures", "top_k", "top_p", "min_p") if n in inputs})
        return {"tokens": "tokens", "logprobs": "logprobs"}

    def run(self):
        self.runtime.run(self.env)
        return self.outputs


def prepare(case, seed):
    """The inputs; for the framework in its own buffers (the one memory its programs run on),
    with the compiled program."""
    inputs = _inputs(case, seed)
    if own:
        return _Program(case, inputs)
    if case["op"] == "rotary":  # what a program works out once
        inputs["frequencies"] = torch.tensor(_frequencies(case), dtype=torch.float64).cuda()
    return case, inputs


def run(state):
    if own:
        return state.run()
    case, t = state
    return {"pages": _pages, "rotary": _rotary, "adapters": _adapters, "sample": _sample}[case["op"]](case, **t)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _pages(case, pages, free, lengths, counts):
    p, rows = case["page_size"], case["tokens"]
    begin, count = lengths.long(), counts.long()
    end = begin + count
    have = (begin + p - 1) // p
    need = (end + p - 1) // p - have
    upto = need.cumsum(0)
    at = torch.arange(pages.shape[1], device=pages.device) - have[:, None]  # of a sequence's new pages
    new = (at >= 0) & (at < need[:, None])
    index = ((upto - need)[:, None] + at).clamp_(0, max(0, free.shape[0] - 1))
    pages.copy_(torch.where(new, free[index], pages))
    last = count.cumsum(0)
    row = torch.arange(rows, device=pages.device)
    owner = torch.searchsorted(last, row, right=True)
    live = owner < last.shape[0]
    owner = owner.clamp(max=last.shape[0] - 1)
    position = begin[owner] + row - (last - count)[owner]
    position = torch.where(live, position, 0)
    slot = pages[owner, position // p] * p + position % p
    return {"table": pages, "slots": torch.where(live, slot, -1).int(), "positions": torch.where(live, position, -1).int(),
            "ends": end.int(), "used": upto[-1:].int()}


def _rotary(case, q, k, positions, frequencies):
    angle = positions.double()[:, None] * frequencies
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    found = {}
    for name, x in (("q", q), ("k", k)):
        x = x.view(x.shape[0], -1, case["dim"])
        turned, rest = x[..., : case["part"]], x[..., case["part"] :]
        if case["layout"] == "half":
            one, two = turned.chunk(2, dim=-1)
            turned = torch.cat((one * cos - two * sin, two * cos + one * sin), dim=-1)
        else:
            one, two = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack((one * cos - two * sin, two * cos + one * sin), dim=-1).flatten(-2)
        found[name] = torch.cat((turned, rest), dim=-1).flatten(1)
    return found


def _adapters(case, x, base, a, b, ids, scales):
    m, n, k, r, s = case["rows"], case["cols"], case["inner"], case["rank"], case["held"]
    a, b = a.view(s, r, k), b.view(s, n, r)
    if m * r * (k + n) <= 2**26:  # few rows: each fetches its own
        at = ids.clamp(min=0).long()
        down = (a[at] * x[:, None]).sum(-1)
        more = (b[at] * down[:, None]).sum(-1) * scales[at][:, None]
        return {"y": base + torch.where(ids[:, None] >= 0, more, 0)}
    y = base.clone()
    for i in range(s):
        y += torch.where((ids == i)[:, None], x @ a[i].T @ b[i].T * scales[i], 0)
    return {"y": y}


def _sample(case, logits, uniforms, temperatures, top_k=None, top_p=None, min_p=None):
    cols = case["cols"]
    ordered, order = torch.sort(logits, dim=1, descending=True, stable=True)
    greedy = temperatures <= 0
    # in 64 bits: sums of many weights, next to the border that a random number draws
    t = torch.where(greedy, 1, temperatures).double()[:, None]
    w = torch.exp((ordered.double() - ordered[:, :1].double()) / t)
    kept = torch.ones_like(w, dtype=torch.bool)
    if top_k is not None:
        most = torch.where(top_k > 0, top_k, cols)
        kept &= torch.arange(cols, device=w.device) < most[:, None]
    if top_p is not None:
        live = torch.where(kept, w, 0)
        before = live.cumsum(1) - live
        p = top_p.double()[:, None]
        kept &= (p >= 1) | (before < p * live.sum(1, keepdim=True))
        kept[:, 0] = True
    if min_p is not None:
        kept &= w >= min_p.double()[:, None]
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0))  # by index again
    upto = w.cumsum(1)
    token = (upto > uniforms.double()[:, None] * upto[:, -1:]).int().argmax(1)
    drawn = torch.log(w.gather(1, token[:, None])[:, 0] / upto[:, -1])  # the probability that it was drawn with
    return {"tokens": torch.where(greedy, order[:, 0], token).int(), "logprobs": torch.where(greedy, 0, drawn).float()}


# ---------------------------------------------------------------------------
# what a pass needs, and what it should give
# ---------------------------------------------------------------------------


def work(case):
    """Inputs read once, outputs written once; 2 flops a multiply-add, one an elementwise
    operation."""
    if case["op"] == "pages":
        moved = 2 * sum(_pages_needed(case)) + 4 * case["sequences"] + 2 * case["tokens"] + 1
        return {"bytes": 4 * moved, "flops": 4 * (case["sequences"] + case["tokens"])}
    if case["op"] == "rotary":
        n = case["rows"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 8 * n * case["dim"] + 4 * case["rows"], "flops": 3 * n * case["part"]}
    if case["op"] == "adapters":
        ids = _ids(case)
        live = sum(ids[q] >= 0 for q in _row_request(case))
        weights = len({i for i in ids if i >= 0}) * case["rank"] * (case["inner"] + case["cols"])
        moved = live * case["inner"] + 2 * case["rows"] * case["cols"] + weights + case["rows"]
        return {"bytes": 4 * moved, "flops": 2 * live * case["rank"] * (case["inner"] + case["cols"])}
    n = case["rows"] * case["cols"]
    return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}


def exact(case, seed):
    """The outputs of ``run`` in 64 bits, from the definitions."""
    t = _inputs(case, seed)
    if case["op"] == "pages":
        p, table, free = case["page_size"], t["pages"].cpu().numpy(), t["free"].tolist()
        slots, positions, ends, used = [], [], [], 0
        for b, (begin, count) in enumerate(zip(t["lengths"].tolist(), t["counts"].tolist())):
            for at in range(begin, begin + count):
                if at % p == 0:
                    table[b, at // p] = free[used]
                    used += 1
                slots.append(int(table[b, at // p]) * p + at % p)
                positions.append(at)
            ends.append(begin + count)
        pad = [-1] * (case["tokens"] - len(slots))
        made = {"slots": slots + pad, "positions": positions + pad, "ends": ends, "used": [used]}
        return {"table": torch.from_numpy(table), **{n: torch.tensor(v, dtype=torch.int32) for n, v in made.items()}}
    if case["op"] == "rotary":
        f = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), t["positions"].double()[:, None] * f)[:, None]
        found = {}
        for name in ("q", "k"):
            x = t[name].view(case["rows"], -1, case["dim"]).double()
            y, h = x.clone(), case["part"] // 2
            one, two = (slice(0, h), slice(h, 2 * h)) if case["layout"] == "half" else (slice(0, 2 * h, 2), slice(1, 2 * h, 2))
            z = torch.complex(x[..., one], x[..., two]) * turn
            y[..., one], y[..., two] = z.real, z.imag
            found[name] = y.flatten(1)
        return found
    if case["op"] == "adapters":
        n, r = case["cols"], case["rank"]
        y = t["base"].double()
        ids = t["ids"].long()
        for i in range(case["held"]):
            rows = torch.nonzero(ids == i)[:, 0]
            if rows.numel():
                down = t["x"][rows].double() @ t["a"][i * r : (i + 1) * r].double().T
                y[rows] += t["scales"][i].double() * (down @ t["b"][i * n : (i + 1) * n].double().T)
        return {"y": y}
    tokens, logprobs = [], []
    for row in range(case["rows"]):
        x = t["logits"][row].double()
        temperature = float(t["temperatures"][row])
        top = float(x.max())
        if temperature <= 0:
            tokens.append(int(torch.nonzero(x == top)[0, 0]))
            logprobs.append(0.0)
            continue
        order = torch.argsort(-x, stable=True)
        if case["filters"] in ("all", "mixed", "top_k") and int(t["top_k"][row]) > 0:
            order = order[: int(t["top_k"][row])]
        w = torch.exp((x[order] - top) / temperature)
        if case["filters"] in ("all", "mixed", "top_p") and float(t["top_p"][row]) < 1:
            total = float(w.sum())
            n = 1 + int((w.cumsum(0) < float(t["top_p"][row]) * total).sum())
            order, w = order[:n], w[:n]
        if case["filters"] in ("all", "mixed", "min_p"):
            n = int((w >= float(t["min_p"][row])).sum())
            order, w = order[:n], w[:n]
        order, by = torch.sort(order)
        upto = w[by].cumsum(0)
        at = min(int((upto <= float(t["uniforms"][row]) * float(upto[-1])).sum()), order.numel() - 1)
        tokens.append(int(order[at]))
        logprobs.append((float(x[order[at]]) - top) / temperature - math.log(float(upto[-1])))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}
