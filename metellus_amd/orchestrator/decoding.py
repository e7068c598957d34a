"""The decoding ops: what a decode step does around its products and attention.

No counterpart in the reference.  Serving ops like those of
``orchestrator.serving`` (whole operators, a kernel each, tensors of other types
than fp32):

* ``PageTablesOp``  block tables, slots and positions of a step's tokens, in place
* ``RotaryOp``      queries and keys turned by their positions
* ``AdapterDownOp``, ``AdapterUpOp``
                    low-rank adapters of many requests, added to a shared product
* ``SampleScanOp``, ``SampleOp``
                    tokens from logits and given random numbers

``Rotary`` describes a rotation: which elements of a head are pairs, and their
angles.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from decimal import Decimal, localcontext

import numpy as np

from metellus_amd.orchestrator.ir import Tensor
from metellus_amd.orchestrator.serving import HEAD_DIM_MAX, _INT32_MAX, ServingOp, _dense, _rows, _want

ROTARY_LAYOUTS = ("half", "interleaved")
POSITIONS_MAX = _INT32_MAX - 1024  # of a table's row (its positions and a step's rows are int32)
ADAPTER_RANK_MAX = 256
VOCABULARY_MAX = 2**20
SAMPLE_CHUNK = 4096  # logits, and the smallest share of a workgroup
SAMPLE_BINS_FINE = 131072  # columns up to which there are 512 bins
SAMPLE_LIST = 7168  # logits that a row has listed at most

# pi to 64 digits: 2 pi has to outlast a double's 53 bits twice
_PI = Decimal("3.141592653589793238462643383279502884197169399375105820974944592")


@dataclass(frozen=True)
class Rotary:
    """The rotation of heads of ``dim``: the first ``part`` of its elements (all
    unless given) are pairs, (i, i + part / 2) in the ``half`` layout and
    (2 i, 2 i + 1) in the ``interleaved`` one; pair i turns by position times
    frequency i, base^(-2 i / part), and is then ``magnitude`` times as long.

    ``factor`` slows the frequencies down for contexts longer than a model was
    trained for: all of them alike, or, with the trained length ``original``, by
    parts: a pair that turns t = original * frequency / (2 pi) times within it keeps
    its frequency for t >= ``high``, has it divided by ``factor`` for t <= ``low``,
    and in between a mix, linear in t.  ``frequencies`` are taken as they are
    instead, for schedules other than these."""

    dim: int
    part: int | None = None
    base: float = 10000.0
    layout: str = "half"
    factor: float = 1.0
    original: int | None = None
    low: float = 1.0
    high: float = 32.0
    magnitude: float = 1.0
    frequencies: tuple[float, ...] | None = None

    def __post_init__(self) -> None:
        if self.part is None:
            object.__setattr__(self, "part", self.dim)
        for name in ("dim", "part"):
            v = getattr(self, name)
            if isinstance(v, bool) or not isinstance(v, (int, np.integer)) or v <= 0:
                raise ValueError(f"rotary: {name} must be a positive int; got {v!r}")
            object.__setattr__(self, name, int(v))
        for name in ("base", "factor", "low", "high", "magnitude"):
            v = getattr(self, name)
            try:
                if isinstance(v, (str, bytes)):
                    raise TypeError
                object.__setattr__(self, name, float(v))  # (in 64 bits, whatever numpy's type is)
            except (TypeError, ValueError, OverflowError):
                raise ValueError(f"rotary: {name} must be a number of 64 bits; got {v!r}") from None
        if self.dim > HEAD_DIM_MAX:
            raise ValueError(f"rotary: dim must be at most {HEAD_DIM_MAX}; got {self.dim}")
        if self.part % 2 or self.part > self.dim:
            raise ValueError(f"rotary: part must be even and at most dim = {self.dim}; got {self.part}")
        if self.layout not in ROTARY_LAYOUTS:
            raise ValueError(f"rotary: layout must be one of {ROTARY_LAYOUTS}; got {self.layout!r}")
        if not 1.0 <= self.base < math.inf:
            raise ValueError(f"rotary: base must be finite and at least 1; got {self.base}")
        if not 0.0 < self.factor < math.inf:
            raise ValueError(f"rotary: factor must be finite and above 0; got {self.factor}")
        if self.original is not None:
            if isinstance(self.original, bool) or not isinstance(self.original, (int, np.integer)) or self.original <= 0:
                raise ValueError(f"rotary: original must be a positive int; got {self.original!r}")
            object.__setattr__(self, "original", int(self.original))
            if not 0.0 <= self.low < self.high < math.inf:
                raise ValueError(f"rotary: low and high must be finite, 0 <= low < high; got {self.low} and {self.high}")
        if not 0.0 < self.magnitude <= 2.0**60:
            raise ValueError(f"rotary: magnitude must be above 0 and at most 2^60; got {self.magnitude}")
        if self.frequencies is not None:
            given = tuple(float(f) for f in self.frequencies)
            if len(given) != self.part // 2:
                raise ValueError(f"rotary: {self.part // 2} pairs need as many frequencies; got {len(given)}")
            object.__setattr__(self, "frequencies", given)
        if not all(abs(f) <= 2.0**20 for f in self.angles):
            raise ValueError("rotary: frequencies must be finite and within 2^20")

    @property
    def angles(self) -> tuple[float, ...]:
        """Radians that each pair turns for a step of position."""
        if self.frequencies is not None:
            return self.frequencies
        plain = [self.base ** (-2 * i / self.part) for i in range(self.part // 2)]
        if self.original is None:
            return tuple(f / self.factor for f in plain)
        made = []
        for f in plain:
            kept = (self.original * f / (2 * math.pi) - self.low) / (self.high - self.low)
            kept = min(1.0, max(0.0, kept))
            made.append((1 - kept) * f / self.factor + kept * f)
        return tuple(made)

    @property
    def turns(self) -> tuple[tuple[float, float], ...]:
        """``angles`` in whole turns, each as the sum of two doubles."""
        found = []
        with localcontext() as ctx:
            ctx.prec = 60
            for f in self.angles:
                t = Decimal(f) / (2 * _PI)
                head = float(t)
                found.append((head, float(t - Decimal(head))))
        return tuple(found)


ADAPTER_DOWN_WAVES = 4  # a workgroup's
ADAPTER_ORDER_ROWS = 128  # from here on rows of many adapters are put in order first


def adapter_many(rows: int, inner: int, cols: int, rank: int) -> bool:
    """Whether tiles have 64 rows, for which adapters are read less often, or 16, of which there
    are more workgroups.  (us, 64 and 16, ids of 8 prompts, and drawn from 64: rank 64, 1100 rows
    of 4096 x 4096 58 and 64, 110 and 86; 1500 58 and 73, 96 and 96; 2048 52 and 78, 73 and 89; 4096
    of 1024 x 1024 45 and 33, 52 and 41; 12000 of 256 x 256 41 and 37, 56 and 58; rank 16, 4096 of
    4096 x 4096 57 and 57, 64 and 67; 1500 36 and 34, 50 and 39.)"""
    return rows * min(inner, cols) * min(rank, 64) >= 5 << 26


def adapter_splits(rows: int, inner: int, many: bool) -> int:
    """Shares of x's columns that workgroups take apart, where rows alone are too few
    workgroups to fill the GPU: of 512 columns at least, and not so many that adding them
    up takes longer (us: 1 row of 4096 columns, rank 16, whole 17, in 4 9.4, 8 9.6; 32 rows 30,
    13.4, 12.3, in 16 12.8; 77 of 5003, rank 23, 37, 21, 18, 20; 8 of 11008, rank 64, in 8
    23, 12 20, 20 32; 600 of 4096, rank 64, in 3 49, 5 43, 6 43), or that some come after
    others (3000 rows of 4096 columns, rank 64: in 6 98, in 5 87).  Two workgroups of large tiles
    fit a compute unit, and take longer than one (4096 rows of 4096 columns, rank 64, in 4 and
    in 8: this kernel 32 and 41, the second, with twice the parts, 39 and 49)."""
    wanted = 256 // -(-rows // 64) if many else min(12, 3000 // rows)
    return max(1, min(-(-inner // 512), wanted))


# ---------------------------------------------------------------------------
# ops
# ---------------------------------------------------------------------------


def _list(label: str, t: Tensor, dtype: str, n: int | None = None) -> int:
    """A dense 1-D tensor of ``dtype``; its length."""
    if len(t.shape) != 1:
        raise ValueError(f"{label} must be 1D; got shape {t.shape} ({t.name!r})")
    _want(label, t, dtype, t.shape if n is None else (n,))
    _dense(label, t)
    return t.shape[0]


@dataclass(frozen=True)
class PageTablesOp(ServingOp):
    """With L = lengths clamped to the table's room, C = max(counts, 0) and E = L + C
    clamped to it (``ends``): sequence b has the first ceil(L / page_size) entries of
    its row of ``pages``, and gets those up to ceil(E / page_size) from ``free``, whose
    numbers go to the sequences in turn from the ``taken``-th on (the first, where not
    given or below 0), -1 behind its end.  ``used`` is ``taken`` and how many were needed,
    2^31 - 1 at the most.  Token rows are packed, C of each sequence after the other: the i-th of
    sequence b has position L + i and that position's slot; -1 for both beyond the
    room and behind the last sequence, and for a slot whose page is below 0."""

    written: Tensor
    slots: Tensor
    positions: Tensor
    ends: Tensor
    used: Tensor
    pages: Tensor
    free: Tensor
    lengths: Tensor
    counts: Tensor
    page_size: int
    taken: Tensor | None = None
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        if len(self.pages.shape) != 2:
            raise ValueError(f"page_tables pages must be 2D; got shape {self.pages.shape} ({self.pages.name!r})")
        _want("page_tables pages", self.pages, "int32", self.pages.shape)
        _dense("page_tables pages", self.pages)
        rows, width = self.pages.shape
        if isinstance(self.page_size, bool) or not isinstance(self.page_size, (int, np.integer)) or self.page_size <= 0:
            raise ValueError(f"page_tables page_size must be a positive int; got {self.page_size!r}")
        object.__setattr__(self, "page_size", int(self.page_size))  # (numpy's products wrap)
        if width * self.page_size > POSITIONS_MAX or rows * width > _INT32_MAX:
            raise ValueError(f"page_tables: {rows} rows of {width} pages of {self.page_size}; positions and entries are int32")
        _list("page_tables free", self.free, "int32")
        _list("page_tables lengths", self.lengths, "int32", rows)
        _list("page_tables counts", self.counts, "int32", rows)
        if self.taken is not None:
            _list("page_tables taken", self.taken, "int32", 1)

    @property
    def overwrites(self) -> Tensor:
        return self.pages

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return (self.written, self.slots, self.positions, self.ends, self.used)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.pages, self.free, self.lengths, self.counts, self.taken) if t is not None)


@dataclass(frozen=True)
class RotaryOp(ServingOp):
    """Row t of ``x`` (and of ``k``) by ``positions[t]``, every head alike."""

    y: Tensor
    x: Tensor
    positions: Tensor
    spec: Rotary
    k: Tensor | None = None
    k_out: Tensor | None = None
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows = 0
        for label, t in (("rotary x", self.x), ("rotary k", self.k)):
            if t is None:
                continue
            n, cols = _rows(label, t, "float32")
            if cols % self.spec.dim:
                raise ValueError(f"{label} must have whole heads of {self.spec.dim}; got shape {t.shape} ({t.name!r})")
            if rows and n != rows:
                raise ValueError(f"{label} must have {rows} rows; got shape {t.shape} ({t.name!r})")
            rows = n
        _list("rotary positions", self.positions, "int32", rows)
        if (self.k is None) != (self.k_out is None):
            raise ValueError("rotary: k and k_out go together")

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.y, self.k_out) if t is not None)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.x, self.k, self.positions) if t is not None)



@dataclass(frozen=True)
class AdapterDownOp(ServingOp):
    """Part s of ``down`` (``splits`` parts of x's rows): x[m] . A[ids[m]] over the
    s-th share of the columns, ranks in whole fours; rows whose id is no adapter's are not
    written."""

    down: Tensor
    x: Tensor
    a: Tensor
    ids: Tensor
    rank: int
    splits: int
    many: bool
    name: str  # of the operator's output
    order: Tensor | None = None  # the rows and their ids as they are taken in turn
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows, inner = _rows("adapters x", self.x, "float32")
        if len(self.a.shape) != 2 or self.a.shape[1] != inner or self.a.shape[0] % self.rank:
            raise ValueError(f"adapters a must have shape (adapters * {self.rank}, {inner}); got {self.a.shape} ({self.a.name!r})")
        _want("adapters a", self.a, "float32", self.a.shape)
        _dense("adapters a", self.a)
        _list("adapters ids", self.ids, "int32", rows)

    @property
    def held(self) -> int:
        return self.a.shape[0] // self.rank

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return (self.down,) if self.order is None else (self.down, self.order)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return (self.x, self.a, self.ids)


@dataclass(frozen=True)
class AdapterUpOp(ServingOp):
    """y[m] = base[m] + scales[ids[m]] * B[ids[m]] (the parts of down[m] added)."""

    y: Tensor
    base: Tensor
    down: Tensor
    b: Tensor
    ids: Tensor
    rank: int
    splits: int
    many: bool
    scales: Tensor | None = None
    order: Tensor | None = None
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows, cols = _rows("adapters base", self.base, "float32")
        held = self.b.shape[0] // cols
        _want("adapters b", self.b, "float32", (held * cols, self.rank))
        _dense("adapters b", self.b)
        _list("adapters ids", self.ids, "int32", rows)
        if self.scales is not None:
            _list("adapters scales", self.scales, "float32", held)

    @property
    def held(self) -> int:
        return self.b.shape[0] // self.base.shape[1]

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return (self.y,)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.base, self.down, self.b, self.ids, self.scales, self.order) if t is not None)


def sample_chunks(rows: int, cols: int) -> tuple[int, int]:
    """Logits of a chunk, and the chunks of a row: as many as make 512 workgroups of all
    rows, but at most 16, for each workgroup adds all of a row's bins up."""
    chunk = SAMPLE_CHUNK
    while cols > chunk and (rows * -(-cols // chunk) > 512 or cols > 16 * chunk):
        chunk *= 2
    return chunk, -(-cols // chunk)


def sample_bins(cols: int) -> int:
    """Bins of 32 temperatures: the finer, the shorter the lists of what is in one, and the
    longer adding them up takes (us a call with 512 and 1024: 64 rows of 131072 cut by k 30.4 and
    32.4, by p 45.1 and 44.3, filters mixed 40.6 and 40.0; one row by k 15.6 and 17.0, by p 20.0
    and 20.7)."""
    return 512 if cols <= SAMPLE_BINS_FINE else 1024 if cols <= 2 * SAMPLE_BINS_FINE else 2048


@dataclass(frozen=True)
class SampleScanOp(ServingOp):
    """The largest logit of each chunk (int64s, as two int32), and its bins for rows that
    ``top_k`` or ``top_p`` cut; the rows' counts of arrivals and listed logits are cleared."""

    best: Tensor
    counts: Tensor
    logits: Tensor
    name: str  # of the operator's output
    bins: Tensor | None = None
    temperatures: Tensor | None = None
    top_k: Tensor | None = None
    top_p: Tensor | None = None
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows, _ = _rows("sample logits", self.logits, "float32")
        for label, t, dtype in (("temperatures", self.temperatures, "float32"), ("top_k", self.top_k, "int32"),
                                ("top_p", self.top_p, "float32")):
            if t is not None:
                _list(f"sample {label}", t, dtype, rows)

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.best, self.counts, self.bins) if t is not None)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.logits, self.temperatures, self.top_k, self.top_p) if t is not None)


@dataclass(frozen=True)
class SampleOp(ServingOp):
    """For a row x with temperature T: w_i = exp((x_i - max x) / T).  In the order of
    x descending, the lower index first among equals: the first ``top_k`` stay; of
    those, the ones before which there is less than ``top_p`` of their weight; of
    those, the ones of weight ``min_p`` at least.  The token is the first index, in
    index order, up to which more than u times the weight that stayed has come by."""

    tokens: Tensor
    logits: Tensor
    uniforms: Tensor
    # what rows of several chunks have between the kernels and between workgroups
    best: Tensor | None = None
    counts: Tensor | None = None
    sums: Tensor | None = None
    bins: Tensor | None = None
    listed: Tensor | None = None
    logprobs: Tensor | None = None
    temperatures: Tensor | None = None
    top_k: Tensor | None = None
    top_p: Tensor | None = None
    min_p: Tensor | None = None
    after: tuple[Tensor, ...] = ()

    def __post_init__(self) -> None:
        rows, cols = _rows("sample logits", self.logits, "float32")
        if cols > VOCABULARY_MAX:
            raise ValueError(f"sample logits: at most {VOCABULARY_MAX} columns; got shape {self.logits.shape}")
        for label, t, dtype in (("uniforms", self.uniforms, "float32"), ("temperatures", self.temperatures, "float32"),
                                ("top_k", self.top_k, "int32"), ("top_p", self.top_p, "float32"),
                                ("min_p", self.min_p, "float32")):
            if t is not None:
                _list(f"sample {label}", t, dtype, rows)

    @property
    def outs(self) -> tuple[Tensor, ...]:
        return tuple(t for t in (self.tokens, self.logprobs, self.sums, self.listed) if t is not None)

    @property
    def reads(self) -> tuple[Tensor, ...]:
        return tuple(
            t
            for t in (self.logits, self.uniforms, self.temperatures, self.top_k, self.top_p, self.min_p, self.best, self.bins,
                      self.counts)
            if t is not None
        )
