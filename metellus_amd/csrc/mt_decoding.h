// mt_decoding.h -- device code of the decoding operators (gfx950): what a decode
// step does around its products and attention.  Follows mt_device.h and
// mt_serving.h in the kernels of these operators only; a generated kernel is one
// call of one function here.
//
//   * mt_page_tables    block tables, slots and positions of a step's tokens
//   * mt_rotary         queries and keys turned by their positions
//   * mt_adapter_down / mt_adapter_up
//                       low-rank adapters of many requests beside a shared product
//   * mt_sample_scan / mt_sample_pick
//                       tokens from logits and given random numbers

// ---------------------------------------------------------------------------
// Sums over lanes.
// ---------------------------------------------------------------------------

typedef unsigned long long mt_u64;

// The sum of v over this lane and those before it, by adding from one lane, two, four and
// eight before in rows of 16, then from the ends of the rows before.
template <int FROM, int ROWS>
MT_INLINE mt_u64 mt_from(mt_u64 v) {  // (0 where there is no such lane)
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, FROM, ROWS, 15, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), FROM, ROWS, 15, false);
    return ((mt_u64)hi << 32) | lo;
}
template <int FROM, int ROWS>
MT_INLINE mt_u64 mt_add_from(mt_u64 v) {
    return v + mt_from<FROM, ROWS>(v);
}
template <int FROM, int ROWS>
MT_INLINE mt_u64 mt_most_from(mt_u64 v) {
    const mt_u64 other = mt_from<FROM, ROWS>(v);
    return other > v ? other : v;
}
MT_INLINE mt_u64 mt_wave_upto(mt_u64 v) {
    v = mt_add_from<0x111, 15>(v);  // row_shr:1
    v = mt_add_from<0x112, 15>(v);
    v = mt_add_from<0x114, 15>(v);
    v = mt_add_from<0x118, 15>(v);
    v = mt_add_from<0x142, 10>(v);  // row_bcast:15 into rows 1 and 3
    return mt_add_from<0x143, 12>(v);  // row_bcast:31 into rows 2 and 3
}
// The last lane's word.
MT_INLINE mt_u64 mt_wave_last(mt_u64 v) {
    return ((mt_u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), 63) << 32) |
           (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, 63);
}
MT_INLINE mt_u64 mt_wave_sum(mt_u64 v) { return mt_wave_last(mt_wave_upto(v)); }

// The largest of a wave's, and of a workgroup's.
MT_INLINE mt_u64 mt_wave_most(mt_u64 v) {
    v = mt_most_from<0x112, 15>(mt_most_from<0x111, 15>(v));
    v = mt_most_from<0x118, 15>(mt_most_from<0x114, 15>(v));
    return mt_wave_last(mt_most_from<0x143, 12>(mt_most_from<0x142, 10>(v)));
}
template <unsigned WAVES>
MT_INLINE mt_u64 mt_group_most(mt_u64 v, mt_u64* lds) {
    v = mt_wave_most(v);
    __syncthreads();
    if (mt_lane() == 0u) lds[mt_wave()] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (unsigned w = 1; w < WAVES; ++w) v = lds[w] > v ? lds[w] : v;
    return v;
}

// The sum of v over the workgroup.
template <unsigned WAVES>
MT_INLINE mt_u64 mt_group_sum(mt_u64 v, mt_u64* lds) {
    v = mt_wave_sum(v);
    __syncthreads();
    if (mt_lane() == 0u) lds[mt_wave()] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (unsigned w = 0; w < WAVES; ++w) v += lds[w];
    return v;
}

// The sum of v over the lanes before this one; `all`: over all of them.
template <unsigned WAVES>
MT_INLINE mt_u64 mt_group_before(mt_u64 v, mt_u64* lds, mt_u64& all) {
    const mt_u64 sum = mt_wave_upto(v);
    __syncthreads();
    if (mt_lane() == 63u) lds[mt_wave()] = sum;
    __syncthreads();
    mt_u64 before = 0;
    all = 0;
#pragma unroll
    for (unsigned w = 0; w < WAVES; ++w) {
        before += w < mt_wave() ? lds[w] : 0;
        all += lds[w];
    }
    return before + sum - v;
}

// ---------------------------------------------------------------------------
// Block tables.  A sequence goes from `begin` positions to `end`: of its table's row it
// has `have` entries and needs `need` more.  Every workgroup adds up all sequences
// (8 bytes each), lane t the `each` sequences from t each on, and keeps the sums before
// each lane in LDS; a token row, or a new entry, finds its lane there and its sequence
// behind it.  So no workgroup waits for another, and the numbers do not depend on how
// many there are.  A launch reads entries below `have` alone and writes those from there
// on, so the table can be written in place.
// Bound by the latency of a launch and of loads in turn -- lengths, then a row's own -- of a few
// KB (32 sequences, a token each: kernel 3.2 us, call 4.9; 1021 sequences and 16384 tokens,
// 5.5 and 5.4).
// ---------------------------------------------------------------------------

// Sums of rows stop at 2^31 - 1, behind any row.
MT_INLINE unsigned mt_add_rows(unsigned a, unsigned b) {
    const unsigned sum = a + b;
    return sum > 0x7FFFFFFFu ? 0x7FFFFFFFu : sum;
}

template <unsigned P>
struct mt_growth {
    unsigned begin, end, rows, have, need;
    MT_INLINE mt_growth(int length, int count, unsigned room) {
        begin = length < 0 ? 0u : (unsigned)length < room ? (unsigned)length : room;
        rows = count < 0 ? 0u : (unsigned)count;
        end = begin + (rows < room - begin ? rows : room - begin);
        have = (begin + P - 1u) / P;
        need = (end + P - 1u) / P - have;
    }
};

// The last lane whose sum `before` is not above v.
template <unsigned LANES>
MT_INLINE unsigned mt_lane_of(const unsigned* before, unsigned v) {
    unsigned lo = 0u, hi = LANES;
#pragma unroll 1
    while (hi - lo > 1u) {
        const unsigned mid = (lo + hi) / 2u;
        if (before[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <unsigned P, unsigned LANES>
MT_INLINE void mt_page_tables(int* pages, const int* free, const int* taken, const int* lengths, const int* counts,
                              int* slots, int* positions, int* ends, int* used, unsigned rows, unsigned sequences,
                              unsigned width, unsigned frees, unsigned* lds) {
    constexpr unsigned WAVES = LANES / 64u;
    const unsigned gone = taken != nullptr && *taken > 0 ? (unsigned)*taken : 0u;  // (and the needed: below 2^32)
    unsigned *rows_before = lds, *need_before = lds + LANES + 1u, *sums = lds + 2u * (LANES + 1u);
    const unsigned t = threadIdx.x, room = width * P, each = (sequences + LANES - 1u) / LANES;
    const unsigned first = t * each < sequences ? t * each : sequences;
    const unsigned last = first + each < sequences ? first + each : sequences;
    unsigned made = 0u, need = 0u;
    for (unsigned b = first; b < last; ++b) {
        const mt_growth<P> s(lengths[b], counts[b], room);
        made = mt_add_rows(made, s.rows);
        need += s.need;
        if (blockIdx.x == 0u) ends[b] = (int)s.end;
    }
    // sums up to this lane
#pragma unroll
    for (unsigned off = 1u; off < 64u; off *= 2u) {
        const unsigned a = __shfl_up(made, off, 64), b = __shfl_up(need, off, 64);
        if (mt_lane() >= off) made = mt_add_rows(made, a), need += b;
    }
    if (mt_lane() == 63u) sums[mt_wave()] = made, sums[WAVES + mt_wave()] = need;
    __syncthreads();
    for (unsigned w = 0; w < mt_wave(); ++w) made = mt_add_rows(made, sums[w]), need += sums[WAVES + w];
    rows_before[t + 1u] = made, need_before[t + 1u] = need;
    if (t == 0u) rows_before[0] = 0u, need_before[0] = 0u;
    __syncthreads();

    const unsigned all_rows = rows_before[LANES], all_need = need_before[LANES], stride = gridDim.x * LANES;
    for (unsigned row = blockIdx.x * LANES + t; row < rows; row += stride) {
        int slot = -1, position = -1;
        if (row < all_rows) {
            const unsigned lane = mt_lane_of<LANES>(rows_before, row);
            unsigned b = lane * each, i = row - rows_before[lane], page = need_before[lane];
            mt_growth<P> s(lengths[b], counts[b], room);
            while (i >= s.rows) {
                i -= s.rows, page += s.need, ++b;
                s = mt_growth<P>(lengths[b], counts[b], room);
            }
            if (i < s.end - s.begin) {
                const unsigned at = s.begin + i, entry = at / P;
                position = (int)at;
                page += gone + entry - s.have;  // (where the entry is new)
                const int number = entry < s.have ? pages[(size_t)b * width + entry] : page < frees ? free[page] : -1;
                const long long found = (long long)number * P + at % P;
                if (number >= 0 && found <= 0x7FFFFFFFll) slot = (int)found;
            }
        }
        slots[row] = slot, positions[row] = position;
    }
    for (unsigned e = blockIdx.x * LANES + t; e < all_need; e += stride) {
        const unsigned lane = mt_lane_of<LANES>(need_before, e);
        unsigned b = lane * each, i = e - need_before[lane];
        mt_growth<P> s(lengths[b], counts[b], room);
        while (i >= s.need) {
            i -= s.need, ++b;
            s = mt_growth<P>(lengths[b], counts[b], room);
        }
        pages[(size_t)b * width + s.have + i] = gone + e < frees ? free[gone + e] : -1;
    }
    if (blockIdx.x == 0u && t == 0u) *used = (int)mt_add_rows(gone, all_need);
}

// ---------------------------------------------------------------------------
// Rotary positions: y1 = c x1 - s x2, y2 = c x2 + s x1 for the pairs of a head's first R
// elements, (i, i + R / 2) or, NEAR, (2 i, 2 i + 1); the others are copied.
//
// c and s belong to a position and a pair, and all heads share them: a workgroup works
// them out for its TOK rows once, in 64 bits, and keeps them in LDS in 32.  The angle is
// counted in turns, position times a turn's share per position, as the exact sum of two
// doubles, of which whole turns are taken away before anything is rounded to the size of
// the rest: an angle is right to 2^-51 of a turn at any int32 position.
// Bound by memory: every element is read and written once (8192 rows of 40 heads of 128 58 us,
// 5.8 TB/s, where a copy of 1 GiB has 5.1), or by the launch (a row 4.7 us, of which the kernel 2.2).
// ---------------------------------------------------------------------------

template <unsigned D, unsigned R, bool NEAR, unsigned V, unsigned XH, unsigned XRS, unsigned XCS, unsigned KH,
          unsigned KRS, unsigned KCS, unsigned TOK>
MT_INLINE void mt_rotary(const float* x, const float* k, const int* positions, const double (*turns)[2],
                         double magnitude, float* y, float* k_out, unsigned rows, mt_f32x2* lds) {
    constexpr unsigned HALF = R / 2u, LANES = 256u;
    // What a lane takes at once: V pairs of elements R / 2 apart, V / 2 (one at the least) of
    // neighbours, or V elements that stay.
    constexpr unsigned PAIRS = NEAR ? (V == 1u ? 1u : V / 2u) : V, TURNED = HALF / PAIRS, ITEMS = TURNED + (D - R) / V;
    const unsigned first = blockIdx.x * TOK;
    for (unsigned i = threadIdx.x; i < TOK * HALF; i += LANES) {
        const unsigned row = first + i / HALF, pair = i % HALF;
        if (row < rows) {
            const double at = (double)positions[row], turn = turns[pair][0];
            const double whole = at * turn, rest = __builtin_fma(at, turn, -whole) + at * turns[pair][1];
            double s, c;
            sincospi(2.0 * ((whole - __builtin_rint(whole)) + rest), &s, &c);
            lds[i] = mt_f32x2{(float)(c * magnitude), (float)(s * magnitude)};
        }
    }
    __syncthreads();
    for (unsigned at = threadIdx.x; at < TOK * (XH + KH) * ITEMS; at += LANES) {
        const unsigned item = at % ITEMS, head = at / ITEMS % (XH + KH), t = at / (ITEMS * (XH + KH)), row = first + t;
        if (row >= rows) break;  // (the rows of what follows are no smaller)
        const bool key = KH != 0u && head >= XH;
        const unsigned h = key ? head - XH : head;
        const float* from = key ? k + (size_t)row * KRS : x + (size_t)row * XRS;
        const size_t cs = key ? KCS : XCS;
        float* to = key ? k_out + ((size_t)row * KH + h) * D : y + ((size_t)row * XH + h) * D;
        const auto load = [&](unsigned e) {
            mt_f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if constexpr (V == 4u) v = mt_ld4u(from + h * D + e);
            else v[0] = from[(h * D + e) * cs];
            return v;
        };
        const auto store = [&](unsigned e, mt_f32x4 v) {
            if constexpr (V == 4u) __builtin_nontemporal_store(v, reinterpret_cast<mt_f32x4u*>(to + e));
            else to[e] = v[0];
        };
        if (item >= TURNED) {
            const unsigned e = R + (item - TURNED) * V;
            store(e, load(e));
            continue;
        }
        const mt_f32x2* cs_of = lds + t * HALF + item * PAIRS;
        if constexpr (!NEAR) {
            const unsigned e = item * V;
            const mt_f32x4 one = load(e), two = load(HALF + e);
            mt_f32x4 a = one, b = two;
#pragma unroll
            for (unsigned j = 0; j < V; ++j) {
                const mt_f32x2 w = cs_of[j];
                a[j] = __builtin_fmaf(one[j], w.x, -(two[j] * w.y));
                b[j] = __builtin_fmaf(two[j], w.x, one[j] * w.y);
            }
            store(e, a);
            store(HALF + e, b);
        } else if constexpr (V == 4u) {
            const mt_f32x4 v = load(4u * item);
            const mt_f32x2 w0 = cs_of[0], w1 = cs_of[1];
            store(4u * item, mt_f32x4{__builtin_fmaf(v[0], w0.x, -(v[1] * w0.y)), __builtin_fmaf(v[1], w0.x, v[0] * w0.y),
                                      __builtin_fmaf(v[2], w1.x, -(v[3] * w1.y)), __builtin_fmaf(v[3], w1.x, v[2] * w1.y)});
        } else {
            const float one = load(2u * item)[0], two = load(2u * item + 1u)[0];
            const mt_f32x2 w = cs_of[0];
            store(2u * item, mt_f32x4{__builtin_fmaf(one, w.x, -(two * w.y)), 0.f, 0.f, 0.f});
            store(2u * item + 1u, mt_f32x4{__builtin_fmaf(two, w.x, one * w.y), 0.f, 0.f, 0.f});
        }
    }
}

// ---------------------------------------------------------------------------
// Low-rank adapters: out[m] = base[m] + s[id] B[id] (A[id] x[m]), id = ids[m].
//
// Rows are taken in tiles of 16 MB.  Of a tile's, those with the same id are a group, led
// by its first row: a group reads its adapter once and multiplies all of the 16-row blocks
// that have rows of it (an MFMA's columns do not mix), of which it stores its own.  So a
// batch whose rows each have an adapter reads each of them once, and so does one whose rows
// share one.  TURNS workgroups take a tile's groups in turn, or with none a workgroup does the
// one that its row leads, if it does.
// fp32 MFMAs 16x16x4: with (n, g) = (lane % 16, lane / 16) a lane has 4 consecutive k of
// row n of both operands, k = 4 g + i in the i-th of four MFMAs; the order of k is the
// same for both, so the sum is the product's.  An element (row 4 g + i, column n) of the
// result is lane (n, g)'s i-th: rows are ranks, or columns of the output, so a lane has
// four neighbours of row m = n of `down` or `out`.
// Bound by two launches and the latency of loads in turn for few rows (us: 1 row of 4096 x
// 4096, rank 16, kernels 3.8 and 3.1, call 8.4; 32 rows of 4096 x 11008, an adapter each, 4.4 and
// 8.0, of which 29 MB take 5.7; 77 of 5003 x 4099, rank 23, 7.1 and 6.5); for
// prompts by MFMAs, half of their rate in the first kernel, and by base and out in the second
// (4096 rows of 4096 x 4096, rank 64: 32 and 43).
// ---------------------------------------------------------------------------

// Rows are put in order before they are cut into tiles, MT_ADAPTER_ORDERED at a time: by id
// (by a part of it: rows in one part stay as they are), and rows of an id in their own order,
// so that all workgroups find the same.  Where ids change less than twice a tile they stay as
// they are.  Each workgroup counts all of the rows' ids for itself and keeps the rows of its
// tile: rows[m], m < TILE, or nothing behind the last.  (us, rank 64 of 4096 x 4096, in
// the order they come in and in this: of 64 adapters in turn, shuffled, 150 rows 54, 45; 600 rows
// 211, 60; 2048 rows 560, 72; of 8 prompts 150 rows 20.7, 23.2; 600 rows 36.3, 37.7; 4096 rows 72, 74.)
// `lds`: WAVES words of sums, WAVES times BINS numbers, and a byte a row.
constexpr unsigned MT_ADAPTER_BINS = 256u, MT_ADAPTER_ORDERED = 4096u;
constexpr unsigned MT_ADAPTER_ROWS = 64u;  // words of LDS, in front of all others, for a tile's rows
template <unsigned TILE, unsigned WAVES>
MT_INLINE void mt_adapter_order(const int* ids, unsigned tile, unsigned all_rows, unsigned* rows, mt_u64* lds) {
    constexpr unsigned LANES = 64u * WAVES, BINS = MT_ADAPTER_BINS;
    static_assert(LANES == BINS, "a lane for each bin");
    unsigned* counts = reinterpret_cast<unsigned*>(lds + WAVES);
    unsigned char* keys = reinterpret_cast<unsigned char*>(counts + WAVES * BINS);
    const unsigned from = tile * TILE / MT_ADAPTER_ORDERED * MT_ADAPTER_ORDERED, begin = tile * TILE - from;
    const unsigned n = all_rows - from < MT_ADAPTER_ORDERED ? all_rows - from : MT_ADAPTER_ORDERED;
    const unsigned t = threadIdx.x, wave = mt_wave();
    constexpr unsigned EACH = MT_ADAPTER_ORDERED / LANES;
    unsigned id[EACH], last[EACH], changes = 0u;  // (all loaded before the first is looked at)
#pragma unroll
    for (unsigned e = 0; e < EACH; ++e) {
        id[e] = last[e] = 0u;
        if (e * LANES < n) {
            const unsigned i = e * LANES + t < n ? e * LANES + t : n - 1u;
            id[e] = (unsigned)ids[from + i], last[e] = (unsigned)ids[from + (i != 0u ? i - 1u : 0u)];
        }
    }
#pragma unroll
    for (unsigned e = 0; e < EACH; ++e)
        if (e * LANES + t < n) {
            changes += id[e] != last[e] ? 1u : 0u;
            keys[e * LANES + t] = (unsigned char)(id[e] % BINS);
        }
    for (unsigned c = t; c < WAVES * BINS; c += LANES) counts[c] = 0u;
    mt_u64 all;
    mt_group_before<WAVES>(changes, lds, all);
    if (all < 2u * ((n + TILE - 1u) / TILE)) {  // (the same in all workgroups)
        if (t < TILE) rows[t] = from + begin + t;
        __syncthreads();
        return;
    }
    // wave w counts the w-th share of the rows, and goes through it in order
    const unsigned share = (n + LANES - 1u) / LANES * 64u, first = wave * share, end = first + share < n ? first + share : n;
    for (unsigned i = first + mt_lane(); i < end; i += 64u) atomicAdd(counts + wave * BINS + keys[i], 1u);
    __syncthreads();
    unsigned number = 0u;
#pragma unroll
    for (unsigned w = 0; w < WAVES; ++w) number += counts[w * BINS + t];
    unsigned place = (unsigned)mt_group_before<WAVES>(number, lds, all);
#pragma unroll
    for (unsigned w = 0; w < WAVES; ++w) {
        const unsigned own = counts[w * BINS + t];
        counts[w * BINS + t] = place;
        place += own;
    }
    __syncthreads();
    for (unsigned i0 = first; i0 < end; i0 += 64u) {
        const unsigned i = i0 + mt_lane();
        const unsigned key = i < end ? keys[i] : 0u;
        mt_u64 alike = __ballot(i < end);
#pragma unroll
        for (unsigned bit = 1u; bit < BINS; bit *= 2u) {
            const mt_u64 has = __ballot((key & bit) != 0u);
            alike &= (key & bit) != 0u ? has : ~has;
        }
        const unsigned before = __builtin_amdgcn_mbcnt_hi((unsigned)(alike >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)alike, 0u));
        const unsigned base = counts[wave * BINS + key];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (i < end) {
            if (before == 0u) counts[wave * BINS + key] = base + (unsigned)__builtin_popcountll(alike);
            if (base + before - begin < TILE) rows[base + before - begin] = from + i;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
}

// The rows of a tile, and the groups that they lead.
template <unsigned MB, unsigned HELD, bool ORDER>
struct mt_adapter_rows {
    static constexpr unsigned TILE = 16u * MB;
    unsigned row0, mine;       // the tile's first row, the id of this lane's (-1: none, -2: no row)
    const unsigned* in_order;  // the rows, in LDS
    MT_INLINE mt_adapter_rows(unsigned tile, const unsigned* lds) : row0(tile * TILE), mine(0xFFFFFFFEu), in_order(lds) {}
    MT_INLINE void of(const int* ids, unsigned rows) {
        if (row0 + mt_lane() % TILE < rows) {
            const int found = ids[row(mt_lane() % TILE)];
            mine = found < 0 || (unsigned)found >= HELD ? 0xFFFFFFFFu : (unsigned)found;
        }
    }
    // The m-th row.
    MT_INLINE unsigned row(unsigned m) const { return ORDER ? in_order[m] : row0 + m; }
    // Of the tile's rows: bit m says whether row m is of the group that row j leads; 0 where
    // j leads none.
    MT_INLINE unsigned long long group(unsigned j, int& id) const {
        id = __builtin_amdgcn_readlane((int)mine, (int)j);
        const unsigned long long all = __ballot((int)mine == id) & (TILE == 64u ? ~0ull : (1ull << TILE) - 1ull);
        return id != -2 && (unsigned)__builtin_ctzll(all) == j ? all : 0ull;
    }
};

// A workgroup's tile and its share of the columns (blockIdx.x; blockIdx.y is the row of the
// tile that may lead, so that those of first rows, which all do, go first).  With turns the GPU's
// eight parts, which take workgroups in turn, have neighbouring tiles each, whose rows are
// likely to share adapters; there are eight times a whole number of tiles then, and the
// last may not be there.
template <bool LOOP>
struct mt_adapter_place {
    unsigned tile, share;
    MT_INLINE explicit mt_adapter_place(unsigned tiles) {
        const unsigned around = LOOP ? (tiles + 7u) / 8u * 8u : tiles, at = blockIdx.x % around;
        tile = LOOP ? at % 8u * (around / 8u) + at / 8u : at;
        share = blockIdx.x / around;
    }
};

// Elements c .. c + 3 of a row of COLS elements CS apart, 0 behind its end, without a branch.
// (MFMAs take all lanes' registers, whichever lanes are at them: lanes that may part on their
// way through a loop of MFMAs, at a condition of their own that the compiler knows from the
// round before, must not.)
template <unsigned COLS, unsigned CS, bool LOOP>
MT_INLINE mt_f32x4 mt_quad(const float* row, unsigned c) {
    mt_f32x4 v;
    if constexpr (LOOP) asm volatile("" : "+v"(c));  // (known to no other round; 77 rows, without: 15 us, with 17)
    if constexpr (CS == 1u && COLS >= 4u) {
        const unsigned at = c < COLS - 4u ? c : COLS - 4u, by = c - at;
        const mt_f32x4 w = mt_ld4u(row + at);
        if constexpr (COLS % 4u == 0u) {
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j) v[j] = by == 0u ? w[j] : 0.f;
        } else {
            v[0] = by == 0u ? w[0] : by == 1u ? w[1] : by == 2u ? w[2] : by == 3u ? w[3] : 0.f;
            v[1] = by == 0u ? w[1] : by == 1u ? w[2] : by == 2u ? w[3] : 0.f;
            v[2] = by == 0u ? w[2] : by == 1u ? w[3] : 0.f;
            v[3] = by == 0u ? w[3] : 0.f;
        }
    } else {
#pragma unroll
        for (unsigned j = 0; j < 4u; ++j) {
            const float one = row[(size_t)(c + j < COLS ? c + j : COLS - 1u) * CS];
            v[j] = c + j < COLS ? one : 0.f;
        }
    }
    return v;
}
// All four in the row.
template <unsigned CS>
MT_INLINE mt_f32x4 mt_quad_in(const float* row, unsigned c) {
    if constexpr (CS == 1u) return mt_ld4u(row + c);
    return mt_f32x4{row[(size_t)c * CS], row[(size_t)(c + 1u) * CS], row[(size_t)(c + 2u) * CS], row[(size_t)(c + 3u) * CS]};
}

// A row of `down`, in whole quads.
MT_INLINE constexpr unsigned mt_quads(unsigned ranks) { return (ranks + 3u) / 4u * 4u; }

// A's part: blocks of RB x 16 ranks; the waves of the SPLITS workgroups of a group take
// 64 columns of x in turn and add up in LDS; each split stores its part.  Loads of 16
// columns go out as the registers of those 64 before are free, so MFMAs and memory go on
// together.  Lanes of rows of other groups load the leader's, which are loaded anyway.
template <unsigned K, unsigned R, unsigned RB, unsigned MB, unsigned TURNS, bool ORDER, unsigned SPLITS, unsigned HELD,
          unsigned WAVES, unsigned XRS, unsigned XCS>
MT_INLINE void mt_adapter_down(const float* x, const float* a, const int* ids, float* down, int* order, unsigned rows,
                               mt_f32x4* lds) {
    constexpr bool LOOP = TURNS != 0u;
    constexpr unsigned TILE = 16u * MB, STEP = 64u * SPLITS * WAVES, WHOLE = K / 64u * 64u;
    // Sums that an MFMA does not wait for the one before with, added at the end: few tiles are
    // too few MFMAs to wait in turn (and shorter sums round less).
    constexpr unsigned SUMS = MB == 1u ? 4u : 1u;
    const unsigned tiles = (rows + TILE - 1u) / TILE, lane = mt_lane(), n = lane & 15u, g = lane >> 4;
    const mt_adapter_place<LOOP> at(tiles);
    const unsigned split = at.share % SPLITS, r0 = at.share / SPLITS * RB * 16u;
    if (at.tile >= tiles) return;
    unsigned* in_order = reinterpret_cast<unsigned*>(lds);
    if constexpr (ORDER) {
        lds += MT_ADAPTER_ROWS / 4u;
        mt_adapter_order<TILE, WAVES>(ids, at.tile, rows, in_order, reinterpret_cast<mt_u64*>(lds));
    }
    mt_adapter_rows<MB, HELD, ORDER> tile(at.tile, in_order);
    tile.of(ids, rows);
    if (ORDER && at.share == 0u && blockIdx.y == 0u && threadIdx.x < TILE && tile.row0 + lane < rows) {  // for the second kernel
        order[2u * (size_t)(tile.row0 + lane)] = (int)in_order[lane];
        order[2u * (size_t)(tile.row0 + lane) + 1u] = (int)tile.mine;
    }
#pragma unroll 1
    for (unsigned j = LOOP ? 0u : blockIdx.y, taken = 0u; j < TILE; ++j) {
        int id;
        const unsigned long long group = tile.group(j, id);
        if (group != 0ull && (TURNS <= 1u || taken++ % TURNS == blockIdx.y) && id >= 0) {
            const float *xr[MB], *ar[RB];
            mt_f32x4 acc[SUMS][MB][RB], xv[4][MB], av[4][RB];
#pragma unroll
            for (unsigned m = 0; m < MB; ++m) {
                const unsigned row = (group >> (16u * m + n)) & 1ull ? 16u * m + n : j;
                xr[m] = x + (size_t)tile.row(row) * XRS;
#pragma unroll
                for (unsigned b = 0; b < RB; ++b)
#pragma unroll
                    for (unsigned q = 0; q < SUMS; ++q) acc[q][m][b] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (unsigned b = 0; b < RB; ++b) {
                const unsigned r = r0 + 16u * b + n;
                ar[b] = a + ((size_t)(unsigned)id * R + (r < R ? r : R - 1u)) * K;
            }
            const auto load = [&](unsigned k0, unsigned u) {
                const unsigned k = k0 + 16u * u + 4u * g;
#pragma unroll
                for (unsigned m = 0; m < MB; ++m) xv[u][m] = mt_quad_in<XCS>(xr[m], k);
#pragma unroll
                for (unsigned b = 0; b < RB; ++b) av[u][b] = mt_quad_in<1u>(ar[b], k);
            };
            const auto multiply = [&](unsigned u) {
#pragma unroll
                for (unsigned m = 0; m < MB; ++m)
                    if (MB == 1u || ((group >> (16u * m)) & 0xFFFFull))  // (a block with rows of the group)
#pragma unroll
                        for (unsigned b = 0; b < RB; ++b)
#pragma unroll
                            for (unsigned i = 0; i < 4u; ++i)
                                acc[i % SUMS][m][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[u][b][i], xv[u][m][i],
                                                                                           acc[i % SUMS][m][b], 0, 0, 0);
            };
            unsigned k0 = 64u * (split * WAVES + mt_wave());
            if (k0 < WHOLE) {
#pragma unroll
                for (unsigned u = 0; u < 4u; ++u) load(k0, u);
#pragma unroll 1
                for (; k0 + STEP < WHOLE; k0 += STEP) {
#pragma unroll
                    for (unsigned u = 0; u < 4u; ++u) {
                        __builtin_amdgcn_sched_barrier(0);
                        multiply(u);
                        load(k0 + STEP, u);
                    }
                }
#pragma unroll
                for (unsigned u = 0; u < 4u; ++u) multiply(u);
            }
            if (WHOLE != K && WHOLE / 64u % (SPLITS * WAVES) == split * WAVES + mt_wave()) {  // the last columns
#pragma unroll
                for (unsigned u = 0; u < 4u; ++u) {
                    const unsigned k = WHOLE + 16u * u + 4u * g;
#pragma unroll
                    for (unsigned m = 0; m < MB; ++m) xv[u][m] = mt_quad<K, XCS, LOOP>(xr[m], k);
#pragma unroll
                    for (unsigned b = 0; b < RB; ++b) av[u][b] = mt_quad<K, 1u, LOOP>(ar[b], k);
                    multiply(u);
                }
            }
            if (LOOP) __syncthreads();  // (the group before has been added up)
#pragma unroll
            for (unsigned m = 0; m < MB; ++m)
#pragma unroll
                for (unsigned b = 0; b < RB; ++b) {
                    mt_f32x4 v = acc[0][m][b];
#pragma unroll
                    for (unsigned q = 1; q < SUMS; ++q) v = v + acc[q][m][b];
                    lds[((mt_wave() * MB + m) * RB + b) * 64u + lane] = v;
                }
            __syncthreads();
            for (unsigned e = threadIdx.x; e < MB * RB * 64u; e += WAVES * 64u) {
                mt_f32x4 v = lds[e];
#pragma unroll
                for (unsigned w = 1; w < WAVES; ++w) v = v + lds[w * MB * RB * 64u + e];
                const unsigned m = e / (64u * RB) * 16u + e % 16u, r = r0 + e / 64u % RB * 16u + e / 16u % 4u * 4u;
                if ((group >> m) & 1ull) {
                    // (nothing behind R: the last of A's rows stood in for those)
#pragma unroll
                    for (unsigned i = 1; i < 4u; ++i) v[i] = r + i < R ? v[i] : 0.f;
                    if (r < R) mt_st4(down + ((size_t)split * rows + tile.row(m)) * mt_quads(R) + r, v);
                }
            }
        }
        if (!LOOP) break;
    }
}

// B's part and the sum: the waves of a workgroup take BL blocks of 16 columns of the output
// in turn, PER times.  `down`'s parts are added up in LDS, once for all waves.  A block of 16
// rows goes through LDS on its way out, where rows become what lanes next to each other have:
// base is read and the output written 64 BL bytes of a row at a time, and by the four waves
// 256 BL (4096 rows of 4096, rank 64: 64 bytes of a row at a time 58 us).
template <unsigned N, unsigned R, unsigned MB, unsigned TURNS, bool ORDER, unsigned SPLITS, unsigned HELD, unsigned WAVES,
          unsigned PER, unsigned BL, unsigned YRS, unsigned YCS>
MT_INLINE void mt_adapter_up(const float* base, const float* down, const float* b, const int* ids, const int* order,
                             const float* scales, float* out, unsigned rows, float* lds) {
    constexpr bool LOOP = TURNS != 0u;
    constexpr unsigned RC = (R + 15u) / 16u, TILE = 16u * MB, PITCH = 16u * RC + 4u, WIDE = 16u * BL, OUT_PITCH = WIDE + 4u;
    constexpr unsigned ALONG = 4u * BL, ABREAST = 64u / ALONG;  // lanes along a row, and rows at a time
    const unsigned tiles = (rows + TILE - 1u) / TILE, lane = mt_lane(), n = lane & 15u, g = lane >> 4;
    const mt_adapter_place<LOOP> at(tiles);
    if (at.tile >= tiles) return;
    unsigned* in_order = reinterpret_cast<unsigned*>(lds);
    mt_adapter_rows<MB, HELD, ORDER> tile(at.tile, in_order);
    if constexpr (ORDER) {
        lds += MT_ADAPTER_ROWS;
        const unsigned m = lane % TILE;
        if (tile.row0 + m < rows) {
            const int* one = order + 2u * (size_t)(tile.row0 + m);
            tile.mine = (unsigned)one[1];
            if (threadIdx.x < TILE) in_order[m] = (unsigned)one[0];
        }
        __syncthreads();
    } else
        tile.of(ids, rows);
    float* turn = lds + TILE * PITCH + mt_wave() * 16u * OUT_PITCH;  // this wave's block of rows
#pragma unroll 1
    for (unsigned j = LOOP ? 0u : blockIdx.y, taken = 0u; j < TILE; ++j) {
        int id;
        const unsigned long long group = tile.group(j, id);
        if (group != 0ull && (TURNS <= 1u || taken++ % TURNS == blockIdx.y)) {
            mt_f32x4 bv[BL][RC], v[BL];
            const auto columns = [&](unsigned p) { return ((at.share * PER + p) * WAVES + mt_wave()) * WIDE; };
            const auto load = [&](unsigned from) {
                if (id < 0) return;
#pragma unroll
                for (unsigned q = 0; q < BL; ++q) {
                    const unsigned col = from + 16u * q + n;
                    const float* br = b + ((size_t)(unsigned)id * N + (col < N ? col : N - 1u)) * R;
#pragma unroll
                    for (unsigned c = 0; c < RC; ++c)
                        bv[q][c] = 16u * c + 16u <= R ? mt_quad_in<1u>(br, 16u * c + 4u * g) : mt_quad<R, 1u, LOOP>(br, 16u * c + 4u * g);
                }
            };
            // base's part of block m, as it goes out (rows of other groups: the leader's)
            const auto load_base = [&](unsigned from, unsigned m) {
                const unsigned col = from + 4u * (lane % ALONG);
#pragma unroll
                for (unsigned q = 0; q < BL; ++q) {
                    const unsigned row = 16u * m + q * ABREAST + lane / ALONG;
                    const float* yr = base + (size_t)tile.row((group >> row) & 1ull ? row : j) * YRS;
                    if (from + WIDE <= N) v[q] = mt_quad_in<YCS>(yr, col);
                    else v[q] = mt_quad<N, YCS, LOOP>(yr, col);
                }
            };
            if (columns(0u) < N) load(columns(0u));
            // the sums of down's parts; nothing for rows of other groups
            if (LOOP) __syncthreads();  // (the group before has been multiplied)
            for (unsigned e = threadIdx.x; e < TILE * RC * 4u; e += WAVES * 64u) {
                const unsigned m = e / (RC * 4u), r = e % (RC * 4u) * 4u;
                mt_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
                if (((group >> m) & 1ull) && id >= 0 && r < R) {
#pragma unroll
                    for (unsigned s = 0; s < SPLITS; ++s)
                        sum = sum + mt_ld4(down + ((size_t)s * rows + tile.row(m)) * mt_quads(R) + r);
                }
                *reinterpret_cast<mt_f32x4*>(lds + m * PITCH + r) = sum;
            }
            const float scale = scales != nullptr && id >= 0 ? scales[id] : 1.f;
            __syncthreads();
#pragma unroll 1
            for (unsigned p = 0; p < PER && columns(p) < N; ++p) {
                const unsigned from = columns(p);
                if (p != 0u) load(from);
#pragma unroll 1
                for (unsigned m = 0; m < MB; ++m) {
                    if (!((group >> (16u * m)) & 0xFFFFull)) continue;
                    load_base(from, m);
                    if (id >= 0) {
                        mt_f32x4 acc[BL];
#pragma unroll
                        for (unsigned q = 0; q < BL; ++q) acc[q] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (unsigned c = 0; c < RC; ++c) {
                            const mt_f32x4 t = *reinterpret_cast<const mt_f32x4*>(lds + (16u * m + n) * PITCH + 16u * c + 4u * g);
#pragma unroll
                            for (unsigned i = 0; i < 4u; ++i)
#pragma unroll
                                for (unsigned q = 0; q < BL; ++q)
                                    acc[q] = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[q][c][i], t[i], acc[q], 0, 0, 0);
                        }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the block before has been read)
#pragma unroll
                        for (unsigned q = 0; q < BL; ++q)
                            *reinterpret_cast<mt_f32x4*>(turn + n * OUT_PITCH + 16u * q + 4u * g) = acc[q];
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                        for (unsigned q = 0; q < BL; ++q) {
                            const mt_f32x4 sum = *reinterpret_cast<const mt_f32x4*>(
                                turn + (q * ABREAST + lane / ALONG) * OUT_PITCH + 4u * (lane % ALONG));
#pragma unroll
                            for (unsigned i = 0; i < 4u; ++i) v[q][i] = __builtin_fmaf(scale, sum[i], v[q][i]);
                        }
                    }
#pragma unroll
                    for (unsigned q = 0; q < BL; ++q) {
                        const unsigned row = 16u * m + q * ABREAST + lane / ALONG, col = from + 4u * (lane % ALONG);
                        unsigned stores = ((group >> row) & 1ull) && col < N;
                        asm volatile("" : "+v"(stores));  // (known to no other round)
                        if (stores) mt_put_row4<N>(out + (size_t)tile.row(row) * N, col, v[q]);
                    }
                }
            }
        }
        if (!LOOP) break;
    }
}

// ---------------------------------------------------------------------------
// Sampling.  w_i = exp((x_i - max) / T), worked out in 64 bits and held as a whole
// number of 2^-SHIFT: sums of whole numbers are the same in any order, so every cut and
// the token are too.  A weight is off by 2^-SHIFT-1 of the largest at most.
//
// A cut -- the k largest, or the largest that weigh p of all -- is where the amount (ones,
// or weights) that lies above a key first reaches what is asked for: it is looked for a
// byte of the key at a time, the amounts of the 256 values of a byte added up in LDS.
// Among equals at the cut the first indexes stay.
// ---------------------------------------------------------------------------

// A float's place in the order of floats; -0 is 0.
MT_INLINE unsigned mt_order_key(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
MT_INLINE float mt_order_value(unsigned key) {
    return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// e^z for z <= 0, right to about 2^-50 of itself; 0 below -700, and for a NaN.  z = n log 2 +
// r, and the series of e^r: for |r| up to log(2) / 2 its 13th term is under 2^-51.
MT_INLINE double mt_exp_below(double z) {
    const double n = __builtin_rint(z * 0x1.71547652b82fep+0);  // 1 / log 2
    const double r = __builtin_fma(n, -0x1.abc9e3b39803fp-56, __builtin_fma(n, -0x1.62e42fefa39efp-1, z));  // (log 2 in two parts)
    double e = 1.0 / 479001600.0;
    e = __builtin_fma(e, r, 1.0 / 39916800.0);
    e = __builtin_fma(e, r, 1.0 / 3628800.0);
    e = __builtin_fma(e, r, 1.0 / 362880.0);
    e = __builtin_fma(e, r, 1.0 / 40320.0);
    e = __builtin_fma(e, r, 1.0 / 5040.0);
    e = __builtin_fma(e, r, 1.0 / 720.0);
    e = __builtin_fma(e, r, 1.0 / 120.0);
    e = __builtin_fma(e, r, 1.0 / 24.0);
    e = __builtin_fma(e, r, 1.0 / 6.0);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    const bool some = z >= -700.0;
    // (e is 0.7 to 1.5: its exponent takes n as it is)
    const mt_u64 bits = __builtin_bit_cast(mt_u64, e) + ((mt_u64)(unsigned)(some ? (int)n : 0) << 52);
    return some ? __builtin_bit_cast(double, bits) : 0.0;
}

// 2^(l / 64) for the lanes l of a wave, for mt_weights.
constexpr unsigned MT_POWERS = 64u;
MT_INLINE double mt_power(unsigned l) { return 2.0 * mt_exp_below(0x1.62e42fefa39efp-7 * ((double)l - 64.0)); }

// The weights of a row.
template <unsigned SHIFT>
struct mt_weights {
    float top;
    double from;           // as `top`, and for +inf a number that +inf is above
    double by;             // one over the temperature
    const double* powers;  // 2^(l / 64), in LDS
    MT_INLINE mt_weights(float largest, float temperature, const double* lds)
        : top(largest), from(largest == INFINITY ? 1e308 : (double)largest), by(__builtin_fmax(1.0 / (double)temperature, 1e-300)),
          powers(lds) {}
    // (an x that is -inf weighs nothing, and beside a top of +inf so do all others, whatever
    // the temperature)
    MT_INLINE double scaled(float x) const { return __builtin_fmin(((double)x - from) * by, 0.0); }
    // e^z, z being x scaled, right to about 2^-50 of itself; nothing is a multiple of 2^-44
    // below e^-708.  z = n log(2) / 64 + r, and the series of e^r: for |r| up to log(2) / 128
    // its sixth term is under 2^-54.  (n is in the last bits of a sum with 1.5 2^52.  A series
    // alone, of twelve products in turn, took 60 % longer.)
    MT_INLINE double weight(float x) const {
        const double z = __builtin_fmax(scaled(x), -708.0);
        const double sum = __builtin_fma(z, 0x1.71547652b82fep+6, 0x1.8p52), n = sum - 0x1.8p52;
        const unsigned whole_n = (unsigned)__builtin_bit_cast(mt_u64, sum);
        const double power = powers[whole_n % MT_POWERS];
        const double r = __builtin_fma(n, -0x1.abc9e3b39803fp-62, __builtin_fma(n, -0x1.62e42fefa39efp-7, z));  // (log 2 in two parts)
        double e = __builtin_fma(1.0 / 120.0, r, 1.0 / 24.0);
        e = __builtin_fma(e, r, 1.0 / 6.0);
        e = __builtin_fma(e, r, 0.5);
        e = __builtin_fma(e, r, 1.0);
        e = __builtin_fma(e, r, 1.0) * power;
        // (e is 0.99 to 2: its exponent takes the rest of n as it is)
        return __builtin_bit_cast(double, __builtin_bit_cast(mt_u64, e) + ((mt_u64)((whole_n & ~(MT_POWERS - 1u)) << 14) << 32));
    }
    // The nearest whole number of 2^-SHIFT: in the last bits of a sum with 1.5 2^52.
    MT_INLINE static mt_u64 whole(double w) {
        const double sum = __builtin_fma(w, (double)(1ull << SHIFT), 0x1.8p52);
        return __builtin_bit_cast(mt_u64, sum) - __builtin_bit_cast(mt_u64, 0x1.8p52);
    }
    MT_INLINE mt_u64 held(float x) const { return whole(weight(x)); }
    // 0 for a weight below e^least, told by its logarithm: weights that differ by less than
    // they are rounded by still do.
    MT_INLINE mt_u64 kept(float x, double least) const {
        return scaled(x) < least ? 0 : whole(weight(x));
    }
    MT_INLINE static double log_of(mt_u64 total) { return log((double)total * (1.0 / (double)(1ull << SHIFT))); }
    MT_INLINE void answer(unsigned row, unsigned i, float x, double log_total, int* tokens, float* logprobs) const {
        tokens[row] = (int)i;
        if (logprobs != nullptr) logprobs[row] = (float)(scaled(x) - log_total);
    }
};

// A cut of a row: what stays lies above `key`, or is one of its equals up to index `last`.
struct mt_cut_at {
    unsigned key, last;
    MT_INLINE bool stays(unsigned k, unsigned i) const { return k > key || (k == key && i <= last); }
};

// each(f) calls f(index, x) for this lane's elements.  The cut where amount(index, x),
// added up from the largest x on, first reaches `asked` (1 at the least, all of it at the
// most); `above`: the amount above its key, `at`: of its equals.
template <unsigned WAVES, typename EACH, typename AMOUNT>
MT_INLINE unsigned mt_find_cut(EACH each, AMOUNT amount, mt_u64 asked, mt_u64& above, mt_u64& at, mt_u64* lds) {
    mt_u64* bins = lds + 2u * WAVES;
    unsigned key = 0u;
    above = 0;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256u) bins[threadIdx.x] = 0;
        __syncthreads();
        const unsigned known = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        each([&](unsigned i, float x) {
            const unsigned k = mt_order_key(x);
            if ((k & known) == key) {
                const mt_u64 v = amount(i, x);
                if (v != 0) atomicAdd(bins + ((k >> shift) & 255u), v);
            }
        });
        __syncthreads();
        // lane t: bin 255 - t, so that sums before it are of larger keys
        mt_u64 all;
        const mt_u64 mine = threadIdx.x < 256u ? bins[255u - threadIdx.x] : 0;
        const mt_u64 before = above + mt_group_before<WAVES>(mine, lds, all);
        if (threadIdx.x < 256u && before < asked && asked <= before + mine) {
            lds[WAVES] = 255u - threadIdx.x;
            lds[WAVES + 1u] = before;
            lds[WAVES + 2u] = mine;
        }
        __syncthreads();
        key |= (unsigned)lds[WAVES] << shift;
        above = lds[WAVES + 1u], at = lds[WAVES + 2u];
    }
    return key;
}

// A row's numbers.
struct mt_asked {
    float temperature, p, u;
    double least;  // a weight's logarithm
    int k;
    MT_INLINE mt_asked(unsigned row, const float* uniforms, const float* temperatures, const int* top_k, const float* top_p,
                       const float* min_p) {
        temperature = temperatures != nullptr ? temperatures[row] : 1.f;
        k = top_k != nullptr ? top_k[row] : 0;
        p = top_p != nullptr ? top_p[row] : 1.f;
        u = uniforms[row];
        const float m = min_p != nullptr ? min_p[row] : 0.f;
        least = m > 0.f ? log((double)__builtin_fminf(m, 1.f)) : -INFINITY;
        if (temperature == INFINITY) least = __builtin_fmin(least, -1e-200);  // (what is finite is scaled to less than that)
    }
    // The weight before which the largest stay, of `total`: the first always does.
    MT_INLINE mt_u64 weight_asked(mt_u64 total) const {
        const mt_u64 asked = p > 0.f ? (mt_u64)__builtin_ceil((double)p * (double)total) : 1;
        return asked < 1 ? 1 : asked < total ? asked : total;
    }
    // The weight before the token, of `total`.
    MT_INLINE mt_u64 target(mt_u64 total) const {
        const mt_u64 found = u > 0.f ? (mt_u64)((double)__builtin_fminf(u, 1.f) * (double)total) : 0;
        return found < total ? found : total - 1;
    }
};

// Where a cut falls among equals: of those equal to cut.key, which weigh or count `one` each
// and `at` together, those stay that it takes to reach what is asked for; nth(key, n) is the
// index of the n-th.
template <typename NTH>
MT_INLINE void mt_cut_equals(mt_cut_at& cut, mt_u64 asked, mt_u64 above, mt_u64 at, mt_u64 one, NTH nth) {
    const mt_u64 n = (asked - above + one - 1) / one;
    if (n < at / one) cut.last = nth(cut.key, n);
}

// The first of a row's largest, by key and index: larger is better, and nothing is above a NaN.
MT_INLINE mt_u64 mt_best(unsigned i, float v) {
    return v == v ? ((mt_u64)mt_order_key(v) << 32) | (0xFFFFFFFFu - i) : ~0ull;
}

// The answer for a row that has no choice; false for one that has.
MT_INLINE bool mt_sample_plain(mt_u64 best, float temperature, unsigned row, bool writes, int* tokens, float* logprobs) {
    const bool none = best == ~0ull || mt_order_value((unsigned)(best >> 32)) == -INFINITY;
    if (!none && temperature > 0.f) return false;
    if (writes) {
        tokens[row] = none ? -1 : (int)(0xFFFFFFFFu - (unsigned)best);
        if (logprobs != nullptr) logprobs[row] = none ? NAN : 0.f;
    }
    return true;
}

// One workgroup draws from a whole row, in as many passes over it as it takes: for rows
// that the two kernels below do not have in pieces small enough.
template <unsigned V, unsigned SHIFT, unsigned WAVES, unsigned CS>
MT_INLINE void mt_sample_whole(const float* x, const mt_asked& asked, const mt_weights<SHIFT>& weights, unsigned row,
                               int* tokens, float* logprobs, mt_u64* lds) {
    constexpr unsigned LANES = 64u * WAVES, STEP = 4u * LANES;
    const unsigned t = threadIdx.x;
    const auto each = [&](auto f) {
#pragma unroll 1
        for (unsigned c0 = 4u * t; c0 < V; c0 += 4u * STEP) {
            mt_f32x4 v[4];
#pragma unroll
            for (unsigned q = 0; q < 4u; ++q) {
                v[q] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
                if (c0 + q * STEP < V) v[q] = mt_row4<V, CS>(x, c0 + q * STEP);
            }
#pragma unroll
            for (unsigned q = 0; q < 4u; ++q)
#pragma unroll
                for (unsigned j = 0; j < 4u; ++j)
                    if (c0 + q * STEP + j < V) f(c0 + q * STEP + j, v[q][j]);
        }
    };
    // The index of the n-th of those equal to `key`, of which there are more.
    const auto nth = [&](unsigned key, mt_u64 n) {
        mt_u64 seen = 0;
#pragma unroll 1
        for (unsigned c0 = 0; c0 < V; c0 += STEP) {
            const unsigned c = c0 + 4u * t;
            unsigned hits = 0u;
            if (c < V) {
                const mt_f32x4 v = mt_row4<V, CS>(x, c);
#pragma unroll
                for (unsigned j = 0; j < 4u; ++j)
                    if (c + j < V && mt_order_key(v[j]) == key) hits |= 1u << j;
            }
            mt_u64 all, before = seen + mt_group_before<WAVES>(__builtin_popcount(hits), lds, all);
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j)
                if ((hits >> j) & 1u) {
                    if (++before == n) lds[WAVES] = c + j;
                }
            seen += all;
            if (seen >= n) break;  // (the same in all lanes)
        }
        __syncthreads();
        const unsigned found = (unsigned)lds[WAVES];
        __syncthreads();
        return found;
    };
    mt_cut_at cut{0u, 0xFFFFFFFFu};
    mt_u64 above, at;
    if (asked.k > 0 && (unsigned)asked.k < V) {
        cut.key = mt_find_cut<WAVES>(each, [](unsigned, float) { return (mt_u64)1; }, (mt_u64)asked.k, above, at, lds);
        mt_cut_equals(cut, (mt_u64)asked.k, above, at, 1, nth);
    }
    if (asked.p < 1.f) {
        const mt_cut_at by_k = cut;
        const auto amount = [&](unsigned i, float v) { return by_k.stays(mt_order_key(v), i) ? weights.held(v) : (mt_u64)0; };
        mt_u64 total = 0;
        each([&](unsigned i, float v) { total += amount(i, v); });
        total = mt_group_sum<WAVES>(total, lds);
        const mt_u64 wanted = asked.weight_asked(total);
        cut.key = mt_find_cut<WAVES>(each, amount, wanted, above, at, lds);
        if (cut.key != by_k.key) cut.last = 0xFFFFFFFFu;
        mt_cut_equals(cut, wanted, above, at, weights.held(mt_order_value(cut.key)), nth);
    }
    const auto amount = [&](unsigned i, float v) { return cut.stays(mt_order_key(v), i) ? weights.kept(v, asked.least) : (mt_u64)0; };
    mt_u64 total = 0;
    each([&](unsigned i, float v) { total += amount(i, v); });
    total = mt_group_sum<WAVES>(total, lds);
    const mt_u64 target = asked.target(total);
    const double log_total = weights.log_of(total);
    mt_u64 seen = 0;
#pragma unroll 1
    for (unsigned c0 = 0; c0 < V; c0 += STEP) {
        const unsigned c = c0 + 4u * t;
        mt_u64 w[4] = {0, 0, 0, 0};
        mt_f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (c < V) v = mt_row4<V, CS>(x, c);
#pragma unroll
        for (unsigned j = 0; j < 4u; ++j)
            if (c + j < V) w[j] = amount(c + j, v[j]);
        mt_u64 all, before = seen + mt_group_before<WAVES>(w[0] + w[1] + w[2] + w[3], lds, all);
#pragma unroll
        for (unsigned j = 0; j < 4u; ++j) {
            if (before <= target && target < before + w[j]) weights.answer(row, c + j, v[j], log_total, tokens, logprobs);
            before += w[j];
        }
        seen += all;
        if (seen > target) break;  // (the same in all lanes)
    }
}

// ---------------------------------------------------------------------------
// Two kernels draw from rows of which S chunks are in as many workgroups; of one chunk, the
// second alone, which does the first's part for itself.
//
// The first finds a chunk's largest and, for rows that k or p cut, counts its logits by how
// far below it they are: 512 bins of a sixteenth of the temperature, or more and finer ones
// of long rows, on a grid that all chunks share (bin f of x is floor(16 x / T)), each with its
// number of logits and about what they weigh.  What lies further below, 31.9 temperatures
// and more, weighs less than 2^-45 of the largest, and is 0 as it is held.
// The second adds the chunks' bins up, in every workgroup for itself, and so knows in which
// bin the cut is.  What lies above it stays, and is only added up; what lies in it -- or,
// where k and p both cut, everything from k's bin on, for p's cut depends on where k's is --
// is listed, in any order.  The last of a row's workgroups to arrive finds the cut in the
// list, adds what stays to the sums of the chunks, and looks through the chunk that the
// random number falls into.
// All of it counts with the same whole numbers as one workgroup alone, and what the bins
// say about weights, in 32 bits, is checked; rows that do not fit -- a list beyond LIST, a
// cut by p next to a bin's edge, logits so large that the grid has no bin for them -- are
// drawn from by one workgroup.
//
// The list takes half a compute unit's LDS, so there are two workgroups on each, of eight
// waves (us a call, eight waves in 512, 256 and 1024 workgroups, four in 512 and 1024: 64 rows of
// 131072 cut by p 45, 50, 59, 55, 67; cut by k 30, 33, 42, 34, 43; filters mixed 41, 48, 42, 51,
// 45; not cut 22, 22, 22, 23, 22; one row 17.5, 17.6, 17.6, 19.2, 19.0).
// Many rows are bound by what each does in turn, and a batch by its rows that p alone cuts, which
// take longest while the others' compute units are done (64 rows of 131072, us: the scan 9.6, with
// bins 11.6, of 6.5 to read them; the second kernel 15 with no cut, 19 by k, 36 by p, of
// which the pass over the logits takes 8, 2 and 16, and the last workgroup's list, from its
// arrival on, 3, 7 and 13; vector instructions are 6 of the 30 of mixed filters).  Few rows are
// bound by two launches and that list (one of 131072 5.3 and 12).
// ---------------------------------------------------------------------------

constexpr unsigned MT_SAMPLE_WAVES = 8u, MT_SAMPLE_LANES = 512u;
constexpr unsigned MT_SAMPLE_LIST = 7168u;
constexpr unsigned MT_SAMPLE_PARTS = 1024u;  // of a list's range, where its cut is looked for
constexpr unsigned MT_SAMPLE_CLOSE = 256u;   // logits that are compared one by one
constexpr unsigned MT_SAMPLE_SHORT = 128u;   // ... all of a list, for both cuts and the token
constexpr unsigned MT_SAMPLE_COUNT_AT = 43u;  // a bin's word: up to 2^20 logits from this bit on, 2^20 of their weights below

// The bin of x on the grid of a temperature, a thirty-second of the bins to each.
template <unsigned BINS>
struct mt_grid {
    float by;
    MT_INLINE explicit mt_grid(float temperature) : by((float)(BINS / 32u) / temperature) {}
    MT_INLINE float bin(float x) const { return __builtin_floorf(x * by); }
};

// Four logits from i on, -inf behind the row's end.
template <unsigned V, unsigned CS>
MT_INLINE mt_f32x4 mt_sample_quad(const float* x, unsigned i) {
    mt_f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (i < V) {
        v = mt_row4<V, CS>(x, i);
#pragma unroll
        for (unsigned j = 1; j < 4u; ++j)
            if (V % 4u != 0u && i + j >= V) v[j] = -INFINITY;
    }
    return v;
}

// Calls f(q, i, v) for this lane's quads of the chunk from i0 on, of which the q-th of all
// lanes are 2048 neighbours: i is the first one's index, v the four.  Four quads are loaded
// while the four before are looked at.
template <unsigned V, unsigned CHUNK, unsigned CS, typename F>
MT_INLINE void mt_sample_each(const float* x, unsigned i0, F f) {
    constexpr unsigned QUADS = CHUNK / (4u * MT_SAMPLE_LANES);
    constexpr unsigned DEEP = QUADS < 4u ? QUADS : 4u;
    static_assert(QUADS % DEEP == 0u, "whole sets of quads");
    const auto index = [&](unsigned q) { return i0 + 4u * (threadIdx.x + MT_SAMPLE_LANES * q); };
    const auto load = [&](unsigned q) { return mt_sample_quad<V, CS>(x, q < QUADS ? index(q) : V); };
    mt_f32x4 next[DEEP];
#pragma unroll
    for (unsigned q = 0; q < DEEP; ++q) next[q] = load(q);
#pragma unroll 1
    for (unsigned q0 = 0; q0 < QUADS; q0 += DEEP) {
        mt_f32x4 now[DEEP];
#pragma unroll
        for (unsigned q = 0; q < DEEP; ++q) now[q] = next[q], next[q] = load(q0 + DEEP + q);
#pragma unroll
        for (unsigned q = 0; q < DEEP; ++q) f(q0 + q, index(q0 + q), now[q]);
    }
}

// mt_sample_each as an object, called as often as its logits are looked at; the second has
// what a lane looks at in registers where that is eight quads or less, and loads them once.
template <unsigned V, unsigned CHUNK, unsigned CS>
struct mt_sample_again {
    const float* x;
    unsigned i0;
    template <typename F>
    MT_INLINE void operator()(F f) const { mt_sample_each<V, CHUNK, CS>(x, i0, f); }
};
template <unsigned V, unsigned CHUNK, unsigned CS>
struct mt_sample_kept {
    static constexpr unsigned QUADS = CHUNK / (4u * MT_SAMPLE_LANES);
    static constexpr bool KEEPS = QUADS <= 8u;
    const float* x;
    unsigned i0;
    mt_f32x4 held[KEEPS ? QUADS : 1u];
    MT_INLINE mt_sample_kept(const float* row, unsigned from) : x(row), i0(from) {
        if constexpr (KEEPS)
#pragma unroll
            for (unsigned q = 0; q < QUADS; ++q) held[q] = mt_sample_quad<V, CS>(x, index(q));
    }
    MT_INLINE unsigned index(unsigned q) const { return i0 + 4u * (threadIdx.x + MT_SAMPLE_LANES * q); }
    template <typename F>
    MT_INLINE void operator()(F f) const {
        if constexpr (KEEPS) {
#pragma unroll
            for (unsigned q = 0; q < QUADS; ++q) f(q, index(q), held[q]);
        } else
            mt_sample_each<V, CHUNK, CS>(x, i0, f);
    }
};

// The first of a chunk's largest, in all lanes.
template <unsigned V, typename EACH>
MT_INLINE mt_u64 mt_sample_best(EACH each, mt_u64* lds) {
    mt_u64 best = 0;
    each([&](unsigned, unsigned i, mt_f32x4 v) {
#pragma unroll
        for (unsigned j = 0; j < 4u; ++j) {
            const mt_u64 found = i + j < V ? mt_best(i + j, v[j]) : 0;
            best = found > best ? found : best;
        }
    });
    return mt_group_most<MT_SAMPLE_WAVES>(best, lds);
}

// A chunk's logits, and about what they weigh where asked, added to the bins in LDS, which are 0;
// `first`: the bin of its largest.
template <unsigned BINS, typename EACH>
MT_INLINE void mt_sample_count(EACH each, const mt_grid<BINS>& grid, float first, bool weigh, mt_u64* bins) {
    each([&](unsigned, unsigned, mt_f32x4 v) {
#pragma unroll
        for (unsigned j = 0; j < 4u; ++j) {
            const float f = grid.bin(v[j]), below = first - f;
            if (below >= 0.f && below < (float)BINS) {
                mt_u64 word = 1ull << MT_SAMPLE_COUNT_AT;
                if (weigh) word += (unsigned)(__builtin_amdgcn_exp2f((v[j] * grid.by - f) * (1.44269504f * 32.f / (float)BINS)) * 1048576.f);
                atomicAdd(bins + (unsigned)below, word);
            }
        }
    });
}

// best: [row][S]; bins: [row][S][BINS]; counts: [row][2], the row's arrivals and the length of
// its list.
template <unsigned V, unsigned CHUNK, unsigned S, unsigned BINS, unsigned RS, unsigned CS, bool CUT>
MT_INLINE void mt_sample_scan(const float* logits, const float* temperatures, const int* top_k, const float* top_p,
                              mt_u64* best_out, mt_u64* bins_out, unsigned* counts, mt_u64* lds) {
    constexpr unsigned LANES = MT_SAMPLE_LANES;
    const unsigned row = blockIdx.x / S, part = blockIdx.x % S, t = threadIdx.x;
    if (part == 0u && t < 2u) counts[2u * row + t] = 0u;
    const float* x = logits + (size_t)row * RS;
    mt_u64* bins = lds + MT_SAMPLE_WAVES;
    if (CUT)
        for (unsigned b = t; b < BINS; b += LANES) bins[b] = 0;
    const mt_sample_kept<V, CHUNK, CS> each(x, part * CHUNK);
    const mt_u64 best = mt_sample_best<V>(each, lds);
    if (t == 0u) best_out[(size_t)row * S + part] = best;
    if constexpr (CUT) {
        const float temperature = temperatures != nullptr ? temperatures[row] : 1.f;
        const bool by_p = top_p != nullptr && top_p[row] < 1.f, by_k = top_k != nullptr && top_k[row] > 0;
        if (!(temperature > 0.f) || !(by_p || by_k)) return;
        const mt_grid<BINS> grid(temperature);
        mt_sample_count(each, grid, grid.bin(mt_order_value((unsigned)(best >> 32))), by_p, bins);
        __syncthreads();
        for (unsigned b = t; b < BINS; b += LANES) bins_out[((size_t)row * S + part) * BINS + b] = bins[b];
    }
}

// The cut of a list: an entry is a key and, below it, the index upside down, so that larger
// is earlier, and no two are the same.  Where amount(entry), added up from the largest on,
// first reaches `asked`: up to 64 are compared one by one; of more, those in the cut's part of
// the list's range, whose parts place(entry) numbers from the largest on -- and while they
// are more than MT_SAMPLE_CLOSE, as with equal logits, those in the cut's part of the range
// from the least to the largest of them, ten bits of which that takes off.  False where the
// amounts are less than asked.  `lds`: results, MT_SAMPLE_PARTS and two times
// MT_SAMPLE_CLOSE words.
template <typename AMOUNT, typename PLACE>
MT_INLINE bool mt_list_cut(const mt_u64* list, unsigned n, AMOUNT amount, PLACE place, mt_u64 asked, mt_cut_at& cut,
                           mt_u64* lds) {
    constexpr unsigned WAVES = MT_SAMPLE_WAVES, LANES = MT_SAMPLE_LANES, EACH = MT_SAMPLE_PARTS / LANES;
    mt_u64 *found = lds + WAVES, *parts = found + 8u, *close = parts + MT_SAMPLE_PARTS, *weighs = close + MT_SAMPLE_CLOSE;
    const unsigned t = threadIdx.x;
    mt_u64 over = 0, least = 0, most = ~0ull;
    unsigned m = n;
    __syncthreads();
    if (t < 8u) found[t] = 0;
    if (n <= 64u) {
        if (t < n) close[t] = list[t], weighs[t] = amount(list[t]);
    } else {
#pragma unroll 1
        for (bool again = false;; again = true) {
            const unsigned bits = 64u - (unsigned)__builtin_clzll((most - least) | 1ull), shift = bits > 10u ? bits - 10u : 0u;
            const auto part = [&](mt_u64 e) { return again ? (unsigned)((most - e) >> shift) : place(e); };
            for (unsigned b = t; b < MT_SAMPLE_PARTS; b += LANES) parts[b] = 0;
            if (t < 8u) found[t] = t == 4u ? ~0ull : 0;
            __syncthreads();
            for (unsigned l = t; l < n; l += LANES) {
                const mt_u64 e = list[l];
                if (e >= least && e <= most) {
                    const mt_u64 w = amount(e);
                    if (w != 0) atomicAdd(parts + part(e), w);
                }
            }
            __syncthreads();
            mt_u64 mine[EACH], sum = 0, all;
#pragma unroll
            for (unsigned b = 0; b < EACH; ++b) mine[b] = parts[t * EACH + b], sum += mine[b];
            mt_u64 before = over + mt_group_before<WAVES>(sum, lds, all);
            if (over + all < asked) return false;  // (the same in all lanes)
#pragma unroll
            for (unsigned b = 0; b < EACH; ++b) {
                if (before < asked && asked <= before + mine[b]) found[0] = t * EACH + b, found[1] = before;
                before += mine[b];
            }
            __syncthreads();
            const unsigned at = (unsigned)found[0];
            over = found[1];
            for (unsigned l = t; l < n; l += LANES) {
                const mt_u64 e = list[l];
                if (e >= least && e <= most && part(e) == at) {
                    const unsigned to = (unsigned)atomicAdd(found + 2, 1ull);
                    if (to < MT_SAMPLE_CLOSE) close[to] = e, weighs[to] = amount(e);
                    atomicMin(found + 4, e);
                    atomicMax(found + 5, e);
                }
            }
            __syncthreads();
            m = (unsigned)found[2], least = found[4], most = found[5];
            if (m <= MT_SAMPLE_CLOSE) break;  // (at the latest with a part for each)
            __syncthreads();
        }
    }
    __syncthreads();
    if (t < m) {
        const mt_u64 own = close[t], weight = weighs[t];
        mt_u64 before = over;
#pragma unroll 8
        for (unsigned j = 0; j < m; ++j) {
            const mt_u64 other = close[j], more = weighs[j];  // (both loaded whatever the first is)
            before += other > own ? more : 0;
        }
        if (before < asked && asked <= before + weight) found[3] = own;
    }
    __syncthreads();
    cut.key = (unsigned)(found[3] >> 32), cut.last = 0xFFFFFFFFu - (unsigned)found[3];
    return found[3] != 0;
}

// A cut by k, one by p if asked, and the token, of a list of up to 128 that has everything
// that may stay: each entry is compared with all, a share of them by each of the lanes that
// have it, and the weights of those that are larger, or have an earlier index, are added up.
// `lds`: WAVES words, and twice 128.
template <unsigned SHIFT>
MT_INLINE void mt_sample_short(const mt_u64* list, unsigned n, const mt_asked& asked, const mt_weights<SHIFT>& weights,
                               unsigned row, int* tokens, float* logprobs, mt_u64* lds) {
    constexpr unsigned WAVES = MT_SAMPLE_WAVES, LANES = MT_SAMPLE_LANES, MOST = MT_SAMPLE_SHORT;
    const unsigned width = n <= 64u ? 64u : MOST, shares = LANES / width;
    const unsigned t = threadIdx.x, l = t % width, share = t / width;
    const unsigned begin = n * share / shares, end = n * (share + 1u) / shares;
    mt_u64 *sums = lds + WAVES, *amount = sums + MOST;
    const mt_u64 one = l < n ? list[l] : 0;
    const double w = weights.weight(mt_order_value((unsigned)(one >> 32)));
    // the sum of what more(entry, its amount) says of each entry
    const auto before = [&](auto more) {
        __syncthreads();
        if (t < MOST) sums[t] = 0;
        __syncthreads();
        mt_u64 sum = 0;
#pragma unroll 8
        for (unsigned j = begin; j < end; ++j) sum += more(list[j], amount[j]);
        atomicAdd(sums + l, sum);
        __syncthreads();
        return sums[l];
    };
    const mt_u64 rank = before([&](mt_u64 other, mt_u64) { return (mt_u64)(other > one ? 1 : 0); });
    mt_u64 weight = share == 0u && one != 0 && rank < (mt_u64)asked.k ? weights.whole(w) : 0;
    if (asked.p < 1.f) {
        if (share == 0u) amount[l] = weight;
        const mt_u64 wanted = asked.weight_asked(mt_group_sum<WAVES>(weight, lds));
        const mt_u64 larger = before([&](mt_u64 other, mt_u64 more) { return other > one ? more : 0; });
        if (!(larger < wanted)) weight = 0;
    }
    if (weights.scaled(mt_order_value((unsigned)(one >> 32))) < asked.least) weight = 0;
    __syncthreads();
    if (share == 0u) amount[l] = weight;
    const mt_u64 total = mt_group_sum<WAVES>(weight, lds), target = asked.target(total);
    const double log_total = weights.log_of(total);
    // (the index is upside down: larger is earlier)
    const mt_u64 earlier = before([&](mt_u64 other, mt_u64 more) { return (unsigned)other > (unsigned)one ? more : 0; });
    if (earlier <= target && target < earlier + weight)
        weights.answer(row, 0xFFFFFFFFu - (unsigned)one, mt_order_value((unsigned)(one >> 32)), log_total, tokens, logprobs);
}

// sums: [row][S][2], all weights and those above the cut, behind them for each row, the
// weights that stay of each segment of 256; list: [row][MT_SAMPLE_LIST].
template <unsigned V, unsigned CHUNK, unsigned S, unsigned BINS, unsigned SHIFT, unsigned RS, unsigned CS, bool CUT>
MT_INLINE void mt_sample_pick(const float* logits, const float* uniforms, const float* temperatures, const int* top_k,
                              const float* top_p, const float* min_p, const mt_u64* best_in, const mt_u64* bins_in,
                              unsigned* counts, mt_u64* sums, mt_u64* list, int* tokens, float* logprobs, mt_u64* lds) {
    constexpr unsigned LANES = MT_SAMPLE_LANES, WAVES = MT_SAMPLE_WAVES, EACH = BINS / LANES;
    constexpr unsigned SEGMENTS = CHUNK / 256u, ROW = 2u * S + S * SEGMENTS;  // a chunk's, and the words of a row's sums
    const unsigned row = blockIdx.x / S, part = blockIdx.x % S, t = threadIdx.x;
    const float* x = logits + (size_t)row * RS;
    const auto put = [](mt_u64* to, mt_u64 value) { __hip_atomic_store(to, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    const auto get = [](const mt_u64* from) {
        return __hip_atomic_load(const_cast<mt_u64*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    // LDS: powers, the folds' words and some results, four more, what stays of each segment; for cuts,
    // mt_list_cut's, and the list
    const double* powers = reinterpret_cast<const double*>(lds);
    if (t < MT_POWERS) lds[t] = __builtin_bit_cast(mt_u64, mt_power(t));  // (read behind the next barrier)
    lds += MT_POWERS;
    mt_u64 *words = lds + WAVES + 4u, *kept = words + 4u, *cut_lds = kept + S * SEGMENTS;
    mt_u64* held = cut_lds + WAVES + 8u + MT_SAMPLE_PARTS + 2u * MT_SAMPLE_CLOSE;
    const mt_asked asked(row, uniforms, temperatures, top_k, top_p, min_p);
    mt_u64 best = 0;
    if constexpr (S == 1u) {
        best = mt_sample_best<V>(mt_sample_again<V, CHUNK, CS>{x, 0u}, lds);
    } else {
        for (unsigned c = mt_lane(); c < S; c += 64u) {
            const mt_u64 one = best_in[(size_t)row * S + c];
            best = one > best ? one : best;
            if (CUT && t < 64u) kept[c] = one;
        }
        best = mt_wave_most(best);
    }
    if (mt_sample_plain(best, asked.temperature, row, part == 0u && t == 0u, tokens, logprobs)) return;
    const mt_weights<SHIFT> weights(mt_order_value((unsigned)(best >> 32)), asked.temperature, powers);
    const mt_grid<BINS> grid(asked.temperature);
    const float first = grid.bin(weights.top);

    // From which bin on logits are listed, and up to which: those above the first stay, those
    // below the last go.
    bool by_k = asked.k > 0 && (unsigned)asked.k < V, by_p = asked.p < 1.f, whole = false;
    unsigned from = BINS, upto = BINS;  // (none listed, all stay)
    mt_u64 above_k = 0;                                     // logits above `from`
    if (t < 4u) words[t] = 0;
    __syncthreads();
    if constexpr (CUT) {
        if (by_k || by_p) {
            // this lane's bins, EACH neighbours: their logits and weights, and those before them
            mt_u64 number[EACH], mass[EACH], numbers = 0, masses = 0;
#pragma unroll
            for (unsigned b = 0; b < EACH; ++b) number[b] = mass[b] = 0;
            if constexpr (S == 1u) {
                mt_u64* bins = held;  // (the list comes later)
                for (unsigned b = t; b < BINS; b += LANES) bins[b] = 0;
                __syncthreads();
                mt_sample_count(mt_sample_again<V, CHUNK, CS>{x, 0u}, grid, first, by_p, bins);
                __syncthreads();
#pragma unroll
                for (unsigned b = 0; b < EACH; ++b) {
                    const mt_u64 word = bins[t * EACH + b];
                    number[b] = word >> MT_SAMPLE_COUNT_AT, mass[b] = word & ((1ull << MT_SAMPLE_COUNT_AT) - 1ull);
                }
                __syncthreads();
            } else
#pragma unroll
            for (unsigned c = 0; c < S; ++c) {  // (loads that do not wait for each other)
                const float shift = first - grid.bin(mt_order_value((unsigned)(kept[c] >> 32)));
                const int by = shift >= 0.f && shift < (float)BINS ? (int)shift : (int)BINS;
#pragma unroll
                for (unsigned b = 0; b < EACH; ++b) {
                    const int at = (int)(t * EACH + b) - by;
                    const mt_u64 word = bins_in[((size_t)row * S + c) * BINS + (at < 0 ? 0 : at)];
                    number[b] += at < 0 ? 0 : word >> MT_SAMPLE_COUNT_AT;
                    mass[b] += at < 0 ? 0 : word & ((1ull << MT_SAMPLE_COUNT_AT) - 1ull);
                }
            }
#pragma unroll
            for (unsigned b = 0; b < EACH; ++b) {
                numbers += number[b];
                // in 2^-40 of the first bin's lower edge
                mass[b] = (mt_u64)((double)mass[b] * mt_exp_below(-32.0 / (double)BINS * (double)(t * EACH + b)) * 1048576.0);
                masses += mass[b];
            }
            mt_u64 *found = lds + WAVES, all;
            if (t == 0u) found[0] = found[1] = BINS;
            if (by_k) {
                mt_u64 before = mt_group_before<WAVES>(numbers, lds, all);
                const mt_u64 k = (mt_u64)asked.k;
#pragma unroll
                for (unsigned b = 0; b < EACH; ++b) {
                    if (before < k && k <= before + number[b]) found[0] = t * EACH + b, found[2] = before, found[3] = number[b];
                    before += number[b];
                }
                __syncthreads();
                upto = (unsigned)found[0];
                by_k = upto != BINS;  // (else what weighs anything stays)
                if (by_k) {
                    // (of few, all are listed: nothing else stays then)
                    const bool every = by_p || found[2] + found[3] <= MT_SAMPLE_SHORT;
                    from = every ? 0u : upto, above_k = every ? 0 : found[2];
                    whole = found[2] + found[3] - above_k > MT_SAMPLE_LIST;
                }
            }
            if (by_p && !by_k) {
                __syncthreads();
                mt_u64 before = mt_group_before<WAVES>(masses, lds, all);
                const mt_u64 wanted = asked.weight_asked(all);
#pragma unroll
                for (unsigned b = 0; b < EACH; ++b) {
                    if (before < wanted && wanted <= before + mass[b]) found[1] = t * EACH + b, found[3] = number[b];
                    before += mass[b];
                }
                __syncthreads();
                from = upto = (unsigned)found[1];
                whole = from == BINS || found[3] > MT_SAMPLE_LIST;
            }
            whole = whole || !(__builtin_fabsf(first) < 1048576.f);
            __syncthreads();
        }
    }
    if (whole && part != 0u) return;  // (the same in all workgroups of the row)
    const bool cuts = from < BINS;
    if (!whole) {
        mt_u64 all = 0, above = 0;
        const bool weigh_all = by_p && !by_k;
        // Logits of bins before `whole_from` stay as far as the bins say, those of bins before `weighed`
        // are weighed.  (NaN where nothing cuts, which no bin is at or behind, not the infinite and NaN
        // ones of logits off the grid either: all are weighed, the largest too, and a row's total is never 0.)
        const float whole_from = cuts ? (float)from : NAN, weighed = weigh_all ? INFINITY : whole_from;
        for (unsigned c = t; c < SEGMENTS; c += LANES) kept[c] = 0;
        __syncthreads();
        mt_sample_each<V, CHUNK, CS>(x, part * CHUNK, [&](unsigned q, unsigned i, mt_f32x4 v) {
            float below[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (CUT)
#pragma unroll
                for (unsigned j = 0; j < 4u; ++j) below[j] = first - grid.bin(v[j]);
            const float nearest = __builtin_fminf(__builtin_fminf(below[0], below[1]), __builtin_fminf(below[2], below[3]));
            mt_u64 stay = 0;
            if (!CUT || __ballot(!(nearest >= weighed)) != 0) {
#pragma unroll
                for (unsigned j = 0; j < 4u; ++j) {
                    const double w = weights.weight(v[j]);
                    const mt_u64 h = weights.whole(w);
                    const bool in = !CUT || !(below[j] >= whole_from);
                    all += h, above += in ? h : 0, stay += in && weights.scaled(v[j]) >= asked.least ? h : 0;
                }
            }
            if (CUT && cuts && __ballot(nearest <= (float)upto) != 0) {
                // one place in the list for all of the wave's, then each its own
                mt_u64 listed[4];
                unsigned number = 0u, to = 0u;
#pragma unroll
                for (unsigned j = 0; j < 4u; ++j) {
                    listed[j] = __ballot(below[j] >= (float)from && below[j] <= (float)upto);
                    number += (unsigned)__builtin_popcountll(listed[j]);
                }
                if (mt_lane() == 0u && number != 0u) to = atomicAdd((unsigned*)(words + 3), number);
                to = (unsigned)__builtin_amdgcn_readfirstlane((int)to);
#pragma unroll
                for (unsigned j = 0; j < 4u; ++j) {
                    const unsigned own = __builtin_amdgcn_mbcnt_hi((unsigned)(listed[j] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)listed[j], to));
                    if (below[j] >= (float)from && below[j] <= (float)upto && own < MT_SAMPLE_LIST) held[own] = mt_best(i + j, v[j]);
                    to += (unsigned)__builtin_popcountll(listed[j]);
                }
            }
            if (from != 0u) {  // (else nothing stays before the list is looked at)
                stay = mt_add_from<0x112, 15>(mt_add_from<0x111, 15>(stay));  // over four lanes
                unsigned to = q * WAVES + mt_wave();
                asm volatile("" : "+v"(to));  // (else lanes are added up one after another before the atomic)
                if ((mt_lane() & 3u) == 3u) atomicAdd(kept + to, stay);
            }
        });
        if (weigh_all) {
            all = mt_wave_sum(all), above = mt_wave_sum(above);
            if (mt_lane() == 0u) atomicAdd(words, all), atomicAdd(words + 1, above);
        }
        __syncthreads();
        unsigned n = (unsigned)words[3];  // (at most LIST, as the bins said)
        n = n < MT_SAMPLE_LIST ? n : MT_SAMPLE_LIST;
        mt_u64 row_all = words[0], row_above = words[1];
        if constexpr (S > 1u) {
            mt_u64 *of = sums + (size_t)row * ROW, *segments = of + 2u * S;
            if (weigh_all && t < 2u) put(of + 2u * part + t, words[t]);
            if (from != 0u)
                for (unsigned c = t; c < SEGMENTS; c += LANES) put(segments + part * SEGMENTS + c, kept[c]);
            if (CUT && n != 0u) {
                __syncthreads();
                if (t == 0u) words[3] = __hip_atomic_fetch_add(counts + 2u * row + 1u, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __syncthreads();
                for (unsigned l = t; l < n; l += LANES)
                    if ((unsigned)words[3] + l < MT_SAMPLE_LIST) put(list + (size_t)row * MT_SAMPLE_LIST + (unsigned)words[3] + l, held[l]);
            }
            __builtin_amdgcn_s_waitcnt(0);  // every lane's stores have reached memory
            __syncthreads();
            if (t == 0u) words[3] = __hip_atomic_fetch_add(counts + 2u * row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (words[3] + 1u != S) return;
            // the last workgroup of the row: what stays of each segment, and the list
            for (unsigned c = t; c < S * SEGMENTS; c += LANES) kept[c] = from != 0u ? get(segments + c) : 0;
            if (CUT && cuts) {
                n = __hip_atomic_load(counts + 2u * row + 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                n = n < MT_SAMPLE_LIST ? n : MT_SAMPLE_LIST;
                for (unsigned l = t; l < n; l += LANES) held[l] = get(list + (size_t)row * MT_SAMPLE_LIST + l);
                if (weigh_all) {
                    mt_u64 one_all = 0, one_above = 0;
                    for (unsigned c = mt_lane(); c < S; c += 64u) one_all += get(of + 2u * c), one_above += get(of + 2u * c + 1u);
                    row_all = mt_wave_sum(one_all), row_above = mt_wave_sum(one_above);
                }
            }
        }
        __syncthreads();
        if (CUT && by_k && from == 0u && n <= MT_SAMPLE_SHORT) {
            mt_sample_short<SHIFT>(held, n, asked, weights, row, tokens, logprobs, cut_lds);
            return;
        }
        mt_cut_at cut{0u, 0xFFFFFFFFu};
        if (CUT && cuts) {
            const auto value = [](mt_u64 one) { return mt_order_value((unsigned)(one >> 32)); };
            const auto stays = [&](mt_u64 one) { return cut.stays((unsigned)(one >> 32), 0xFFFFFFFFu - (unsigned)one); };
            // the part of bins `from` .. `upto` that a logit is in
            const float scale = (float)MT_SAMPLE_PARTS / (float)(upto - from + 1u), edge = first - (float)from + 1.f;
            const auto place = [&](mt_u64 one) {
                const float at = (edge - value(one) * grid.by) * scale;
                return at < 0.f ? 0u : at < (float)MT_SAMPLE_PARTS ? (unsigned)at : MT_SAMPLE_PARTS - 1u;
            };
            if (by_k)
                whole = !mt_list_cut(held, n, [](mt_u64) { return (mt_u64)1; }, place, (mt_u64)asked.k - above_k, cut, cut_lds);
            if (by_p && !whole) {
                if (by_k) {
                    mt_u64 total = 0;
                    for (unsigned l = t; l < n; l += LANES) total += stays(held[l]) ? weights.held(value(held[l])) : 0;
                    row_all = mt_group_sum<WAVES>(total, lds), row_above = 0;
                }
                const mt_u64 wanted = asked.weight_asked(row_all);
                const mt_cut_at by = cut;
                whole = wanted <= row_above ||
                        !mt_list_cut(held, n, [&](mt_u64 one) {
                            return by.stays((unsigned)(one >> 32), 0xFFFFFFFFu - (unsigned)one) ? weights.held(value(one)) : (mt_u64)0;
                        }, place, wanted - row_above, cut, cut_lds);
            }
            for (unsigned l = t; l < n; l += LANES)
                if (stays(held[l])) {
                    const mt_u64 h = weights.kept(value(held[l]), asked.least);
                    if (h != 0) atomicAdd(kept + (0xFFFFFFFFu - (unsigned)held[l]) / 256u, h);
                }
            __syncthreads();
        }
        if (!whole) {
            // The segment that the random number falls into, and the token in it.
            constexpr unsigned PER = (S * SEGMENTS + LANES - 1u) / LANES;
            mt_u64 mine = 0, total;
            for (unsigned c = t * PER; c < (t + 1u) * PER && c < S * SEGMENTS; ++c) mine += kept[c];
            mt_u64 before = mt_group_before<WAVES>(mine, lds, total);
            const mt_u64 target = asked.target(total);
            if (before <= target && target < before + mine) {
                unsigned c = t * PER;
                while (before + kept[c] <= target) before += kept[c++];
                words[0] = c, words[1] = before;
            }
            __syncthreads();
            if (t >= 64u) return;
            const unsigned i = (unsigned)words[0] * 256u + 4u * t;
            before = words[1];
            mt_f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (i < V) v = mt_row4<V, CS>(x, i);
            double log_total = weights.log_of(total);
            asm volatile("" : "+v"(log_total));  // (here, while the load is on its way)
            mt_u64 w[4];
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j)
                w[j] = i + j < V && cut.stays(mt_order_key(v[j]), i + j) ? weights.kept(v[j], asked.least) : 0;
            before += mt_wave_upto(w[0] + w[1] + w[2] + w[3]) - (w[0] + w[1] + w[2] + w[3]);
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j) {
                if (before <= target && target < before + w[j]) weights.answer(row, i + j, v[j], log_total, tokens, logprobs);
                before += w[j];
            }
            return;
        }
    }
    mt_sample_whole<V, SHIFT, WAVES, CS>(x, asked, weights, row, tokens, logprobs, lds);
}
