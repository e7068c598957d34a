// mt_decoding.h -- device code of the decoding operators (gfx950): what a decode
// step does around its products and attention.  Follows mt_device.h and
// mt_serving.h in the kernels of these operators only; a generated kernel is one
// call of one function here.
//
//   * mt_page_tables    block tables, slots and positions of a step's tokens
//   * mt_rotary         queries and keys turned by their positions
//   * mt_adapter_down / mt_adapter_up
//                       low-rank adapters of many requests beside a shared product
//   * mt_sample         tokens from logits and given random numbers

// ---------------------------------------------------------------------------
// Block tables.  A sequence goes from `begin` positions to `end`: of its table's row it
// has `have` entries and needs `need` more.  Every workgroup adds up all sequences
// (8 bytes each), lane t the `each` sequences from t each on, and keeps the sums before
// each lane in LDS; a token row, or a new entry, finds its lane there and its sequence
// behind it.  So no workgroup waits for another, and the numbers do not depend on how
// many there are.  A launch reads entries below `have` alone and writes those from there
// on, so the table can be written in place.
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
MT_INLINE void mt_page_tables(int* pages, const int* free, const int* lengths, const int* counts, int* slots,
                              int* positions, int* ends, int* used, unsigned rows, unsigned sequences, unsigned width,
                              unsigned frees, unsigned* lds) {
    constexpr unsigned WAVES = LANES / 64u;
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
                page += entry - s.have;  // (where the entry is new)
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
        pages[(size_t)b * width + s.have + i] = e < frees ? free[e] : -1;
    }
    if (blockIdx.x == 0u && t == 0u) *used = (int)all_need;
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
// share one.  LOOP: a workgroup does all groups of a tile, otherwise a workgroup does the
// one that its row leads, if it does.
// fp32 MFMAs 16x16x4: with (n, g) = (lane % 16, lane / 16) a lane has 4 consecutive k of
// row n of both operands, k = 4 g + i in the i-th of four MFMAs; the order of k is the
// same for both, so the sum is the product's.  An element (row 4 g + i, column n) of the
// result is lane (n, g)'s i-th: rows are ranks, or columns of the output, so a lane has
// four neighbours of row m = n of `down` or `out`.
// ---------------------------------------------------------------------------

// Tiles and the rows that lead their groups.  Workgroups in turn go to the GPU's eight
// parts in turn, so tiles, not leaders, are next to each other: few of a tile's rows lead.
template <unsigned MB, unsigned HELD>
struct mt_adapter_rows {
    static constexpr unsigned TILE = 16u * MB;
    unsigned row0, mine;  // the tile's first row, the id of this lane's (-1: none, -2: no row)
    MT_INLINE mt_adapter_rows(const int* ids, unsigned tile, unsigned rows) : row0(tile * TILE) {
        const unsigned row = row0 + mt_lane() % TILE;
        int found = -2;
        if (row < rows) {
            found = ids[row];
            if (found < 0 || (unsigned)found >= HELD) found = -1;
        }
        mine = (unsigned)found;
    }
    // Of the tile's rows: bit m says whether row m is of the group that row j leads; 0 where
    // j leads none.
    MT_INLINE unsigned long long group(unsigned j, int& id) const {
        id = __builtin_amdgcn_readlane((int)mine, (int)j);
        const unsigned long long all = __ballot((int)mine == id) & (TILE == 64u ? ~0ull : (1ull << TILE) - 1ull);
        return id != -2 && (unsigned)__builtin_ctzll(all) == j ? all : 0ull;
    }
};

MT_INLINE mt_f32x4 mt_mfma16_f32(mt_f32x4 a, mt_f32x4 b, mt_f32x4 c) {
#pragma unroll
    for (unsigned i = 0; i < 4u; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

// The tile of a workgroup.  LOOP: the GPU's eight parts, which take workgroups in turn, have
// neighbouring tiles each, whose rows are likely to share adapters; there are eight times
// a whole number of workgroups then, and the last may have no tile.
template <bool LOOP>
MT_INLINE unsigned mt_adapter_tile(unsigned tiles) {
    return LOOP ? blockIdx.x % 8u * (gridDim.x / 8u) + blockIdx.x / 8u : blockIdx.x % tiles;
}

// A's part: blocks of RB x 16 ranks; the waves of the SPLITS workgroups of a group take
// 64 columns of x in turn and add up in LDS; each split stores its part.  Loads of 16
// columns go out as the registers of those 64 before are free, so MFMAs and memory go on
// together.
template <unsigned K, unsigned R, unsigned RB, unsigned MB, bool LOOP, unsigned SPLITS, unsigned HELD, unsigned WAVES,
          unsigned XRS, unsigned XCS>
MT_INLINE void mt_adapter_down(const float* x, const float* a, const int* ids, float* down, unsigned rows,
                               mt_f32x4* lds) {
    constexpr unsigned TILE = 16u * MB;
    const unsigned tiles = (rows + TILE - 1u) / TILE, split = blockIdx.y % SPLITS, r0 = blockIdx.y / SPLITS * RB * 16u;
    const unsigned lane = mt_lane(), n = lane & 15u, g = lane >> 4, at = mt_adapter_tile<LOOP>(tiles);
    if (at >= tiles) return;
    const mt_adapter_rows<MB, HELD> tile(ids, at, rows);
#pragma unroll 1
    for (unsigned j = LOOP ? 0u : blockIdx.x / tiles; j < TILE; ++j) {
        int id;
        const unsigned long long group = tile.group(j, id);
        if (group != 0ull && id >= 0) {
            const float* ar = a + ((size_t)(unsigned)id * R + r0 + n) * K;
            mt_f32x4 acc[MB][RB], xv[4][MB], av[4][RB];
#pragma unroll
            for (unsigned m = 0; m < MB; ++m)
#pragma unroll
                for (unsigned b = 0; b < RB; ++b) acc[m][b] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
            const auto load = [&](unsigned k0, unsigned u) {
                const unsigned k = k0 + 16u * u + 4u * g;
#pragma unroll
                for (unsigned m = 0; m < MB; ++m) {
                    xv[u][m] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
                    if (((group >> (16u * m + n)) & 1ull) && (K % 64u == 0u || k < K))
                        xv[u][m] = mt_row4<K, XCS>(x + (size_t)(tile.row0 + 16u * m + n) * XRS, k);
                }
#pragma unroll
                for (unsigned b = 0; b < RB; ++b) {
                    av[u][b] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
                    if ((R % 16u == 0u && RB * 16u >= R || r0 + 16u * b + n < R) && (K % 64u == 0u || k < K))
                        av[u][b] = mt_row4<K, 1u>(ar + (size_t)(16u * b) * K, k);
                }
            };
            unsigned k0 = 64u * (split * WAVES + mt_wave());
            if (k0 < K) {
#pragma unroll
                for (unsigned u = 0; u < 4u; ++u) load(k0, u);
            }
            for (; k0 < K; k0 += 64u * SPLITS * WAVES) {
                const unsigned next = k0 + 64u * SPLITS * WAVES;
#pragma unroll
                for (unsigned u = 0; u < 4u; ++u) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (unsigned m = 0; m < MB; ++m)
                        if (MB == 1u || ((group >> (16u * m)) & 0xFFFFull))
#pragma unroll
                            for (unsigned b = 0; b < RB; ++b) acc[m][b] = mt_mfma16_f32(av[u][b], xv[u][m], acc[m][b]);
                    if (next < K) load(next, u);
                }
            }
            if (LOOP) __syncthreads();  // (the group before has been added up)
#pragma unroll
            for (unsigned m = 0; m < MB; ++m)
#pragma unroll
                for (unsigned b = 0; b < RB; ++b) lds[((mt_wave() * MB + m) * RB + b) * 64u + lane] = acc[m][b];
            __syncthreads();
            for (unsigned e = threadIdx.x; e < MB * RB * 64u; e += WAVES * 64u) {
                mt_f32x4 v = lds[e];
#pragma unroll
                for (unsigned w = 1; w < WAVES; ++w) v = v + lds[w * MB * RB * 64u + e];
                const unsigned m = e / (64u * RB) * 16u + e % 16u, r = r0 + e / 64u % RB * 16u + e / 16u % 4u * 4u;
                if ((group >> m) & 1ull) {
                    float* to = down + ((size_t)split * rows + tile.row0 + m) * R;
                    if (R % 4u == 0u) {
                        if (r < R) mt_st4(to + r, v);
                    } else {
#pragma unroll
                        for (unsigned i = 0; i < 4u; ++i)
                            if (r + i < R) to[r + i] = v[i];
                    }
                }
            }
        }
        if (!LOOP) break;
    }
}

// B's part and the sum: a wave takes PER blocks of 16 columns of the output, and loads
// AHEAD of them, of B and of base, before it needs them.  Tiles of several blocks of rows
// have `down`'s parts added up in LDS, once for all waves.
template <unsigned N, unsigned R, unsigned MB, bool LOOP, unsigned SPLITS, unsigned HELD, unsigned WAVES, unsigned PER,
          unsigned AHEAD, unsigned YRS, unsigned YCS>
MT_INLINE void mt_adapter_up(const float* base, const float* down, const float* b, const int* ids, const float* scales,
                             float* out, unsigned rows, float* lds) {
    constexpr unsigned RC = (R + 15u) / 16u, TILE = 16u * MB, PITCH = 16u * RC + 4u;
    static_assert(PER % AHEAD == 0u, "blocks in whole sets");
    const unsigned tiles = (rows + TILE - 1u) / TILE, lane = mt_lane(), n = lane & 15u, g = lane >> 4;
    const unsigned n0 = (blockIdx.y * WAVES + mt_wave()) * PER * 16u, at = mt_adapter_tile<LOOP>(tiles);
    if (at >= tiles) return;
    const mt_adapter_rows<MB, HELD> tile(ids, at, rows);
#pragma unroll 1
    for (unsigned j = LOOP ? 0u : blockIdx.x / tiles; j < TILE; ++j) {
        int id;
        const unsigned long long group = tile.group(j, id);
        if (group != 0ull) {
            mt_f32x4 bv[AHEAD][RC], v[AHEAD][MB], t[MB][RC];
            const auto load = [&](unsigned from, unsigned p) {
                const float* br = b + ((size_t)(unsigned)(id < 0 ? 0 : id) * N + from + n) * R;
#pragma unroll
                for (unsigned c = 0; c < RC; ++c) {
                    bv[p][c] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
                    if (id >= 0 && (N % 16u == 0u || from + n < N) && (R % 16u == 0u || 16u * c + 4u * g < R))
                        bv[p][c] = mt_row4<R, 1u>(br, 16u * c + 4u * g);
                }
                const unsigned col = from + 4u * g;
#pragma unroll
                for (unsigned m = 0; m < MB; ++m) {
                    v[p][m] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
                    if (((group >> (16u * m + n)) & 1ull) && (N % 16u == 0u || col < N))
                        v[p][m] = mt_row4<N, YCS>(base + (size_t)(tile.row0 + 16u * m + n) * YRS, col);
                }
            };
#pragma unroll
            for (unsigned p = 0; p < AHEAD; ++p)
                if (n0 + 16u * p < N) load(n0 + 16u * p, p);
            // the sums of down's parts; nothing for rows of other groups
            const auto parts = [&](unsigned m, unsigned r) {
                mt_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
                if (((group >> m) & 1ull) && id >= 0 && r < R) {
#pragma unroll
                    for (unsigned s = 0; s < SPLITS; ++s)
                        sum = sum + mt_row4<R, 1u>(down + ((size_t)s * rows + tile.row0 + m) * R, r);
                }
                return sum;
            };
            if constexpr (MB > 1u) {
                if (LOOP) __syncthreads();  // (the group before has been multiplied)
                for (unsigned e = threadIdx.x; e < TILE * RC * 4u; e += WAVES * 64u) {
                    const unsigned m = e / (RC * 4u), r = e % (RC * 4u) * 4u;
                    *reinterpret_cast<mt_f32x4*>(lds + m * PITCH + r) = parts(m, r);
                }
                __syncthreads();
            }
#pragma unroll
            for (unsigned m = 0; m < MB; ++m)
#pragma unroll
                for (unsigned c = 0; c < RC; ++c) {
                    if constexpr (MB > 1u) {
                        t[m][c] = *reinterpret_cast<const mt_f32x4*>(lds + (16u * m + n) * PITCH + 16u * c + 4u * g);
                    } else {
                        t[m][c] = parts(n, 16u * c + 4u * g);
                    }
                }
            const float scale = scales != nullptr && id >= 0 ? scales[id] : 1.f;
#pragma unroll 1
            for (unsigned p0 = 0; p0 < PER; p0 += AHEAD) {
#pragma unroll
                for (unsigned p = 0; p < AHEAD; ++p) {
                    const unsigned from = n0 + 16u * (p0 + p), col = from + 4u * g;
                    if (from >= N) break;
#pragma unroll
                    for (unsigned m = 0; m < MB; ++m) {
                        if (MB > 1u && !((group >> (16u * m)) & 0xFFFFull)) continue;
                        if (id >= 0) {
                            mt_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (unsigned c = 0; c < RC; ++c) acc = mt_mfma16_f32(bv[p][c], t[m][c], acc);
#pragma unroll
                            for (unsigned i = 0; i < 4u; ++i) v[p][m][i] = __builtin_fmaf(scale, acc[i], v[p][m][i]);
                        }
                        if (((group >> (16u * m + n)) & 1ull) && (N % 16u == 0u || col < N))
                            mt_put_row4<N>(out + (size_t)(tile.row0 + 16u * m + n) * N, col, v[p][m]);
                    }
                    if (p0 + p + AHEAD < PER && from + 16u * AHEAD < N) load(from + 16u * AHEAD, p);
                    __builtin_amdgcn_sched_barrier(0);
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

typedef unsigned long long mt_u64;

// A float's place in the order of floats; -0 is 0.
MT_INLINE unsigned mt_order_key(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
MT_INLINE float mt_order_value(unsigned key) {
    return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

template <typename OP>
MT_INLINE mt_u64 mt_wave_fold(mt_u64 v, OP op) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = op(v, (mt_u64)__shfl_xor(v, off, 64));
    return v;
}

// v (op) over the workgroup's waves; `lds` holds a word a wave.
template <unsigned WAVES, typename OP>
MT_INLINE mt_u64 mt_group_fold(mt_u64 v, mt_u64* lds, OP op) {
    v = mt_wave_fold(v, op);
    __syncthreads();
    if (mt_lane() == 0u) lds[mt_wave()] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (unsigned w = 1; w < WAVES; ++w) v = op(v, lds[w]);
    return v;
}

// The sum of v over the lanes before this one; `all`: over all of them.
template <unsigned WAVES>
MT_INLINE mt_u64 mt_group_before(mt_u64 v, mt_u64* lds, mt_u64& all) {
    mt_u64 sum = v;
#pragma unroll
    for (unsigned off = 1u; off < 64u; off *= 2u) {
        const mt_u64 other = __shfl_up(sum, off, 64);
        if (mt_lane() >= off) sum += other;
    }
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

// The weights of a row.
template <unsigned SHIFT>
struct mt_weights {
    float top;
    double by;  // the temperature
    MT_INLINE double scaled(float x) const { return ((double)x - (double)top) / by; }
    MT_INLINE double weight(float x) const {
        if (x == top) return 1.0;
        return x == -INFINITY || top == INFINITY ? 0.0 : exp(scaled(x));  // (whatever the temperature)
    }
    MT_INLINE static mt_u64 whole(double w) { return (mt_u64)__builtin_rint(w * (double)(1ull << SHIFT)); }
    MT_INLINE mt_u64 held(float x) const { return whole(weight(x)); }
    // 0 for a weight below `least`.
    MT_INLINE mt_u64 kept(float x, double least) const {
        const double w = weight(x);
        return w < least ? 0 : whole(w);
    }
    MT_INLINE void answer(unsigned row, unsigned i, float x, mt_u64 total, int* tokens, float* logprobs) const {
        tokens[row] = (int)i;
        if (logprobs != nullptr)
            logprobs[row] = (float)((x == top ? 0.0 : scaled(x)) - log((double)total / (double)(1ull << SHIFT)));
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
    double least;
    int k;
    MT_INLINE mt_asked(unsigned row, const float* uniforms, const float* temperatures, const int* top_k, const float* top_p,
                       const float* min_p) {
        temperature = temperatures != nullptr ? temperatures[row] : 1.f;
        k = top_k != nullptr ? top_k[row] : 0;
        p = top_p != nullptr ? top_p[row] : 1.f;
        u = uniforms[row];
        const float m = min_p != nullptr ? min_p[row] : 0.f;
        least = m > 0.f ? (double)__builtin_fminf(m, 1.f) : 0.0;
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
    const auto sum = [](mt_u64 a, mt_u64 b) { return a + b; };
    const auto each = [&](auto f) {
#pragma unroll 1
        for (unsigned c = 4u * t; c < V; c += STEP) {
            const mt_f32x4 v = mt_row4<V, CS>(x, c);
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j)
                if (c + j < V) f(c + j, v[j]);
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
        total = mt_group_fold<WAVES>(total, lds, sum);
        const mt_u64 wanted = asked.weight_asked(total);
        cut.key = mt_find_cut<WAVES>(each, amount, wanted, above, at, lds);
        if (cut.key != by_k.key) cut.last = 0xFFFFFFFFu;
        mt_cut_equals(cut, wanted, above, at, weights.held(mt_order_value(cut.key)), nth);
    }
    const auto amount = [&](unsigned i, float v) { return cut.stays(mt_order_key(v), i) ? weights.kept(v, asked.least) : (mt_u64)0; };
    mt_u64 total = 0;
    each([&](unsigned i, float v) { total += amount(i, v); });
    total = mt_group_fold<WAVES>(total, lds, sum);
    const mt_u64 target = asked.target(total);
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
            if (before <= target && target < before + w[j]) weights.answer(row, c + j, v[j], total, tokens, logprobs);
            before += w[j];
        }
        seen += all;
        if (seen > target) break;  // (the same in all lanes)
    }
}

// ---------------------------------------------------------------------------
// Two kernels draw from rows of which S chunks are in as many workgroups, PER neighbours to
// a lane.
//
// The first finds a chunk's largest and, for rows that k or p cut, counts its logits by how
// far below it they are: 512 bins of a sixteenth of the temperature, on a grid that all
// chunks share (bin f of x is floor(16 x / T)), each with its number of logits and about
// what they weigh.  What lies further below, 31.9 temperatures and more, weighs less than
// 2^-45 of the largest, and is 0 as it is held.
// The second adds the chunks' bins up, in every workgroup for itself, and so knows in which
// bin the cut is.  What lies above it stays, and is only added up; what lies in it -- or,
// where k and p both cut, everything from k's bin on, for p's cut depends on where k's is --
// is listed, in the order of the indexes.  The last of a row's workgroups to arrive finds
// the cut in the list, adds what stays to the sums of the chunks, and looks through the
// chunk that the random number falls into.
// All of it counts with the same whole numbers as one workgroup alone, and what the bins
// say about weights, in 32 bits, is checked; rows that do not fit -- a list beyond LIST, a
// bin that p's cut is next to, logits so large that a bin is none of theirs -- are drawn
// from by one workgroup.
// ---------------------------------------------------------------------------

constexpr unsigned MT_SAMPLE_BINS = 512u, MT_SAMPLE_LIST = 8192u;
constexpr unsigned MT_SAMPLE_COUNT_AT = 48u;  // a bin's word: its logits from this bit on, 2^20 of their weights below

// The bin of x on the grid of a temperature.
struct mt_grid {
    float by;
    MT_INLINE explicit mt_grid(float temperature) : by(16.0f / temperature) {}
    MT_INLINE float bin(float x) const { return __builtin_floorf(x * by); }
};

// This lane's PER logits of a chunk; -inf behind the row's end.
template <unsigned V, unsigned PER, unsigned CS>
MT_INLINE void mt_sample_load(const float* x, unsigned i0, float (&v)[PER]) {
#pragma unroll
    for (unsigned q = 0; q < PER; q += 4u) {
        mt_f32x4 four = {0.f, 0.f, 0.f, 0.f};
        if (i0 + q < V) four = mt_row4<V, CS>(x, i0 + q);
#pragma unroll
        for (unsigned j = 0; j < 4u; ++j) v[q + j] = i0 + q + j < V ? four[j] : -INFINITY;
    }
}

constexpr unsigned MT_SAMPLE_CLOSE = 256u;  // logits that are compared one by one

// The cut of a list of n logits: an entry is a key and, below it, the index upside down, so
// that larger is earlier; `amount`s, of which `asked` is at most the sum.  Up to 64 are
// compared one by one; of more, those that fall into the cut's part of 1024 even parts of
// the list's range of keys.  False where these are too many.
template <unsigned WAVES, unsigned DEEP>
MT_INLINE bool mt_list_cut(const mt_u64 (&entry)[DEEP], const mt_u64 (&amount)[DEEP], unsigned n, mt_u64 asked,
                           mt_cut_at& cut, mt_u64* lds) {
    constexpr unsigned LANES = 64u * WAVES;
    mt_u64 *bins = lds + 2u * WAVES, *close = bins + LANES, *close_amount = close + MT_SAMPLE_CLOSE;
    const unsigned t = threadIdx.x;
    mt_u64 over = 0;
    unsigned m = n;
    if (n <= 64u) {
        __syncthreads();
        if (t < n) close[t] = entry[0], close_amount[t] = amount[0];
    } else {
        // the largest key, and the least upside down
        mt_u64 span = 0;
        const auto both = [](mt_u64 a, mt_u64 b) {
            const mt_u64 low = 0xFFFFFFFFull, high = (a > b ? a : b) & ~low, x = a & low, y = b & low;
            return high | (x > y ? x : y);
        };
#pragma unroll
        for (unsigned d = 0; d < DEEP; ++d)
            if (amount[d] != 0) span = both(span, (entry[d] & ~0xFFFFFFFFull) | (0xFFFFFFFFull - (entry[d] >> 32)));
        span = mt_group_fold<WAVES>(span, lds, both);
        const unsigned top = (unsigned)(span >> 32), range = top - (0xFFFFFFFFu - (unsigned)span);
        const unsigned shift = range >= LANES ? 32u - __builtin_clz(range / LANES) : 0u;
        bins[t] = 0;
        if (t == 0u) lds[WAVES] = 0, lds[WAVES + 1u] = 0, lds[WAVES + 2u] = 0;
        __syncthreads();
#pragma unroll
        for (unsigned d = 0; d < DEEP; ++d)
            if (amount[d] != 0) atomicAdd(bins + ((top - (unsigned)(entry[d] >> 32)) >> shift), amount[d]);
        __syncthreads();
        mt_u64 all;
        const mt_u64 mine = bins[t], before = mt_group_before<WAVES>(mine, lds, all);
        if (before < asked && asked <= before + mine) lds[WAVES] = t, lds[WAVES + 1u] = before;
        __syncthreads();
        const unsigned bin = (unsigned)lds[WAVES];
        over = lds[WAVES + 1u];
#pragma unroll
        for (unsigned d = 0; d < DEEP; ++d)
            if (amount[d] != 0 && (top - (unsigned)(entry[d] >> 32)) >> shift == bin) {
                const unsigned at = (unsigned)atomicAdd(lds + WAVES + 2u, 1ull);
                if (at < MT_SAMPLE_CLOSE) close[at] = entry[d], close_amount[at] = amount[d];
            }
        __syncthreads();
        m = (unsigned)lds[WAVES + 2u];
        if (m > MT_SAMPLE_CLOSE) return false;  // (the same in all lanes)
    }
    __syncthreads();
    if (t < m) {
        const mt_u64 own = close[t], weighs = close_amount[t];
        mt_u64 before = over;
#pragma unroll 4
        for (unsigned j = 0; j < m; ++j) before += close[j] > own ? close_amount[j] : 0;
        if (before < asked && asked <= before + weighs) lds[WAVES + 3u] = own;
    }
    __syncthreads();
    cut.key = (unsigned)(lds[WAVES + 3u] >> 32), cut.last = 0xFFFFFFFFu - (unsigned)lds[WAVES + 3u];
    return true;
}

template <unsigned V, unsigned PER, unsigned S, unsigned WAVES, unsigned RS, unsigned CS, bool CUT>
MT_INLINE void mt_sample_scan(const float* logits, const float* temperatures, const int* top_k, const float* top_p,
                              mt_u64* best_out, mt_u64* bins_out, unsigned* arrivals, mt_u64* lds) {
    constexpr unsigned LANES = 64u * WAVES;
    const unsigned row = blockIdx.x / S, chunk = blockIdx.x % S, t = threadIdx.x, i0 = (chunk * LANES + t) * PER;
    if (chunk == 0u && t == 0u) arrivals[row] = 0u;
    float v[PER];
    mt_sample_load<V, PER, CS>(logits + (size_t)row * RS, i0, v);
    mt_u64* bins = lds + WAVES;
    if (CUT)
        for (unsigned b = t; b < MT_SAMPLE_BINS; b += LANES) bins[b] = 0;
    mt_u64 best = 0;
#pragma unroll
    for (unsigned e = 0; e < PER; ++e)
        if (i0 + e < V) {
            const mt_u64 found = mt_best(i0 + e, v[e]);
            best = found > best ? found : best;
        }
    best = mt_group_fold<WAVES>(best, lds, [](mt_u64 a, mt_u64 b) { return a > b ? a : b; });
    if (t == 0u) best_out[(size_t)row * S + chunk] = best;
    if constexpr (CUT) {
        const float temperature = temperatures != nullptr ? temperatures[row] : 1.f;
        const bool by_p = top_p != nullptr && top_p[row] < 1.f, by_k = top_k != nullptr && top_k[row] > 0;
        if (!(temperature > 0.f) || !(by_p || by_k)) return;
        const mt_grid grid(temperature);
        const float first = grid.bin(mt_order_value((unsigned)(best >> 32)));
#pragma unroll
        for (unsigned e = 0; e < PER; ++e) {
            const float f = grid.bin(v[e]), below = first - f;
            if (i0 + e < V && below >= 0.f && below < (float)MT_SAMPLE_BINS) {
                mt_u64 word = 1ull << MT_SAMPLE_COUNT_AT;
                if (by_p) word += (mt_u64)(__builtin_amdgcn_exp2f((v[e] * grid.by - f) * (1.44269504f / 16.f)) * 1048576.f);
                atomicAdd(bins + (unsigned)below, word);
            }
        }
        __syncthreads();
        for (unsigned b = t; b < MT_SAMPLE_BINS; b += LANES) bins_out[((size_t)row * S + chunk) * MT_SAMPLE_BINS + b] = bins[b];
    }
}

template <unsigned V, unsigned PER, unsigned S, unsigned SHIFT, unsigned WAVES, unsigned RS, unsigned CS, bool CUT>
MT_INLINE void mt_sample_pick(const float* logits, const float* uniforms, const float* temperatures, const int* top_k,
                              const float* top_p, const float* min_p, const mt_u64* best_in, const mt_u64* bins_in,
                              unsigned* arrivals, mt_u64* sums, mt_u64* list, int* tokens, float* logprobs, mt_u64* lds) {
    constexpr unsigned LANES = 64u * WAVES, ROOM = PER * LANES < MT_SAMPLE_LIST ? PER * LANES : MT_SAMPLE_LIST;
    constexpr unsigned DEEP = MT_SAMPLE_LIST / LANES;
    const unsigned row = blockIdx.x / S, chunk = blockIdx.x % S, t = threadIdx.x, i0 = (chunk * LANES + t) * PER;
    const float* x = logits + (size_t)row * RS;
    const auto sum = [](mt_u64 a, mt_u64 b) { return a + b; };
    const mt_asked asked(row, uniforms, temperatures, top_k, top_p, min_p);
    float v[PER];
    mt_sample_load<V, PER, CS>(x, i0, v);
    mt_u64 best = 0;
    for (unsigned c = mt_lane(); c < S; c += 64u) {
        const mt_u64 found = best_in[(size_t)row * S + c];
        best = found > best ? found : best;
    }
    best = mt_wave_fold(best, [](mt_u64 a, mt_u64 b) { return a > b ? a : b; });
    if (mt_sample_plain(best, asked.temperature, row, chunk == 0u && t == 0u, tokens, logprobs)) return;
    const mt_weights<SHIFT> weights{mt_order_value((unsigned)(best >> 32)), (double)asked.temperature};
    const mt_grid grid(asked.temperature);
    const float first = grid.bin(weights.top);

    // From which bin on logits are listed, and up to which: those above the first stay, those
    // below the last go.
    bool by_k = asked.k > 0 && (unsigned)asked.k < V, by_p = asked.p < 1.f, whole = false;
    unsigned from = MT_SAMPLE_BINS, upto = MT_SAMPLE_BINS;  // (none listed, all stay)
    mt_u64 above_k = 0;                                     // logits above `from`
    if constexpr (CUT) {
        if (by_k || by_p) {
            // lane t: bin t of the row, the sums up to it
            constexpr unsigned EACH = LANES / MT_SAMPLE_BINS;
            static_assert(EACH >= 1u && LANES % MT_SAMPLE_BINS == 0u, "a lane to a bin at the least");
            mt_u64 number = 0, mass = 0;
            const unsigned bin = t % MT_SAMPLE_BINS;
            for (unsigned c = t / MT_SAMPLE_BINS; c < S; c += EACH) {
                const float shift = first - grid.bin(mt_order_value((unsigned)(best_in[(size_t)row * S + c] >> 32)));
                if (shift >= 0.f && shift <= (float)bin) {
                    const mt_u64 word = bins_in[((size_t)row * S + c) * MT_SAMPLE_BINS + (bin - (unsigned)shift)];
                    number += word >> MT_SAMPLE_COUNT_AT, mass += word & ((1ull << MT_SAMPLE_COUNT_AT) - 1ull);
                }
            }
            if constexpr (EACH > 1u) {
                mt_u64* other = lds + 2u * WAVES;
                for (unsigned h = 1; h < EACH; ++h) {
                    __syncthreads();
                    if (t / MT_SAMPLE_BINS == h) other[2u * bin] = number, other[2u * bin + 1u] = mass;
                    __syncthreads();
                    if (t < MT_SAMPLE_BINS) number += other[2u * bin], mass += other[2u * bin + 1u];
                }
                if (t >= MT_SAMPLE_BINS) number = 0, mass = 0;
            }
            // weights of the bin in 2^-20 of the first bin's edge, as a whole number of 2^-40
            mass = (mt_u64)((double)mass * exp(-0.0625 * (double)bin) * 1048576.0);
            mt_u64 all_number, all_mass;
            const mt_u64 n0 = mt_group_before<WAVES>(number, lds, all_number), m0 = mt_group_before<WAVES>(mass, lds, all_mass);
            if (t == 0u) lds[WAVES] = MT_SAMPLE_BINS, lds[WAVES + 1u] = MT_SAMPLE_BINS, lds[WAVES + 2u] = 0, lds[WAVES + 3u] = 0;
            __syncthreads();
            const mt_u64 k = (mt_u64)asked.k;
            if (by_k && n0 < k && k <= n0 + number) lds[WAVES] = bin, lds[WAVES + 2u] = n0, lds[WAVES + 3u] = n0 + number;
            if (by_p) {
                const mt_u64 wanted = asked.weight_asked(all_mass);
                if (m0 < wanted && wanted <= m0 + mass) lds[WAVES + 1u] = bin, lds[WAVES + 4u] = number;
            }
            __syncthreads();
            const unsigned k_bin = (unsigned)lds[WAVES], p_bin = (unsigned)lds[WAVES + 1u];
            mt_u64 listed = 0;
            if (k_bin == MT_SAMPLE_BINS) by_k = false;  // (what weighs anything stays)
            if (by_k) {
                from = by_p ? 0u : k_bin, upto = k_bin;
                above_k = by_p ? 0 : lds[WAVES + 2u];
                listed = lds[WAVES + 3u] - above_k;
            } else if (by_p) {
                from = upto = p_bin;
                listed = lds[WAVES + 4u];
                whole = p_bin == MT_SAMPLE_BINS;
            }
            whole = whole || listed > MT_SAMPLE_LIST || !(__builtin_fabsf(first) < 1048576.f);
            __syncthreads();
        }
    }
    if (whole && chunk != 0u) return;  // (the same in all workgroups of the row)
    const bool cuts = from < MT_SAMPLE_BINS;
    if (!whole) {
        mt_u64 all = 0, above = 0, kept = 0;
        unsigned marks = 0u;  // which of this lane's are listed
#pragma unroll
        for (unsigned e = 0; e < PER; ++e) {
            if (i0 + e >= V) continue;
            bool stays = true;
            if (CUT && cuts) {
                const float below = first - grid.bin(v[e]);
                stays = below < (float)from;
                if (!stays && below <= (float)upto) marks |= 1u << e;
            }
            if (stays || (by_p && !by_k)) {
                const double w = weights.weight(v[e]);
                const mt_u64 h = weights.whole(w);
                all += h;
                if (stays) above += h, kept += w < asked.least ? 0 : h;
            }
        }
        mt_u64* mine = sums + ((size_t)row * S + chunk) * 4u;
        const auto put = [](mt_u64* to, mt_u64 value) { __hip_atomic_store(to, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        const auto get = [](const mt_u64* from_) {
            return __hip_atomic_load(const_cast<mt_u64*>(from_), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        mt_u64 listed = 0;
        if (CUT && cuts) {
            mt_u64 at = mt_group_before<WAVES>(__builtin_popcount(marks), lds, listed);
#pragma unroll
            for (unsigned e = 0; e < PER; ++e)
                if ((marks >> e) & 1u) {
                    if (at < ROOM) put(list + ((size_t)row * S + chunk) * ROOM + at, mt_best(i0 + e, v[e]));
                    ++at;
                }
        }
        if (CUT && by_p && !by_k) all = mt_group_fold<WAVES>(all, lds, sum), above = mt_group_fold<WAVES>(above, lds, sum);
        kept = mt_group_fold<WAVES>(kept, lds, sum);
        if (t == 0u) put(mine, all), put(mine + 1, above), put(mine + 2, kept), put(mine + 3, listed);
        if constexpr (S > 1u) {
            __builtin_amdgcn_s_waitcnt(0);  // every lane's stores have reached memory
            __syncthreads();
            if (t == 0u) lds[0] = __hip_atomic_fetch_add(arrivals + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (lds[0] + 1u != S) return;
        } else {
            __builtin_amdgcn_s_waitcnt(0);
        }
        __syncthreads();

        // The last workgroup of the row.  In LDS: what stays of each chunk, and where each
        // chunk's part of the list begins.
        mt_u64 *chunk_kept = lds + 2u * WAVES + LANES + 2u * MT_SAMPLE_CLOSE, *begins = chunk_kept + S;
        mt_u64 row_all = 0, row_above = 0;
        unsigned n = 0u;
        for (unsigned c = 0; c < S; c += 64u) {  // (each wave for itself)
            const bool live = c + mt_lane() < S;
            const mt_u64* at = sums + ((size_t)row * S + c + mt_lane()) * 4u;
            const mt_u64 part = live ? get(at + 3) : 0;
            if (CUT && by_p && !by_k) {
                row_all += mt_wave_fold(live ? get(at) : 0, sum);
                row_above += mt_wave_fold(live ? get(at + 1) : 0, sum);
            }
            mt_u64 before = part;
#pragma unroll
            for (unsigned off = 1u; off < 64u; off *= 2u) {
                const mt_u64 other = __shfl_up(before, off, 64);
                if (mt_lane() >= off) before += other;
            }
            if (live && t < 64u) begins[c + mt_lane()] = n + before - part, chunk_kept[c + mt_lane()] = get(at + 2);
            n += (unsigned)__shfl(before, 63, 64);
        }
        __syncthreads();
        mt_cut_at cut{0u, 0xFFFFFFFFu};
        if (CUT && cuts) {
            // lane t: entries t, t + LANES .. of the list, and what they count or weigh
            mt_u64 entry[DEEP], amount[DEEP];
#pragma unroll
            for (unsigned d = 0; d < DEEP; ++d) {
                const unsigned l = t + d * LANES;
                entry[d] = 0, amount[d] = 0;
                if (l < n) {
                    unsigned lo = 0u, hi = S;
                    while (hi - lo > 1u) {
                        const unsigned mid = (lo + hi) / 2u;
                        if (begins[mid] <= l) lo = mid;
                        else hi = mid;
                    }
                    entry[d] = get(list + ((size_t)row * S + lo) * ROOM + (l - (unsigned)begins[lo]));
                    amount[d] = 1;
                }
            }
            const auto stays = [&](mt_u64 one) { return cut.stays((unsigned)(one >> 32), 0xFFFFFFFFu - (unsigned)one); };
            if (by_k) whole = !mt_list_cut<WAVES>(entry, amount, n, (mt_u64)asked.k - above_k, cut, lds);
            mt_u64 total = 0;
            unsigned light = 0u;  // those below min_p
#pragma unroll
            for (unsigned d = 0; d < DEEP; ++d) {
                if (amount[d] != 0) {
                    const double w = weights.weight(mt_order_value((unsigned)(entry[d] >> 32)));
                    amount[d] = stays(entry[d]) ? weights.whole(w) : 0;
                    total += amount[d];
                    if (w < asked.least) light |= 1u << d;
                }
            }
            if (by_p && !whole) {
                total = mt_group_fold<WAVES>(total, lds, sum);
                const mt_u64 wanted = asked.weight_asked(by_k ? total : row_all);
                if (by_k || (row_above < wanted && wanted <= row_above + total))
                    whole = !mt_list_cut<WAVES>(entry, amount, n, wanted - row_above, cut, lds);
                else
                    whole = true;  // (next to a bin's edge)
            }
#pragma unroll
            for (unsigned d = 0; d < DEEP; ++d)
                if (amount[d] != 0 && !((light >> d) & 1u) && stays(entry[d]))
                    atomicAdd(chunk_kept + (0xFFFFFFFFu - (unsigned)entry[d]) / (PER * LANES), amount[d]);
            __syncthreads();
        }
        if (!whole) {
            // The chunk that the random number falls into, and the token in it.
            mt_u64 total = 0;
            for (unsigned c = 0; c < S; ++c) total += chunk_kept[c];
            const mt_u64 target = asked.target(total);
            mt_u64 before = 0;
            unsigned in = 0u;
            while (in + 1u < S && before + chunk_kept[in] <= target) before += chunk_kept[in], ++in;
            const unsigned k0 = (in * LANES + t) * PER;
            mt_sample_load<V, PER, CS>(x, k0, v);
            mt_u64 w[PER], lane_all = 0, every;
#pragma unroll
            for (unsigned e = 0; e < PER; ++e) {
                w[e] = k0 + e < V && cut.stays(mt_order_key(v[e]), k0 + e) ? weights.kept(v[e], asked.least) : 0;
                lane_all += w[e];
            }
            before += mt_group_before<WAVES>(lane_all, lds, every);
#pragma unroll
            for (unsigned e = 0; e < PER; ++e) {
                if (before <= target && target < before + w[e]) weights.answer(row, k0 + e, v[e], total, tokens, logprobs);
                before += w[e];
            }
            return;
        }
    }
    mt_sample_whole<V, SHIFT, WAVES, CS>(x, asked, weights, row, tokens, logprobs, lds);
}
