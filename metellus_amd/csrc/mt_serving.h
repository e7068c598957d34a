// mt_serving.h -- device code of the serving operators (gfx950): one decode
// step of a model with a paged cache.  Follows mt_device.h in the kernels of
// these operators only; a generated kernel is one call of one function here.
//
//   * mt_rms_norm          residual addition, RMS norm, output in 32 or 8 bits
//   * mt_dequantize        rows of 8 bits back to 32
//   * mt_cache_write/read  rows of keys and values into the paged cache and back
//   * mt_paged_attention   one new token per sequence over that cache
//   * mt_matmul_int4       few rows against 4-bit weights with group scales
//
// Sizes and strides are template parameters: a program is compiled for its
// shapes, and divisions by page or row sizes become multiplications.

typedef int mt_i32x4 __attribute__((ext_vector_type(4)));

// Elements c .. c + 3 of a row of COLS elements CS apart, 0 behind its end.
template <unsigned COLS, unsigned CS>
MT_INLINE mt_f32x4 mt_row4(const float* row, unsigned c) {
    if constexpr (CS == 1u) {
        if (COLS % 4u == 0u || c + 4u <= COLS) return mt_ld4u(row + c);
    }
    mt_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (unsigned j = 0; j < 4u; ++j)
        if (c + j < COLS) v[j] = row[(size_t)(c + j) * CS];
    return v;
}
template <unsigned COLS>
MT_INLINE void mt_put_row4(float* row, unsigned c, mt_f32x4 v) {
    if (COLS % 4u == 0u || c + 4u <= COLS) {
        *reinterpret_cast<mt_f32x4u*>(row + c) = v;
        return;
    }
#pragma unroll
    for (unsigned j = 0; j < 4u; ++j)
        if (c + j < COLS) row[c + j] = v[j];
}

// ---------------------------------------------------------------------------
// h = x + residual;  y = h / sqrt(mean(h^2) + eps) * w, in 32 bits, or as
// q = rint(y / s) with s = max|y| / 127 of the row.
//
// T lanes (a power of two of at least 64) share a row, which they keep in PER
// float4s each, so x and the residual are read once; rows longer than that
// (PER 0) are read again for each pass.  Squares, the mean and y are in 64
// bits: HBM bounds the kernel many times over, no square overflows, y is
// rounded once, and q falls on the side of its border that the formula says.
// A row with a value that is not finite has no scale: it is stored as zeros
// with the scale NaN, and reads back as NaN.
// ---------------------------------------------------------------------------

template <unsigned T, typename OP>
MT_INLINE double mt_row_fold(double v, double* lds, OP op) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off, 64));
    if constexpr (T > 64u) {
        __syncthreads();
        if (mt_lane() == 0u) lds[mt_wave()] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (unsigned w = 1; w < T / 64u; ++w) v = op(v, lds[w]);
    }
    return v;
}

template <unsigned COLS, unsigned T, unsigned PER, unsigned XRS, unsigned XCS, unsigned RRS, unsigned RCS, bool RES,
          bool SUM, bool WEIGHT, bool EIGHT>
MT_INLINE void mt_rms_norm(const float* x, const float* res, const float* w, double eps, float* h_out, float* y_out,
                           signed char* q_out, float* s_out, unsigned rows, double* lds) {
    constexpr unsigned NQ = (COLS + 3u) / 4u, N = PER ? PER : (NQ + T - 1u) / T, KEEP = PER ? PER : 1u;
    const unsigned t = T == 64u ? mt_lane() : threadIdx.x;
    const unsigned row = T == 64u ? blockIdx.x * 4u + mt_wave() : blockIdx.x;
    if (T == 64u && row >= rows) return;  // (no barrier where a wave has its own row)
    const float* xr = x + (size_t)row * XRS;
    const float* rr = RES ? res + (size_t)row * RRS : nullptr;
    const auto load = [&](unsigned c) {
        mt_f32x4 v = mt_row4<COLS, XCS>(xr, c);
        if constexpr (RES) v = v + mt_row4<COLS, RCS>(rr, c);
        return v;
    };
    mt_f32x4 h[KEEP];
    if constexpr (PER != 0u) {
#pragma unroll
        for (unsigned i = 0; i < PER; ++i) {
            const unsigned c = 4u * (t + T * i);
            h[i] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
            if (c < COLS) h[i] = load(c);
        }
    }
    // Calls f(c, values) for this lane's quads; `again` where they are kept.
    const auto each = [&](auto f) {
        if constexpr (PER != 0u) {
#pragma unroll
            for (unsigned i = 0; i < PER; ++i) {
                const unsigned c = 4u * (t + T * i);
                if (c < COLS) f(c, h[i]);
            }
        } else {
            for (unsigned i = 0; i < N; ++i) {
                const unsigned c = 4u * (t + T * i);
                if (c < COLS) f(c, load(c));
            }
        }
    };
    double sum = 0.0;
    each([&](unsigned c, mt_f32x4 v) {
        if constexpr (SUM) mt_put_row4<COLS>(h_out + (size_t)row * COLS, c, v);
#pragma unroll
        for (unsigned j = 0; j < 4u; ++j) sum = __builtin_fma((double)v[j], (double)v[j], sum);
    });
    sum = mt_row_fold<T>(sum, lds, [](double a, double b) { return a + b; });
    const double r = 1.0 / __builtin_sqrt(sum / (double)COLS + eps);
    const auto norm = [&](unsigned c, mt_f32x4 v, double (&y)[4]) {
        mt_f32x4 g = {1.f, 1.f, 1.f, 1.f};
        if constexpr (WEIGHT) g = mt_row4<COLS, 1u>(w, c);
#pragma unroll
        for (unsigned j = 0; j < 4u; ++j) y[j] = (double)v[j] * r * (double)g[j];
    };
    if constexpr (!EIGHT) {
        each([&](unsigned c, mt_f32x4 v) {
            double y[4];
            norm(c, v, y);
            mt_put_row4<COLS>(y_out + (size_t)row * COLS, c,
                              mt_f32x4{(float)y[0], (float)y[1], (float)y[2], (float)y[3]});
        });
    } else {
        double top = 0.0;
        each([&](unsigned c, mt_f32x4 v) {
            double y[4];
            norm(c, v, y);
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j) {
                const double a = __builtin_fabs(y[j]);
                if (c + j < COLS) top = a < (double)INFINITY ? __builtin_fmax(top, a) : (double)INFINITY;
            }
        });
        top = mt_row_fold<T>(top, lds, [](double a, double b) { return __builtin_fmax(a, b); });
        const bool fine = top < (double)INFINITY;
        const float s = fine ? (float)(top / 127.0) : NAN;
        const double inv = s > 0.f ? 1.0 / (double)s : 0.0;
        if (t == 0u) s_out[row] = s;
        each([&](unsigned c, mt_f32x4 v) {
            double y[4];
            norm(c, v, y);
            unsigned word = 0u;
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j) {
                double q = __builtin_rint(y[j] * inv);
                q = __builtin_fmin(__builtin_fmax(q, -127.0), 127.0);  // (a subnormal scale has few bits)
                word |= ((unsigned)(fine ? (int)q : 0) & 255u) << (8u * j);
            }
            signed char* to = q_out + (size_t)row * COLS + c;
            if constexpr (COLS % 4u == 0u) {
                *reinterpret_cast<unsigned*>(to) = word;
            } else {
#pragma unroll
                for (unsigned j = 0; j < 4u; ++j)
                    if (c + j < COLS) to[j] = (signed char)(word >> (8u * j));
            }
        });
    }
}

// ---------------------------------------------------------------------------
// y[r, c] = q[r, c] * s[r].  The matrix is dense, so lanes take 16 elements of
// the flat array each, aligned whatever the row length.
// ---------------------------------------------------------------------------

template <unsigned COLS>
MT_INLINE void mt_dequantize(const signed char* q, const float* s, float* y, size_t n) {
    const size_t at = ((size_t)blockIdx.x * 256u + threadIdx.x) * 16u;
    if (at >= n) return;
    size_t row = at / COLS;
    unsigned c = (unsigned)(at - row * COLS);
    if (at + 16u <= n) {
        const mt_u32x4 v = *reinterpret_cast<const mt_u32x4*>(q + at);
        float scale = s[row];
#pragma unroll
        for (unsigned i = 0; i < 4u; ++i) {
            mt_f32x4 o;
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j) {
                if (c == COLS) c = 0u, scale = s[++row];
                o[j] = (float)(int)(signed char)(v[i] >> (8u * j)) * scale;
                ++c;
            }
            mt_st4(y + at + 4u * i, o);
        }
    } else {
        for (size_t i = at; i < n; ++i) y[i] = (float)(int)q[i] * s[i / COLS];
    }
}

// ---------------------------------------------------------------------------
// The paged cache.  A page is a row of PAGE_BYTES: [keys | values], each
// [HK heads][PS rows][D], then (8-bit types) a fp32 scale for each of those
// rows, keys first.  KIND 0: fp32, 1: int8, 2: e4m3 (OCP).
// ---------------------------------------------------------------------------

template <int KIND, unsigned HK, unsigned PS, unsigned D>
struct mt_cache {
    static constexpr unsigned ITEM = KIND == 0 ? 4u : 1u;
    static constexpr unsigned HALF = HK * PS * D * ITEM;  // bytes of a page's keys (or values)
    static constexpr unsigned SCALES = 2u * HALF;
    static constexpr unsigned PAGE = (2u * HALF + (KIND == 0 ? 0u : 8u * HK * PS) + 15u) / 16u * 16u;
    MT_INLINE static size_t row(unsigned page, unsigned part, unsigned head, unsigned r) {
        return (size_t)page * PAGE + (size_t)part * HALF + (size_t)((head * PS + r) * D) * ITEM;
    }
    MT_INLINE static size_t scale(unsigned page, unsigned part, unsigned head, unsigned r) {
        return (size_t)page * PAGE + SCALES + (size_t)((part * HK + head) * PS + r) * 4u;
    }
};

// Four values of a held type from one word.
template <int KIND>
MT_INLINE mt_f32x4 mt_held4(unsigned w) {
    if constexpr (KIND == 1) {
        return mt_f32x4{(float)(int)(signed char)w, (float)(int)(signed char)(w >> 8),
                        (float)(int)(signed char)(w >> 16), (float)((int)w >> 24)};
    } else {
        const mt_f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        const mt_f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return mt_f32x4{lo.x, lo.y, hi.x, hi.y};
    }
}

// x / s rounded once to a whole number (KIND 1) or to e4m3's steps (KIND 2),
// ties to even, for a scale s that brings |x / s| to at most 127 or 448.
// The quotient from a reciprocal is off by about 2^-22 of itself, enough to
// fall on the wrong side of a border between two steps.  The remainder
// x - n st s of the nearest multiple n st is exact in fp32 (it is a multiple of
// x's last place or of st times s's, and below st s, so it has 24 bits), and
// decides: more than half a step, or exactly half with n odd, moves n by one.
template <int KIND>
MT_INLINE float mt_step_round(float x, float s, float inv) {
    const float t = x * inv;
    float st = 1.0f, per = 1.0f;  // the step, and steps per unit
    if constexpr (KIND == 2) {
        // e4m3: three bits behind the leading one, the last step 2^-9
        const int e = (int)((__float_as_uint(t) >> 23) & 255u) - 127, b = (e < -6 ? -6 : e) - 3;
        st = __uint_as_float((unsigned)(127 + b) << 23);
        per = __uint_as_float((unsigned)(127 - b) << 23);
    }
    float n = __builtin_rintf(t * per);
    const float rest = __builtin_fmaf(-(n * st), s, x);
    const float twice = 2.0f * __builtin_fabsf(rest), one = st * s;
    if (twice > one || (twice == one && ((int)n & 1))) n += rest > 0.0f ? 1.0f : -1.0f;
    const float most = KIND == 2 ? 448.0f : 127.0f;
    return __builtin_fminf(__builtin_fmaxf(n * st, -most), most);
}

// One row of D values held by 16 lanes (lane j has dims 64 c + 4 j .. + 3) into
// the cache.  `live`: whether the row is stored at all; every lane takes part
// in the exchange of the maximum.
template <int KIND, unsigned HK, unsigned PS, unsigned D>
MT_INLINE void mt_cache_put(unsigned char* cache, const mt_f32x4 (&v)[(D + 63u) / 64u], unsigned j, bool live,
                            unsigned page, unsigned part, unsigned head, unsigned r) {
    using C = mt_cache<KIND, HK, PS, D>;
    constexpr unsigned NC = (D + 63u) / 64u;
    if constexpr (KIND == 0) {
        if (!live) return;
        float* to = reinterpret_cast<float*>(cache + C::row(page, part, head, r));
#pragma unroll
        for (unsigned c = 0; c < NC; ++c)
            if (D % 64u == 0u || 64u * c + 4u * j < D) mt_st4(to + 64u * c + 4u * j, v[c]);
    } else {
        float top = 0.f;
#pragma unroll
        for (unsigned c = 0; c < NC; ++c)
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                const float a = __builtin_fabsf(v[c][i]);
                top = a < INFINITY ? __builtin_fmaxf(top, a) : INFINITY;
            }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) top = __builtin_fmaxf(top, mt_shfl_xor(top, off));
        const bool fine = top < INFINITY;
        const float s = fine ? top / (KIND == 2 ? 448.0f : 127.0f) : NAN;
        // Near the smallest scales the reciprocal overflows and steps times the
        // scale lose bits: there both sides of the quotient are taken 2^64 larger.
        const float up = s < 0x1.0p-100f ? 0x1.0p+64f : 1.0f;
        const float big = s * up, inv = s > 0.f ? 1.0f / big : 0.f;
        if (!live) return;
        unsigned char* to = cache + C::row(page, part, head, r);
#pragma unroll
        for (unsigned c = 0; c < NC; ++c) {
            if (D % 64u != 0u && 64u * c + 4u * j >= D) continue;
            float q[4];
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i)
                q[i] = fine && s > 0.f ? mt_step_round<KIND>(v[c][i] * up, big, inv) : 0.f;
            unsigned word = 0u;
            if constexpr (KIND == 1) {
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i) word |= ((unsigned)(int)q[i] & 255u) << (8u * i);
            } else {
                word = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
                word = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], (int)word, true);
            }
            *reinterpret_cast<unsigned*>(to + 64u * c + 4u * j) = word;
        }
        if (j == 0u) *reinterpret_cast<float*>(cache + C::scale(page, part, head, r)) = s;
    }
}

// Token t's keys and values go to slot slots[t] (page slot / PS, row slot % PS);
// a slot outside the cache is passed over, and of tokens that name the same
// slot the last is stored, whole: a token looks through the slots behind it
// for its own.  A workgroup takes TB tokens, so those slots are read T / TB
// times in all; 16 lanes take a row of one head.
template <int KIND, unsigned HK, unsigned PS, unsigned D, unsigned PAGES, unsigned TB, unsigned KRS, unsigned KCS,
          unsigned VRS, unsigned VCS>
MT_INLINE void mt_cache_write(const float* k, const float* v, const int* slots, unsigned char* cache, unsigned tokens,
                              unsigned* dead) {
    constexpr unsigned long long ALL = (unsigned long long)PAGES * PS;
    constexpr unsigned SLOTS = ALL > 0x80000000ull ? 0x80000000u : (unsigned)ALL;
    constexpr unsigned NC = (D + 63u) / 64u;
    const unsigned t0 = blockIdx.x * TB;
    unsigned mine[TB], hit = 0u;
#pragma unroll
    for (unsigned i = 0; i < TB; ++i) mine[i] = t0 + i < tokens ? (unsigned)slots[t0 + i] : 0xFFFFFFFFu;
    if (threadIdx.x == 0u) *dead = 0u;
    for (unsigned j = t0 + 1u + threadIdx.x; j < tokens; j += 256u) {
        const unsigned other = (unsigned)slots[j];
#pragma unroll
        for (unsigned i = 0; i < TB; ++i)
            if (other == mine[i] && j > t0 + i) hit |= 1u << i;
    }
    __syncthreads();
    if (hit) atomicOr(dead, hit);
    __syncthreads();
    const unsigned lost = *dead, j = threadIdx.x & 15u;
    for (unsigned at = threadIdx.x >> 4; at < TB * 2u * HK; at += 16u) {
        const unsigned i = at / (2u * HK), part = (at / HK) % 2u, head = at % HK, t = t0 + i;
        // (no mine[i]: an index that is not constant would put the array into memory)
        const unsigned slot = t < tokens ? (unsigned)slots[t] : 0xFFFFFFFFu;
        const bool live = slot < SLOTS && !((lost >> i) & 1u);
        mt_f32x4 x[NC];
#pragma unroll
        for (unsigned c = 0; c < NC; ++c) {
            x[c] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
            const unsigned d = 64u * c + 4u * j;
            if (live && (D % 64u == 0u || d < D))
                x[c] = part ? mt_row4<HK * D, VCS>(v + (size_t)t * VRS, head * D + d)
                            : mt_row4<HK * D, KCS>(k + (size_t)t * KRS, head * D + d);
        }
        mt_cache_put<KIND, HK, PS, D>(cache, x, j, live, slot / PS, part, head, slot % PS);
    }
}

// Row r of k and v is slot slots[r] of the cache in 32 bits, zeros for a slot
// outside it.  16 lanes take a row of one head.
template <int KIND, unsigned HK, unsigned PS, unsigned D, unsigned PAGES>
MT_INLINE void mt_cache_read(const unsigned char* cache, const int* slots, float* k, float* v, unsigned rows) {
    using C = mt_cache<KIND, HK, PS, D>;
    constexpr unsigned long long ALL = (unsigned long long)PAGES * PS;
    constexpr unsigned SLOTS = ALL > 0x80000000ull ? 0x80000000u : (unsigned)ALL;
    constexpr unsigned NC = (D + 63u) / 64u;
    const size_t at = (size_t)blockIdx.x * 16u + (threadIdx.x >> 4);
    const unsigned j = threadIdx.x & 15u;
    const size_t r = at / (2u * HK);
    if (r >= rows) return;
    const unsigned part = (unsigned)(at / HK) % 2u, head = (unsigned)(at % HK);
    const unsigned slot = (unsigned)slots[r];
    const bool live = slot < SLOTS;
    const unsigned page = live ? slot / PS : 0u, in = live ? slot % PS : 0u;
    const unsigned char* from = cache + C::row(page, part, head, in);
    float s = 1.f;
    if constexpr (KIND != 0) s = *reinterpret_cast<const float*>(cache + C::scale(page, part, head, in));
    float* to = (part ? v : k) + r * (HK * D) + head * D;
#pragma unroll
    for (unsigned c = 0; c < NC; ++c) {
        const unsigned d = 64u * c + 4u * j;
        if (D % 64u != 0u && d >= D) continue;
        mt_f32x4 x;
        if constexpr (KIND == 0) x = mt_ld4(reinterpret_cast<const float*>(from) + d);
        else x = mt_held4<KIND>(*reinterpret_cast<const unsigned*>(from + d)) * s;
        if (!live) x = mt_f32x4{0.f, 0.f, 0.f, 0.f};
        mt_st4(to + d, x);
    }
}

// ---------------------------------------------------------------------------
// Attention of one new token per sequence over the paged cache.
//
// A workgroup takes one sequence, one key head with the (at most 16) query
// heads that share it, and one part of the sequence's length; each of its waves
// takes every WAVES-th tile of 16 positions on its own, and they meet at the end.
//
//   scores  S[position, head] = K . q: fp32 MFMAs 16x16x4, K the rows.  Lane
//     (n, g) = (lane % 16, lane / 16) loads row n's dims VK (4 jj + g) .. + VK - 1
//     whole, and element e of load jj is its operand of MFMA (jj, e): the four
//     dims of that product are the ones at e in each g's piece, for K and q alike.
//   softmax S comes back with lane (n, g) holding head n at positions 4 g + i,
//     i < 4; the running maximum m (in units of log 2: the scale carries
//     log2(e)) is shared by the four g of a head, the sum l is each lane's own
//     until the end.  The sums so far are rescaled only when some head's
//     maximum grows.
//   output  O[head, dim] += P . V: MFMA i takes positions {4 g + i}, so p[i] is
//     its P operand where it stands, and lane (n, g) loads row 4 g + i's dims
//     VV (16 c + n) .. + VV - 1 of V, element e being the operand for the dims
//     that stand at e.  No value changes lanes and nothing is transposed.
//
// 8-bit values are widened in registers; a position's scales multiply its score
// and its weight.  A position that is masked (behind the length, or in a page
// outside the cache) scores -inf and its values are replaced by zeros, whatever
// its bytes hold.
//
// Bound: HBM, K and V once.  The fp32 MFMAs take 64 elements in 32 cycles
// whatever the number of heads that share them, 4.9e12 elements a second, which
// exceeds HBM for fp32 and about matches it for 8 bits.
// ---------------------------------------------------------------------------

template <unsigned W>
MT_INLINE void mt_ld_words(unsigned (&to)[W], const unsigned char* p) {
    if constexpr (W == 4u) {
        const mt_u32x4 v = *reinterpret_cast<const mt_u32x4*>(p);
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
    } else if constexpr (W == 2u) {
        typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 v = *reinterpret_cast<const u32x2*>(p);
        to[0] = v.x, to[1] = v.y;
    } else {
        to[0] = *reinterpret_cast<const unsigned*>(p);
    }
}
// Four values of a held type from the words at 4 e of a row.
template <int KIND, unsigned W>
MT_INLINE mt_f32x4 mt_four(const unsigned (&w)[W], unsigned e) {
    if constexpr (KIND == 0)
        return mt_f32x4{__uint_as_float(w[4u * e]), __uint_as_float(w[4u * e + 1u]), __uint_as_float(w[4u * e + 2u]),
                        __uint_as_float(w[4u * e + 3u])};
    else
        return mt_held4<KIND>(w[e]);
}

template <int KIND, unsigned HK, unsigned PS, unsigned D, unsigned PAGES, unsigned WIDTH, unsigned SHARE, unsigned WAVES,
          unsigned SPLITS, unsigned EACH, unsigned BATCH, unsigned QRS, unsigned QCS>
MT_INLINE void mt_paged_attention(const float* q, const unsigned char* cache, const int* pages, const int* lengths,
                                  float* o, double scale, float* ws, unsigned rows, unsigned char* lds) {
    using C = mt_cache<KIND, HK, PS, D>;
    constexpr unsigned ITEM = C::ITEM, PARTS = (SHARE + 15u) / 16u, HELD = SHARE < 16u ? SHARE : 16u;
    constexpr unsigned VK = KIND == 0 ? 4u : D % 64u == 0u ? 16u : D % 32u == 0u ? 8u : 4u, NJ = D / (4u * VK);
    constexpr unsigned VV = KIND == 0 || D <= 64u ? 4u : 8u, NV = (D + 16u * VV - 1u) / (16u * VV);
    constexpr unsigned KW = VK * ITEM / 4u, VW = VV * ITEM / 4u, FLOATS = HELD * (D + 2u);
    constexpr bool ONE_PAGE = PS % 16u == 0u;  // a tile lies in one page
    const unsigned lane = mt_lane(), n = lane & 15u, g = lane >> 4, wave = mt_wave();
    const unsigned split = blockIdx.x % SPLITS, pair = blockIdx.x / SPLITS;
    const unsigned part = pair % PARTS, head = pair / PARTS % HK, b = pair / (PARTS * HK);
    // (a batch larger than the workspace was laid out for is not split)
    const bool joined = SPLITS > 1u && gridDim.z <= BATCH;
    const int asked = lengths[b];
    const unsigned len = asked < 0 ? 0u : (unsigned)asked < WIDTH * PS ? (unsigned)asked : WIDTH * PS;
    const unsigned active = joined && len > EACH ? (len + EACH - 1u) / EACH : 1u;
    if (split >= active) return;
    const unsigned first = active > 1u ? split * EACH : 0u;
    const unsigned last = active > 1u && len - first > EACH ? first + EACH : len;
    const unsigned tiles = (last - first + 15u) / 16u;

    mt_f32x4 qf[NJ][VK / 4u];
    {
        const unsigned h = part * 16u + n;
        const float by = (float)(scale * 1.4426950408889634);
#pragma unroll
        for (unsigned jj = 0; jj < NJ; ++jj)
#pragma unroll
            for (unsigned e = 0; e < VK / 4u; ++e) {
                qf[jj][e] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
                if (n < HELD && h < SHARE)
                    qf[jj][e] = mt_row4<HK * SHARE * D, QCS>(q + (size_t)b * QRS,
                                                             (head * SHARE + h) * D + VK * (4u * jj + g) + 4u * e) * by;
            }
    }

    const int* table = pages + (size_t)b * WIDTH;
    // The page of this lane's row n of a tile (of the tile, where it lies in one).
    const auto page_of = [&](unsigned ti) -> int {
        if constexpr (ONE_PAGE) {
            return ti < tiles ? __builtin_amdgcn_readfirstlane(table[(first + 16u * ti) / PS]) : -1;
        } else {
            const unsigned at = first + 16u * ti + n;
            return ti < tiles && at < last ? table[at / PS] : -1;
        }
    };
    const auto row_page = [&](int page, unsigned i) -> int { return ONE_PAGE ? page : __shfl(page, (int)(4u * g + i), 64); };
    const auto safe = [&](int page) -> unsigned { return (unsigned)page < PAGES ? (unsigned)page : 0u; };

    unsigned kw[NJ][KW], vw[4][NV][VW];
    float ks[4], vs[4];
    const auto load_k = [&](unsigned ti, int page) {
        const unsigned t0 = first + 16u * ti;
        const unsigned char* p = cache + C::row(safe(page), 0u, head, (t0 + n) % PS) + g * (VK * ITEM);
#pragma unroll
        for (unsigned jj = 0; jj < NJ; ++jj) mt_ld_words<KW>(kw[jj], p + jj * (4u * VK * ITEM));
        if constexpr (KIND != 0) {
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i)
                ks[i] = *reinterpret_cast<const float*>(
                    cache + C::scale(safe(row_page(page, i)), 0u, head, (t0 + 4u * g + i) % PS));
        }
    };
    const auto load_v = [&](unsigned ti, int page) {
        const unsigned t0 = first + 16u * ti;
#pragma unroll
        for (unsigned i = 0; i < 4u; ++i) {
            const unsigned pg = safe(row_page(page, i)), r = (t0 + 4u * g + i) % PS;
            const unsigned char* p = cache + C::row(pg, 1u, head, r);
#pragma unroll
            for (unsigned c = 0; c < NV; ++c) {
                unsigned d = VV * (16u * c + n);
                if (D % (16u * VV) != 0u && d >= D) d = 0u;  // (columns that no output takes)
                mt_ld_words<VW>(vw[i][c], p + d * ITEM);
            }
            if constexpr (KIND != 0) vs[i] = *reinterpret_cast<const float*>(cache + C::scale(pg, 1u, head, r));
        }
    };

    mt_f32x4 acc[NV * VV];
#pragma unroll
    for (unsigned i = 0; i < NV * VV; ++i) acc[i] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool seen = false;
    int page = -1, page_next = -1;
    if (wave < tiles) {
        page = page_of(wave);
        load_k(wave, page);
        load_v(wave, page);
        page_next = page_of(wave + WAVES);
    }
    for (unsigned ti = wave; ti < tiles; ti += WAVES) {
        const int page_after = page_of(ti + 2u * WAVES);
        const bool more = ti + WAVES < tiles;
        mt_f32x4 s = {0.f, 0.f, 0.f, 0.f}, s2 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (unsigned jj = 0; jj < NJ; ++jj)
#pragma unroll
            for (unsigned e = 0; e < VK / 4u; ++e) {
                const mt_f32x4 k4 = mt_four<KIND, KW>(kw[jj], e);
                s = __builtin_amdgcn_mfma_f32_16x16x4f32(k4.x, qf[jj][e].x, s, 0, 0, 0);
                s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(k4.y, qf[jj][e].y, s2, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_16x16x4f32(k4.z, qf[jj][e].z, s, 0, 0, 0);
                s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(k4.w, qf[jj][e].w, s2, 0, 0, 0);
            }
        s = s + s2;
        if constexpr (KIND != 0) {
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) s[i] *= ks[i];
        }
        if (more) load_k(ti + WAVES, page_next);
        bool ok[4], any = false, all = true;
#pragma unroll
        for (unsigned i = 0; i < 4u; ++i) {
            ok[i] = (unsigned)row_page(page, i) < PAGES && first + 16u * ti + 4u * g + i < last;
            if (!ok[i]) s[i] = -INFINITY;
            any = any || ok[i];
            all = all && ok[i];
        }
        seen = seen || __any(any);
        float top = __builtin_fmaxf(__builtin_fmaxf(s[0], s[1]), __builtin_fmaxf(s[2], s[3]));
        top = __builtin_fmaxf(top, mt_shfl_xor(top, 16));
        top = __builtin_fmaxf(top, mt_shfl_xor(top, 32));
        if (__any(top > m)) {
            const float grown = __builtin_fmaxf(m, top);
            const float by = grown > m ? __builtin_amdgcn_exp2f(m - grown) : 1.f;
            m = grown;
            l *= by;
            mt_f32x4 rows_by;
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) rows_by[i] = __shfl(by, (int)(4u * g + i), 64);
#pragma unroll
            for (unsigned i = 0; i < NV * VV; ++i) acc[i] = acc[i] * rows_by;
        }
        const float base = m == -INFINITY ? 0.f : m;
        float p[4];
#pragma unroll
        for (unsigned i = 0; i < 4u; ++i) {
            p[i] = __builtin_amdgcn_exp2f(s[i] - base);
            l += p[i];
            if constexpr (KIND != 0) p[i] *= vs[i];
        }
        if (!__all(all)) {
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                if (ok[i]) continue;
                p[i] = 0.f;
#pragma unroll
                for (unsigned c = 0; c < NV; ++c)
#pragma unroll
                    for (unsigned w = 0; w < VW; ++w) vw[i][c][w] = 0u;
            }
        }
#pragma unroll
        for (unsigned i = 0; i < 4u; ++i)
#pragma unroll
            for (unsigned c = 0; c < NV; ++c)
#pragma unroll
                for (unsigned e = 0; e < VV / 4u; ++e) {
                    const mt_f32x4 v4 = mt_four<KIND, VW>(vw[i][c], e);
#pragma unroll
                    for (unsigned u = 0; u < 4u; ++u)
                        acc[VV * c + 4u * e + u] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                            p[i], v4[u], acc[VV * c + 4u * e + u], 0, 0, 0);
                }
        if (more) load_v(ti + WAVES, page_next);
        page = page_next;
        page_next = page_after;
    }
    l += mt_shfl_xor(l, 16);
    l += mt_shfl_xor(l, 32);
    if (m == -INFINITY) l = seen ? 1.f : 0.f;

    // The waves' parts: [WAVES][HELD][D] sums, then [WAVES][HELD] of m and of l.  A
    // part weighs 2^(m - the largest m); one whose scores are all -inf weighs nothing
    // and says in l whether it has positions: a softmax over such scores alone is
    // 0 / 0, one over no positions gives zeros.
    float* sums = reinterpret_cast<float*>(lds);
    float* ms = sums + WAVES * HELD * D;
    float* ls = ms + WAVES * HELD;
    float* by = ls + WAVES * HELD;  // [SPLITS][HELD] weights
    unsigned* flag = reinterpret_cast<unsigned*>(by + SPLITS * HELD);
#pragma unroll
    for (unsigned c = 0; c < NV; ++c)
#pragma unroll
        for (unsigned e = 0; e < VV; ++e) {
            const unsigned d = VV * (16u * c + n) + e;
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                const unsigned h = 4u * g + i;
                if (h < HELD && (D % (16u * VV) == 0u || d < D)) sums[(wave * HELD + h) * D + d] = acc[VV * c + e][i];
            }
        }
    if (g == 0u && n < HELD) {
        ms[wave * HELD + n] = m;
        ls[wave * HELD + n] = l;
    }
    __syncthreads();

    float* mine = nullptr;
    if (active > 1u) mine = ws + MT_WS_HEAD + (((size_t)blockIdx.z * (rows * HK * PARTS) + pair) * SPLITS + split) * FLOATS;
    for (unsigned at = threadIdx.x; at < HELD * D; at += 64u * WAVES) {
        const unsigned h = at / D, d = at % D;
        float top = -INFINITY, empty = 0.f, total = 0.f, value = 0.f;
#pragma unroll
        for (unsigned w = 0; w < WAVES; ++w) top = __builtin_fmaxf(top, ms[w * HELD + h]);
#pragma unroll
        for (unsigned w = 0; w < WAVES; ++w) {
            const float mw = ms[w * HELD + h], lw = ls[w * HELD + h];
            if (mw == -INFINITY) {
                empty += lw;
                continue;
            }
            const float u = __builtin_amdgcn_exp2f(mw - top);
            total += u * lw;
            value += u * sums[(w * HELD + h) * D + d];
        }
        if (top == -INFINITY) total = empty;
        if (active > 1u) {
            mt_sn_put(mine + at, value);
            if (d == 0u) {
                mt_sn_put(mine + HELD * D + h, top);
                mt_sn_put(mine + HELD * D + HELD + h, total);
            }
        } else if (part * 16u + h < SHARE) {
            const float r = top == -INFINITY ? (total > 0.f ? NAN : 0.f) : value / total;
            o[((size_t)b * HK * SHARE + head * SHARE + part * 16u + h) * D + d] = r;
        }
    }
    if (active <= 1u) return;

    // The last workgroup of the sequence's head joins the parts: maxima into `by`,
    // sums of weights into `sums` (at most 64 parts, which is no more than WAVES * D).
    unsigned* counter = reinterpret_cast<unsigned*>(ws) + blockIdx.z * (rows * HK * PARTS) + pair;
    if (!mt_sn_arrive(counter, active, flag)) return;
    const float* all = mine - (size_t)split * FLOATS;
    for (unsigned at = threadIdx.x; at < HELD * active; at += 64u * WAVES) {
        const unsigned s = at / HELD, h = at % HELD;
        by[at] = mt_sn_get(all + (size_t)s * FLOATS + HELD * D + h);
        sums[at] = mt_sn_get(all + (size_t)s * FLOATS + HELD * D + HELD + h);
    }
    __syncthreads();
    for (unsigned at = threadIdx.x; at < HELD * D; at += 64u * WAVES) {
        const unsigned h = at / D, d = at % D;
        float top = -INFINITY, empty = 0.f, total = 0.f, value = 0.f;
        for (unsigned s = 0; s < active; ++s) top = __builtin_fmaxf(top, by[s * HELD + h]);
#pragma unroll 8
        for (unsigned s = 0; s < active; ++s) {
            const float v = mt_sn_get(all + (size_t)s * FLOATS + at);
            const float mw = by[s * HELD + h], lw = sums[s * HELD + h];
            const bool none = mw == -INFINITY;
            const float u = none ? 0.f : __builtin_amdgcn_exp2f(mw - top);
            empty += none ? lw : 0.f;
            total += none ? 0.f : u * lw;
            value += none ? 0.f : u * v;
        }
        if (part * 16u + h < SHARE) {
            const float r = top == -INFINITY ? (empty > 0.f ? NAN : 0.f) : value / total;
            o[((size_t)b * HK * SHARE + head * SHARE + part * 16u + h) * D + d] = r;
        }
    }
}

// ---------------------------------------------------------------------------
// y[m, n] = sum over groups of s[n, group] * sum_k x[m, k] (q[n, k] - z[n, group])
// for 4-bit q: whole numbers on the int8 matrix cores, exact within a group.
//
// x in fp32 becomes whole numbers too: the 128 values of a row's block are
// multiples of 2^-30 of a power of two above the largest, x = 2^(E-156) X, and
// X = 2^24 d3 + 2^16 d2 + 2^8 d1 + d0 with digits of 8 bits.  The digits of 4
// rows of x are the 16 rows of an MFMA 16x16x64; 16 weight rows are its columns.
// What is lost is 2^-30 of the block's largest value per element; a block that
// holds an infinity or a NaN is summed in fp32 as the formula says.  x in 8 bits
// is 16 rows as it stands.
//
// A lane's 16 bytes of weights are q of 32 consecutive k, even ones in the low
// nibbles: xor 0x88 turns q into q - 8 in two's complement, and in the high
// nibble of a byte that is 16 (q - 8) as int8, so w & 0xF0.. are the odd k and
// (w << 4) & 0xF0.. the even k: two MFMAs, with x's digits in the same order.  A
// block of 128 k is four lanes' pieces of a row; with groups of 32 or 64 the
// pieces of the other groups are zeroed in x.
//
// Bound: HBM, the weights once.  The waves of a workgroup share its weight rows
// and split k, so that few rows of weights still keep many loads in flight; each
// makes the digits of its own part of k (LDS of its own, no barrier).
// ---------------------------------------------------------------------------

// Byte i of a, b, c, d together in to[i].
MT_INLINE void mt_bytes4(unsigned a, unsigned b, unsigned c, unsigned d, unsigned (&to)[4]) {
    const unsigned ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
    const unsigned cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
    to[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u);
    to[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
    to[2] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u);
    to[3] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
}

// The whole number that an MFMA's four digit rows stand for.
MT_INLINE float mt_digits(mt_i32x4 c) {
    const int hi = c[0] * 256 + c[1], lo = c[2] * 256 + c[3];
    return __builtin_fmaf((float)hi, 65536.0f, (float)lo);
}

template <bool EIGHT, unsigned SETS, unsigned K, unsigned N, unsigned GROUP, bool ZEROS, unsigned R, unsigned WAVES,
          unsigned XRS, unsigned XCS>
MT_INLINE void mt_matmul_int4(const float* x, const signed char* x8, const float* xs, const unsigned char* w,
                              const float* scales, const float* zeros, float* y, unsigned rows, unsigned char* lds) {
    constexpr unsigned NB = (K + 127u) / 128u, NG = K / GROUP, GB = 128u / GROUP, ACC = EIGHT ? 4u : SETS;
    constexpr bool RAGGED = K % 128u != 0u;
    const unsigned lane = mt_lane(), n = lane & 15u, g = lane >> 4, wave = mt_wave();
    const unsigned n0 = blockIdx.x * (16u * R), m0 = blockIdx.y * 16u;
    const unsigned b0 = NB * wave / WAVES, b1 = NB * (wave + 1u) / WAVES;

    const unsigned char* wr[R];
    size_t sr[R];
#pragma unroll
    for (unsigned r = 0; r < R; ++r) {
        const unsigned row = n0 + 16u * r + n < N ? n0 + 16u * r + n : N - 1u;
        wr[r] = w + (size_t)row * (K / 2u) + 16u * g;
        sr[r] = (size_t)row * NG;
    }
    struct block {
        mt_u32x4 q[R];
        float s[R][GB], z[R][ZEROS ? GB : 1u];
        mt_f32x4 f[EIGHT ? 1u : SETS][2];  // x: rows 4 t + g, k 8 n .. + 7
        mt_u32x4 e[EIGHT ? 2u : 1u];       // x in 8 bits: row n, k 32 g .. + 31
    };
    const auto load = [&](unsigned blk, block& to) {
        const bool in = !RAGGED || blk * 128u + 32u * g < K;
#pragma unroll
        for (unsigned r = 0; r < R; ++r) {
            to.q[r] = mt_u32x4{0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u};
            if (in) to.q[r] = __builtin_nontemporal_load(reinterpret_cast<const mt_u32x4*>(wr[r] + (size_t)blk * 64u));
#pragma unroll
            for (unsigned j = 0; j < GB; ++j) {
                const unsigned gr = blk * GB + j;
                to.s[r][j] = !RAGGED || gr < NG ? scales[sr[r] + gr] : 0.f;
                if constexpr (ZEROS) to.z[r][j] = !RAGGED || gr < NG ? zeros[sr[r] + gr] : 0.f;
            }
        }
        if constexpr (EIGHT) {
            to.e[0] = to.e[1] = mt_u32x4{0u, 0u, 0u, 0u};
            if (in && m0 + n < rows) {
                const mt_u32x4* p = reinterpret_cast<const mt_u32x4*>(x8 + (size_t)(m0 + n) * K + blk * 128u + 32u * g);
                to.e[0] = p[0];
                to.e[1] = p[1];
            }
        } else {
#pragma unroll
            for (unsigned t = 0; t < SETS; ++t) {
                to.f[t][0] = to.f[t][1] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
                const unsigned row = m0 + 4u * t + g, k = blk * 128u + 8u * n;
                if (row < rows && (!RAGGED || k < K)) {
                    to.f[t][0] = mt_row4<K, XCS>(x + (size_t)row * XRS, k);
                    to.f[t][1] = mt_row4<K, XCS>(x + (size_t)row * XRS, k + 4u);
                }
            }
        }
    };

    float acc[R][ACC];
#pragma unroll
    for (unsigned r = 0; r < R; ++r)
#pragma unroll
        for (unsigned a = 0; a < ACC; ++a) acc[r][a] = 0.f;
    unsigned char* own = lds + wave * (2048u * SETS);
    const mt_i32x4 zero4 = {0, 0, 0, 0}, ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};

    block now;
    if (b0 < b1) load(b0, now);
    for (unsigned blk = b0; blk < b1; ++blk) {
        block next = now;
        if (blk + 1u < b1) load(blk + 1u, next);
        mt_i32x4 ae[SETS], ao[SETS];  // x of the even and the odd k, as the MFMA's rows
        int ex[SETS];                 // E of this lane group's row of each set
        bool odd = false;             // a block with values that are not finite
        if constexpr (EIGHT) {
            unsigned ev[4], od[4];
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                const unsigned lo = now.e[i / 2u][2u * (i % 2u)], hi = now.e[i / 2u][2u * (i % 2u) + 1u];
                ev[i] = __builtin_amdgcn_perm(hi, lo, 0x06040200u);
                od[i] = __builtin_amdgcn_perm(hi, lo, 0x07050301u);
            }
            ae[0] = mt_i32x4{(int)ev[0], (int)ev[1], (int)ev[2], (int)ev[3]};
            ao[0] = mt_i32x4{(int)od[0], (int)od[1], (int)od[2], (int)od[3]};
            ex[0] = 0;
        } else {
#pragma unroll
            for (unsigned t = 0; t < SETS; ++t) {
                unsigned top = 0u;  // the bits of |x| order as the values do, infinities and NaN last
                float v[8];
#pragma unroll
                for (unsigned j = 0; j < 8u; ++j) {
                    v[j] = now.f[t][j / 4u][j % 4u];
                    const unsigned a = __float_as_uint(v[j]) & 0x7FFFFFFFu;
                    top = top > a ? top : a;
                }
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) {
                    const unsigned a = (unsigned)__shfl_xor((int)top, off, 64);
                    top = top > a ? top : a;
                }
                const int e = (int)(top >> 23);
                ex[t] = e < 1 ? 1 : e;
                odd = odd || e == 255;
                unsigned d[8];
#pragma unroll
                for (unsigned j = 0; j < 8u; ++j) {
                    const int whole = e == 255 ? 0 : (int)__builtin_ldexpf(v[j], 156 - ex[t]);
                    d[j] = ((unsigned)whole + 0x00808080u) ^ 0x00808080u;
                }
                unsigned ev[4], od[4];
                mt_bytes4(d[0], d[2], d[4], d[6], ev);
                mt_bytes4(d[1], d[3], d[5], d[7], od);
                unsigned char* to = own + 2048u * t + 4u * n + 256u * g;
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i) {
                    *reinterpret_cast<unsigned*>(to + 64u * i) = ev[3u - i];
                    *reinterpret_cast<unsigned*>(to + 1024u + 64u * i) = od[3u - i];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (unsigned t = 0; t < SETS; ++t) {
                ae[t] = *reinterpret_cast<const mt_i32x4*>(own + 2048u * t + 64u * n + 16u * g);
                ao[t] = *reinterpret_cast<const mt_i32x4*>(own + 2048u * t + 1024u + 64u * n + 16u * g);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        mt_i32x4 we[R], wo[R];
#pragma unroll
        for (unsigned r = 0; r < R; ++r)
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                const unsigned v = now.q[r][i] ^ 0x88888888u;
                we[r][i] = (int)((v << 4) & 0xF0F0F0F0u);
                wo[r][i] = (int)(v & 0xF0F0F0F0u);
            }
#pragma unroll
        for (unsigned j = 0; j < GB; ++j) {
            const bool mine = GB == 1u || 32u * g / GROUP == j;
#pragma unroll
            for (unsigned t = 0; t < SETS; ++t) {
                const mt_i32x4 je = mine ? ae[t] : zero4, jo = mine ? ao[t] : zero4;
                mt_i32x4 cz = zero4;
                if constexpr (ZEROS) {
                    cz = __builtin_amdgcn_mfma_i32_16x16x64_i8(je, ones, cz, 0, 0, 0);
                    cz = __builtin_amdgcn_mfma_i32_16x16x64_i8(jo, ones, cz, 0, 0, 0);
                }
#pragma unroll
                for (unsigned r = 0; r < R; ++r) {
                    mt_i32x4 c = __builtin_amdgcn_mfma_i32_16x16x64_i8(je, we[r], zero4, 0, 0, 0);
                    c = __builtin_amdgcn_mfma_i32_16x16x64_i8(jo, wo[r], c, 0, 0, 0);
                    const float s = now.s[r][j];
                    if constexpr (EIGHT) {
#pragma unroll
                        for (unsigned i = 0; i < 4u; ++i) {
                            float f = (float)c[i];
                            if constexpr (ZEROS) f = __builtin_fmaf((float)cz[i], 128.f - 16.f * now.z[r][j], f);
                            acc[r][i] = __builtin_fmaf(f, s, acc[r][i]);
                        }
                    } else {
                        float f = mt_digits(c);
                        if constexpr (ZEROS) f = __builtin_fmaf(mt_digits(cz), 128.f - 16.f * now.z[r][j], f);
                        acc[r][t] += __builtin_ldexpf(f * s, ex[t] - 160);
                    }
                }
            }
        }
        if constexpr (!EIGHT) {
            if (__any(odd)) {
                // Rare: the rows of this block that hold infinities or NaN, in fp32.  Every
                // lane sums its 32 k of its weight rows, the four pieces meet.
#pragma unroll
                for (unsigned t = 0; t < SETS; ++t)
                    for (unsigned mm = 0; mm < 4u; ++mm) {
                        if (__shfl(ex[t], (int)(16u * mm), 64) != 255) continue;
                        const float* xr = x + (size_t)(m0 + 4u * t + mm) * XRS;
#pragma unroll
                        for (unsigned r = 0; r < R; ++r) {
                            float part = 0.f;
                            float z = 8.f, s = now.s[r][0];
#pragma unroll
                            for (unsigned j = 0; j < GB; ++j)
                                if (32u * g / GROUP == j) {
                                    s = now.s[r][j];
                                    if constexpr (ZEROS) z = now.z[r][j];
                                }
                            for (unsigned i = 0; i < 32u; ++i) {
                                const unsigned k = blk * 128u + 32u * g + i;
                                const unsigned word = i < 8u ? now.q[r].x : i < 16u ? now.q[r].y
                                                      : i < 24u ? now.q[r].z : now.q[r].w;
                                const float q = (float)((word >> (4u * (i % 8u))) & 15u);
                                if (!RAGGED || k < K) part += xr[(size_t)k * XCS] * (q - z);
                            }
                            if (!RAGGED || blk * 128u + 32u * g < K) part *= s;
                            part += mt_shfl_xor(part, 16);
                            part += mt_shfl_xor(part, 32);
                            if (g == mm) acc[r][t] += part;
                        }
                    }
            }
        }
        now = next;
    }

    // The waves' sums, [WAVES][R][ACC][64 lanes].
    float* sums = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (unsigned r = 0; r < R; ++r)
#pragma unroll
        for (unsigned a = 0; a < ACC; ++a) sums[((wave * R + r) * ACC + a) * 64u + lane] = acc[r][a];
    __syncthreads();
    for (unsigned at = threadIdx.x; at < R * ACC * 64u; at += 64u * WAVES) {
        float v = 0.f;
#pragma unroll
        for (unsigned i = 0; i < WAVES; ++i) v += sums[i * (R * ACC * 64u) + at];
        const unsigned r = at / (ACC * 64u), a = at / 64u % ACC, ln = at % 64u;
        const unsigned col = n0 + 16u * r + (ln & 15u), row = m0 + (EIGHT ? 4u * (ln >> 4) + a : 4u * a + (ln >> 4));
        if (col < N && row < rows) y[(size_t)row * N + col] = EIGHT ? v * (xs[row] * 0.0625f) : v;
    }
}
