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

// 32 bits where they hold every value, 64 otherwise.
template <bool SMALL>
struct mt_count {
    using type = unsigned;
};
template <>
struct mt_count<false> {
    using type = unsigned long long;
};

// Elements c .. c + 3 of a row of COLS elements CS apart, 0 behind its end.  NT: loads
// that keep nothing in the caches, for rows that are read once.
template <unsigned COLS, unsigned CS, bool NT = false>
MT_INLINE mt_f32x4 mt_row4(const float* row, unsigned c) {
    if constexpr (CS == 1u) {
        if (COLS % 4u == 0u || c + 4u <= COLS) return NT ? mt_ld4u_nt(row + c) : mt_ld4u(row + c);
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
        __builtin_nontemporal_store(v, reinterpret_cast<mt_f32x4u*>(row + c));
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
// (PER 0) are read again for each pass.  What is read and written once goes past the
// caches (4096 rows of 4096 with a residual and 8 bits: outputs 47 -> 44 us, inputs too,
// with the pass that reads y back, 58 -> 55).  Squares, the mean and y are in 64
// bits: HBM bounds the kernel many times over, no square overflows, y is
// rounded once, and q falls on the side of its border that the formula says.
// A row with a value that is not finite has no scale: it is stored as zeros
// with the scale NaN, and reads back as NaN.
//
// Measured: 4096 rows of 4096, residual, 8 bits: 41 us, 5.3 TB/s of a copy's 5.5; 777
// rows of 5003: 7.4 us (4.2 TB/s; 777 workgroups on 256 compute units); one row 3 us.
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
        mt_f32x4 v = mt_row4<COLS, XCS, PER != 0u>(xr, c);
        if constexpr (RES) v = v + mt_row4<COLS, RCS, PER != 0u>(rr, c);
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
// y[r, c] = q[r, c] * s[r].  The matrix is dense, so lanes take four elements of the
// flat array at a time, aligned whatever the row length; a wave's stores are
// contiguous, and its four loads are on the way together.  4096 x 4096: 13 us, 6.3 TB/s
// (what was just written is in the last-level cache).
// ---------------------------------------------------------------------------

template <unsigned COLS>
MT_INLINE void mt_dequantize(const signed char* q, const float* s, float* y, size_t n) {
    const size_t base = (size_t)blockIdx.x * 4096u + 4u * threadIdx.x;
    unsigned v[4];
    float scale[4];
#pragma unroll
    for (unsigned i = 0; i < 4u; ++i) {
        const size_t at = base + 1024u * i;
        v[i] = 0u, scale[i] = 0.f;
        if (at + 4u <= n) {
            v[i] = *reinterpret_cast<const unsigned*>(q + at);
            scale[i] = s[at / COLS];
        }
    }
#pragma unroll
    for (unsigned i = 0; i < 4u; ++i) {
        const size_t at = base + 1024u * i;
        if (at + 4u <= n) {
            mt_f32x4 o;
#pragma unroll
            for (unsigned j = 0; j < 4u; ++j) {
                float by = scale[i];
                if (COLS % 4u != 0u && (at + j) / COLS != at / COLS) by = s[(at + j) / COLS];
                o[j] = (float)(int)(signed char)(v[i] >> (8u * j)) * by;
            }
            mt_st4_nt(y + at, o);
        } else {
            for (size_t e = at; e < n; ++e) y[e] = (float)(int)q[e] * s[e / COLS];
        }
    }
}

// ---------------------------------------------------------------------------
// The paged cache.  A page is a row of PAGE_BYTES: [keys | values], each
// [HK heads][PS rows][D], then (8-bit types) a fp32 scale for each of those
// rows, keys first.  KIND 0: fp32, 1: int8, 2: e4m3 (OCP).
// ---------------------------------------------------------------------------

template <int KIND, unsigned HK, unsigned PS, unsigned D, unsigned PAGES>
struct mt_cache {
    static constexpr unsigned ITEM = KIND == 0 ? 4u : 1u;
    static constexpr unsigned HALF = HK * PS * D * ITEM;  // bytes of a page's keys (or values)
    static constexpr unsigned SCALES = 2u * HALF;
    static constexpr unsigned PAGE = (2u * HALF + (KIND == 0 ? 0u : 8u * HK * PS) + 15u) / 16u * 16u;
    // Offsets in the cache: 32 bits (a register less, one base) up to 4 GiB of it.
    using offset = typename mt_count<((unsigned long long)PAGES * PAGE < (1ull << 32))>::type;
    MT_INLINE static offset row(unsigned page, unsigned part, unsigned head, unsigned r) {
        return (offset)page * PAGE + part * HALF + ((head * PS + r) * D) * ITEM;
    }
    MT_INLINE static offset scale(unsigned page, unsigned part, unsigned head, unsigned r) {
        return (offset)page * PAGE + SCALES + ((part * HK + head) * PS + r) * 4u;
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

// Four of them in the held type's bytes.
template <int KIND>
MT_INLINE unsigned mt_step_word_slow(mt_f32x4 v, float s, float inv) {
    unsigned word = 0u;
#pragma unroll 1
    for (unsigned i = 0; i < 4u; ++i) {
        const float q = mt_step_round<KIND>(i < 2u ? (i == 0u ? v[0] : v[1]) : (i == 2u ? v[2] : v[3]), s, inv);
        const unsigned byte = KIND == 1 ? (unsigned)(int)q : (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false);
        word |= (byte & 255u) << (8u * i);
    }
    return word;
}

// Four of a row's values in a held type's bytes, for a scale s of at least 2^-100 and
// its reciprocal.  Both are off by 2^-22 of the quotient at most, so it lies between the
// quotients by scales 2^-20 smaller and larger: where those round to the same four
// bytes (all but one in thousands), these are it; where not, the remainders decide
// (8192 tokens of 8 heads of 128 in e4m3: 28 us -> 22).
template <int KIND>
MT_INLINE unsigned mt_step_word(mt_f32x4 v, float s, float inv) {
    const auto word = [&](float by) {
        if constexpr (KIND == 1) {
            unsigned b[4];  // a whole number in a float's last byte, rounded there by the addition
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) b[i] = __float_as_uint(__builtin_fmaf(v[i], by, 12582912.0f));
            return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u),
                                         __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), 0x05040100u);
        } else {
            const unsigned lo = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[0] * by, v[1] * by, 0, false);
            return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * by, v[3] * by, (int)lo, true);
        }
    };
    const unsigned low = word(inv * (1.0f - 0x1.0p-20f));
    return low == word(inv * (1.0f + 0x1.0p-20f)) ? low : mt_step_word_slow<KIND>(v, s, inv);
}

// One row of D values held by 16 lanes (lane j has dims 64 c + 4 j .. + 3) into
// the cache.  `live`: whether the row is stored at all; every lane takes part
// in the exchange of the maximum.
template <int KIND, unsigned HK, unsigned PS, unsigned D, unsigned PAGES>
MT_INLINE void mt_cache_put(unsigned char* cache, const mt_f32x4 (&v)[(D + 63u) / 64u], unsigned j, bool live,
                            unsigned page, unsigned part, unsigned head, unsigned r) {
    using C = mt_cache<KIND, HK, PS, D, PAGES>;
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
        // The largest times fp32's 1 / peak, as a division by a scalar is elsewhere on GPUs (torch's
        // among them): two roundings, within 2^-23 of the quotient.  Caches that others
        // wrote are then the same bytes.  Values are rounded against the scale that is stored.
        const float s = fine ? top * (1.0f / (KIND == 2 ? 448.0f : 127.0f)) : NAN;
        // Near the smallest scales the reciprocal overflows and steps times the
        // scale lose bits: there both sides of the quotient are taken 2^64 larger.
        const float up = s < 0x1.0p-100f ? 0x1.0p+64f : 1.0f;
        const float big = s * up, inv = s > 0.f ? 1.0f / big : 0.f;
        if (!live) return;
        unsigned char* to = cache + C::row(page, part, head, r);
#pragma unroll
        for (unsigned c = 0; c < NC; ++c) {
            if (D % 64u != 0u && 64u * c + 4u * j >= D) continue;
            unsigned word = 0u;
            if (fine && s > 0.f) word = up == 1.0f ? mt_step_word<KIND>(v[c], s, inv) : mt_step_word_slow<KIND>(v[c] * up, big, inv);
            *reinterpret_cast<unsigned*>(to + 64u * c + 4u * j) = word;
        }
        if (j == 0u) *reinterpret_cast<float*>(cache + C::scale(page, part, head, r)) = s;
    }
}

// Bound: HBM, or the launch for few tokens.  8192 tokens of 8 heads of 128 in e4m3: 22.7
// us, 3.7 TB/s (15.3 us at a copy's rate), of which the look through the slots is about 4 us;
// in fp32 27 us, 5.0 TB/s.  The look grows with the square of the tokens: 32768 take 98 us.
//
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
    constexpr unsigned ROWS = TB * 2u * HK, MANY = ROWS >= 64u ? 4u : 1u;  // rows whose loads are on the way together
    const unsigned t0 = blockIdx.x * TB, j = threadIdx.x & 15u;
    unsigned lost = 0u;
    if (threadIdx.x == 0u) *dead = 0u;
    for (unsigned first = 0; first < ROWS; first += 16u * MANY) {
        mt_f32x4 x[MANY][NC];
        unsigned slot[MANY];
#pragma unroll
        for (unsigned u = 0; u < MANY; ++u) {
            const unsigned at = first + 16u * u + (threadIdx.x >> 4), part = at / HK % 2u, head = at % HK;
            const unsigned t = t0 + at / (2u * HK);
            const bool in = at < ROWS && t < tokens;
            slot[u] = in ? (unsigned)slots[t] : 0xFFFFFFFFu;
#pragma unroll
            for (unsigned c = 0; c < NC; ++c) {
                x[u][c] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
                const unsigned d = 64u * c + 4u * j;
                if (in && (D % 64u == 0u || d < D))
                    x[u][c] = part ? mt_row4<HK * D, VCS, true>(v + (size_t)t * VRS, head * D + d)
                                   : mt_row4<HK * D, KCS, true>(k + (size_t)t * KRS, head * D + d);
            }
        }
        if (first == 0u) {  // while the first rows are on the way
            unsigned mine[TB], hit = 0u;
            bool same[TB];
#pragma unroll
            for (unsigned i = 0; i < TB; ++i) mine[i] = t0 + i < tokens ? (unsigned)slots[t0 + i] : 0xFFFFFFFFu, same[i] = false;
            // Slots behind this workgroup's, four at a time (eight loads on the way): one
            // comparison for each of its tokens.  Then the ones around its own and the last.
            const unsigned from = (t0 + TB + 3u) / 4u, whole = tokens / 4u;
            for (unsigned q0 = from + threadIdx.x; q0 < whole; q0 += 8u * 256u) {
                mt_u32x4 s4[8];
#pragma unroll
                for (unsigned u = 0; u < 8u; ++u) {
                    s4[u] = mt_u32x4{0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
                    if (q0 + 256u * u < whole) s4[u] = reinterpret_cast<const mt_u32x4*>(slots)[q0 + 256u * u];
                }
#pragma unroll
                for (unsigned u = 0; u < 8u; ++u)
#pragma unroll
                    for (unsigned e = 0; e < 4u; ++e)
#pragma unroll
                        for (unsigned i = 0; i < TB; ++i) same[i] = same[i] | (s4[u][e] == mine[i]);
            }
            const auto look = [&](unsigned at) {
                const unsigned other = at < tokens ? (unsigned)slots[at] : 0xFFFFFFFFu;
#pragma unroll
                for (unsigned i = 0; i < TB; ++i) same[i] = same[i] | (other == mine[i] && at > t0 + i);
            };
            if (threadIdx.x < TB + 3u) look(t0 + 1u + threadIdx.x);
            if (threadIdx.x < 4u && 4u * whole + threadIdx.x > t0) look(4u * whole + threadIdx.x);
#pragma unroll
            for (unsigned i = 0; i < TB; ++i) hit |= same[i] ? 1u << i : 0u;
            __syncthreads();
            if (hit) atomicOr(dead, hit);
            __syncthreads();
            lost = *dead;
        }
#pragma unroll
        for (unsigned u = 0; u < MANY; ++u) {
            const unsigned at = first + 16u * u + (threadIdx.x >> 4);
            const bool live = slot[u] < SLOTS && !((lost >> (at / (2u * HK) % 32u)) & 1u);
            mt_cache_put<KIND, HK, PS, D, PAGES>(cache, x[u], j, live, slot[u] / PS, at / HK % 2u, at % HK, slot[u] % PS);
        }
    }
}

// Row r of k and v is slot slots[r] of the cache in 32 bits, zeros for a slot
// outside it.  16 lanes take a row of one head.  16384 slots of 8 heads of 128 in e4m3:
// 27 us, 6.2 TB/s (what was just written is in the last-level cache).
template <int KIND, unsigned HK, unsigned PS, unsigned D, unsigned PAGES>
MT_INLINE void mt_cache_read(const unsigned char* cache, const int* slots, float* k, float* v, unsigned rows) {
    using C = mt_cache<KIND, HK, PS, D, PAGES>;
    constexpr unsigned long long ALL = (unsigned long long)PAGES * PS;
    constexpr unsigned SLOTS = ALL > 0x80000000ull ? 0x80000000u : (unsigned)ALL;
    constexpr unsigned NC = (D + 63u) / 64u;
    constexpr unsigned MANY = 4u;  // rows whose loads are on the way together
    const unsigned j = threadIdx.x & 15u;
    unsigned slot[MANY], w[MANY][NC];
    mt_f32x4 x[MANY][NC];
    float s[MANY];
    bool live[MANY];
#pragma unroll
    for (unsigned u = 0; u < MANY; ++u) {
        const size_t at = ((size_t)blockIdx.x * MANY + u) * 16u + (threadIdx.x >> 4), r = at / (2u * HK);
        slot[u] = r < rows ? (unsigned)slots[r] : 0xFFFFFFFFu;
    }
#pragma unroll
    for (unsigned u = 0; u < MANY; ++u) {
        const size_t at = ((size_t)blockIdx.x * MANY + u) * 16u + (threadIdx.x >> 4);
        const unsigned part = (unsigned)(at / HK) % 2u, head = (unsigned)(at % HK);
        live[u] = slot[u] < SLOTS;
        const unsigned page = live[u] ? slot[u] / PS : 0u, in = live[u] ? slot[u] % PS : 0u;
        const unsigned char* from = cache + C::row(page, part, head, in);
        s[u] = 1.f;
        if constexpr (KIND != 0) s[u] = *reinterpret_cast<const float*>(cache + C::scale(page, part, head, in));
#pragma unroll
        for (unsigned c = 0; c < NC; ++c) {
            const unsigned d = 64u * c + 4u * j;
            if (D % 64u != 0u && d >= D) continue;
            if constexpr (KIND == 0) x[u][c] = mt_ld4(reinterpret_cast<const float*>(from) + d);
            else w[u][c] = *reinterpret_cast<const unsigned*>(from + d);
        }
    }
#pragma unroll
    for (unsigned u = 0; u < MANY; ++u) {
        const size_t at = ((size_t)blockIdx.x * MANY + u) * 16u + (threadIdx.x >> 4), r = at / (2u * HK);
        if (r >= rows) return;
        float* to = ((unsigned)(at / HK) % 2u ? v : k) + r * (HK * D) + (unsigned)(at % HK) * D;
#pragma unroll
        for (unsigned c = 0; c < NC; ++c) {
            const unsigned d = 64u * c + 4u * j;
            if (D % 64u != 0u && d >= D) continue;
            mt_f32x4 o;
            if constexpr (KIND == 0) o = x[u][c];
            else o = mt_held4<KIND>(w[u][c]) * s[u];
            if (!live[u]) o = mt_f32x4{0.f, 0.f, 0.f, 0.f};
            mt_st4_nt(to + d, o);
        }
    }
}

// ---------------------------------------------------------------------------
// Attention of one new token per sequence over the paged cache.
//
// The work is a row of units, STEP positions each of one sequence and one key head
// with HELD (at most 16) of the query heads that share it, sequence after sequence.
// The lengths are known on the device alone, so the workgroups of the launch cut
// that row into equal ranges there: a workgroup has the same share of a ragged batch
// as the others, and a table with room for far more positions costs nothing.  Where
// a range begins or ends inside a sequence's head, the parts go to the workspace and
// the last workgroup to arrive joins them, in their order.  Where the heads divide the
// workgroups well each has a row of units of its own (SIDES of them), cut alike: the
// heads of a page are then read at about one time (key heads of 128 in int8, 32 ragged
// sequences: 8 heads, up to 8192 keys 64 -> 63 us; 32 heads, up to 2048 69 -> 65).
//
// A piece is what a range has of one sequence's head.  Each costs as long as about
// 64 KB of the cache (its q, the waves' meeting), so it counts for as many units more
// where ranges are long (these two 65 -> 63 and 69 -> 65 us).  Its place, q and pages
// are there before the piece ahead of it ends, whose waves load its first tiles as they
// finish.  All of a piece's places are in scalar registers: loads of pages by lanes
// would wait for the tiles on the way before them (78 -> 63 us).
//
// Within a piece each of the workgroup's waves takes every WAVES-th tile of positions
// on its own, and they meet at the end.  With (n, g) = (lane % 16, lane / 16):
//
//   scores  S[position, column] = K . q by MFMAs whose rows are 16 positions:
//     lane (n, g) loads row n's dims VK (4 jj + g) .. + VK - 1 whole, and they are
//     its operands as they stand: which dims one MFMA takes together is the same
//     for K and q, so nothing is rearranged.
//   softmax S comes back with lane (n, g) holding column n at positions 4 g + i,
//     i < 4.  The running maximum m (in units of log 2: the scale carries
//     log2(e)) is shared by the four g of a head, the sum l is each lane's own
//     until the end.  The sums so far are rescaled only when some head's maximum
//     grows.
//   output  O[row, dim] += P . V: p[i] of positions 4 g + i is the P operand where
//     it stands, and lane (n, g) loads rows 4 g + i's dims VV (16 c + n) .. + VV - 1
//     of V.  No value changes lanes.
//
// KIND 0 (fp32): MFMAs 16x16x4 in fp32, tiles of 16 positions, and each value of V an
// operand by itself.
// 8 bits: the values are exact in bf16, and q and p are three bf16 parts each (hi, mid,
// lo: their 24 bits), an MFMA 16x16x32 for each in turn: tiles of 32 positions.  The fp32
// MFMAs take 64 values of the cache in 32 cycles, 4.9e12 a second on the GPU -- no more
// than HBM brings at one byte each; these take 512 in 48.  (The parts in columns of their
// own, four heads to an MFMA, took as long for 4 heads, and every lane's softmax once more
// for each further four: 8 heads 74 us for 58, 16 129 for 62.)  Four rows of V are
// exchanged byte by byte in registers, so that a dim's positions stand together.  (Weights
// below 2^-110 lose low parts.)
//
// A position's scales multiply its score and its weight.  A position that is
// masked (behind the length, or in a page outside the cache) scores -inf and its
// values are replaced by zeros, whatever its bytes hold.
//
// Bound: HBM, K and V once (32 sequences of 4080 keys, 8 key heads of 128, a copy's rate 50
// us: int8 with 1 to 8 query heads each 55 to 58, 16 62; e4m3 54 to 57; fp32 of a quarter
// of the keys 50 to 53).  Heads of 64 in 8 bits take as many vector instructions a position
// as longer ones' halves and are bound by them (40 to 43 us for 26), and rows of 16
// positions in two pages take more (pages of 20: 72 in int8).  One sequence of 131071 keys
// in e4m3 59 us, 4.7 TB/s; 2048 keys of 32 heads in fp32 15 us.  Beyond the stream a launch
// takes 5 us and a join over workgroups 4.
// ---------------------------------------------------------------------------

typedef short mt_i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned mt_u32x2 __attribute__((ext_vector_type(2)));

template <unsigned W>
MT_INLINE void mt_ld_words(unsigned (&to)[W], const unsigned char* p) {
    if constexpr (W == 4u) {
        const mt_u32x4 v = *reinterpret_cast<const mt_u32x4*>(p);
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
    } else if constexpr (W == 2u) {
        const mt_u32x2 v = *reinterpret_cast<const mt_u32x2*>(p);
        to[0] = v.x, to[1] = v.y;
    } else {
        to[0] = *reinterpret_cast<const unsigned*>(p);
    }
}

// Byte i of a, b, c, d together in to[i].
MT_INLINE void mt_bytes4(unsigned a, unsigned b, unsigned c, unsigned d, unsigned (&to)[4]) {
    const unsigned ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
    const unsigned cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
    to[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u);
    to[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
    to[2] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u);
    to[3] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
}

// Four 8-bit values as four bf16 in two words (exact).
template <int KIND>
MT_INLINE mt_u32x2 mt_held4_bf16(unsigned w) {
    if constexpr (KIND == 1) {
        const mt_f32x4 f = mt_held4<1>(w);
        return mt_u32x2{__builtin_amdgcn_perm(__float_as_uint(f.y), __float_as_uint(f.x), 0x07060302u),
                        __builtin_amdgcn_perm(__float_as_uint(f.w), __float_as_uint(f.z), 0x07060302u)};
    } else {
        return mt_u32x2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
    }
}

// What the upper half of x, a bf16, leaves of it.  Three times that is all of x: 8 bits of
// its 24 each, hi, mid and lo.
MT_INLINE float mt_bf16_rest(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }
// The upper halves of two floats in one word.
MT_INLINE unsigned mt_bf16_pair(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

MT_INLINE mt_f32x4 mt_mfma16_bf16(mt_u32x4 a, mt_u32x4 b, mt_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mt_bf16x8, a), __builtin_bit_cast(mt_bf16x8, b),
                                                   c, 0, 0, 0);
}

// v (op) over the four lanes of the same n.
template <typename OP>
MT_INLINE float mt_fold_g(float v, OP op) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The parts of a launch in the workspace, at device scope.
struct mt_parts : mt_sn_part {
    using mt_sn_part::mt_sn_part;
    MT_INLINE void put1(unsigned at, float v) const {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, at, 0, 16);
    }
    MT_INLINE float get1(unsigned at) const { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 16)); }
};

// A part (its maximum, sum of weights and sums) added to the joined ones, whose maximum is `top`.
MT_INLINE void mt_join(mt_f32x4& value, float& total, float& empty, float top, float m, float l, mt_f32x4 v) {
    const bool none = m == -INFINITY;
    const float u = none ? 0.f : __builtin_amdgcn_exp2f(m - top);
    empty += none ? l : 0.f;
    total += none ? 0.f : u * l;
#pragma unroll
    for (unsigned e = 0; e < 4u; ++e) value[e] += none ? 0.f : u * v[e];
}

// A value that is the same in all lanes, in scalar registers.
MT_INLINE unsigned mt_uniform(unsigned v) { return (unsigned)__builtin_amdgcn_readfirstlane((int)v); }
MT_INLINE unsigned long long mt_uniform(unsigned long long v) {
    return ((unsigned long long)mt_uniform((unsigned)(v >> 32)) << 32) | mt_uniform((unsigned)v);
}

// The units of a launch: which sequence and head they belong to, and which
// workgroup has them.  The first `extra` ones of a sequence's head hold nothing: where
// a workgroup has four or more (with fewer, equal numbers of real ones count).  Whole
// waves call its functions; their results are uniform.
template <unsigned ROWS, unsigned STEP, unsigned MOST, unsigned HEADS, unsigned GROUPS, unsigned EXTRA>
struct mt_units {
    // Every product of units and workgroups fits in N.
    static constexpr unsigned long long ROOM = (unsigned long long)ROWS * HEADS * ((MOST + STEP - 1ull) / STEP + EXTRA);
    using N = typename mt_count<(ROOM * (GROUPS + 1ull) < (1ull << 32))>::type;
    static constexpr int LAST = ROWS < 64u ? (int)ROWS - 1 : 63;  // the lane whose sum is a scan's whole
    const int* lengths;
    // The 64 sequences from from_, before_ units behind the first: the steps of this
    // lane's, and the sum of those up to it.
    unsigned steps_, sum_, from_;
    N before_;
    unsigned workgroups, extra;
    N all;

    MT_INLINE static unsigned length(int asked) { return asked < 0 ? 0u : (unsigned)asked < MOST ? (unsigned)asked : MOST; }
    // The steps of this lane's sequence of the 64 from b0, and the sum of those up to
    // it.  A sequence without keys has a step too: its zeros are somebody's.
    MT_INLINE void scan(unsigned b0, unsigned& steps, unsigned& sum) const {
        const unsigned b = b0 + mt_lane();
        const unsigned n = b < ROWS ? (length(lengths[b]) + STEP - 1u) / STEP : 0u;
        steps = b < ROWS && n == 0u ? 1u : n;
        sum = steps;
#pragma unroll
        for (unsigned off = 1u; off < (ROWS < 64u ? ROWS : 64u); off <<= 1) {
            const unsigned v = (unsigned)__shfl_up((int)sum, off, 64);
            if (mt_lane() >= off) sum += v;
        }
    }
    MT_INLINE void init(const int* lengths_, unsigned most) {
        lengths = lengths_;
        all = 0u, extra = 0u;
        for (unsigned b0 = 0; b0 < ROWS; b0 += 64u) {
            scan(b0, steps_, sum_);
            all += (N)(unsigned)__builtin_amdgcn_readlane((int)sum_, LAST) * HEADS;
        }
        if (all >= (N)4u * most) {
            extra = EXTRA;
            all += (N)ROWS * EXTRA * HEADS;
        }
        workgroups = all < most ? (unsigned)all : most;
        from_ = 0u, before_ = 0u;
        if (ROWS > 64u) scan(0u, steps_, sum_);
    }
    // The sequence that unit u < all belongs to, the units before it and its steps; from
    // call to call u grows.
    MT_INLINE unsigned find(N u, N& at, unsigned& steps) {
        for (;;) {
            const unsigned sum = sum_ + extra * (mt_lane() + 1u);
            const unsigned long long past = __ballot(before_ + (N)sum * HEADS > u);
            if (past || from_ + 64u >= ROWS) {
                const int who = __builtin_ctzll(past);
                steps = (unsigned)__builtin_amdgcn_readlane((int)steps_, who);
                at = before_ + (N)((unsigned)__builtin_amdgcn_readlane((int)sum, who) - steps - extra) * HEADS;
                return from_ + (unsigned)who;
            }
            before_ += (N)(unsigned)__builtin_amdgcn_readlane((int)sum, LAST) * HEADS;
            from_ += 64u;
            scan(from_, steps_, sum_);
        }
    }
    MT_INLINE N first(unsigned w) const { return mt_uniform(all * w / workgroups); }
    MT_INLINE unsigned owner(N u) const { return (unsigned)(((u + 1u) * workgroups - 1u) / all); }
};

template <int KIND, unsigned HK, unsigned PS, unsigned D, unsigned PAGES, unsigned WIDTH, unsigned SHARE, unsigned HELD,
          unsigned WAVES, unsigned GROUPS, unsigned BATCH, unsigned ROWS, unsigned QRS, unsigned QCS>
MT_INLINE void mt_paged_attention(const float* q, const unsigned char* cache, const int* pages, const int* lengths,
                                  float* o, double scale, float* ws, unsigned char* lds) {
    using C = mt_cache<KIND, HK, PS, D, PAGES>;
    constexpr unsigned ITEM = C::ITEM, PARTS = (SHARE + HELD - 1u) / HELD;
    constexpr bool WIDE = KIND == 0;
    constexpr unsigned BLOCKS = WIDE ? 1u : 2u, TILE = 16u * BLOCKS;       // positions of a tile
    constexpr unsigned SPLIT = WIDE ? 1u : 3u;                             // operands a value of q or p makes
    constexpr unsigned VK = WIDE ? 4u : D % 64u == 0u ? 16u : D % 32u == 0u ? 8u : 4u, NJ = D / (4u * VK);
    constexpr unsigned VV = WIDE || D <= 64u ? 4u : 8u, NV = (D + 16u * VV - 1u) / (16u * VV);
    constexpr unsigned KW = VK * ITEM / 4u, VW = VV * ITEM / 4u, FLOATS = (HELD * (D + 2u) + 3u) / 4u * 4u;
    constexpr unsigned STEP = TILE * WAVES;
    constexpr bool ONE_PAGE = PS % 16u == 0u;  // 16 positions lie in one page
    const unsigned lane = mt_lane(), n = lane & 15u, g = lane >> 4, wave = mt_wave();

    // LDS: the operands of q, 16 bytes a lane each, of two pieces in turn; then the waves'
    // parts, [WAVES][HELD][D] sums and [WAVES][HELD] of m and of l.
    constexpr unsigned KO = WIDE ? 4u : VK < 8u ? VK : 8u, NO = VK / KO, OPS = NJ * NO;
    mt_u32x4* q2 = reinterpret_cast<mt_u32x4*>(lds);  // [2][SPLIT][OPS][64]
    float* sums = reinterpret_cast<float*>(lds + 2u * SPLIT * OPS * 1024u);
    float* ms = sums + WAVES * HELD * D;
    float* ls = ms + WAVES * HELD;
    unsigned* flag = reinterpret_cast<unsigned*>(ls + WAVES * HELD);

    constexpr unsigned UNIT = STEP * 2u * D * ITEM, EXTRA = (65536u + UNIT / 2u) / UNIT;
    constexpr unsigned HEADS = HK * PARTS, SIDES = GROUPS / HEADS * HEADS * 16u >= GROUPS * 15u ? HEADS : 1u;
    constexpr unsigned RANGES = GROUPS / SIDES;
    using U = mt_units<ROWS, STEP, WIDTH * PS, HEADS / SIDES, RANGES, EXTRA>;
    const unsigned range = blockIdx.x / SIDES, side = blockIdx.x % SIDES;
    U units;
    // (a batch larger than the workspace was laid out for is not split)
    units.init(lengths, gridDim.z <= BATCH ? RANGES : 1u);
    if (range >= units.workgroups) return;
    const typename U::N end = units.first(range + 1u);

    // A piece of the range: `taken` of the `steps` of a sequence's head, from `step` on
    // (positions first .. last - 1), the head's first unit being `begins`.
    struct piece {
        typename U::N begins;
        unsigned b, head, part, step, steps, taken, first, last, tiles;
        const int* table;
    };
    typename U::N unit = units.first(range);
    const auto piece_at = [&]() {
        piece p;
        typename U::N before;
        p.b = units.find(unit, before, p.steps);
        const unsigned in = (unsigned)(unit - before), wide = p.steps + units.extra;
        const unsigned pair = HEADS == SIDES ? side : mt_uniform(in / wide), at = HEADS == SIDES ? in : mt_uniform(in % wide);
        p.part = pair % PARTS, p.head = pair / PARTS;
        p.begins = unit - at + units.extra;
        p.step = at > units.extra ? at - units.extra : 0u;
        unit = p.begins + p.step;
        const typename U::N left = unit < end ? end - unit : 0u;
        p.taken = left < p.steps - p.step ? (unsigned)left : p.steps - p.step;
        unit += p.taken;
        const unsigned len = units.length(lengths[p.b]);
        p.first = p.step * STEP;
        p.last = len < (p.step + p.taken) * STEP ? len : (p.step + p.taken) * STEP;
        p.last = p.last < p.first ? p.first : p.last;
        p.tiles = (p.last - p.first + TILE - 1u) / TILE;
        p.table = pages + (size_t)p.b * WIDTH;
        return p;
    };
    // The page of row n of block `bi` of a tile (of the block, where it lies in one).
    const auto page_of = [&](const piece& p, unsigned ti, unsigned bi) -> int {
        const unsigned t0 = p.first + TILE * ti + 16u * bi;
        if constexpr (ONE_PAGE) {
            return t0 < p.last ? __builtin_amdgcn_readfirstlane(p.table[t0 / PS]) : -1;
        } else {
            return t0 + n < p.last ? p.table[(t0 + n) / PS] : -1;
        }
    };
    const auto row_page = [&](int page, unsigned i) -> int { return ONE_PAGE ? page : __shfl(page, (int)(4u * g + i), 64); };
    const auto safe = [&](int page) -> unsigned { return (unsigned)page < PAGES ? (unsigned)page : 0u; };

    unsigned kw[BLOCKS][NJ][KW], vw[BLOCKS][4][NV][VW];
    float ks[BLOCKS][4], vs[BLOCKS][4];
    const auto load_k = [&](unsigned start, unsigned head, unsigned ti, const int (&page)[BLOCKS]) {
#pragma unroll
        for (unsigned bi = 0; bi < BLOCKS; ++bi) {
            const unsigned t0 = start + TILE * ti + 16u * bi;
            const typename C::offset p = C::row(safe(page[bi]), 0u, head, (t0 + n) % PS) + g * (VK * ITEM);
#pragma unroll
            for (unsigned jj = 0; jj < NJ; ++jj) mt_ld_words<KW>(kw[bi][jj], cache + p + jj * (4u * VK * ITEM));
            if constexpr (!WIDE) {
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i)
                    ks[bi][i] = *reinterpret_cast<const float*>(
                        cache + C::scale(safe(row_page(page[bi], i)), 0u, head, (t0 + 4u * g + i) % PS));
            }
        }
    };
    const auto load_v = [&](unsigned start, unsigned head, unsigned ti, const int (&page)[BLOCKS]) {
#pragma unroll
        for (unsigned bi = 0; bi < BLOCKS; ++bi) {
            const unsigned t0 = start + TILE * ti + 16u * bi;
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                const unsigned pg = safe(row_page(page[bi], i)), r = (t0 + 4u * g + i) % PS;
                const typename C::offset p = C::row(pg, 1u, head, r);
#pragma unroll
                for (unsigned c = 0; c < NV; ++c) {
                    unsigned d = VV * (16u * c + n);
                    if (D % (16u * VV) != 0u && d >= D) d = 0u;  // (columns that no output takes)
                    mt_ld_words<VW>(vw[bi][i][c], cache + (p + d * ITEM));
                }
                if constexpr (!WIDE) vs[bi][i] = *reinterpret_cast<const float*>(cache + C::scale(pg, 1u, head, r));
            }
        }
    };

    // Slot 2 w of the workspace is the part of workgroup w that began before it, 2 w + 1
    // the part that begins in it: [HELD][D] sums, [HELD] of m, [HELD] of l.  Four dims a
    // lane, written and read at device scope.
    const unsigned own = blockIdx.z * gridDim.x + side * RANGES;  // this side's counters and slots
    float* slots = ws + MT_WS_HEAD + (size_t)own * 2u * FLOATS;
    constexpr unsigned QUADS = HELD * D / 4u, LANES = 64u * WAVES;
    // Lanes that share four dims of a head when the parts of other workgroups are joined,
    // and parts of each whose loads are on the way together.
    constexpr unsigned SHARED = QUADS * WAVES <= LANES ? WAVES : LANES / QUADS > 0u ? LANES / QUADS : 1u;
    constexpr unsigned DEEP = SHARED > 2u ? 4u : 16u;
    const auto put = [&](unsigned b_, unsigned head_, unsigned part_, unsigned at, mt_f32x4 value, float top, float total) {
        const unsigned h = at / (D / 4u);
        if (part_ * HELD + h >= SHARE) return;
        const float by = 1.0f / total, none = total > 0.f ? NAN : 0.f;
        mt_f32x4 r = value * by;
        if (top == -INFINITY) r = mt_f32x4{none, none, none, none};
        mt_st4(o + ((size_t)b_ * HK * SHARE + head_ * SHARE + part_ * HELD + h) * D + 4u * (at % (D / 4u)), r);
    };

    // q, times the scale, as the MFMAs take it: column h, dim d element d % VK % KO of operand
    // (d / (4 VK), d % VK / KO) in the lanes of g = d / VK % 4; for 8 bits hi, mid and lo.
    const auto put_q = [&](const piece& p, mt_u32x4* qs) {
        const float by = (float)(scale * 1.4426950408889634);
        const float* qr = q + (size_t)p.b * QRS;
        for (unsigned at = threadIdx.x; at < 16u * D; at += 64u * WAVES) {
            const unsigned h = at / D, d = at % D, op = d / (4u * VK) * NO + d % VK / KO, e = d % KO, gd = d / VK % 4u;
            float v = 0.f;
            if (h < HELD && p.part * HELD + h < SHARE) v = qr[(size_t)((p.head * SHARE + p.part * HELD + h) * D + d) * QCS] * by;
            mt_u32x4* to = qs + op * 64u + gd * 16u + h;
            if constexpr (WIDE) {
                reinterpret_cast<float*>(to)[e] = v;
            } else {
#pragma unroll
                for (unsigned j = 0; j < SPLIT; ++j, v = mt_bf16_rest(v))
                    reinterpret_cast<unsigned short*>(to + j * (OPS * 64u))[e] = (unsigned short)(__float_as_uint(v) >> 16);
            }
        }
    };

    piece now = piece_at();
    if (now.taken == 0u) return;
    int page[BLOCKS], page_next[BLOCKS];
#pragma unroll
    for (unsigned bi = 0; bi < BLOCKS; ++bi) page[bi] = page_of(now, wave, bi), page_next[bi] = page_of(now, wave + WAVES, bi);
    load_k(now.first, now.head, wave, page);
    load_v(now.first, now.head, wave, page);
    put_q(now, q2);
    for (unsigned turn = 0;; turn ^= 1u) {
    // The piece after this one: known, its pages and q there, from this one's start, and
    // its first tile on the way from each wave's last one.  (Pages that are not there are
    // -1, whose loads are page 0's and whose rows are masked: a wave without a tile of a
    // piece passes through one of those.)
    piece next = now;
    next.taken = next.tiles = next.first = next.last = 0u;
    if (unit < end) next = piece_at();
    const bool again = next.taken > 0u;
    int page_then[BLOCKS], page_then_next[BLOCKS];
#pragma unroll
    for (unsigned bi = 0; bi < BLOCKS; ++bi)
        page_then[bi] = page_of(next, wave, bi), page_then_next[bi] = page_of(next, wave + WAVES, bi);
    if (again) put_q(next, q2 + (turn ^ 1u) * (SPLIT * OPS * 64u));
    const mt_u32x4* qs = q2 + turn * (SPLIT * OPS * 64u);
    __syncthreads();

    mt_f32x4 acc[NV * VV];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (unsigned i = 0; i < NV * VV; ++i) acc[i] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
    bool seen = false;
#pragma unroll 1
    for (unsigned ti = wave;; ti += WAVES) {
        int page_after[BLOCKS];
#pragma unroll
        for (unsigned bi = 0; bi < BLOCKS; ++bi) page_after[bi] = page_of(now, ti + 2u * WAVES, bi);
        const bool more = ti + WAVES < now.tiles;
        const unsigned start = more ? now.first : next.first, head = more ? now.head : next.head, tn = more ? ti + WAVES : wave;
        mt_f32x4 s[BLOCKS];
        if constexpr (WIDE) {
            mt_f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (unsigned jj = 0; jj < NJ; ++jj) {
                const mt_f32x4 qv = __builtin_bit_cast(mt_f32x4, qs[jj * 64u + lane]);
#pragma unroll
                for (unsigned e = 0; e < 4u; e += 2u) {
                    s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[0][jj][e]), qv[e], s0, 0, 0, 0);
                    s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[0][jj][e + 1u]), qv[e + 1u], s1, 0, 0, 0);
                }
            }
            s[0] = s0 + s1;
        } else {
            // hi's products in one sum, mid's and lo's, 2^-8 of them, in another: each
            // rounds to its own size.
            mt_f32x4 sum[BLOCKS][2];
#pragma unroll
            for (unsigned bi = 0; bi < BLOCKS; ++bi) sum[bi][0] = sum[bi][1] = mt_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (unsigned op = 0; op < OPS; ++op) {
                mt_u32x4 k8[BLOCKS];  // (the first two words where KO is 4)
#pragma unroll
                for (unsigned bi = 0; bi < BLOCKS; ++bi) {
                    const unsigned* k = &kw[bi][op / NO][KO / 4u * (op % NO)];
                    const mt_u32x2 lo = mt_held4_bf16<KIND>(k[0]), hi = KO == 8u ? mt_held4_bf16<KIND>(k[KO / 8u]) : lo;
                    k8[bi] = mt_u32x4{lo.x, lo.y, hi.x, hi.y};
                }
#pragma unroll
                for (unsigned j = 0; j < SPLIT; ++j) {
                    const mt_u32x4 q8 = qs[(j * OPS + op) * 64u + lane];
#pragma unroll
                    for (unsigned bi = 0; bi < BLOCKS; ++bi) {
                        mt_f32x4& to = sum[bi][j ? 1u : 0u];
                        if constexpr (KO == 8u)
                            to = mt_mfma16_bf16(k8[bi], q8, to);
                        else
                            to = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(mt_i16x4, mt_u32x2(k8[bi].xy)),
                                                                           __builtin_bit_cast(mt_i16x4, mt_u32x2(q8.xy)), to, 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (unsigned bi = 0; bi < BLOCKS; ++bi)
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i) s[bi][i] = (sum[bi][0][i] + sum[bi][1][i]) * ks[bi][i];
        }
        if (!more) {
#pragma unroll
            for (unsigned bi = 0; bi < BLOCKS; ++bi) page_next[bi] = page_then[bi], page_after[bi] = page_then_next[bi];
        }
        if (more || again) load_k(start, head, tn, page_next);
        bool ok[BLOCKS][4], any = false, all = true;
#pragma unroll
        for (unsigned bi = 0; bi < BLOCKS; ++bi)
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                ok[bi][i] = (unsigned)row_page(page[bi], i) < PAGES && now.first + TILE * ti + 16u * bi + 4u * g + i < now.last;
                any = any || ok[bi][i];
                all = all && ok[bi][i];
            }
        seen = seen || __any(any);
        const bool whole = __all(all);
        if (!whole) {
#pragma unroll
            for (unsigned bi = 0; bi < BLOCKS; ++bi)
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i)
                    if (!ok[bi][i]) s[bi][i] = -INFINITY;
        }
        float p[BLOCKS][4], top = -INFINITY;
#pragma unroll
        for (unsigned bi = 0; bi < BLOCKS; ++bi)
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) top = __builtin_fmaxf(top, s[bi][i]);
        top = mt_fold_g(top, [](float x, float y) { return __builtin_fmaxf(x, y); });
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
#pragma unroll
        for (unsigned bi = 0; bi < BLOCKS; ++bi)
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                const float e = __builtin_amdgcn_exp2f(s[bi][i] - base);
                l += e;
                p[bi][i] = WIDE ? e : e * vs[bi][i];
            }
        if (!whole) {
#pragma unroll
            for (unsigned bi = 0; bi < BLOCKS; ++bi)
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i) {
                    if (ok[bi][i]) continue;
                    p[bi][i] = 0.f;
#pragma unroll
                    for (unsigned c = 0; c < NV; ++c)
#pragma unroll
                        for (unsigned w = 0; w < VW; ++w) vw[bi][i][c][w] = 0u;
                }
        }
        if constexpr (WIDE) {
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i)
#pragma unroll
                for (unsigned c = 0; c < NV; ++c)
#pragma unroll
                    for (unsigned e = 0; e < VV; ++e)
                        acc[VV * c + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[0][i], __uint_as_float(vw[0][i][c][e]),
                                                                               acc[VV * c + e], 0, 0, 0);
        } else {
            mt_u32x4 pb[SPLIT];
#pragma unroll
            for (unsigned j = 0; j < SPLIT; ++j) {
                pb[j] = mt_u32x4{mt_bf16_pair(p[0][0], p[0][1]), mt_bf16_pair(p[0][2], p[0][3]),
                                 mt_bf16_pair(p[BLOCKS - 1u][0], p[BLOCKS - 1u][1]), mt_bf16_pair(p[BLOCKS - 1u][2], p[BLOCKS - 1u][3])};
#pragma unroll
                for (unsigned bi = 0; bi < BLOCKS; ++bi)
#pragma unroll
                    for (unsigned i = 0; i < 4u; ++i) p[bi][i] = mt_bf16_rest(p[bi][i]);
            }
#pragma unroll
            for (unsigned c = 0; c < NV; ++c)
#pragma unroll
                for (unsigned w = 0; w < VW; ++w) {
                    unsigned lo[4], hi[4];
                    mt_bytes4(vw[0][0][c][w], vw[0][1][c][w], vw[0][2][c][w], vw[0][3][c][w], lo);
                    mt_bytes4(vw[BLOCKS - 1u][0][c][w], vw[BLOCKS - 1u][1][c][w], vw[BLOCKS - 1u][2][c][w],
                              vw[BLOCKS - 1u][3][c][w], hi);
#pragma unroll
                    for (unsigned u = 0; u < 4u; ++u) {
                        const mt_u32x2 v0 = mt_held4_bf16<KIND>(lo[u]), v1 = mt_held4_bf16<KIND>(hi[u]);
                        const mt_u32x4 v8 = {v0.x, v0.y, v1.x, v1.y};
#pragma unroll
                        for (unsigned j = 0; j < SPLIT; ++j)
                            acc[VV * c + 4u * w + u] = mt_mfma16_bf16(pb[j], v8, acc[VV * c + 4u * w + u]);
                    }
                }
        }
        if (more || again) load_v(start, head, tn, page_next);
#pragma unroll
        for (unsigned bi = 0; bi < BLOCKS; ++bi) page[bi] = page_next[bi], page_next[bi] = page_after[bi];
        if (!more) break;
    }

    const bool opening = now.step == 0u, entire = now.taken == now.steps;

    // A part weighs 2^(m - the largest m); one whose scores are all -inf weighs nothing
    // and says in l whether it has positions: a softmax over such scores alone is 0 / 0,
    // one over no positions gives zeros.  Maxima pass over scores that are NaN, sums do not:
    // a part whose sum is NaN joins as one with a maximum, so that its NaN comes through.
    l = mt_fold_g(l, [](float x, float y) { return x + y; });
    if (l != l) m = 0.f;
    else if (m == -INFINITY) l = seen ? 1.f : 0.f;
    if (g == 0u && n < HELD) {
        ms[wave * HELD + n] = m;
        ls[wave * HELD + n] = l;
    }
#pragma unroll
    for (unsigned c = 0; c < NV; ++c)
#pragma unroll
        for (unsigned e = 0; e < VV; ++e) {
            const unsigned d = VV * (16u * c + n) + e;
            if (D % (16u * VV) != 0u && d >= D) continue;
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i)
                if (4u * g + i < HELD) sums[(wave * HELD + 4u * g + i) * D + d] = acc[VV * c + e][i];
        }
    __syncthreads();

#pragma unroll 1
    for (bool others = false;; others = true) {
        // The waves' parts, or those of the workgroups as SHARED lanes joined them.
        const mt_parts mine(slots + (size_t)(2u * range + (opening ? 1u : 0u)) * FLOATS, FLOATS * 4u);
#pragma unroll 1
        for (unsigned at = threadIdx.x; at < QUADS; at += LANES) {
            const unsigned h = at / (D / 4u);
            float top = -INFINITY, empty = 0.f, total = 0.f;
            mt_f32x4 value = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (unsigned w = 0; w < WAVES; ++w) top = __builtin_fmaxf(top, ms[w * HELD + h]);
#pragma unroll
            for (unsigned w = 0; w < WAVES; ++w)
                mt_join(value, total, empty, top, ms[w * HELD + h], ls[w * HELD + h],
                        *reinterpret_cast<const mt_f32x4*>(sums + w * HELD * D + 4u * at));
            if (top == -INFINITY) total = empty;
            if (entire || others) {
                put(now.b, now.head, now.part, at, value, top, total);
            } else {
                mine.put(16u * at, value);
                if (at % (D / 4u) == 0u) {
                    mine.put1(4u * (HELD * D + h), top);
                    mine.put1(4u * (HELD * D + HELD + h), total);
                }
            }
        }
        if (entire || others) break;

        // The last workgroup of the sequence's head to arrive joins the parts.
        const unsigned from = units.owner(now.begins), parts = units.owner(now.begins + now.steps - 1u) - from + 1u;
        unsigned* counter = reinterpret_cast<unsigned*>(ws) + own + from;
        if (!mt_sn_arrive(counter, parts, flag)) break;
        const mt_parts all_parts(slots, RANGES * 2u * FLOATS * 4u);
        const unsigned who = SHARED > 1u ? threadIdx.x / QUADS : 0u;
        for (unsigned at = SHARED > 1u ? threadIdx.x % QUADS : threadIdx.x; at < QUADS && who < SHARED; at += LANES) {
            const unsigned h = at / (D / 4u);
            float top = -INFINITY, empty = 0.f, total = 0.f;
            mt_f32x4 value = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (unsigned i0 = who; i0 < parts; i0 += DEEP * SHARED) {
                float pm[DEEP], pl[DEEP], most = top;
                mt_f32x4 pv[DEEP];
#pragma unroll
                for (unsigned k = 0; k < DEEP; ++k) {
                    const unsigned i = i0 + k * SHARED < parts ? i0 + k * SHARED : i0;
                    const unsigned p = (2u * (from + i) + (i == 0u ? 1u : 0u)) * FLOATS * 4u;
                    pm[k] = all_parts.get1(p + 4u * (HELD * D + h));
                    pl[k] = all_parts.get1(p + 4u * (HELD * D + HELD + h));
                    pv[k] = all_parts.get(p + 16u * at);
                }
#pragma unroll
                for (unsigned k = 0; k < DEEP; ++k) most = __builtin_fmaxf(most, pm[k]);
                if (most > top) {
                    const float by = __builtin_amdgcn_exp2f(top - most);
                    total *= by, value = value * by;
                    top = most;
                }
#pragma unroll
                for (unsigned k = 0; k < DEEP; ++k)
                    if (k == 0u || i0 + k * SHARED < parts) mt_join(value, total, empty, top, pm[k], pl[k], pv[k]);
            }
            *reinterpret_cast<mt_f32x4*>(sums + who * HELD * D + 4u * at) = value;
            if (at % (D / 4u) == 0u) {
                ms[who * HELD + h] = top;
                ls[who * HELD + h] = top == -INFINITY ? empty : total;
            }
        }
        for (unsigned at = threadIdx.x; at < (WAVES - SHARED) * HELD; at += LANES)
            ms[SHARED * HELD + at] = -INFINITY, ls[SHARED * HELD + at] = 0.f;
        __syncthreads();
    }
    if (!again) return;
    now = next;
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
// What is lost is under 2^-30 of that power of two per element.  Where four values in a
// row, not all zero, lie below 2^-9 of it -- a few outliers stand far above the rest --
// the rest could do with more, and the block goes without digits: it is added in fp32, as
// is one that holds an infinity or a NaN.  So an element is off by at most 2^-21 of the
// largest of its four, whatever the outliers' weights are.  Such a block costs about as
// much again (one channel 1e4 times the others: 1 row, 11008 x 4096 8.2 -> 8.7 us; 4 rows,
// 131072 x 4096 62 -> 75, in four blocks of the 32 112; all 32 blocks of one row 19); the
// look for them costs others up to 4 % (8 rows, 11008 x 8192: 23.3 -> 24.3).  (A group's sum, up to 2^44, is times its scale
// before x's exponent comes in: scales below 2^83.)  One or two rows of x (XR) make the
// digits of four or two blocks at once instead.  x in 8 bits is 16 rows as it stands.
//
// With (n, g) = (lane % 16, lane / 16): lane (n, g) loads 16 bytes of weight row n, q of
// k = 32 g .. + 31 of a block of 128, even ones in the low nibbles.  xor 0x88 turns q
// into q - 8 in two's complement, and in the high nibble of a byte that is 16 (q - 8)
// as int8: (v << 4) & 0xF0.. are a word's four even k, v & 0xF0.. its odd ones, and
// those two words in turn are the operand, in weights and digits alike.  Groups of 64
// or 32: the words of a group are spread over all g first, by exchanges of halves and
// rows of the wave (permlane swaps: 2 or 4 for 32 k a lane), so that an MFMA takes
// one group whole.
//
// SHARED: the digits of x stay in LDS, PB blocks of k at a time, and every wave takes
// weight tiles of its own, row after row; otherwise the waves of a workgroup share its
// weight rows and split k, each making the digits of its part as it goes, so that few
// weight rows still keep many loads in flight.
//
// Bound: HBM, the weights once, for many weight rows (n x k: 4 rows of x, 131072 x 4096:
// 54 us, 5.3 TB/s).  For few a wave's share of k is a handful of blocks, and the waits for
// them and the making of digits (about 12 vector instructions a value, in every workgroup)
// count: 1 row, 11008 x 4096 7.3 us; 16 rows in 8 bits, 4096 x 11008 10.5; 5 rows, 4099 x
// 5024 in groups of 32 15, of which vector instructions are 8; 11008 x 8192 in groups of 128
// (48 MB, a copy's rate 8.7 us) 1 row 14, 8 rows 24, 16 rows 35, in 8 bits 15 and 22.
// ---------------------------------------------------------------------------

// The whole number that an MFMA's four digit rows stand for.
MT_INLINE float mt_digits(mt_i32x4 c) {
    const int hi = c[0] * 256 + c[1], lo = c[2] * 256 + c[3];
    return __builtin_fmaf((float)hi, 65536.0f, (float)lo);
}

// The largest of a value's bits over 16 lanes (DPP: quads, halves, rows mirrored).
MT_INLINE unsigned mt_max16(unsigned v) {
    const auto step = [&](unsigned other) { v = v > other ? v : other; };
    step((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    step((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
    step((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
    step((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
    return v;
}

// The larger of two; NaN where one is.
MT_INLINE float mt_maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// a's upper half of the wave for b's lower half; a's odd rows of 16 for b's even ones.
MT_INLINE void mt_swap32(unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
}
MT_INLINE void mt_swap16(unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
}

// What one MFMA of a block takes: 16 bytes a lane of 64 k, or 8 of 32.  A block is two
// of the first kind (both of one group of 128, or one of each group of 64), or four.
template <unsigned GB>
struct mt_operand {
    static constexpr unsigned COUNT = GB == 4u ? 4u : 2u, WORDS = GB == 4u ? 2u : 4u;
    // Where in a row's 128 bytes of a block, in digits (the even and the odd k of 8 in turn).
    MT_INLINE static unsigned at(unsigned i, unsigned g) {
        return GB == 1u ? 32u * g + 16u * i : GB == 2u ? 64u * i + 32u * (g % 2u) + 16u * (g / 2u) : 32u * i + 8u * g;
    }
    // This lane's words of weights, k 32 g .. + 31, so that words WORDS / 2 * i .. make operand i.
    MT_INLINE static void spread(unsigned (&w)[4]) {
        if constexpr (GB > 1u) {
            mt_swap32(w[0], w[2]);
            mt_swap32(w[1], w[3]);
        }
        if constexpr (GB == 4u) {
            mt_swap16(w[0], w[1]);
            mt_swap16(w[2], w[3]);
        }
    }
    MT_INLINE static mt_i32x4 product(const unsigned (&a)[WORDS], const unsigned (&b)[WORDS], mt_i32x4 c) {
        if constexpr (GB == 4u) {
            return __builtin_amdgcn_mfma_i32_16x16x32_i8((long)(((unsigned long long)a[1] << 32) | a[0]),
                                                         (long)(((unsigned long long)b[1] << 32) | b[0]), c, 0, 0, 0);
        } else {
            return __builtin_amdgcn_mfma_i32_16x16x64_i8(mt_i32x4{(int)a[0], (int)a[1], (int)a[2], (int)a[3]},
                                                         mt_i32x4{(int)b[0], (int)b[1], (int)b[2], (int)b[3]}, c, 0, 0, 0);
        }
    }
};

template <bool EIGHT, bool SHARED, unsigned PB, unsigned XR, unsigned SETS, unsigned K, unsigned N, unsigned GROUP, bool ZEROS, unsigned R,
          unsigned U, unsigned WAVES, unsigned XRS, unsigned XCS>
MT_INLINE void mt_matmul_int4(const float* x, const signed char* x8, const float* xs, const unsigned char* w,
                              const float* scales, const float* zeros, float* y, unsigned rows, unsigned char* lds) {
    constexpr unsigned NB = (K + 127u) / 128u, NG = K / GROUP, GB = 128u / GROUP, GU = GB * U, ACC = EIGHT ? 4u : SETS;
    constexpr unsigned NC = (NB + U - 1u) / U;        // chunks of U blocks, whose loads are in flight together
    constexpr unsigned BL = EIGHT ? 1u : 4u / XR;     // blocks of x made into digits at once
    constexpr unsigned DIGITS = 512u * XR * SETS;     // bytes of a block's digits: [SETS][4 XR rows][128]
    constexpr bool RAGGED = K % (128u * U) != 0u;
    static_assert(SHARED || U / BL * SETS <= 16u, "a bit for each row of a chunk's blocks");
    static_assert(U % BL == 0u && (!SHARED || PB % U == 0u), "makings of digits are whole in a chunk, chunks in a phase");
    using OP = mt_operand<GB>;
    const unsigned lane = mt_lane(), n = lane & 15u, g = lane >> 4, wave = mt_wave();
    const unsigned m0 = blockIdx.y * 16u;
    const unsigned c0 = SHARED ? 0u : NC * wave / WAVES, c1 = SHARED ? NC : NC * (wave + 1u) / WAVES;
    constexpr unsigned PHASES = SHARED ? (NB + PB - 1u) / PB : 1u;

    // x for one making of digits: rows 4 t + g % XR of block blk + g / XR, k 8 n .. + 7; x
    // in 8 bits: row n's share of the operands of block blk.
    constexpr unsigned XV = EIGHT ? 2u : 2u * SETS;
    const auto load_x = [&](unsigned blk, mt_u32x4 (&to)[XV]) {
        if constexpr (EIGHT && SHARED) {
            const unsigned k = blk * 128u + 32u * g;
            const bool in = m0 + n < rows && k < K;
#pragma unroll
            for (unsigned i = 0; i < 2u; ++i) {
                to[i] = mt_u32x4{0u, 0u, 0u, 0u};
                if (in) to[i] = *reinterpret_cast<const mt_u32x4*>(x8 + (size_t)(m0 + n) * K + k + 16u * i);
            }
        } else if constexpr (EIGHT) {
            const signed char* row = x8 + (size_t)(m0 + n < rows ? m0 + n : m0) * K;
#pragma unroll
            for (unsigned i = 0; i < OP::COUNT; ++i) {
                const unsigned k = blk * 128u + OP::at(i, g);
                const bool in = m0 + n < rows && (!RAGGED || k < K);
                if constexpr (GB == 4u) {
                    mt_u32x2 v = {0u, 0u};
                    if (in) v = *reinterpret_cast<const mt_u32x2*>(row + k);
                    to[i / 2u][2u * (i % 2u)] = v.x, to[i / 2u][2u * (i % 2u) + 1u] = v.y;
                } else {
                    to[i] = mt_u32x4{0u, 0u, 0u, 0u};
                    if (in) to[i] = *reinterpret_cast<const mt_u32x4*>(row + k);
                }
            }
        } else {
#pragma unroll
            for (unsigned t = 0; t < SETS; ++t) {
                to[2u * t] = to[2u * t + 1u] = mt_u32x4{0u, 0u, 0u, 0u};
                const unsigned row = m0 + 4u * t + g % XR, k = (blk + g / XR) * 128u + 8u * n;
                if (row < rows && k < K) {
                    to[2u * t] = __builtin_bit_cast(mt_u32x4, mt_row4<K, XCS>(x + (size_t)row * XRS, k));
                    to[2u * t + 1u] = __builtin_bit_cast(mt_u32x4, mt_row4<K, XCS>(x + (size_t)row * XRS, k + 4u));
                }
            }
        }
    };
    // Row r's 16 bytes c of a block's digits stand at c ^ (r / 2 % 8): the 16 rows that a
    // quarter of a wave reads lie in different banks.
    const auto place = [](unsigned r, unsigned byte) { return 128u * r + (byte ^ (16u * (r / 2u % 8u))); };
    // The digits of BL blocks to `to`, and E of this lane group's row and block (255: no
    // digits, a block that is added in fp32).
    const auto make_digits = [&](const mt_u32x4 (&xv)[XV], unsigned char* to, int (&made)[SETS]) {
#pragma unroll
        for (unsigned t = 0; t < SETS; ++t) {
            float v[8], top[2];  // (NaN above all, as infinities are)
#pragma unroll
            for (unsigned j = 0; j < 8u; ++j) v[j] = __uint_as_float(xv[EIGHT ? 0u : 2u * t + j / 4u][j % 4u]);
#pragma unroll
            for (unsigned h = 0; h < 2u; ++h)
                top[h] = mt_maximum(mt_maximum(mt_maximum(__builtin_fabsf(v[4u * h]), __builtin_fabsf(v[4u * h + 1u])),
                                               __builtin_fabsf(v[4u * h + 2u])), __builtin_fabsf(v[4u * h + 3u]));
            const int e = (int)((mt_max16(__float_as_uint(mt_maximum(top[0], top[1]))) >> 23) & 255u);
            // Four values that are not all zero, all below 2^(E-135)?  The smallest top but 0 is
            // the largest negated.  (Up to E = 8 a step is at most 2^-148.)
            const unsigned a = 0u - __float_as_uint(top[0]), b = 0u - __float_as_uint(top[1]);
            const int least = (e - 8) * 0x800000;
            const bool wide = mt_max16(a > b ? a : b) > 0u - (unsigned)(least > 1 ? least : 1);
            made[t] = wide ? 255 : e < 1 ? 1 : e;
            unsigned d[8];
#pragma unroll
            for (unsigned j = 0; j < 8u; ++j) {
                const int whole = made[t] == 255 ? 0 : (int)__builtin_ldexpf(v[j], 156 - made[t]);
                d[j] = (unsigned)whole + 0x00808080u;
            }
            unsigned ev[4], od[4];
            mt_bytes4(d[0], d[2], d[4], d[6], ev);
            mt_bytes4(d[1], d[3], d[5], d[7], od);
#pragma unroll
            for (unsigned i = 0; i < 3u; ++i) ev[i] ^= 0x80808080u, od[i] ^= 0x80808080u;
            unsigned char* block = to + (g / XR) * DIGITS + t * (512u * XR);
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i)
                *reinterpret_cast<mt_u32x2*>(block + place(4u * (g % XR) + i, 8u * n)) = mt_u32x2{ev[3u - i], od[3u - i]};
        }
    };

    bool lacks = false;  // SHARED: whether a row has a block without digits in this phase
    int* es = reinterpret_cast<int*>(lds + (SHARED ? PB * DIGITS : 0u));  // SHARED: E, [PB][SETS][4]
    // SHARED: the digits of blocks p0 .. p0 + PB - 1.
    const auto make_phase = [&](unsigned p0) {
        lacks = false;
        for (unsigned at = wave * BL; at < PB && p0 + at < NB; at += WAVES * BL) {
            mt_u32x4 xv[XV];
            load_x(p0 + at, xv);
            if constexpr (EIGHT) {
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i) {  // 8 k at a time, the even and the odd ones
                    const unsigned lo = xv[i / 2u][2u * (i % 2u)], hi = xv[i / 2u][2u * (i % 2u) + 1u];
                    *reinterpret_cast<mt_u32x2*>(lds + at * DIGITS + place(n, 32u * g + 8u * i)) =
                        mt_u32x2{__builtin_amdgcn_perm(hi, lo, 0x06040200u), __builtin_amdgcn_perm(hi, lo, 0x07050301u)};
                }
            } else {
                int made[SETS];
                make_digits(xv, lds + at * DIGITS, made);
#pragma unroll
                for (unsigned t = 0; t < SETS; ++t) {
                    lacks = lacks || made[t] == 255;
                    if (n == 0u) es[((at + g / XR) * SETS + t) * 4u + g % XR] = made[t];
                }
            }
        }
        if constexpr (EIGHT) __syncthreads();
        else lacks = __syncthreads_or(lacks);
    };

    constexpr unsigned TILES = (N + 16u * R - 1u) / (16u * R);
    // (all waves of a workgroup go round together where they share digits)
    for (unsigned at = blockIdx.x; at * (SHARED ? WAVES : 1u) < TILES; at += gridDim.x) {
        const unsigned tile = SHARED ? at * WAVES + wave : at;
        const unsigned n0 = tile * (16u * R);
        const unsigned char* wr[R];
        size_t sr[R];
#pragma unroll
        for (unsigned r = 0; r < R; ++r) {
            const unsigned row = n0 + 16u * r + n < N ? n0 + 16u * r + n : N - 1u;
            wr[r] = w + (size_t)row * (K / 2u) + 16u * g;
            sr[r] = (size_t)row * NG;
        }
        const auto load_w = [&](unsigned c, mt_u32x4 (&q)[U][R], float (&s)[R][GU], float (&z)[R][ZEROS ? GU : 1u]) {
#pragma unroll
            for (unsigned u = 0; u < U; ++u)
#pragma unroll
                for (unsigned r = 0; r < R; ++r) {
                    q[u][r] = mt_u32x4{0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u};
                    if (!RAGGED || (c * U + u) * 128u + 32u * g < K)
                        q[u][r] = *reinterpret_cast<const mt_u32x4*>(wr[r] + (size_t)(c * U + u) * 64u);
                }
#pragma unroll
            for (unsigned r = 0; r < R; ++r) {
                const auto some = [&](const float* from, float* to) {
                    if (GU % 4u == 0u && (!RAGGED || (c + 1u) * GU <= NG)) {
#pragma unroll
                        for (unsigned i = 0; i + 3u < GU; i += 4u) {
                            const mt_f32x4 v = mt_ld4u(from + i);
                            to[i] = v.x, to[i + 1u] = v.y, to[i + 2u] = v.z, to[i + 3u] = v.w;
                        }
                    } else {
#pragma unroll
                        for (unsigned i = 0; i < GU; ++i) to[i] = !RAGGED || c * GU + i < NG ? from[i] : 0.f;
                    }
                };
                some(scales + sr[r] + c * GU, s[r]);
                if constexpr (ZEROS) some(zeros + sr[r] + c * GU, z[r]);
            }
        };

        float acc[R][ACC];
#pragma unroll
        for (unsigned r = 0; r < R; ++r)
#pragma unroll
            for (unsigned a = 0; a < ACC; ++a) acc[r][a] = 0.f;
        // The products of row m of x in block blk in fp32: a lane sums its 32 k of its weight
        // rows (weights first, as a value of W is, so that nothing is larger on the way), the
        // four pieces meet.
        const auto add_plain = [&](unsigned blk, unsigned m) {
            const float* xr = x + (size_t)(m0 + m) * XRS;
            const unsigned k0 = blk * 128u + 32u * g;
            float part[R];
#pragma unroll
            for (unsigned r = 0; r < R; ++r) part[r] = 0.f;
            if (k0 < K) {
                mt_f32x4 v[8];  // (all loads on the way together)
                mt_u32x4 word[R];
#pragma unroll
                for (unsigned i = 0; i < 8u; ++i) v[i] = mt_row4<K, XCS>(xr, k0 + 4u * i);
#pragma unroll
                for (unsigned r = 0; r < R; ++r) word[r] = *reinterpret_cast<const mt_u32x4*>(wr[r] + (size_t)blk * 64u);
#pragma unroll
                for (unsigned r = 0; r < R; ++r) {
                    const float by = scales[sr[r] + k0 / GROUP];
                    float zero = 8.f;
                    if constexpr (ZEROS) zero = zeros[sr[r] + k0 / GROUP];
#pragma unroll
                    for (unsigned i = 0; i < 32u; ++i)
                        part[r] = __builtin_fmaf(v[i / 4u][i % 4u], ((float)((word[r][i / 8u] >> (4u * (i % 8u))) & 15u) - zero) * by, part[r]);
                }
            }
#pragma unroll
            for (unsigned r = 0; r < R; ++r) {
                part[r] += mt_shfl_xor(part[r], 16);
                part[r] += mt_shfl_xor(part[r], 32);
#pragma unroll
                for (unsigned t = 0; t < SETS; ++t)
                    if (m / 4u == t && m % 4u == g) acc[r][t] += part[r];
            }
        };
        const mt_i32x4 zero4 = {0, 0, 0, 0};
        mt_u32x4 q[U][R], xv[XV];
        float s[R][GU], z[R][ZEROS ? GU : 1u];
        if (c0 < c1) {
            // x first where digits are made of it for one tile: while the weights arrive (1 row,
            // 11008 x 4096: 7.2 us, weights first 7.5).  Of more tiles weights first (8 rows, 8192
            // x 11008: 25 and 28), and for x in 8 bits, which is used with them.
            constexpr bool AHEAD = !SHARED && !EIGHT && R == 1u;
            if constexpr (AHEAD) load_x(c0 * U, xv);
            load_w(c0, q, s, z);
            if constexpr (!SHARED && !AHEAD) load_x(c0 * U, xv);
        }
#pragma unroll 1
        for (unsigned phase = 0; phase < PHASES; ++phase) {
        if constexpr (SHARED) {
            if (PHASES > 1u || at == blockIdx.x) {
                if (phase > 0u || at != blockIdx.x) __syncthreads();
                make_phase(phase * PB);
            }
        }
        const unsigned cp = SHARED ? phase * (PB / U) : c0;
        const unsigned cq = SHARED ? (cp + PB / U < c1 ? cp + PB / U : c1) : c1;
#pragma unroll 1
        for (unsigned c = cp; c < cq; ++c) {
            mt_u32x4 qn[U][R];
            float sn[R][GU], zn[R][ZEROS ? GU : 1u];
            if (c + 1u < c1) load_w(c + 1u, qn, sn, zn);
            // Rows of the chunk's blocks that have no digits: bit 16 i + SETS b + t for E of set t
            // and lane group i of making b.
            unsigned long long plain = 0ull;
#pragma unroll
            for (unsigned pu = 0; pu < U; pu += BL) {
                mt_u32x4 xn[XV];
                unsigned char* digits = SHARED ? lds + (c * U + pu - phase * PB) * DIGITS : lds + wave * (2048u * SETS);
                int made[SETS];
                if constexpr (!SHARED) {
                    const unsigned after = c * U + pu + BL;
                    if (after < c1 * U) load_x(after, xn);
                    if constexpr (!EIGHT) {
                        make_digits(xv, digits, made);
#pragma unroll
                        for (unsigned t = 0; t < SETS; ++t)
                            plain |= (__ballot(made[t] == 255) & 0x0001000100010001ull) << (pu / BL * SETS + t);
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        __builtin_amdgcn_wave_barrier();
                    }
                }
#pragma unroll
                for (unsigned bl = 0; bl < BL; ++bl) {
                    const unsigned u = pu + bl;
                    if (RAGGED && (c * U + u) >= NB) continue;
                    unsigned a[SETS][OP::COUNT][OP::WORDS];
                    int ex[SETS];  // E of this lane group's row of the products
#pragma unroll
                    for (unsigned t = 0; t < SETS; ++t) {
                        if constexpr (EIGHT && !SHARED) {
#pragma unroll
                            for (unsigned i = 0; i < 4u; ++i) {  // 8 k at a time, the even and the odd ones
                                const unsigned lo = xv[i / 2u][2u * (i % 2u)], hi = xv[i / 2u][2u * (i % 2u) + 1u];
                                constexpr unsigned PER = OP::WORDS / 2u;
                                a[0][i / PER][2u * (i % PER)] = __builtin_amdgcn_perm(hi, lo, 0x06040200u);
                                a[0][i / PER][2u * (i % PER) + 1u] = __builtin_amdgcn_perm(hi, lo, 0x07050301u);
                            }
                        } else {
                            const unsigned char* from = digits + bl * DIGITS + t * (512u * XR);
#pragma unroll
                            for (unsigned i = 0; i < OP::COUNT; ++i)
                                mt_ld_words<OP::WORDS>(a[t][i], from + place(n % (4u * XR), OP::at(i, g)));
                            if constexpr (EIGHT) ex[t] = 0;
                            else if constexpr (SHARED) ex[t] = es[((c * U + u - phase * PB) * SETS + t) * 4u + g % XR];
                            else
                                ex[t] = XR == 4u ? made[t]
                                        : XR == 1u ? __builtin_amdgcn_readlane(made[t], (int)(16u * bl))
                                                   : __shfl(made[t], (int)(16u * (bl * XR + g % XR)), 64);
                        }
                    }
                    float cz[SETS][GB][EIGHT ? 4u : 1u];  // the sums of x by group, for the zeros
                    if constexpr (ZEROS) {
                        unsigned one[OP::WORDS];
#pragma unroll
                        for (unsigned i = 0; i < OP::WORDS; ++i) one[i] = 0x01010101u;
#pragma unroll
                        for (unsigned t = 0; t < SETS; ++t)
#pragma unroll
                            for (unsigned j = 0; j < GB; ++j) {
                                mt_i32x4 o = OP::product(a[t][j], one, zero4);
                                if constexpr (GB == 1u) o = OP::product(a[t][1], one, o);
                                if constexpr (EIGHT) {
#pragma unroll
                                    for (unsigned i = 0; i < 4u; ++i) cz[t][j][i] = (float)o[i];
                                } else {
                                    cz[t][j][0] = mt_digits(o);
                                }
                            }
                    }
#pragma unroll
                    for (unsigned r = 0; r < R; ++r) {
                        unsigned v[4], b[OP::COUNT][OP::WORDS];
#pragma unroll
                        for (unsigned i = 0; i < 4u; ++i) v[i] = q[u][r][i] ^ 0x88888888u;
                        OP::spread(v);
#pragma unroll
                        for (unsigned i = 0; i < 4u; ++i) {
                            constexpr unsigned PER = OP::WORDS / 2u;
                            b[i / PER][2u * (i % PER)] = (v[i] << 4) & 0xF0F0F0F0u;
                            b[i / PER][2u * (i % PER) + 1u] = v[i] & 0xF0F0F0F0u;
                        }
#pragma unroll
                        for (unsigned t = 0; t < SETS; ++t) {
                            float sum = 0.f;
#pragma unroll
                            for (unsigned j = 0; j < GB; ++j) {
                                mt_i32x4 p = OP::product(a[t][j], b[j], zero4);
                                if constexpr (GB == 1u) p = OP::product(a[t][1], b[1], p);
                                const float by = s[r][u * GB + j];
                                if constexpr (EIGHT) {
#pragma unroll
                                    for (unsigned i = 0; i < 4u; ++i) {
                                        float f = (float)p[i];
                                        if constexpr (ZEROS) f = __builtin_fmaf(cz[t][j][i], 128.f - 16.f * z[r][u * GB + j], f);
                                        acc[r][i] = __builtin_fmaf(f, by, acc[r][i]);
                                    }
                                } else {
                                    float f = mt_digits(p);
                                    if constexpr (ZEROS) f = __builtin_fmaf(cz[t][j][0], 128.f - 16.f * z[r][u * GB + j], f);
                                    sum = GB == 1u ? f * by : __builtin_fmaf(f, by, sum);
                                }
                            }
                            if constexpr (!EIGHT) acc[r][t] += __builtin_ldexpf(sum, ex[t] - 160);
                        }
                    }
                }
                if constexpr (!SHARED) {
                    if constexpr (!EIGHT) {
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        __builtin_amdgcn_wave_barrier();
                    }
#pragma unroll
                    for (unsigned i = 0; i < XV; ++i) xv[i] = xn[i];
                }
            }
            if constexpr (!EIGHT && !SHARED) {
                if (__builtin_expect(plain != 0ull, 0)) {
                    while (plain) {
                        const unsigned bit = (unsigned)__builtin_ctzll(plain), i = bit / 16u, at = bit % 16u;
                        plain &= plain - 1ull;
                        add_plain(c * U + at / SETS * BL + i / XR, 4u * (at % SETS) + i % XR);
                    }
                    // What was on the way is loaded again: nothing of it is kept over these products.
                    if (c + 1u < c1) {
                        load_w(c + 1u, qn, sn, zn);
                        load_x((c + 1u) * U, xv);
                    }
                }
            }
#pragma unroll
            for (unsigned r = 0; r < R; ++r) {
#pragma unroll
                for (unsigned u = 0; u < U; ++u) q[u][r] = qn[u][r];
#pragma unroll
                for (unsigned i = 0; i < GU; ++i) {
                    s[r][i] = sn[r][i];
                    if constexpr (ZEROS) z[r][i] = zn[r][i];
                }
            }
        }
        if constexpr (SHARED && !EIGHT) {
            if (__builtin_expect(lacks, 0)) {
                constexpr unsigned MANY = 16u / SETS;  // blocks whose E the lanes look at together
                for (unsigned b = phase * PB; b < NB && b < phase * PB + PB; b += MANY) {
                    const unsigned blk = b + n / SETS;
                    bool none = n < MANY * SETS && g < XR && blk < NB && blk < phase * PB + PB;
                    if (none) none = es[((blk - phase * PB) * SETS + n % SETS) * 4u + g] == 255;
                    for (unsigned long long plain = __ballot(none); plain; plain &= plain - 1ull) {
                        const unsigned bit = (unsigned)__builtin_ctzll(plain);
                        add_plain(b + bit % 16u / SETS, 4u * (bit % 16u % SETS) + bit / 16u);
                    }
                }
                if (cq < c1) load_w(cq, q, s, z);  // (as above)
            }
        }
        }
        const auto put = [&](unsigned r, unsigned a, unsigned ln, float v) {
            const unsigned col = n0 + 16u * r + (ln & 15u), row = m0 + (EIGHT ? 4u * (ln >> 4) + a : 4u * a + (ln >> 4));
            if (col < N && row < rows && (EIGHT || ln / 16u < XR))
                y[(size_t)row * N + col] = EIGHT ? (v * 0.0625f) * xs[row] : v;  // (a 16th of a subnormal scale loses bits)
        };
        if constexpr (SHARED) {
#pragma unroll
            for (unsigned r = 0; r < R; ++r)
#pragma unroll
                for (unsigned a = 0; a < ACC; ++a) put(r, a, lane, acc[r][a]);
        } else {
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
                put(at / (ACC * 64u), at / 64u % ACC, at % 64u, v);
            }
            __syncthreads();
        }
    }
}
