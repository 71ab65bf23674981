// Rows into and out of a paged KV cache, gfx950.
//
//   kuiops_kv_paged_append  per-head norm and rotation of new tokens' queries and keys,
//       keys and values into the sequences' pages, quantised as they are written
//   kuiops_kv_paged_read    the sequences' rows gathered out of their pages as numbers
//
// 8-bit pages hold a row x as x_i = scale * s_i with scale = m / M, s_i = nearest(x_i M / m),
// m = max |x_i|, M the type's largest value (int8 127, e4m3 448).
#include <algorithm>
#include <type_traits>

#include "paged.hpp"

namespace kuiops {

int check_cache(const kuiops_paged_layout *at, int dtype, const void *K, const void *V, const float *ks, const float *vs,
                const int32_t *table, PagedCache &c) {
    if (at->pages < 0 || at->page <= 0 || at->hkv <= 0 || at->hd <= 0 || at->width < 0) return KUIOPS_E_INVALID;
    if (at->width > 0 && !table) return KUIOPS_E_INVALID;
    if (at->pages > 0 && (!K || !V)) return KUIOPS_E_INVALID;
    if (dtype != KUIOPS_BF16 && dtype != KUIOPS_F16) return KUIOPS_E_UNSUPPORTED;
    const bool bytes = at->dtype == KUIOPS_I8 || at->dtype == KUIOPS_F8E4M3;
    if (!bytes && at->dtype != KUIOPS_BF16 && at->dtype != KUIOPS_F16) return KUIOPS_E_UNSUPPORTED;
    if (!bytes && at->dtype != dtype) return KUIOPS_E_INVALID;
    if (bytes && at->pages > 0 && (!ks || !vs)) return KUIOPS_E_INVALID;
    // rows in 16-byte pieces, 16 rows of a page at a time, 32-bit slots
    if (at->hd % 16 || at->hd > 128 || at->page % 16 || at->page > (1 << 20) || at->pages >= ((int64_t)1 << 31) ||
        at->width * at->page >= ((int64_t)1 << 30) || at->hkv >= (1 << 20))
        return KUIOPS_E_UNSUPPORTED;
    const int64_t unit = bytes ? 16 : 8;
    if (!aligned16(K) || !aligned16(V) || (bytes && (!aligned16(ks) || !aligned16(vs)))) return KUIOPS_E_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (at->sk[i] % unit || at->sv[i] % unit || at->sk[i] < 0 || at->sv[i] < 0) return KUIOPS_E_UNSUPPORTED;
    if (at->sk[2] < at->hd || at->sv[2] < at->hd || at->sk[2] >= (1 << 24) || at->sv[2] >= (1 << 24)) return KUIOPS_E_UNSUPPORTED;
    for (int i = 0; i < 2 && bytes; ++i)
        if (at->sks[i] % 4 || at->svs[i] % 4 || at->sks[i] < 0 || at->svs[i] < 0) return KUIOPS_E_UNSUPPORTED;
    if (at->ld_table < 0) return KUIOPS_E_UNSUPPORTED;
    c = PagedCache{K, V, bytes ? ks : nullptr, bytes ? vs : nullptr, table,
                   at->sk[0], at->sk[1], at->sk[2], at->sv[0], at->sv[1], at->sv[2],
                   at->sks[0], at->sks[1], at->svs[0], at->svs[1], at->ld_table,
                   (int)at->pages, (int)at->page, (int)at->hkv, (int)at->hd, (int)at->width, paged_div((int)at->page / 16), at->dtype};
    return KUIOPS_OK;
}

namespace {

struct AppendArgs {
    PagedCache c;
    int n, t, hq;
    const void *qkv;
    int64_t ld_tok, ld_batch;
    const int32_t *lens, *pos0;
    const float *inv_freq;
    const void *q_norm, *k_norm;
    double eps, inv_hd;
    void *q;
    int64_t sq0, sq1, sq2;
    int heads;                 // heads that a work-group takes
};

// cos and sin of pos * freq, 64-bit: the angle less the nearest multiple of pi / 2 (in two
// parts, whose product with the multiple is exact enough far past any position), then Taylor's
// series on +- pi / 4, whose first term left out is below 2^-53.
__device__ __forceinline__ void turn_of(int64_t pos, float freq, double &c, double &s) {
    const double a = (double)pos * (double)freq;
    const double n = rint(a * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800, a);
    r = fma(-n, 6.12323399573676603587e-17, r);
    const double x = r * r;
    double sn = -1.0 / 1307674368000.0;
    sn = fma(sn, x, 1.0 / 6227020800.0);
    sn = fma(sn, x, -1.0 / 39916800.0);
    sn = fma(sn, x, 1.0 / 362880.0);
    sn = fma(sn, x, -1.0 / 5040.0);
    sn = fma(sn, x, 1.0 / 120.0);
    sn = fma(sn, x, -1.0 / 6.0);
    sn = fma(sn * x, r, r);
    double cs = 1.0 / 20922789888000.0;
    cs = fma(cs, x, -1.0 / 87178291200.0);
    cs = fma(cs, x, 1.0 / 479001600.0);
    cs = fma(cs, x, -1.0 / 3628800.0);
    cs = fma(cs, x, 1.0 / 40320.0);
    cs = fma(cs, x, -1.0 / 720.0);
    cs = fma(cs, x, 1.0 / 24.0);
    cs = fma(cs, x, -1.0 / 2.0);
    cs = fma(cs, x, 1.0);
    const int64_t quarter = (int64_t)n & 3;
    c = quarter == 0 ? cs : quarter == 1 ? -sn : quarter == 2 ? -cs : sn;
    s = quarter == 0 ? sn : quarter == 1 ? cs : quarter == 2 ? -sn : -cs;
}

// 1 / sqrt(x) and 1 / x in 64 bits: the hardware's first values and Newton's iteration, whose
// error squares from 2^-14 or better each time. (Correctly rounded roots and quotients instead:
// 64 tokens of 32 + 8 heads, normed, 3.85 for 3.77 us, 512 tokens in int8 5.1 for 5.0.) The
// root of an infinity is kept from the iteration's 0 * inf.
__device__ __forceinline__ float inverse_root(float x) { return rsqrtf(x); }
__device__ __forceinline__ double inverse_root(double x) {
    double r = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 3; ++i) r = fma(r * 0.5, fma(-x * r, r, 1.0), r);
    return x < INFINITY || x != x ? r : 0.0;
}
__device__ __forceinline__ double inverse(double x) {
    double r = __builtin_amdgcn_rcp(x);
#pragma unroll
    for (int i = 0; i < 3; ++i) r = fma(r, fma(-x, r, 1.0), r);
    return r;
}

// The value of the lane D away within a group of lanes (the same moves as group_sum's)
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    const u32x2 r = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[0], CTRL, 0xF, 0xF, false),
                     (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[1], CTRL, 0xF, 0xF, false)};
    return __builtin_bit_cast(double, r);
}
template <int N, typename F, typename Op>
__device__ __forceinline__ F over_group(F v, Op op) {
    static_assert(N == 4 || N == 8, "group size");
    v = op(v, dpp<0xB1>(v));
    v = op(v, dpp<0x4E>(v));
    if (N == 8) v = op(v, dpp<0x141>(v));
    return v;
}

// Eight values s = nearest(x M / m) of the 8-bit type, four a dword.
//
// Keys, 64 bits: y = x * r with r = M / m, whose last bit may miss a border that the quotient
// hits, so y is taken to be what lies within 2^-38 of it (int8) or what 32 bits hold to 2^-45
// of it (e4m3).  int8: two additions of a power of two round to those steps and then to a whole
// number, which is the low word of the second.  e4m3: the conversion starts at 32 bits, which
// must not turn y into a border; if one of a wave's values lies on one (or below the type's
// normal ones, where borders are elsewhere), they are cut off with the last bit set instead,
// which rounds as the 64-bit value does.
template <bool INT8>
__device__ __forceinline__ void to_bytes(const double (&x)[8], double r, u32x2 &w) {
    if constexpr (INT8) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            uint32_t got = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double y = fma(x[e + i], r, 0x1.8p14) - 0x1.8p14;
                got |= ((uint32_t)__double2loint(y + 0x1.8p52) & 0xffu) << (8 * i);
            }
            w[e / 4] = got;
        }
    } else {
        float f[8];
        bool border = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f[e] = (float)(x[e] * r);
            border |= (__float_as_uint(f[e]) & 0xfffffu) == 0x80000u || fabsf(f[e]) < 0x1p-6f;
        }
        if (__any(border)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double y = x[e] * r, off = y - (double)f[e];
                if (fabs(off) > fabs(y) * 0x1p-45) {
                    uint32_t u = __float_as_uint(f[e]);
                    if ((off < 0) == (y > 0)) u -= 1;            // the neighbour nearer to zero
                    f[e] = __uint_as_float(u | 1);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e += 4)
            w[e / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(f[e + 2], f[e + 3], __builtin_amdgcn_cvt_pk_fp8_f32(f[e], f[e + 1], 0, false), true);
    }
}
// Values, which come in 16 bits: x M is exact in 32, and its quotient by m, rounded once, is a
// border only where the exact one is (that lies a 2^-12th of a step away from any other, at
// least).  Rows near the type's end are scaled down first.
template <bool INT8>
__device__ __forceinline__ void to_bytes(const float (&x)[8], float m, u32x2 &w) {
    const float down = m > 0x1p100f ? 0x1p-16f : 1.f, M = (INT8 ? 127.f : 448.f) * down, by = m > 0.f ? m * down : 1.f;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = x[e + i] * M / by;
        if constexpr (INT8) {
            uint32_t got = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) got |= ((uint32_t)(int)rintf(f[i]) & 0xffu) << (8 * i);
            w[e / 4] = got;
        } else {
            w[e / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false), true);
        }
    }
}

// ------------------------------------------------------------------------
// paged_append_kernel -- a work-group has one token and `heads` of its heads, one pass:
// HD / 16 lanes have a head, 8 values i and their partners i + hd / 2 each, so a row is read
// and written in 16-byte pieces and the rotation needs no exchange.  The row is on its way
// while its cos / sin are computed for all heads (64 bits, in LDS) and its page looked up.
// Queries, and keys of 16-bit pages, are computed in 32 bits and rounded once; keys of 8-bit
// pages in 64, so that a value next to a border between two quantised ones falls on its own
// side of it.
// What bounds it: the bytes, and for 8 bits the arithmetic about as much; waves at work hide
// both, so registers are kept few (4 ragged prompts of 4001 tokens, 32 + 8 heads of 128, normed:
// 7 waves a SIMD 68 us, 4.8 TB/s, 5 waves 82; two tokens a work-group 74, four 78; heads handed
// out over the threads in turn, 4 tokens a work-group, 73; 6297 tokens in e4m3: 8 / 7 / 6 / 5 waves 55 / 44 / 45 / 49).
constexpr int kAppendThreads = 512;
template <typename T, int PK, int HD>
__global__ __launch_bounds__(kAppendThreads, PK == 0 ? 7 : 6) void paged_append_kernel(AppendArgs a) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    constexpr int LPH = HD / 16, HALF = HD / 2;
    typedef typename std::conditional<PK == 0, float, double>::type K;      // what keys are computed in
    __shared__ __attribute__((aligned(16))) K s_cos[HALF], s_sin[HALF];
    __shared__ int s_id, s_at;
    const int tid = threadIdx.x, hd = a.c.hd, half = hd / 2, hkv = a.c.hkv;
    const int64_t b = blockIdx.y;
    const int t = blockIdx.x, h = blockIdx.z * a.heads + tid / LPH, d = tid % LPH * 8;
    // (the lanes of a head are in one wave, and all of them or none are at work; those past the
    // head's end go along without a value)
    const bool mine = d < half, on = tid / LPH < a.heads && h < a.hq + 2 * hkv;
    u32x4 r1 = {0, 0, 0, 0}, r2 = {0, 0, 0, 0};
    if (mine && on) {
        const T *row = reinterpret_cast<const T *>(a.qkv) + b * a.ld_batch + t * a.ld_tok + (h * hd + d);
        r1 = *reinterpret_cast<const u32x4 *>(row);
        r2 = *reinterpret_cast<const u32x4 *>(row + half);
    }
    const bool query = h < a.hq, key = !query && h < a.hq + hkv;
    const void *norm = query ? a.q_norm : key ? a.k_norm : nullptr;
    u32x4 n1 = {0, 0, 0, 0}, n2 = {0, 0, 0, 0};
    if (norm && mine && on) {
        n1 = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const T *>(norm) + d);
        n2 = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const T *>(norm) + d + half);
    }
    const int there = a.lens ? max(0, min(a.lens[b], a.t)) : a.t;
    const int64_t first = a.pos0 ? a.pos0[b] : 0;
    if (t < there) {
        for (int i = tid; i < half; i += blockDim.x) {
            double c, s;
            turn_of(first + t, a.inv_freq[i], c, s);
            s_cos[i] = (K)c;
            s_sin[i] = (K)s;
        }
    }
    if (tid == 0) {
        const int64_t slot = first + t;
        int at = 0;
        s_id = slot >= 0 && slot < (1 << 30) ? page_of(a.c, b, (int)slot, at) : -1;
        s_at = at;
    }
    __syncthreads();
    if (!on) return;
    T *q = reinterpret_cast<T *>(a.q) + b * a.sq0 + h * a.sq1 + t * a.sq2 + d;
    if (t >= there) {
        // a token that is not there: its query is 0
        if (query && mine) {
            *reinterpret_cast<u32x4 *>(q) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4 *>(q + half) = u32x4{0, 0, 0, 0};
        }
        return;
    }
    const t8 v1 = __builtin_bit_cast(t8, r1), v2 = __builtin_bit_cast(t8, r2), w1 = __builtin_bit_cast(t8, n1), w2 = __builtin_bit_cast(t8, n2);
    auto turned = [&](auto one, auto (&x1)[8], auto (&x2)[8]) __attribute__((always_inline)) {
        typedef decltype(one) F;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x1[e] = (F)to_f32(v1[e]);
            x2[e] = (F)to_f32(v2[e]);
        }
        if (norm) {
            F sum = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += x1[e] * x1[e] + x2[e] * x2[e];
            sum = over_group<LPH>(sum, [](F u, F w) { return u + w; });
            const F ms = sum * (F)a.inv_hd + (F)a.eps;
            // bf16's squares leave fp32's range from 2^64 on and lose bits from 2^-63 down (the
            // latter only seen where eps is as small): such a row's norm in 64 bits.  The same
            // in all lanes of a head.
            if (sizeof(F) == 4 && !(ms > (F)0x1p-100 && ms < (F)0x1p100)) {
                double wide = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) wide += (double)x1[e] * (double)x1[e] + (double)x2[e] * (double)x2[e];
                wide = over_group<LPH>(wide, [](double u, double w) { return u + w; });
                const double r = inverse_root(wide * a.inv_hd + a.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x1[e] = (F)((double)x1[e] * (r * (double)to_f32(w1[e])));
                    x2[e] = (F)((double)x2[e] * (r * (double)to_f32(w2[e])));
                }
            } else {
                const F r = inverse_root(ms);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x1[e] *= r * (F)to_f32(w1[e]);
                    x2[e] *= r * (F)to_f32(w2[e]);
                }
            }
        }
        if (!mine) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const F c = (F)s_cos[d + e], s = (F)s_sin[d + e], y1 = x1[e], y2 = x2[e];
            x1[e] = y1 * c - y2 * s;
            x2[e] = y2 * c + y1 * s;
        }
    };
    auto rounded = [&](const float (&y)[8]) __attribute__((always_inline)) {
        t8 w;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = from_f32<T>(y[e]);
        return __builtin_bit_cast(u32x4, w);
    };
    if (query || (PK == 0 && key)) {
        float x1[8], x2[8];
        turned(1.f, x1, x2);
        r1 = rounded(x1);
        r2 = rounded(x2);
    }
    if (query) {
        if (mine) {
            *reinterpret_cast<u32x4 *>(q) = r1;
            *reinterpret_cast<u32x4 *>(q + half) = r2;
        }
        return;
    }
    const int id = __builtin_amdgcn_readfirstlane(s_id), at = __builtin_amdgcn_readfirstlane(s_at);
    if (id < 0) return;                           // the slot has no page
    const int hk = h - a.hq - (key ? 0 : hkv);
    const int64_t off = key ? id * a.c.sk0 + hk * a.c.sk1 + at * a.c.sk2 : id * a.c.sv0 + hk * a.c.sv1 + at * a.c.sv2;
    char *dst = reinterpret_cast<char *>(const_cast<void *>(key ? a.c.K : a.c.V)) + (off + d) * (PK == 0 ? 2 : 1);
    if constexpr (PK == 0) {
        if (mine) {
            *reinterpret_cast<u32x4 *>(dst) = r1;
            *reinterpret_cast<u32x4 *>(dst + half * 2) = r2;
        }
    } else {
        constexpr bool INT8 = PK == 1;
        constexpr double M = INT8 ? 127.0 : 448.0;
        u32x2 b1, b2;
        float scale;                              // NaN for a row that has one, or an infinity
        bool fine;
        if (key) {
            double x1[8], x2[8], top = 0.0, odd = 0.0;
            turned(1.0, x1, x2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top = fmax(top, fmax(fabs(x1[e]), fabs(x2[e])));
                odd += x1[e] + x2[e];
            }
            top = over_group<LPH>(top, [](double u, double w) { return fmax(u, w); });
            odd = over_group<LPH>(odd, [](double u, double w) { return u + w; });
            fine = odd * 0.0 == 0.0;
            const double r = fine && top > 0.0 ? M * inverse(top) : 0.0;
            scale = (float)(top * (1.0 / M));
            to_bytes<INT8>(x1, r, b1);
            to_bytes<INT8>(x2, r, b2);
        } else {
            float x1[8], x2[8], top = 0.f, odd = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x1[e] = to_f32(v1[e]);
                x2[e] = to_f32(v2[e]);
                top = fmaxf(top, fmaxf(fabsf(x1[e]), fabsf(x2[e])));
                odd = __builtin_fmaf(x1[e], 0.f, __builtin_fmaf(x2[e], 0.f, odd));
            }
            top = over_group<LPH>(top, [](float u, float w) { return fmaxf(u, w); });
            odd = over_group<LPH>(odd, [](float u, float w) { return u + w; });
            fine = odd == 0.f;
            scale = (float)((double)top * (1.0 / M));
            to_bytes<INT8>(x1, top, b1);
            to_bytes<INT8>(x2, top, b2);
        }
        if (mine) {
            *reinterpret_cast<u32x2 *>(dst) = fine ? b1 : u32x2{0, 0};
            *reinterpret_cast<u32x2 *>(dst + half) = fine ? b2 : u32x2{0, 0};
        }
        if (d == 0) {
            float *sc = const_cast<float *>(key ? a.c.ks : a.c.vs);
            sc[key ? id * a.c.sks0 + hk * a.c.sks1 + at : id * a.c.svs0 + hk * a.c.svs1 + at] = fine ? scale : __uint_as_float(0x7fc00000u);
        }
    }
}

struct ReadArgs {
    PagedCache c;
    int s;
    const int32_t *kv_len;
    void *k, *v;
    int64_t ko0, ko1, ko2, vo0, vo1, vo2;
    int fill;
};

// ------------------------------------------------------------------------
// paged_read_kernel -- a work-group has 128 slots of one KV head, keys and values; 8 values of
// a row a lane, so that what is written, the larger part, goes out in 16-byte pieces that
// follow one another.  All loads of a thread are on their way at once, behind its page numbers.
// What bounds it: the bytes; 8 sequences of 4583 to 8000 rows, 8 heads of 128 in int8, to bf16 with
// the rows behind them cleared 78 us, 4.7 TB/s read and written (a large copy 5.1); 16 values
// a lane, stored 8 bytes at a time, 85.6.
template <typename T, int PK, int HD>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadArgs a) {
    constexpr int LPR = HD / 8, RPI = 256 / LPR, ROWS = 128, IT = ROWS / RPI, B = PK == 0 ? 2 : 1;
    typedef typename std::conditional<PK == 0, u32x4, u32x2>::type words;
    const int tid = threadIdx.x, d = tid % LPR * 8;
    const int64_t b = blockIdx.z, hk = blockIdx.y;
    const int L = min(a.s, paged_len(a.c, a.kv_len, b)), s0 = blockIdx.x * ROWS, end = a.fill ? a.s : L;
    if (s0 >= end || d >= a.c.hd) return;
    int id[IT], at[IT];
#pragma unroll
    for (int j = 0; j < IT; ++j) {
        const int slot = s0 + j * RPI + tid / LPR;
        id[j] = slot < L ? page_of(a.c, b, slot, at[j]) : -1;
    }
    words w[2][IT];
    float sc[2][IT];
#pragma unroll
    for (int j = 0; j < IT; ++j) {
        w[0][j] = w[1][j] = words{};
        sc[0][j] = sc[1][j] = 0.f;
        if (id[j] >= 0) {
            w[0][j] = *reinterpret_cast<const words *>(reinterpret_cast<const char *>(a.c.K) + (id[j] * a.c.sk0 + hk * a.c.sk1 + at[j] * a.c.sk2 + d) * B);
            w[1][j] = *reinterpret_cast<const words *>(reinterpret_cast<const char *>(a.c.V) + (id[j] * a.c.sv0 + hk * a.c.sv1 + at[j] * a.c.sv2 + d) * B);
            if constexpr (PK != 0) {
                sc[0][j] = a.c.ks[id[j] * a.c.sks0 + hk * a.c.sks1 + at[j]];
                sc[1][j] = a.c.vs[id[j] * a.c.svs0 + hk * a.c.svs1 + at[j]];
            }
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < IT; ++j) {
            const int slot = s0 + j * RPI + tid / LPR;
            if (slot >= end) continue;
            T *dst = reinterpret_cast<T *>(x ? a.v : a.k) +
                     (x ? b * a.vo0 + hk * a.vo1 + slot * a.vo2 : b * a.ko0 + hk * a.ko1 + slot * a.ko2) + d;
            if constexpr (PK == 0) *reinterpret_cast<u32x4 *>(dst) = w[x][j];
            else {
                typedef T t8 __attribute__((ext_vector_type(8)));
                t8 y;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t u = w[x][j][e / 4];
                    float f;
                    if constexpr (PK == 1) f = (float)(int8_t)(u >> (8 * (e % 4)));
                    else switch (e % 4) {
                            case 0: f = __builtin_amdgcn_cvt_f32_fp8((int)u, 0); break;
                            case 1: f = __builtin_amdgcn_cvt_f32_fp8((int)u, 1); break;
                            case 2: f = __builtin_amdgcn_cvt_f32_fp8((int)u, 2); break;
                            default: f = __builtin_amdgcn_cvt_f32_fp8((int)u, 3); break;
                        }
                    y[e] = from_f32<T>(f * sc[x][j]);
                }
                *reinterpret_cast<t8 *>(dst) = y;
            }
        }
}

// ------------------------------------------------------------- host side

constexpr int64_t kCUs = 256;

template <typename T, int PK, int HD>
void launch_append(AppendArgs &a, hipStream_t st) {
    // up to 512 threads, for 8 bits 256 (6297 tokens of 48 heads of 128, e4m3: 44 -> 42 us)
    constexpr int LPH = HD / 16, most = (PK == 0 ? kAppendThreads : kAppendThreads / 2) / LPH;
    const int heads = a.hq + 2 * a.c.hkv;
    // few tokens: the heads are spread over work-groups until each CU has one, a wave of heads each
    // at least
    const int64_t parts = std::max(cdiv(heads, most), std::min(cdiv(heads * LPH, 64), kCUs / ((int64_t)a.n * a.t)));
    a.heads = (int)cdiv(heads, parts);
    const dim3 grid((unsigned)a.t, (unsigned)a.n, (unsigned)cdiv(heads, a.heads)), threads((unsigned)(cdiv(a.heads * LPH, 64) * 64));
    hipLaunchKernelGGL((paged_append_kernel<T, PK, HD>), grid, threads, 0, st, a);
}

template <typename T>
void launch_append_kind(AppendArgs &a, hipStream_t st) {
    const bool small = a.c.hd <= 64;
    if (a.c.dtype == KUIOPS_I8) small ? launch_append<T, 1, 64>(a, st) : launch_append<T, 1, 128>(a, st);
    else if (a.c.dtype == KUIOPS_F8E4M3) small ? launch_append<T, 2, 64>(a, st) : launch_append<T, 2, 128>(a, st);
    else small ? launch_append<T, 0, 64>(a, st) : launch_append<T, 0, 128>(a, st);
}

template <typename T, int PK>
void launch_read(const ReadArgs &a, unsigned n, hipStream_t st) {
    const dim3 grid((unsigned)cdiv(a.s, 128), (unsigned)a.c.hkv, n);
    if (a.c.hd <= 64) hipLaunchKernelGGL((paged_read_kernel<T, PK, 64>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_read_kernel<T, PK, 128>), grid, dim3(256), 0, st, a);
}

template <typename T>
void launch_read_kind(const ReadArgs &a, unsigned n, hipStream_t st) {
    if (a.c.dtype == KUIOPS_I8) launch_read<T, 1>(a, n, st);
    else if (a.c.dtype == KUIOPS_F8E4M3) launch_read<T, 2>(a, n, st);
    else launch_read<T, 0>(a, n, st);
}

}  // namespace

}  // namespace kuiops

using namespace kuiops;

extern "C" int kuiops_kv_paged_append(int64_t n, int64_t t, int64_t hq, int dtype, const void *qkv, int64_t ld_tok,
                                      int64_t ld_batch, const int32_t *lens, const int32_t *pos0, const float *inv_freq,
                                      const void *q_norm, const void *k_norm, double eps, void *q_out, const int64_t sq[3],
                                      const kuiops_paged_layout *at, void *K, void *V, float *k_scale, float *v_scale,
                                      const int32_t *table, void *stream) {
    if (n < 0 || t < 0 || hq < 0 || !at || !sq) return KUIOPS_E_INVALID;
    AppendArgs a{};
    if (n == 0 || t == 0) return KUIOPS_OK;
    const int bad = check_cache(at, dtype, K, V, k_scale, v_scale, table, a.c);
    if (bad) return bad;
    if (!qkv || !inv_freq || (hq > 0 && !q_out) || !(eps >= 0.0 && eps < INFINITY)) return KUIOPS_E_INVALID;
    if (ld_tok % 8 || ld_batch % 8 || sq[0] % 8 || sq[1] % 8 || sq[2] % 8) return KUIOPS_E_UNSUPPORTED;
    if (!aligned16(qkv) || !aligned16(q_out) || (q_norm && !aligned16(q_norm)) || (k_norm && !aligned16(k_norm)))
        return KUIOPS_E_UNSUPPORTED;
    // grid axes, launches below 2^32 threads
    if (n > 65535 || t >= (1 << 24) || hq + 2 * at->hkv >= (1 << 16) || n * t * cdiv(hq + 2 * at->hkv, 32) >= (1 << 23))
        return KUIOPS_E_UNSUPPORTED;
    a.n = (int)n; a.t = (int)t; a.hq = (int)hq;
    a.qkv = qkv; a.ld_tok = ld_tok; a.ld_batch = ld_batch;
    a.lens = lens; a.pos0 = pos0; a.inv_freq = inv_freq;
    a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps; a.inv_hd = 1.0 / (double)at->hd;
    a.q = q_out; a.sq0 = sq[0]; a.sq1 = sq[1]; a.sq2 = sq[2];
    if (dtype == KUIOPS_BF16) launch_append_kind<bf16_t>(a, as_stream(stream));
    else launch_append_kind<f16_t>(a, as_stream(stream));
    return launch_status();
}

extern "C" int kuiops_kv_paged_read(int64_t n, int64_t s, int dtype, const kuiops_paged_layout *at, const void *K, const void *V,
                                    const float *k_scale, const float *v_scale, const int32_t *table, const int32_t *kv_len,
                                    void *k_out, const int64_t sko[3], void *v_out, const int64_t svo[3], int fill, void *stream) {
    if (n < 0 || s < 0 || !at || !sko || !svo) return KUIOPS_E_INVALID;
    if (n == 0 || s == 0) return KUIOPS_OK;
    ReadArgs a{};
    // (8-bit pages as fp32 too; the cache's check knows the 16-bit types)
    const bool wide = dtype == KUIOPS_F32;
    if (wide && at->dtype != KUIOPS_I8 && at->dtype != KUIOPS_F8E4M3) return KUIOPS_E_UNSUPPORTED;
    const int bad = check_cache(at, wide ? KUIOPS_BF16 : dtype, K, V, k_scale, v_scale, table, a.c);
    if (bad) return bad;
    if (!kv_len || !k_out || !v_out) return KUIOPS_E_INVALID;
    const int64_t unit = wide ? 4 : 8;
    for (int i = 0; i < 3; ++i)
        if (sko[i] % unit || svo[i] % unit) return KUIOPS_E_UNSUPPORTED;
    if (!aligned16(k_out) || !aligned16(v_out)) return KUIOPS_E_UNSUPPORTED;
    // grid axes, launches below 2^32 threads
    if (s >= (1 << 30) || n > 65535 || at->hkv > 65535 || cdiv(s, 128) * n * at->hkv >= (1 << 24)) return KUIOPS_E_UNSUPPORTED;
    a.s = (int)s; a.kv_len = kv_len;
    a.k = k_out; a.v = v_out;
    a.ko0 = sko[0]; a.ko1 = sko[1]; a.ko2 = sko[2];
    a.vo0 = svo[0]; a.vo1 = svo[1]; a.vo2 = svo[2];
    a.fill = fill;
    hipStream_t st = as_stream(stream);
    if (wide) at->dtype == KUIOPS_I8 ? launch_read<float, 1>(a, (unsigned)n, st) : launch_read<float, 2>(a, (unsigned)n, st);
    else if (dtype == KUIOPS_BF16) launch_read_kind<bf16_t>(a, (unsigned)n, st);
    else launch_read_kind<f16_t>(a, (unsigned)n, st);
    return launch_status();
}
