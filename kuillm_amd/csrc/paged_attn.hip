// Attention of the newest tokens over a paged KV cache, gfx950.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i)  over the slots j <= L - l + i
//
// of the sequence's L = kv_len[b] ones; slot j is row j % page of page
// table[b][j / page].  8-bit pages: k_j = ks_j * K_j and v_j = vs_j * V_j with a scale
// per row.  Rows of the query heads that share a KV head are one list (row = head in
// group * l + position), so K and V are read once for all of them.
#include <algorithm>

#include "paged.hpp"

namespace kuiops {

namespace {

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000);
}

constexpr float kLn2 = 0.69314718055994530942f, kLog2e = 1.44269504088896340736f;
constexpr uint32_t kOut = 0x80000000u;        // an offset past every descriptor
constexpr float kSlack = 8.f;                 // a row's maximum may grow by 2^8 before its sums are rescaled
constexpr int kMaxSplits = 64;                // (the merge has a lane for each)
constexpr int kCounterStride = 16;            // words: a cache line's atomics serialise

struct PagedArgs {
    PagedCache c;
    int n, hq, l, splits, row_groups;
    const void *Q;
    void *O;
    int64_t sq0, sq1, sq2, so0, so1, so2;
    float *lse;                // [n][hq][l], or null
    float scale_log2;          // softmax scale * log2(e), > 0
    const int32_t *kv_len;
    // splits > 1: per (sequence, KV head, row group) a counter that is zero between calls, and
    // per split 16 rows of (maximum in the log2 domain, sum) and of the unnormalised output
    unsigned *counters;
    float *ws_ml, *ws_o;
};

enum PageKind { kSame = 0, kInt8 = 1, kE4M3 = 2 };

// A probability as a sum of 16-bit parts, one MFMA each, which keeps fp32's bits: bf16
// three parts, each the leading 8 bits of what is left, cut off; f16 two, rounded, 2^-23
// of it lost and no more than half of f16's smallest step (see Shift).  With the few rows
// of this kernel the K / V stream takes the time, not the MFMAs.
template <typename T> struct Parts;
template <> struct Parts<bf16_t> {
    static constexpr int N = 3;
    static __device__ __forceinline__ float cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
    static __device__ __forceinline__ void split(float p, bf16_t (&x)[N]) {
        const float h = cut(p), r = p - h, m = cut(r);
        x[0] = (bf16_t)h;
        x[1] = (bf16_t)m;
        x[2] = (bf16_t)(r - m);
    }
};
template <> struct Parts<f16_t> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void split(float p, f16_t (&x)[N]) {
        x[0] = from_f32<f16_t>(p);
        x[1] = from_f32<f16_t>(p - to_f32(x[0]));
    }
};
// probabilities are relative to 2^(maximum + value): f16's smallest step is then 2^-39 to
// 2^-31 of the row's largest
template <typename T> struct Shift;
template <> struct Shift<bf16_t> { static constexpr float value = 0.f; };
template <> struct Shift<f16_t> { static constexpr float value = -7.f; };

// Two bf16 (the upper halves of lo and hi) in a dword.
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// Byte I of w as a number (integers up to 127 and e4m3's values are bf16's too, exactly)
template <int PK, int I>
__device__ __forceinline__ float byte_value(uint32_t w) {
    if constexpr (PK == kInt8) return (float)(int8_t)(w >> (8 * I));
    else return __builtin_amdgcn_cvt_f32_fp8((int)w, I);
}
// Bytes 0, 1 (H = 0) or 2, 3 (H = 1) of w as two bf16.
template <int PK, int H>
__device__ __forceinline__ uint32_t pair_of(uint32_t w) {
    return upper_halves(byte_value<PK, 2 * H>(w), byte_value<PK, 2 * H + 1>(w));
}
// Byte I of two words as two bf16.
template <int PK, int I>
__device__ __forceinline__ uint32_t pair_across(uint32_t a, uint32_t b) {
    return upper_halves(byte_value<PK, I>(a), byte_value<PK, I>(b));
}

// W dwords of a lane
template <int W> struct Words;
template <> struct Words<1> { typedef uint32_t type; };
template <> struct Words<2> { typedef u32x2 type; };
template <> struct Words<4> { typedef u32x4 type; };
template <int W>
__device__ __forceinline__ typename Words<W>::type load_words(__amdgpu_buffer_rsrc_t r, uint32_t voff) {
    if constexpr (W == 1) return __builtin_amdgcn_raw_buffer_load_b32(r, (int)voff, 0, 0);
    else if constexpr (W == 2) return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)voff, 0, 0));
    else return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, 0, 0));
}
__device__ __forceinline__ uint32_t word(uint32_t v, int) { return v; }
template <typename V> __device__ __forceinline__ uint32_t word(const V &v, int i) { return v[i]; }

// ------------------------------------------------------------------------
// paged_attn_kernel -- a work-group has up to 16 query rows of a KV head and a run of its
// slots; its 4 waves take 32 slots in turn.  Pages are multiples of 16 rows, so 16 slots
// lie in one page: every load has its page's address in scalar registers, and a buffer
// descriptor that ends with the page's (or the sequence's) last row, so rows behind it and
// absent pages read as zeros and nothing is read there.  The pages' numbers of 32 turns are
// fetched at once, a lane each.
//   S = K Q^T (16x16x32 MFMA): K straight to registers, 16 bytes a lane; a lane then holds
//   8 scores of one row, keys 16 t + 4 G + i (G = lane / 16): the row's maximum crosses
//   lanes 16 and 32 apart only.
//   O^T += V^T P^T: the scores' registers are the second operand as they stand.  The first
//   wants 8 keys of a column in a lane: a lane loads HD / 16 adjacent columns of its 8 keys
//   (16 lanes a whole row) and transposes them in registers, so neither product needs LDS.
// A part that is 0 times an infinite value is NaN, so is a masked NaN: a wave whose sums
// are not finite goes over its keys again with the row maxima that it found, value by value
// for the rows that see them.
template <typename T, int PK, int HD>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedArgs a) {
    typedef typename std::conditional<PK == kSame, T, bf16_t>::type C;       // the products' type
    typedef typename Mfma<C>::frag frag;
    typedef C c8 __attribute__((ext_vector_type(8)));
    constexpr int NWV = 4, KB = 32, R = 16, NP = Parts<C>::N;
    constexpr int B = PK == kSame ? 2 : 1;            // bytes of a cached value
    constexpr int KK = HD / 32, KL = HD * B / 64;     // MFMAs over a key, loads of 16 keys
    constexpr int DT = HD / 16, VW = DT * B / 4;      // columns of V a lane has, in dwords
    constexpr int NQ = PK != kSame && sizeof(T) == 2 && !std::is_same<T, bf16_t>::value ? 2 : 1;
    typedef typename Words<VW>::type vwords;
    constexpr int LD = HD + 4;                        // row stride of the waves' sums in LDS
    __shared__ float so[NWV][R][LD], sm[NWV][R], sl[NWV][R];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, G4 = lane >> 4;

    // the row groups of a (sequence, KV head, split) run on one XCD, whose L2 then has the
    // keys for all but the first
    const int idx = blockIdx.x >> 3, unit = idx / a.row_groups * 8 + (blockIdx.x & 7), rg = idx % a.row_groups;
    if (unit >= a.n * a.c.hkv * a.splits) return;
    const int split = unit % a.splits, bh = unit / a.splits, b = bh / a.c.hkv, hk = bh % a.c.hkv;
    const int G = a.hq / a.c.hkv, rows_kv = G * a.l, r0 = rg * R, nrows = min(R, rows_kv - r0);

    const int L = paged_len(a.c, a.kv_len, b);
    // whole turns of the work-group, spread evenly over the sequence's splits
    const int turns = (L + NWV * KB - 1) / (NWV * KB);
    const int per = max(1, (turns + a.splits - 1) / a.splits), used = max(1, (turns + per - 1) / per);
    if (split >= used) return;
    const int kbeg = split * per * NWV * KB, kend = min(L, kbeg + per * NWV * KB);
    const int free_end = L - a.l + 1;                 // slots below are seen by every row

    // the query: row r0 + lr
    const int rr = r0 + lr;
    const bool row_ok = rr < rows_kv;
    const int h = row_ok ? rr / a.l : 0, pos = row_ok ? rr - h * a.l : 0;
    const int last = L - a.l + pos;                   // the row's last slot
    frag qf[NQ][KK];
    {
        const T *q = reinterpret_cast<const T *>(a.Q) + b * a.sq0 + (hk * G + h) * a.sq1 + pos * a.sq2;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            // (columns in the order of K's loads: 8-bit ones bring 16 columns, for two MFMAs)
            const int d = B == 2 ? kk * 32 + G4 * 8 : (kk >> 1) * 64 + G4 * 16 + (kk & 1) * 8;
            const u32x4 raw = row_ok && d < a.c.hd ? *reinterpret_cast<const u32x4 *>(q + d) : u32x4{0, 0, 0, 0};
            if constexpr (NQ == 1) qf[0][kk] = as_frag<frag>(raw);
            else {
                // f16 as two bf16: 8 bits and the 3 behind them
                typedef T t8 __attribute__((ext_vector_type(8)));
                const t8 v = __builtin_bit_cast(t8, raw);
                c8 hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = to_f32(v[e]), top = Parts<bf16_t>::cut(x);
                    hi[e] = (C)top;
                    lo[e] = (C)(fabsf(x) < INFINITY ? x - top : 0.f);
                }
                qf[0][kk] = __builtin_bit_cast(frag, hi);
                qf[1][kk] = __builtin_bit_cast(frag, lo);
            }
        }
    }

    uint32_t offK[KL];
#pragma unroll
    for (int j = 0; j < KL; ++j) {
        const int d = (j * 64 + G4 * 16) / B;
        offK[j] = d < a.c.hd ? (uint32_t)((lr * a.c.sk2 + d) * B) : kOut;
    }
    uint32_t offV[4];                                 // rows 4 G4 + i of 16
#pragma unroll
    for (int i = 0; i < 4; ++i) offV[i] = lr * DT < a.c.hd ? (uint32_t)(((4 * G4 + i) * a.c.sv2 + lr * DT) * B) : kOut;

    // page numbers (-1: none) and rows of the 16-slot groups of 32 turns, a lane each
    auto group_key = [&](int turn, int g) __attribute__((always_inline)) { return kbeg + (turn * NWV + wave) * KB + 16 * g; };
    auto fetch = [&](int turn0, int &id, int &row) __attribute__((always_inline)) {
        id = paged_find16(a.c.table + b * a.c.ld_table, a.c.page, a.c.pages, group_key(turn0 + (lane >> 1), lane & 1), kend, row);
    };
    int id_now, row_now, id_next, row_next, turn0 = 0;
    fetch(0, id_now, row_now);
    fetch(32, id_next, row_next);

    struct Stage {
        u32x4 k[2][KL];
        vwords v[8];
        f32x4 ks[2], vs[2];
        int n[2];                                     // rows of the two groups that are there
    };
    Stage st[2];
    const char *Kp = reinterpret_cast<const char *>(a.c.K) + hk * a.c.sk1 * B, *Vp = reinterpret_cast<const char *>(a.c.V) + hk * a.c.sv1 * B;
    auto issue = [&](int turn, Stage &s) __attribute__((always_inline)) {
        if (turn >= turn0 + 32) {
            turn0 += 32;
            id_now = id_next;
            row_now = row_next;
            fetch(turn0 + 32, id_next, row_next);
        }
        __amdgpu_buffer_rsrc_t rv[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int from = 2 * (turn - turn0) + t;
            const int id = __builtin_amdgcn_readlane(id_now, from), row = __builtin_amdgcn_readlane(row_now, from);
            const int m = s.n[t] = paged_rows16(id, group_key(turn, t), kend);
            const int64_t page = max(id, 0);
            const __amdgpu_buffer_rsrc_t rk =
                make_rsrc(Kp + (page * a.c.sk0 + row * a.c.sk2) * B, m ? (uint32_t)(((m - 1) * a.c.sk2 + a.c.hd) * B) : 0u);
            rv[t] = make_rsrc(Vp + (page * a.c.sv0 + row * a.c.sv2) * B, m ? (uint32_t)(((m - 1) * a.c.sv2 + a.c.hd) * B) : 0u);
#pragma unroll
            for (int j = 0; j < KL; ++j) s.k[t][j] = load_words<4>(rk, offK[j]);
            if constexpr (PK != kSame) {
                s.ks[t] = __builtin_bit_cast(f32x4, load_words<4>(make_rsrc(a.c.ks + page * a.c.sks0 + hk * a.c.sks1 + row, m * 4), G4 * 16));
                s.vs[t] = __builtin_bit_cast(f32x4, load_words<4>(make_rsrc(a.c.vs + page * a.c.svs0 + hk * a.c.svs1 + row, m * 4), G4 * 16));
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s.v[j] = load_words<VW>(rv[j >> 2], offV[j & 3]);
        __builtin_amdgcn_sched_barrier(0);
    };

    // scores of a turn, scales of K in them: (t, i) is slot k0 + 16 t + 4 G4 + i; unseen ones -inf
    auto scores = [&](int turn, const Stage &s, f32x4 *sc) __attribute__((always_inline)) {
        const int k0 = group_key(turn, 0);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                u32x4 kw;
                if constexpr (PK == kSame) kw = s.k[t][kk];
                else {
                    const uint32_t w0 = s.k[t][kk >> 1][2 * (kk & 1)], w1 = s.k[t][kk >> 1][2 * (kk & 1) + 1];
                    kw = u32x4{pair_of<PK, 0>(w0), pair_of<PK, 1>(w0), pair_of<PK, 0>(w1), pair_of<PK, 1>(w1)};
                }
#pragma unroll
                for (int y = 0; y < NQ; ++y) sc[t] = Mfma<C>::m16(as_frag<frag>(kw), qf[y][kk], sc[t]);
            }
            if constexpr (PK != kSame) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[t][i] *= s.ks[t][i];
            }
        }
        if (k0 + KB > free_end || s.n[0] + s.n[1] < KB) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * G4 + i >= s.n[t] || k0 + 16 * t + 4 * G4 + i > last) sc[t][i] = -INFINITY;
        }
    };

    f32x4 o[DT];                                      // o[c][i]: column (4 G4 + i) * DT + c of row lr
    float m_used = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int c = 0; c < DT; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto step = [&](int turn, const Stage &s) __attribute__((always_inline)) {
        f32x4 sc[2];
        scores(turn, s, sc);
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[t][i]);
        mx = xor_max<32>(xor_max<16>(mx)) * a.scale_log2;
        if (__any(mx > m_used + kSlack)) {
            const float m_new = fmaxf(m_used, mx);
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_used - m_new);
            l_run *= alpha;
#pragma unroll
            for (int c = 0; c < DT; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[c][i] *= alpha;
            m_used = m_new;
        }
        const float mref = m_used == -INFINITY ? 0.f : m_used + Shift<C>::value;
        c8 part[NP];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float p = fast_exp2(__builtin_fmaf(sc[t][i], a.scale_log2, -mref));
                l_run += p;
                if constexpr (PK != kSame) p *= s.vs[t][i];
                C x[NP];
                Parts<C>::split(p, x);
#pragma unroll
                for (int y = 0; y < NP; ++y) part[y][4 * t + i] = x[y];
            }
#pragma unroll
        for (int c = 0; c < DT; ++c) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (PK == kSame) {
                    const uint32_t lo = word(s.v[2 * e], c >> 1), hi = word(s.v[2 * e + 1], c >> 1);
                    w[e] = c & 1 ? __builtin_amdgcn_perm(hi, lo, 0x07060302u) : __builtin_amdgcn_perm(hi, lo, 0x05040100u);
                } else {
                    const uint32_t lo = word(s.v[2 * e], c >> 2), hi = word(s.v[2 * e + 1], c >> 2);
                    switch (c & 3) {
                        case 0: w[e] = pair_across<PK, 0>(lo, hi); break;
                        case 1: w[e] = pair_across<PK, 1>(lo, hi); break;
                        case 2: w[e] = pair_across<PK, 2>(lo, hi); break;
                        default: w[e] = pair_across<PK, 3>(lo, hi); break;
                    }
                }
            }
#pragma unroll
            for (int y = 0; y < NP; ++y) o[c] = Mfma<C>::m16(as_frag<frag>(w), __builtin_bit_cast(frag, part[y]), o[c]);
        }
    };

    // turns of this wave whose first slot is below kend
    const int mine = (kend - kbeg - wave * KB + NWV * KB - 1) / (NWV * KB);
    issue(0, st[0]);
    for (int turn = 0; turn < mine; turn += 2) {
        issue(turn + 1, st[1]);
        step(turn, st[0]);
        __builtin_amdgcn_sched_barrier(0);
        issue(turn + 2, st[0]);
        if (turn + 1 < mine) step(turn + 1, st[1]);
        __builtin_amdgcn_sched_barrier(0);
    }

    float z = 0.f;                  // stays 0 if every sum is finite
#pragma unroll
    for (int c = 0; c < DT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) z = __builtin_fmaf(o[c][i], 0.f, z);
    if (__any(z != 0.f)) {
#pragma unroll
        for (int c = 0; c < DT; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float mref = m_used == -INFINITY ? 0.f : m_used + Shift<C>::value;
        turn0 = 0;
        fetch(0, id_now, row_now);
        fetch(32, id_next, row_next);
        for (int turn = 0; turn < mine; ++turn) {
            issue(turn, st[0]);
            f32x4 sc[2];
            scores(turn, st[0], sc);
            const int k0 = group_key(turn, 0);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                float p = fast_exp2(__builtin_fmaf(sc[x >> 2][x & 3], a.scale_log2, -mref));
                if constexpr (PK != kSame) p *= st[0].vs[x >> 2][x & 3];
                const int from = 2 * (turn - turn0) + (x >> 2);
                const int64_t page = max(0, __builtin_amdgcn_readlane(id_now, from));
                const int row = __builtin_amdgcn_readlane(row_now, from);
                for (int g = 0; g < 4; ++g) {
                    const int at = 4 * g + (x & 3);
                    const float pk = __shfl(p, g * 16 + lr, 64);
                    if (at >= st[0].n[x >> 2] || !row_ok || k0 + 16 * (x >> 2) + at > last) continue;
                    const char *vp = Vp + (page * a.c.sv0 + (int64_t)(row + at) * a.c.sv2) * B;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int c = 0; c < DT; ++c) {
                            const int d = (4 * G4 + i) * DT + c;
                            if (d >= a.c.hd) continue;
                            float v;
                            if constexpr (PK == kSame) v = to_f32(reinterpret_cast<const T *>(vp)[d]);
                            else v = byte_value<PK, 0>((uint32_t)(uint8_t)vp[d]);
                            o[c][i] += pk * v;
                        }
                }
            }
        }
    }

    // the waves' sums merge through LDS; lanes of a row hold disjoint keys
    l_run = xor_add<32>(xor_add<16>(l_run));
    if (G4 == 0) {
        sm[wave][lr] = m_used + Shift<C>::value;
        sl[wave][lr] = l_run;
    }
    if (lr < nrows) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < DT; c += 4)
                *reinterpret_cast<f32x4 *>(&so[wave][lr][(4 * G4 + i) * DT + c]) = f32x4{o[c][i], o[c + 1][i], o[c + 2][i], o[c + 3][i]};
    }
    __syncthreads();

    constexpr int D4 = HD / 4;
    auto store_row = [&](int r, int d, f32x4 v, float m, float ls) __attribute__((always_inline)) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        const int head = hk * G + (r0 + r) / a.l, i = (r0 + r) % a.l;
        const float inv = ls != 0.f ? 1.f / ls : 0.f;
        if (d < a.c.hd) {
            t4 w;
#pragma unroll
            for (int y = 0; y < 4; ++y) w[y] = from_f32<T>(v[y] * inv);
            *reinterpret_cast<t4 *>(reinterpret_cast<T *>(a.O) + b * a.so0 + head * a.so1 + i * a.so2 + d) = w;
        }
        if (a.lse && d == 0) a.lse[((int64_t)b * a.hq + head) * a.l + i] = ls != 0.f ? (m + __log2f(ls)) * kLn2 : -INFINITY;
    };
    // the splits' states of this row group, agent-coherent (sc1): written through the XCD's L2
    // and read past it, as the work-group that merges them may run on another XCD
    const int group = bh * a.row_groups + rg;
    const int64_t slot0 = (int64_t)group * a.splits * R;
    const bool alone = used == 1;
    const __amdgpu_buffer_rsrc_t rs_o = make_rsrc(alone ? nullptr : a.ws_o + slot0 * HD, alone ? 0u : (uint32_t)a.splits * R * HD * 4);
    const __amdgpu_buffer_rsrc_t rs_ml = make_rsrc(alone ? nullptr : a.ws_ml + slot0 * 2, alone ? 0u : (uint32_t)a.splits * R * 8);
    for (int x = tid; x < nrows * D4; x += NWV * 64) {
        const int r = x / D4, d = x % D4 * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < NWV; ++w) mm = fmaxf(mm, sm[w][r]);
        const float mu = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f;
        f32x4 oo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NWV; ++w) {
            const float wgt = fast_exp2(sm[w][r] - mu);
            ll = __builtin_fmaf(sl[w][r], wgt, ll);
            const f32x4 ov = *reinterpret_cast<const f32x4 *>(&so[w][r][d]);
#pragma unroll
            for (int i = 0; i < 4; ++i) oo[i] = __builtin_fmaf(ov[i], wgt, oo[i]);
        }
        if (alone) {
            store_row(r, d, oo, mm, ll);
            continue;
        }
        const int at = split * R + r;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, oo), rs_o, (at * HD + d) * 4, 0, kSc1Aux);
        if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{mm, ll}), rs_ml, at * 8, 0, kSc1Aux);
    }
    if (alone) return;

    // The last of the row group's work-groups to arrive merges the splits, in their order
    // (the same bits whatever the order of arrival).  Every thread waits for its stores'
    // acknowledgements before the barrier that precedes the counter's agent-scope addition.
    __shared__ int s_last;
    __shared__ float s_w[R][kMaxSplits], s_M[R], s_L[R];
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    unsigned *ctr = a.counters + (int64_t)group * kCounterStride;
    if (tid == 0) s_last = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(used - 1);
    __syncthreads();
    if (!s_last) return;
    for (int r = wave; r < nrows; r += NWV) {
        u32x2 ml = {__float_as_uint(-INFINITY), 0u};
        if (lane < used) ml = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs_ml, (lane * R + r) * 8, 0, kSc1Aux));
        const float mz = __uint_as_float(ml[0]), M = wave_max(mz), Mu = M == -INFINITY ? 0.f : M;
        const float w = fast_exp2(mz - Mu);
        s_w[r][lane] = w;
        const float Ls = wave_sum(w * __uint_as_float(ml[1]));
        if (lane == 0) {
            s_M[r] = M;
            s_L[r] = Ls;
        }
    }
    __syncthreads();
    for (int x = tid; x < nrows * D4; x += NWV * 64) {
        const int r = x / D4, d = x % D4 * 4;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int z0 = 0; z0 < used; z0 += 16) {
            f32x4 ov[16];
#pragma unroll
            for (int z = 0; z < 16; ++z)
                // (splits that are not there: past the end of the descriptor, no memory is read)
                ov[z] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                      rs_o, z0 + z < used ? (((z0 + z) * R + r) * HD + d) * 4 : (int)kOut, 0, kSc1Aux));
#pragma unroll
            for (int z = 0; z < 16; ++z) {
                const float w = z0 + z < used ? s_w[r][z0 + z] : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(w, ov[z][i], acc[i]);
            }
        }
        store_row(r, d, acc, s_M[r], s_L[r]);
    }
    if (tid == 0) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ------------------------------------------------------------- host side

struct PagedPlan {
    int row_groups, splits;
    int64_t units;
    size_t counter_bytes, ml_bytes, o_bytes;
};

constexpr int kCUs = 256;
// The counters' part of a workspace, the same for calls of all sizes: groups that are split
// are at most one a CU.
constexpr size_t kCounterBytes = (size_t)kCUs * kCounterStride * 4;

PagedPlan plan_of(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t slots, int64_t hd) {
    PagedPlan p{};
    const int64_t rows = hq / hkv * l;
    p.row_groups = (int)cdiv(rows, 16);
    const int64_t groups = n * hkv * p.row_groups;
    // two work-groups a CU, of a turn (128 slots) at least
    p.splits = (int)std::max<int64_t>(1, std::min({(int64_t)kMaxSplits, 2 * kCUs / std::max<int64_t>(groups, 1), cdiv(slots, 128)}));
    p.units = n * hkv * p.splits;
    if (p.splits > 1) {
        p.counter_bytes = kCounterBytes;
        p.ml_bytes = (size_t)groups * p.splits * 16 * 8;
        p.o_bytes = (size_t)groups * p.splits * 16 * (hd <= 64 ? 64 : 128) * 4;
    }
    return p;
}

template <typename T, int PK>
void launch_paged(const PagedArgs &a, const PagedPlan &p, hipStream_t st) {
    const dim3 grid((unsigned)(cdiv(p.units, 8) * 8 * p.row_groups));
    if (a.c.hd <= 64) hipLaunchKernelGGL((paged_attn_kernel<T, PK, 64>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_attn_kernel<T, PK, 128>), grid, dim3(256), 0, st, a);
}

template <typename T>
void launch_paged_kind(const PagedArgs &a, const PagedPlan &p, hipStream_t st) {
    if (a.c.dtype == KUIOPS_I8) launch_paged<T, kInt8>(a, p, st);
    else if (a.c.dtype == KUIOPS_F8E4M3) launch_paged<T, kE4M3>(a, p, st);
    else launch_paged<T, kSame>(a, p, st);
}

}  // namespace

}  // namespace kuiops

using namespace kuiops;

extern "C" size_t kuiops_sdpa_paged_workspace(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t slots, int64_t hd) {
    if (n <= 0 || hq <= 0 || hkv <= 0 || l <= 0 || slots <= 0 || hd <= 0 || hq % hkv) return 0;
    const PagedPlan p = plan_of(n, hq, hkv, l, slots, hd);
    return p.counter_bytes + p.ml_bytes + p.o_bytes;
}

extern "C" int kuiops_sdpa_paged(int64_t n, int64_t hq, int64_t l, int dtype, const void *Q, const int64_t sq[3],
                                 const kuiops_paged_layout *at, const void *K, const void *V, const float *k_scale,
                                 const float *v_scale, const int32_t *table, const int32_t *kv_len, void *O, const int64_t so[3],
                                 float *lse, float scale, void *workspace, size_t workspace_bytes, void *stream) {
    if (n < 0 || hq < 0 || l < 0 || !sq || !so || !at || at->hkv <= 0 || hq % at->hkv) return KUIOPS_E_INVALID;
    if (n == 0 || hq == 0 || l == 0) return KUIOPS_OK;
    PagedArgs a{};
    const int bad = check_cache(at, dtype, K, V, k_scale, v_scale, table, a.c);
    if (bad) return bad;
    if (!Q || !O || !kv_len) return KUIOPS_E_INVALID;
    if (!(scale > 0.f) || !(scale * kLog2e < INFINITY)) return KUIOPS_E_UNSUPPORTED;
    if (!aligned16(Q) || (reinterpret_cast<uintptr_t>(O) & 7)) return KUIOPS_E_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (sq[i] % 8 || so[i] % 4) return KUIOPS_E_UNSUPPORTED;
    // 32-bit indices of rows and work-groups, launches below 2^32 threads
    const int64_t rows = hq / at->hkv * l;
    if (l >= (1 << 24) || rows >= (1 << 24) || n * hq * l >= ((int64_t)1 << 31) || n * at->hkv >= (1 << 20)) return KUIOPS_E_UNSUPPORTED;
    const PagedPlan p = plan_of(n, hq, at->hkv, l, at->width * at->page, at->hd);
    if (cdiv(p.units, 8) * 8 * p.row_groups >= ((int64_t)1 << 24)) return KUIOPS_E_UNSUPPORTED;
    const size_t need = p.counter_bytes + p.ml_bytes + p.o_bytes;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KUIOPS_E_WORKSPACE;
    a.n = (int)n; a.hq = (int)hq; a.l = (int)l; a.splits = p.splits; a.row_groups = p.row_groups;
    a.Q = Q; a.O = O;
    a.sq0 = sq[0]; a.sq1 = sq[1]; a.sq2 = sq[2];
    a.so0 = so[0]; a.so1 = so[1]; a.so2 = so[2];
    a.lse = lse;
    a.scale_log2 = scale * kLog2e;
    a.kv_len = kv_len;
    char *ws = reinterpret_cast<char *>(workspace);
    a.counters = reinterpret_cast<unsigned *>(ws);
    a.ws_o = reinterpret_cast<float *>(ws + p.counter_bytes);
    a.ws_ml = reinterpret_cast<float *>(ws + p.counter_bytes + p.o_bytes);
    if (dtype == KUIOPS_BF16) launch_paged_kind<bf16_t>(a, p, as_stream(stream));
    else launch_paged_kind<f16_t>(a, p, as_stream(stream));
    return launch_status();
}
