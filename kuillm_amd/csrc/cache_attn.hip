// Attention over a KV cache for drafted trees and for summed weights, gfx950.
//
//   kuiops_sdpa_tree          the last t keys of a sequence are the nodes of a
//       tree of drafted tokens; node i sees the context before the tree, its
//       ancestors and itself.
//   kuiops_sdpa_decode_accum  causal (bottom-right) or full attention that
//       also adds every key's weight, summed over the query rows of its KV
//       head, to a running fp32 sum per key.
//
// Both are o_i = sum_j p_ij v_j, p_ij = exp(scale q_i k_j - lse_i) over the
// keys j that row i sees, and differ in which keys those are:
//   keys below `free_end`  are seen by every row of the sequence,
//   the others             by the rows that a bit of the row's mask (tree) or a
//                          bound per row (causal) says.
// Rows of the query heads that share a KV head are one list (row = head in
// group * l + position), so K and V are read once for all of them.
#include <algorithm>
#include <type_traits>

#include "prob_parts.hpp"

namespace kuiops {

namespace {

typedef __attribute__((address_space(3))) char lds_char;
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ lds_char *to_lds(const void *p) { return (lds_char *)(const_cast<void *>(p)); }
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000);
}
// 16 bytes per lane into dst + 16 * lane; zeros past the descriptor's size
__device__ __forceinline__ void dma16_buf(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff, const void *dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)to_lds(dst), 16, (int)voff, (int)soff,
                                             0, 0);
}

constexpr float kLn2 = 0.69314718055994530942f, kLog2e = 1.44269504088896340736f;
constexpr int kMaxTree = 256;                 // nodes of a tree
constexpr int kTreeWords = kMaxTree / 64;
constexpr uint32_t kOut = 0x80000000u;        // an offset past every descriptor

enum Mode { kFull = 0, kCausal = 1, kTree = 2 };

struct CacheAttnArgs {
    int n, hq, hkv, l, e, ev, mode;
    int64_t s;
    const void *Q, *K, *V;
    void *O;
    int64_t sq0, sq1, sq2, sk0, sk1, sk2, sv0, sv1, sv2, so0, so1, so2;
    float *lse;                // [n][hq][l], or null
    float scale_log2;          // softmax scale * log2(e), > 0
    const int32_t *kv_len;     // [n] device, or null: s
    const int32_t *parent;     // kTree: [n][l]
    int splits, row_groups;    // row groups that work-groups begin with: half of them with `pair`
    int pair;
    int head_tiles;            // cache_rows_kernel: row groups of a head where none crosses heads, else 0
    float *ws_ml;              // [splits][n * hq * l][2]: maximum (log2 domain), sum
    float *ws_o;               // [splits][n * hq * l][HD]: unnormalised output
    float *acc;                // kuiops_sdpa_decode_accum: per key sums, strides sa0, sa1, 1
    int64_t sa0, sa1;
    float *scores;             // [n][hkv][hq / hkv * l][spad]: q k, -inf where not seen; or null
    int sum_here;              // a work-group has all rows and keys of its KV head: it adds up the weights itself
    int64_t spad;
    float *part_sums;          // key_weights_kernel: [parts][n][hkv][spad], or null
};

__device__ __forceinline__ int keys_of(const CacheAttnArgs &a, int b) {
    return a.kv_len ? (int)max((int64_t)0, min((int64_t)a.kv_len[b], a.s)) : (int)a.s;
}

// Which nodes each node of the tree sees (itself and its ancestors), as bits, by
// pointer doubling: after round r a node's word holds its 2^r nearest ancestors
// and `up` the next one, so 6 rounds suffice for 64 nodes, 8 for 256, and a
// shallow tree stops early.  A node is absent if its parent is below -1 or not
// an earlier node, or if an ancestor of it is: it then sees nothing.
//
// Up to 64 nodes: lane i of every wave has node i, no LDS and no barrier, so the
// first keys' loads stay in flight meanwhile.
__device__ __forceinline__ uint64_t tree_bits_wave(const int32_t *parent, int t) {
    const int i = threadIdx.x & 63;
    const int p = i < t ? parent[i] : -1;
    int bad = p < -1 || p >= i;
    int up = bad ? -1 : p;
    uint32_t lo = i < 32 ? 1u << i : 0u, hi = i < 32 ? 0u : 1u << (i - 32);
    while (__any(up >= 0)) {
        const int from = up >= 0 ? up : i;
        const uint32_t l2 = __shfl(lo, from, 64), h2 = __shfl(hi, from, 64);
        const int b2 = __shfl(bad, from, 64), u2 = __shfl(up, from, 64);
        lo |= l2;
        hi |= h2;
        bad |= b2;
        up = up >= 0 ? u2 : -1;
    }
    return bad ? 0 : (uint64_t)hi << 32 | lo;
}
// More nodes: thread i has node i, words in LDS.
struct TreeBits {
    uint64_t w[kMaxTree][kTreeWords];
    int16_t up[kMaxTree];
    int16_t bad[kMaxTree];
};
template <int NT>
__device__ __forceinline__ void tree_bits(TreeBits &tb, const int32_t *parent, int t) {
    static_assert(NT >= kMaxTree, "a thread per node");
    const int i = threadIdx.x;
    const bool mine = i < t;
    uint64_t w[kTreeWords];
    int up = -1, bad = 0;
    if (mine) {
        const int p = parent[i];
        bad = p < -1 || p >= i;
        up = bad ? -1 : p;
#pragma unroll
        for (int x = 0; x < kTreeWords; ++x) {
            w[x] = (i >> 6) == x ? 1ull << (i & 63) : 0;
            tb.w[i][x] = w[x];
        }
        tb.up[i] = (int16_t)up;
        tb.bad[i] = (int16_t)bad;
    }
    while (__syncthreads_or(mine && up >= 0)) {
        int nup = -1;
        if (mine && up >= 0) {
#pragma unroll
            for (int x = 0; x < kTreeWords; ++x) w[x] |= tb.w[up][x];
            bad |= tb.bad[up];
            nup = tb.up[up];
        }
        __syncthreads();
        if (mine && up >= 0) {
#pragma unroll
            for (int x = 0; x < kTreeWords; ++x) tb.w[i][x] = w[x];
            tb.up[i] = (int16_t)nup;
            tb.bad[i] = (int16_t)bad;
        }
        up = nup;
    }
    if (mine && bad) {
#pragma unroll
        for (int x = 0; x < kTreeWords; ++x) tb.w[i][x] = 0;
    }
    __syncthreads();
}

// The row's first n >= 0 of 64 keys.
__device__ __forceinline__ uint64_t first_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// Which of the keys k0 .. k0 + 63 a row sees, as bits: `mine` is its word of the
// tree's nodes where the tree has at most 64, else the words are tb's.
__device__ __forceinline__ uint64_t seen_word(const CacheAttnArgs &a, const TreeBits *tb, uint64_t mine, int pos, int k0, int L) {
    const int first = L - a.l;
    if (a.mode != kTree) return first_bits((a.mode == kCausal ? min(L, first + pos + 1) : L) - k0);
    const int j0 = k0 - first;                // the tree's node of key k0
    if (j0 <= -64) return ~0ull;
    if (a.l <= 64) return j0 < 0 ? mine << -j0 | first_bits(-j0) : j0 < 64 ? mine >> j0 : 0;
    if (j0 < 0) return tb->w[pos][0] << -j0 | first_bits(-j0);
    const int w = j0 >> 6, sh = j0 & 63;
    uint64_t r = w < kTreeWords ? tb->w[pos][w] >> sh : 0;
    if (sh && w + 1 < kTreeWords) r |= tb->w[pos][w + 1] << (64 - sh);
    return r;
}

// How many of the first L keys a row of causal or full attention sees.  Its weights go
// to them alone: a row of NaN leaves the other keys' sums as they are.
__device__ __forceinline__ int keys_seen(const CacheAttnArgs &a, int pos, int L) {
    return a.mode == kCausal ? min(L, L - a.l + pos + 1) : L;
}

// What a work-group works on: the row groups of a (sequence, KV head, split)
// run on one XCD, whose L2 then has the keys for all but the first.
struct Unit {
    int b, hk, split, rg;
    bool any;
};
__device__ __forceinline__ Unit unit_of(const CacheAttnArgs &a) {
    const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
    const int unit = idx / a.row_groups * 8 + xcd;
    Unit u;
    u.any = unit < a.n * a.hkv * a.splits;
    u.rg = idx % a.row_groups;
    u.split = unit % a.splits;
    const int bh = unit / a.splits;
    u.b = bh / a.hkv;
    u.hk = bh % a.hkv;
    return u;
}

// 4 output columns of a row: o * (1 / sum), and the row's log-sum-exp
template <typename T>
__device__ __forceinline__ void store_row(const CacheAttnArgs &a, int64_t b, int head, int i, int d, f32x4 o, float m, float l) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const float inv = l != 0.f ? 1.f / l : 0.f;
    if (d < a.ev) {
        t4 w;
#pragma unroll
        for (int y = 0; y < 4; ++y) w[y] = from_f32<T>(o[y] * inv);
        *reinterpret_cast<t4 *>(reinterpret_cast<T *>(a.O) + b * a.so0 + head * a.so1 + i * a.so2 + d) = w;
    }
    if (a.lse && d == 0) a.lse[(b * a.hq + head) * a.l + i] = l != 0.f ? (m + __log2f(l)) * kLn2 : -INFINITY;
}

// ------------------------------------------------------------------------
// cache_attn_kernel -- few rows per KV head: a work-group has 16 query rows, and
// each of its 4 waves key steps of 32 of its own.
//   S = K Q^T (16x16x32 MFMA): K straight from memory to registers; a lane
//   holds 8 scores of one row, the row's maximum crosses lanes 16 and 32 apart
//   only.  O^T += V^T P^T: V through LDS (DMA), read transposed;
//   the scores' registers are the other operand as they stand, keys numbered
//   in that order.  The probability is the sum of 16-bit parts that keep fp32's
//   bits, one MFMA each (see Parts): with the few rows of this kernel the K / V
//   stream takes the time, not the MFMAs (bf16, two parts against three, calls, us: 8
//   rows over 500 keys 11.1 / 11.1, 16 sequences of 4000 keys with weights 54.5 / 54.6).
// K needs no LDS because a wave shares its keys with no other; V does, as the MFMA
// wants 8 keys of a column in a lane.  Measured: 4 sequences of 1153 to 2013 keys, 32 / 32
// heads of 128, 13 rows: 24.7 us, 4.2 TB/s; 8 rows over 500 keys, one sequence: 7.9 us, all
// of it latency (key count, query, first keys, three steps of them, waves' merge).
// A part that is 0 times an infinite value is NaN, so is a masked NaN: a wave
// whose sums are not finite goes over its keys again with the row maxima that
// it found, multiplying value by value for the rows that see them.
template <typename T, int HD>
__global__ __launch_bounds__(256) void cache_attn_kernel(CacheAttnArgs a) {
    constexpr int NWV = 4, KB = 32, R = 16;
    constexpr int RB = HD * 2, VT = KB * RB;          // bytes per V row / wave tile
    constexpr int KK = HD / 32, DT = HD / 16, DV = VT / 1024, NP = Parts<T>::N;
    typedef typename Mfma<T>::frag frag;
    typedef T t8 __attribute__((ext_vector_type(8)));
    __shared__ __attribute__((aligned(1024))) char sV0[NWV * VT], sV1[NWV * VT];
    __shared__ float sm[NWV][R], sl[NWV][R], s_max[R], s_inv[R];
    __shared__ int s_seen[R];
    __shared__ TreeBits tb;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, G4 = lane >> 4;
    const Unit u = unit_of(a);
    if (!u.any) return;
    const int b = u.b, hk = u.hk, split = u.split;
    const int G = a.hq / a.hkv, rows_kv = G * a.l, r0 = u.rg * R;

    const int L = keys_of(a, b);
    const int steps = (L + KB - 1) / KB;
    // a sequence's steps are spread evenly over its splits, whole steps of the work-group
    const int chunk = (steps + a.splits * NWV - 1) / (a.splits * NWV) * NWV * KB;
    const int kbeg = min(L, split * chunk), kend = min(L, kbeg + chunk);
    // keys below free_end are seen by every row
    const int free_end = a.mode == kFull ? L : a.mode == kCausal ? L - a.l + 1 : L - a.l;

    const T *Kp = reinterpret_cast<const T *>(a.K) + b * a.sk0 + hk * a.sk1 + (int64_t)kbeg * a.sk2;
    const T *Vp = reinterpret_cast<const T *>(a.V) + b * a.sv0 + hk * a.sv1 + (int64_t)kbeg * a.sv2;
    const uint32_t kbytes = kend > kbeg ? (uint32_t)(((int64_t)(kend - kbeg - 1) * a.sk2 + a.e) * 2) : 0u;
    const uint32_t vbytes = kend > kbeg ? (uint32_t)(((int64_t)(kend - kbeg - 1) * a.sv2 + a.ev) * 2) : 0u;

    // V tile: 16-byte chunk c of row r at position c ^ vsw(r): the 16 rows x 32
    // bytes of a transposing read fall on the 64 banks evenly.
    auto vsw = [](int r) { return HD >= 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); };
    uint32_t offV[DV];
#pragma unroll
    for (int j = 0; j < DV; ++j) {
        const int ch = j * 64 + lane, r = ch / (HD / 8), c = (ch % (HD / 8)) ^ vsw(r);
        offV[j] = c * 8 < a.ev ? (uint32_t)((r * a.sv2 + c * 8) * 2) : kOut;
    }
    uint32_t offK[2][KK];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
            offK[t][kk] = kk * 32 + G4 * 8 < a.e ? (uint32_t)(((lr + 16 * t) * a.sk2 + kk * 32 + G4 * 8) * 2) : kOut;
    int offVr[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        const int r = 4 * G4 + (lr >> 2), d = dt * 16 + 4 * (lr & 3);
        offVr[dt] = r * RB + (((d >> 3) ^ vsw(r)) << 4) + ((d >> 2) & 1) * 8;      // vsw(r + 16) == vsw(r)
    }
    u32x4 kr[2][2][KK];
    // keys k0 .. k0 + 31 (nothing past kend): K into registers `slot`, V into tile sv
    auto issue = [&](int k0, int slot, char *sv) __attribute__((always_inline)) {
        const bool on = k0 < kend;
        const uint32_t kb = on ? (uint32_t)((int64_t)(k0 - kbeg) * a.sk2 * 2) : 0u;
        const uint32_t vb = on ? (uint32_t)((int64_t)(k0 - kbeg) * a.sv2 * 2) : 0u;
        const __amdgpu_buffer_rsrc_t rsK = make_rsrc(Kp, on ? kbytes : 0u), rsV = make_rsrc(Vp, on ? vbytes : 0u);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                kr[slot][t][kk] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsK, (int)offK[t][kk], (int)kb, 0));
#pragma unroll
        for (int j = 0; j < DV; ++j) dma16_buf(rsV, offV[j], vb, sv + wave * VT + j * 1024);
        __builtin_amdgcn_sched_barrier(0);
    };

    constexpr int KS = NWV * KB;
    int k0 = kbeg + wave * KB;
    issue(k0, 0, sV0);

    // query row r0 + lr (B operand; rows past the list are 0), loaded before the tree
    // is looked at
    const int rr = r0 + lr;
    bool row_ok = rr < rows_kv;
    const int h = row_ok ? rr / a.l : 0, pos = row_ok ? rr - h * a.l : 0;
    const T *q = reinterpret_cast<const T *>(a.Q) + b * a.sq0 + (hk * G + h) * a.sq1 + pos * a.sq2;
    u32x4 qr[KK];
    frag qf[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        const int d = kk * 32 + G4 * 8;
        qr[kk] = row_ok && d < a.e ? *reinterpret_cast<const u32x4 *>(q + d) : u32x4{0, 0, 0, 0};
    }
    uint64_t mine = 0;
    if (a.mode == kTree) {
        if (a.l <= 64) {
            const uint64_t nodes = tree_bits_wave(a.parent + (int64_t)b * a.l, a.l);
            mine = (uint64_t)__shfl((uint32_t)(nodes >> 32), pos, 64) << 32 | __shfl((uint32_t)nodes, pos, 64);
            row_ok = row_ok && mine != 0;
        } else {
            tree_bits<NWV * 64>(tb, a.parent + (int64_t)b * a.l, a.l);
            row_ok = row_ok && (tb.w[pos][pos >> 6] >> (pos & 63)) & 1;
        }
    }
    // (whatever an absent node's query holds stays out)
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[kk] = as_frag<frag>(row_ok ? qr[kk] : u32x4{0, 0, 0, 0});

    f32x4 o[DT];
    float m_used = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // scores of a step: (t, i) is key k0 + 16 t + 4 G4 + i; unseen keys -inf
    auto scores = [&](int k0, int slot, f32x4 *sc) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) sc[t] = Mfma<T>::m16(as_frag<frag>(kr[slot][t][kk]), qf[kk], sc[t]);
        }
        if (k0 + KB > free_end) {
            const uint32_t seen = (uint32_t)seen_word(a, &tb, mine, pos, k0, L) >> (4 * G4);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!(seen >> (16 * t + i) & 1)) sc[t][i] = -INFINITY;
        }
    };
    float *keep = a.scores ? a.scores + ((int64_t)(b * a.hkv + hk) * rows_kv + rr) * a.spad : nullptr;
    auto step = [&](int k0, int slot, char *sv) __attribute__((always_inline)) {
        f32x4 sc[2];
        scores(k0, slot, sc);
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
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][i] *= alpha;
            m_used = m_new;
        }
        const float mref = m_used == -INFINITY ? 0.f : m_used + Shift<T>::value;
        t8 part[NP];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = fast_exp2(__builtin_fmaf(sc[t][i], a.scale_log2, -mref));
                l_run += p;
                T x[NP];
                Parts<T>::split(p, x);
#pragma unroll
                for (int y = 0; y < NP; ++y) part[y][4 * t + i] = x[y];
            }
        // this step's V tile has landed: only the next step's loads are younger
        constexpr int Y = 2 * KK + DV;
        __builtin_amdgcn_s_waitcnt((Y & 15) | ((Y >> 4) << 14) | (7 << 4) | (15 << 8));
        __builtin_amdgcn_sched_barrier(0);
        // (stored behind that wait, which counts stores too)
        if (keep && row_ok) {
#pragma unroll
            for (int t = 0; t < 2; ++t) *reinterpret_cast<f32x4 *>(keep + k0 + 16 * t + 4 * G4) = sc[t];
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const char *vb = sv + wave * VT + offVr[dt];
            const s16x4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)to_lds(vb));
            const s16x4 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)to_lds(vb + 16 * RB));
            const u32x2 h0 = __builtin_bit_cast(u32x2, t0), h1 = __builtin_bit_cast(u32x2, t1);
            const frag vf = as_frag<frag>(u32x4{h0[0], h0[1], h1[0], h1[1]});
#pragma unroll
            for (int y = 0; y < NP; ++y) o[dt] = Mfma<T>::m16(vf, __builtin_bit_cast(frag, part[y]), o[dt]);
        }
    };

    for (; k0 < kend; k0 += 2 * KS) {
        issue(k0 + KS, 1, sV1);
        step(k0, 0, sV0);
        // (this wave's reads of the tile are done before its refill)
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_sched_barrier(0);
        issue(k0 + 2 * KS, 0, sV0);
        if (k0 + KS < kend) step(k0 + KS, 1, sV1);
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_sched_barrier(0);
    }
    // no DMA is in flight past here
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_sched_barrier(0);
    float z = 0.f;                  // stays 0 if every sum is finite
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) z = __builtin_fmaf(o[t][i], 0.f, z);
    if (__any(z != 0.f)) {
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float mref = m_used == -INFINITY ? 0.f : m_used + Shift<T>::value;
        for (k0 = kbeg + wave * KB; k0 < kend; k0 += KS) {
            issue(k0, 0, sV0);
            __builtin_amdgcn_s_waitcnt(0);
            __builtin_amdgcn_sched_barrier(0);
            f32x4 sc[2];
            scores(k0, 0, sc);
            const uint32_t seen = (uint32_t)seen_word(a, &tb, mine, pos, k0, L);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const float p = fast_exp2(__builtin_fmaf(sc[x >> 2][x & 3], a.scale_log2, -mref));
                for (int g = 0; g < 4; ++g) {
                    const int key = 16 * (x >> 2) + 4 * g + (x & 3);
                    const float pk = __shfl(p, g * 16 + lr, 64);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const int d = dt * 16 + 4 * G4;
                        const T *vp = reinterpret_cast<const T *>(sV0 + wave * VT + key * RB + (((d >> 3) ^ vsw(key)) << 4) + (d & 4) * 2);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (seen >> key & 1) o[dt][i] += pk * to_f32(vp[i]);
                    }
                }
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // the waves' sums merge through LDS, in the first tiles' place
    constexpr int D4 = HD / 4;
    float (*so)[R][HD] = reinterpret_cast<float (*)[R][HD]>(sV0);
    static_assert(R * HD * 4 == VT, "a wave's rows take its V tile");
    // lanes of a row hold disjoint keys: row sums over the lane groups
    l_run = xor_add<32>(xor_add<16>(l_run));
    if (G4 == 0) {
        sm[wave][lr] = row_ok ? m_used + Shift<T>::value : -INFINITY;
        sl[wave][lr] = row_ok ? l_run : 0.f;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<f32x4 *>(&so[wave][lr][dt * 16 + 4 * G4]) = row_ok ? o[dt] : f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    for (int x = tid; x < R * D4; x += NWV * 64) {
        const int r = x / D4, d = x % D4 * 4;
        if (r0 + r >= rows_kv) continue;
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
        const int head = hk * G + (r0 + r) / a.l, i = (r0 + r) % a.l;
        const int64_t st = (int64_t)split * a.n * a.hq * a.l + ((int64_t)b * a.hq + head) * a.l + i;
        if (a.splits == 1) store_row<T>(a, b, head, i, d, oo, mm, ll);
        else *reinterpret_cast<f32x4 *>(&a.ws_o[st * HD + d]) = oo;
        if (d == 0 && a.ws_ml) *reinterpret_cast<f32x2 *>(&a.ws_ml[st * 2]) = f32x2{mm, ll};
        if (d == 0) {
            s_max[r] = mu;
            s_inv[r] = ll != 0.f ? 1.f / ll : 0.f;
            s_seen[r] = keys_seen(a, i, L);
        }
    }
    if (!a.sum_here) return;
    // (the work-group's own scores, written by its other waves)
    __builtin_amdgcn_s_waitcnt(0);
    __threadfence_block();
    __syncthreads();
    const float *sc = a.scores + (int64_t)(b * a.hkv + hk) * rows_kv * a.spad;
    float *acc = a.acc + b * a.sa0 + hk * a.sa1;
    for (int key = tid; key < L; key += NWV * 64) {
        float w = 0.f;
        for (int r = 0; r < rows_kv; ++r) {
            const float p = s_inv[r] * fast_exp2(__builtin_fmaf(sc[r * a.spad + key], a.scale_log2, -s_max[r]));
            w += key < s_seen[r] ? p : 0.f;
        }
        acc[key] += w;
    }
}

// ------------------------------------------------------------------------
// cache_rows_kernel -- many rows per KV head: 4 waves of 32 rows each over the
// same keys, 64 at a time, K and V through LDS (two stages each, DMA).  32x32x16
// MFMAs in the same transposed form: a lane holds 32 scores of one row, and its
// maximum and sum cross lanes 32 apart only.  Step j runs the exponentials of
// block j between the score MFMAs of block j + 1, then O^T += V^T P^T, with the
// probability's parts (see Parts) one behind the other.  One 16-bit value instead would
// cost the weights 2^-9 (bf16) and the outputs 1.4 times the error of an fp32
// product, and which kernel a call runs on would show in its bits; it took, calls, us, one
// part / two / three in bf16: 256 rows a head over 60000 keys 88 / 112 / 130, 16 sequences
// of 8000 145 / 188 / 224, 104 rows over 4000 38 / 41.5 / 45; f16, one / two: a 1999-token
// prompt with weights 61 / 69.
// With two key groups (KG) 8 waves take blocks 2 j and 2 j + 1 and join their sums
// through LDS in the end, half the columns each, in a fixed order.
// Measured: 256 rows per head over 60000 keys, 8 heads of 128: 126 us, 500 TFLOP/s of the
// two products and 2.0 TB/s.  What bounds it: a step of 64 keys is 2048 cycles of MFMA
// (three parts; f16's two: 1536) and about 1200 of exponentials, maxima and the parts'
// splitting, and every wave reads all 32 KB of the step's K and V from LDS for its 32
// rows.  They overlap only in part, as the step's one barrier keeps all waves in the same
// phase: the MFMA pipes are busy 50% of the time (bf16, two key groups; f16 at head dim 64
// 29%), the waves wait 31%.  Found with one part: with all blocks in L2 it took as long,
// deeper prefetch from LDS changed nothing, 512 registers and one wave a SIMD cost 15 to
// 35% (accumulators copied to and fro).
template <typename T, int HD, int KG>
__global__ __launch_bounds__(256 * KG) __attribute__((amdgpu_waves_per_eu(2, 2))) void cache_rows_kernel(CacheAttnArgs a) {
    constexpr int NWV = 4, KB = 64, R = 32 * NWV;
    constexpr int RB = HD * 2, CPR = HD / 8, TILE = KB * RB;
    constexpr int DPW = TILE / 1024 / NWV, RPB = 1024 / RB;
    constexpr int DT = HD / 32, KS = HD / 16, NP = Parts<T>::N;
    typedef typename Mfma<T>::frag frag;
    typedef T t8 __attribute__((ext_vector_type(8)));
    // K rows are read 16 at a time (ds_read_b128), V rows 8 rows x 64 bytes
    // (transposing): chunk c of row r sits at c ^ swizzle(r), all banks evenly
    auto kswz = [](int r) { return CPR == 16 ? (r & 15) : ((r >> 1) & 7); };
    auto vswz = [](int r) { return CPR == 16 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); };
    __shared__ __attribute__((aligned(1024))) char stages[KG * 4 * TILE];
    __shared__ f32x2 s_ml[KG][R];
    __shared__ TreeBits tb;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) % NWV, kg = __builtin_amdgcn_readfirstlane(tid >> 6) / NWV;
    char *const sK0 = stages + kg * 4 * TILE, *const sV0 = sK0 + TILE, *const sK1 = sV0 + TILE, *const sV1 = sK1 + TILE;
    const int lq = lane & 31, lh = lane >> 5, G4 = lane >> 4, qq = lane & 15;
    const Unit u = unit_of(a);
    if (!u.any) return;
    const int b = u.b, hk = u.hk, split = u.split;
    const int G = a.hq / a.hkv, rows_kv = G * a.l;
    const int L = keys_of(a, b), first = L - a.l;
    const int blocks_all = (L + KB * KG - 1) / (KB * KG);
    const int chunk = (blocks_all + a.splits - 1) / a.splits * KB * KG;

    // a.pair: row groups p and last - p, whose causal lengths together are the same for every p
    const int groups = a.head_tiles ? G * a.head_tiles : (rows_kv + R - 1) / R;
    for (int rg = u.rg;;) {
    // rows r0 .. r0 + R - 1 of the KV head's list, up to the head's end with head_tiles
    const int head = a.head_tiles ? rg / a.head_tiles : 0;
    const int r0 = a.head_tiles ? head * a.l + (rg - head * a.head_tiles) * R : rg * R;
    const int rend = min(r0 + R, a.head_tiles ? (head + 1) * a.l : rows_kv), last = rend - 1;
    const int kbeg = min(L, split * chunk);
    int kend = min(L, kbeg + chunk);
    // keys past the last position of the work-group's rows are seen by none
    if (a.mode == kCausal && r0 / a.l == last / a.l) kend = max(kbeg, min(kend, first + last % a.l + 1));
    // keys below free_end are seen by every row of the wave
    const int w0 = r0 + wave * 32, w1 = min(w0 + 31, last);
    const int free_end = a.mode == kFull ? L : a.mode == kCausal ? first + 1 + (w0 / a.l == w1 / a.l ? w0 % a.l : 0) : first;
    const int nkv = (kend - kbeg + KB * KG - 1) / (KB * KG);

    const T *Kp = reinterpret_cast<const T *>(a.K) + b * a.sk0 + hk * a.sk1 + (int64_t)kbeg * a.sk2;
    const T *Vp = reinterpret_cast<const T *>(a.V) + b * a.sv0 + hk * a.sv1 + (int64_t)kbeg * a.sv2;
    const uint32_t kbytes = kend > kbeg ? (uint32_t)(((int64_t)(kend - kbeg - 1) * a.sk2 + a.e) * 2) : 0u;
    const uint32_t vbytes = kend > kbeg ? (uint32_t)(((int64_t)(kend - kbeg - 1) * a.sv2 + a.ev) * 2) : 0u;
    const __amdgpu_buffer_rsrc_t rsK = make_rsrc(Kp, kbytes), rsV = make_rsrc(Vp, vbytes);
    uint32_t offK[DPW], offV[DPW];
#pragma unroll
    for (int j = 0; j < DPW; ++j) {
        const int r = (wave * DPW + j) * RPB + lane / CPR, p = lane % CPR;
        const int ck = (p ^ kswz(r)) * 8, cv = (p ^ vswz(r)) * 8;
        offK[j] = ck < a.e ? (uint32_t)((r * a.sk2 + ck) * 2) : kOut;
        offV[j] = cv < a.ev ? (uint32_t)((r * a.sv2 + cv) * 2) : kOut;
    }
    // (the second key group's last block may begin past the last key: its offset is the
    // descriptor's size then, so every byte of it is past the end, and not beyond, where
    // what is left of the size would be negative)
    auto issue_k = [&](int kt, char *sk) __attribute__((always_inline)) {
        const uint32_t k0 = (uint32_t)((int64_t)(kt * KG + kg) * KB * a.sk2 * 2), kb = KG == 1 ? k0 : min(k0, kbytes);
#pragma unroll
        for (int j = 0; j < DPW; ++j) dma16_buf(rsK, offK[j], kb, sk + (wave * DPW + j) * 1024);
    };
    auto issue_v = [&](int kt, char *sv) __attribute__((always_inline)) {
        const uint32_t v0 = (uint32_t)((int64_t)(kt * KG + kg) * KB * a.sv2 * 2), vb = KG == 1 ? v0 : min(v0, vbytes);
#pragma unroll
        for (int j = 0; j < DPW; ++j) dma16_buf(rsV, offV[j], vb, sv + (wave * DPW + j) * 1024);
    };
    if (nkv > 0) {
        issue_k(0, sK0);
        issue_v(0, sV0);
        if (nkv > 1) issue_k(1, sK1);
    }

    // this lane's row
    const int rr = w0 + lq;
    bool row_ok = rr < rend;
    const bool live = w0 < rend;
    const int h = row_ok ? rr / a.l : 0, pos = row_ok ? rr - h * a.l : 0;
    const T *q = reinterpret_cast<const T *>(a.Q) + b * a.sq0 + (hk * G + h) * a.sq1 + pos * a.sq2;
    u32x4 qr[KS];
    frag qf[KS];
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
        const int d = kk * 16 + lh * 8;
        qr[kk] = row_ok && d < a.e ? *reinterpret_cast<const u32x4 *>(q + d) : u32x4{0, 0, 0, 0};
    }
    uint64_t mine = 0;
    if (a.mode == kTree) {
        if (a.l <= 64) {
            const uint64_t nodes = tree_bits_wave(a.parent + (int64_t)b * a.l, a.l);
            mine = (uint64_t)__shfl((uint32_t)(nodes >> 32), pos, 64) << 32 | __shfl((uint32_t)nodes, pos, 64);
            row_ok = row_ok && mine != 0;
        } else {
            tree_bits<NWV * KG * 64>(tb, a.parent + (int64_t)b * a.l, a.l);
            row_ok = row_ok && (tb.w[pos][pos >> 6] >> (pos & 63)) & 1;
        }
    }
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) qf[kk] = as_frag<frag>(row_ok ? qr[kk] : u32x4{0, 0, 0, 0});

    // LDS offsets: K row 32 t + lq, chunk 2 kk + lh; V^T row d = 32 dt + lq, whose
    // 8 key slots of lane half lh are keys 4 lh .. + 3 and 8 + 4 lh .. + 3 of a
    // 16-key step (the order the scores' registers hold them)
    const int kpos = kswz(lq);                      // == kswz(32 t + lq)
    int offVr[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        const int krow = 4 * (G4 >> 1) + (qq >> 2), d = dt * 32 + 16 * (G4 & 1) + 4 * (qq & 3);
        offVr[dt] = krow * RB + (((d >> 3) ^ vswz(krow)) << 4) + ((d >> 2) & 1) * 8;   // vswz(krow + 8 x) == vswz(krow)
    }
    auto load_k = [&](const char *pk, int kk, int t) __attribute__((always_inline)) {
        return as_frag<frag>(*reinterpret_cast<const u32x4 *>(pk + (t * 32 + lq) * RB + (((2 * kk + lh) ^ kpos) << 4)));
    };
    // scores of a block: sc[t][x] is key kv0 + 32 t + 8 (x / 4) + 4 lh + x % 4
    auto qk = [&](const char *pk, f32x16 *sc) __attribute__((always_inline)) {
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
            for (int t = 0; t < 2; ++t) sc[t] = Mfma<T>::m32(load_k(pk, kk, t), qf[kk], kk == 0 ? f32x16{} : sc[t]);
    };
    auto hide = [&](f32x16 *sc, int kv0) __attribute__((always_inline)) {
        if (kv0 + KB <= free_end) return;
        const uint64_t seen = seen_word(a, &tb, mine, pos, kv0, L) >> (4 * lh);
        const uint32_t w[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 16; ++x)
                if (!(w[t] >> (8 * (x >> 2) + (x & 3)) & 1)) sc[t][x] = -INFINITY;
    };

    f32x16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x16{};
    float m_used = -INFINITY, l_run = 0.f;
    auto step = [&](f32x16 *cur, f32x16 *nxt, const char *pk, const char *pv, int kv0) __attribute__((always_inline)) {
        hide(cur, kv0);
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 16; ++x) mx = fmaxf(mx, cur[t][x]);
        mx = xor_max<32>(mx) * a.scale_log2;
        if (__any(mx > m_used + kSlack)) {
            const float m_new = fmaxf(m_used, mx);
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_used - m_new);
            l_run *= alpha;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int x = 0; x < 16; ++x) o[t][x] *= alpha;
            m_used = m_new;
        }
        const float mref = m_used == -INFINITY ? 0.f : m_used + Shift<T>::value;
        float rs = 0.f;
        constexpr int EPK = 32 / KS, KPF = 3;       // exponentials per MFMA pair; K fragments read ahead
        frag kr[KPF][2];
#pragma unroll
        for (int kk = 0; kk < KPF - 1; ++kk)
#pragma unroll
            for (int t = 0; t < 2; ++t) kr[kk][t] = load_k(pk, kk, t);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            if (kk + KPF - 1 < KS)
#pragma unroll
                for (int t = 0; t < 2; ++t) kr[(kk + KPF - 1) % KPF][t] = load_k(pk, kk + KPF - 1, t);
#pragma unroll
            for (int t = 0; t < 2; ++t) nxt[t] = Mfma<T>::m32(kr[kk % KPF][t], qf[kk], kk == 0 ? f32x16{} : nxt[t]);
#pragma unroll
            for (int y = 0; y < EPK; ++y) {
                const int idx = kk * EPK + y, t = idx >> 4, x = idx & 15;
                const float p = fast_exp2(__builtin_fmaf(cur[t][x], a.scale_log2, -mref));
                cur[t][x] = p;
                rs += p;
            }
        }
        l_run += rs;
        constexpr int NV = 4 * DT, VPF = 2;
        frag vr[VPF];
        auto load_v = [&](int idx, frag &dst) __attribute__((always_inline)) {
            const char *vb = pv + offVr[idx % DT] + idx / DT * 16 * RB;
            const s16x4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)to_lds(vb));
            const s16x4 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)to_lds(vb + 8 * RB));
            const u32x2 h0 = __builtin_bit_cast(u32x2, t0), h1 = __builtin_bit_cast(u32x2, t1);
            dst = as_frag<frag>(u32x4{h0[0], h0[1], h1[0], h1[1]});
        };
#pragma unroll
        for (int x = 0; x < VPF - 1; ++x) load_v(x, vr[x]);
        frag pf[NP];
#pragma unroll
        for (int idx = 0; idx < NV; ++idx) {
            const int b16 = idx / DT;
            if (idx % DT == 0) {
                t8 p8[NP];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    T part[NP];
                    Parts<T>::split(cur[b16 >> 1][8 * (b16 & 1) + x], part);
#pragma unroll
                    for (int y = 0; y < NP; ++y) p8[y][x] = part[y];
                }
#pragma unroll
                for (int y = 0; y < NP; ++y) pf[y] = __builtin_bit_cast(frag, p8[y]);
            }
            if (idx + VPF - 1 < NV) load_v(idx + VPF - 1, vr[(idx + VPF - 1) % VPF]);
#pragma unroll
            for (int y = 0; y < NP; ++y) o[idx % DT] = Mfma<T>::m32(vr[idx % VPF], pf[y], o[idx % DT]);
        }
    };

    // LDS stages: K_j and V_j in stage j % 2.  Step j needs K_{j+1} and V_j; it
    // refills stage j % 2 with K_{j+2} and the other one with V_{j+1}, both
    // consumed a step earlier.  (The last step's next scores are never used.)
    f32x16 scA[2], scB[2];
    if (nkv > 0) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (live) qk(sK0, scA);
    }
    for (int j0 = 0; j0 < nkv; j0 += 2) {
#pragma unroll
        for (int hs = 0; hs < 2; ++hs) {
            const int j = j0 + hs;
            if (j >= nkv) break;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (j + 2 < nkv) issue_k(j + 2, hs ? sK1 : sK0);
            if (j + 1 < nkv) issue_v(j + 1, hs ? sV0 : sV1);
            if (live) step(hs ? scB : scA, hs ? scA : scB, hs ? sK0 : sK1, hs ? sV1 : sV0, kbeg + (j * KG + kg) * KB);
        }
    }
    float z = 0.f;                  // stays 0 if every sum is finite
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int x = 0; x < 16; ++x) z = __builtin_fmaf(o[t][x], 0.f, z);
    if (__syncthreads_or(live && z != 0.f)) {
        // as in cache_attn_kernel: again, value by value, for the rows that see them
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = f32x16{};
        const float mref = m_used == -INFINITY ? 0.f : m_used + Shift<T>::value;
        for (int j = 0; j < nkv; ++j) {
            const int kv0 = kbeg + (j * KG + kg) * KB;
            __syncthreads();
            issue_k(j, sK0);
            issue_v(j, sV0);
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (!live) continue;
            qk(sK0, scA);
            hide(scA, kv0);
            const uint64_t seen = seen_word(a, &tb, mine, pos, kv0, L);
            // 32 keys' weights at a time through the second stages, [key][row]
            float (*pw)[32] = reinterpret_cast<float (*)[32]>((wave < 2 ? sK1 : sV1) + (wave & 1) * 4096);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    pw[8 * (x >> 2) + 4 * lh + (x & 3)][lq] = fast_exp2(__builtin_fmaf(scA[t][x], a.scale_log2, -mref));
                __builtin_amdgcn_s_waitcnt(0xc07f);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
                for (int key = 32 * t; key < 32 * t + 32; ++key) {
                    if (!(seen >> key & 1)) continue;
                    const float pk = pw[key & 31][lq];
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int y = 0; y < 16; ++y) {
                            const int d = dt * 32 + 8 * (y >> 2) + 4 * lh + (y & 3);
                            o[dt][y] += pk * to_f32(*reinterpret_cast<const T *>(sV0 + key * RB + (((d >> 3) ^ vswz(key)) << 4) + (d & 7) * 2));
                        }
                }
                __builtin_amdgcn_s_waitcnt(0xc07f);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    const float l_all = xor_add<32>(l_run);
    float m = row_ok ? m_used + Shift<T>::value : -INFINITY, l = row_ok ? l_all : 0.f;
    const int64_t st = (int64_t)split * a.n * a.hq * a.l + ((int64_t)b * a.hq + hk * G + h) * a.l + pos;
    if constexpr (KG == 2) {
        // each key group has half the columns of both groups' sums in the end
        f32x4 *part = reinterpret_cast<f32x4 *>(stages);        // [wave][DT * 4][lane]
        __syncthreads();
        if (lh == 0) s_ml[kg][wave * 32 + lq] = f32x2{m, l};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (half == kg) continue;
#pragma unroll
            for (int dt = half * DT / 2; dt < (half + 1) * DT / 2; ++dt)
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    part[(wave * DT * 4 + dt * 4 + y) * 64 + lane] = f32x4{o[dt][4 * y], o[dt][4 * y + 1], o[dt][4 * y + 2], o[dt][4 * y + 3]};
        }
        __syncthreads();
        const f32x2 other = s_ml[1 - kg][wave * 32 + lq];
        const float top = fmaxf(m, other[0]), mu = top == -INFINITY ? 0.f : top;
        const float w0 = fast_exp2(m - mu), w1 = fast_exp2(other[0] - mu);
        m = top;
        l = kg == 0 ? __builtin_fmaf(other[1], w1, l * w0) : __builtin_fmaf(l, w0, other[1] * w1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (half != kg) continue;
#pragma unroll
            for (int dt = half * DT / 2; dt < (half + 1) * DT / 2; ++dt)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const f32x4 ov = part[(wave * DT * 4 + dt * 4 + y) * 64 + lane];
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[dt][4 * y + x] = __builtin_fmaf(ov[x], w1, o[dt][4 * y + x] * w0);
                }
        }
    }
    if (rr < rend) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            if (KG == 2 && dt / (DT / 2) != kg) continue;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int d = dt * 32 + 8 * y + 4 * lh;
                const f32x4 v = row_ok ? f32x4{o[dt][4 * y], o[dt][4 * y + 1], o[dt][4 * y + 2], o[dt][4 * y + 3]} : f32x4{0.f, 0.f, 0.f, 0.f};
                if (a.splits == 1) store_row<T>(a, b, hk * G + h, pos, d, v, m, l);
                else *reinterpret_cast<f32x4 *>(&a.ws_o[st * HD + d]) = v;
            }
        }
        if (a.splits > 1 && lh == 0 && kg == 0) *reinterpret_cast<f32x2 *>(&a.ws_ml[st * 2]) = f32x2{m, l};
    }
    if (!a.pair || rg != u.rg || groups - 1 - rg == rg) break;
    rg = groups - 1 - rg;
    __syncthreads();                // (the other group's first keys take the place of the last ones)
    }
}

// 4 columns of a row's splits, merged in split order (the same bits whatever order
// the work-groups ended in); the splits' loads go out together, 8 at a time: 5.6 us
// for 2048 rows of 128 in 16 splits, 4.1 us for fewer (latency).
template <int HD>
__device__ __forceinline__ void merge_splits(const CacheAttnArgs &a, int64_t rows, int64_t row, int d, f32x4 &oo, float &mm, float &ll) {
    oo = f32x4{0.f, 0.f, 0.f, 0.f};
    mm = -INFINITY;
    ll = 0.f;
    for (int z0 = 0; z0 < a.splits; z0 += 8) {
        f32x4 ov[8];
        f32x2 ml[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const int64_t st = (z0 + y) * rows + row;
            ml[y] = f32x2{-INFINITY, 0.f};
            if (z0 + y < a.splits) {
                ml[y] = *reinterpret_cast<const f32x2 *>(&a.ws_ml[st * 2]);
                ov[y] = *reinterpret_cast<const f32x4 *>(&a.ws_o[st * HD + d]);
            }
        }
        float top = mm;
#pragma unroll
        for (int y = 0; y < 8; ++y) top = fmaxf(top, ml[y][0]);
        const float mu = top == -INFINITY ? 0.f : top, old = fast_exp2(mm - mu);
        ll *= old;
#pragma unroll
        for (int i = 0; i < 4; ++i) oo[i] *= old;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            if (z0 + y < a.splits) {
                const float wgt = fast_exp2(ml[y][0] - mu);
                ll = __builtin_fmaf(ml[y][1], wgt, ll);
#pragma unroll
                for (int i = 0; i < 4; ++i) oo[i] = __builtin_fmaf(ov[y][i], wgt, oo[i]);
            }
        }
        mm = top;
    }
}
template <typename T, int HD>
__global__ __launch_bounds__(256) void cache_merge_kernel(CacheAttnArgs a) {
    constexpr int D4 = HD / 4;
    const int64_t rows = (int64_t)a.n * a.hq * a.l;
    const int64_t row = (int64_t)blockIdx.x * (256 / D4) + threadIdx.x / D4;
    if (row >= rows) return;
    const int d = threadIdx.x % D4 * 4;
    f32x4 oo;
    float mm, ll;
    merge_splits<HD>(a, rows, row, d, oo, mm, ll);
    const int i = (int)(row % a.l);
    store_row<T>(a, row / a.l / a.hq, (int)(row / a.l % a.hq), i, d, oo, mm, ll);
}

// accum_merge_kernel -- the weights of a few rows' keys from the scores that
// cache_attn_kernel kept, and the merge of its splits: a work-group has 512 keys
// of a KV head and its share of the rows' outputs.  (Writing and reading the
// scores costs 8 bytes a row and key, reading K again 2 e a key.)  7.9 us for 16 sequences
// of 8 heads, 4 rows, 4000 keys: of which 8 MB of scores take about 2.
constexpr int kScoreRows = 32;
template <typename T, int HD>
__global__ __launch_bounds__(256) void accum_merge_kernel(CacheAttnArgs a) {
    constexpr int D4 = HD / 4, RPB = 256 / D4;
    __shared__ float s_m[kScoreRows], s_l[kScoreRows];
    __shared__ int s_seen[kScoreRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.y / a.hkv, hk = blockIdx.y % a.hkv;
    const int G = a.hq / a.hkv, rows = G * a.l;
    const int64_t all = (int64_t)a.n * a.hq * a.l;
    auto row_of = [&](int r) { return ((int64_t)b * a.hq + hk * G + r / a.l) * a.l + r % a.l; };
    const int L = keys_of(a, b);
    if (blockIdx.x > 0 && (int)blockIdx.x * 512 >= L && (int)blockIdx.x >= (rows + RPB - 1) / RPB) return;
    // the first rows' scores and the sums, before the rows' maxima are known (the
    // scores' rows are padded, with whatever they hold, past the last key)
    const int key = blockIdx.x * 512 + tid * 2;
    const float *sc = a.scores + (int64_t)(b * a.hkv + hk) * rows * a.spad + key;
    float *acc = a.acc + b * a.sa0 + hk * a.sa1 + key;
    f32x2 x[4] = {}, old = {0.f, 0.f};
    if (key < a.s) {
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = *reinterpret_cast<const f32x2 *>(sc + min(y, rows - 1) * a.spad);
        old[0] = acc[0];
        if (key + 1 < a.s) old[1] = acc[1];
    }
    for (int r = wave; r < rows; r += 4) {
        const f32x2 ml = lane < a.splits ? *reinterpret_cast<const f32x2 *>(&a.ws_ml[(lane * all + row_of(r)) * 2]) : f32x2{-INFINITY, 0.f};
        const float mm = wave_max(ml[0]), mu = mm == -INFINITY ? 0.f : mm;
        const float ll = wave_sum(ml[1] * fast_exp2(ml[0] - mu));
        if (lane == 0) {
            s_m[r] = mu;
            s_l[r] = ll != 0.f ? 1.f / ll : 0.f;
            s_seen[r] = keys_seen(a, r % a.l, L);
        }
    }
    // the rows' outputs
    if (a.splits > 1) {
        const int d = tid % D4 * 4;
        for (int r = blockIdx.x * RPB + tid / D4; r < rows; r += gridDim.x * RPB) {
            f32x4 oo;
            float mm, ll;
            merge_splits<HD>(a, all, row_of(r), d, oo, mm, ll);
            store_row<T>(a, b, hk * G + r / a.l, r % a.l, d, oo, mm, ll);
        }
    }
    __syncthreads();
    if (key >= L) return;
    f32x2 w = {0.f, 0.f};
    for (int r = 0; r < rows; r += 4) {
        if (r > 0) {
#pragma unroll
            for (int y = 0; y < 4; ++y) x[y] = *reinterpret_cast<const f32x2 *>(sc + min(r + y, rows - 1) * a.spad);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            if (r + y >= rows) break;
            const float m = s_m[r + y], inv = s_l[r + y];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const float p = inv * fast_exp2(__builtin_fmaf(x[y][z], a.scale_log2, -m));
                w[z] += key + z < s_seen[r + y] ? p : 0.f;
            }
        }
    }
    acc[0] = old[0] + w[0];
    if (key + 1 < L) acc[1] = old[1] + w[1];
}

// key_weights_kernel -- the weights of many rows' keys: acc[key] += sum over the
// rows that see it of exp(scale q k - lse).  A tile is 32 * KT keys, in the
// registers of each of the NWV waves (A operand, 32x32x16 MFMA); the waves take
// the rows in turn, 32 at a time, and a lane adds up its keys of its row position:
// the rows' sum crosses lanes and waves once, at the end, in a fixed order.  Rows
// come through the wave's own LDS stages by DMA, whole rows at a time: loaded from
// memory into the operand's lanes, 16 bytes of 32 rows each, their addresses alone
// took three times the arithmetic's time.  A work-group takes tiles p and last - p:
// causal keys are seen by the fewer rows the later they are, and two such tiles
// always by about as many.  What bounds it: waiting and the exponentials (a turn of 32
// rows and 64 keys, head dim 64: about 770 cycles of vector instructions, 256 of MFMA), and
// for 32-key tiles the rows' traffic from L2, 8 to 10 TB/s.  Waves wait 42% of their cycles:
// the turns' lse values are loads kept in registers across turns, and for the last of a
// group of NS turns the compiler waits for all loads, the next stages' DMA with them; the
// counted wait holds for the others.  33 us for a 1999-token prompt of 32 / 8 heads of 64,
// f16.  With `parts` > 1 that many
// work-groups share a tile's rows, and sum_parts_kernel adds up their sums.
template <typename T, int HD, int KT>
__global__ __launch_bounds__(HD <= 128 ? 512 : 256) void key_weights_kernel(CacheAttnArgs a, int tiles, int parts) {
    constexpr int KS = HD / 16, NWV = HD <= 128 ? 8 : 4, KEYS = 32 * KT, NS = HD <= 64 ? 3 : 2;
    constexpr int RB = HD * 2, CPR = HD / 8, RPB = 1024 / RB, STAGE = 32 * RB, DPT = STAGE / 1024;
    const int part = blockIdx.x % parts, STEP = NWV * parts * 32;
    typedef typename Mfma<T>::frag frag;
    auto swz = [](int r) { return CPR >= 16 ? (r & 15) : ((r >> 1) & 7); };     // as cache_rows_kernel's K
    __shared__ __attribute__((aligned(1024))) char sQ[NS][NWV][STAGE];
    __shared__ float s_sum[NWV][KEYS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lq = lane & 31, lh = lane >> 5;
    const int b = blockIdx.y / a.hkv, hk = blockIdx.y % a.hkv, G = a.hq / a.hkv;
    const int L = keys_of(a, b), first = L - a.l;
    const int p = blockIdx.x / parts, mine = part * NWV + wave;       // the wave among the tile's
    const T *Qp = reinterpret_cast<const T *>(a.Q) + b * a.sq0 + hk * G * a.sq1;
    const float *Lp = a.lse + ((int64_t)b * a.hq + hk * G) * a.l;
    // this lane's row of a stage and its 16 bytes of it, per DMA instruction (columns
    // past the head dim read others: they meet zeros of K)
    int row_j[DPT], col_j[DPT];
    int64_t off_j[DPT];
#pragma unroll
    for (int j = 0; j < DPT; ++j) {
        row_j[j] = j * RPB + lane / CPR;
        const int c = ((lane % CPR) ^ swz(row_j[j])) * 8;
        col_j[j] = c < a.e ? c : 0;
        off_j[j] = row_j[j] * a.sq2 + col_j[j];
    }
    for (int tile = p;; tile = tiles - 1 - p) {
        const int k0 = tile * KEYS;
        if (k0 < L) {
            // rows before position i0 see none of these keys
            const int i0 = a.mode == kCausal ? max(0, k0 - first) : 0, per = a.l - i0, rows = G * per;
            frag kf[KT][KS];
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int key = k0 + 32 * t + lq;
                const T *kp = reinterpret_cast<const T *>(a.K) + b * a.sk0 + hk * a.sk1 + (int64_t)key * a.sk2;
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
                    const int d = kk * 16 + lh * 8;
                    kf[t][kk] = as_frag<frag>(key < L && d < a.e ? *reinterpret_cast<const u32x4 *>(kp + d) : u32x4{0, 0, 0, 0});
                }
            }
            float ln[NS];
            int pn[NS];
            // the wave's next 32 rows into stage z.  Past the list a lane takes its last
            // row (with a weight of 0, and for the keys only that this row sees: a NaN in
            // it reaches no others), so every turn has the same loads.
            int r0 = mine * 32, h0 = r0 / per, p0 = i0 + r0 - h0 * per;
            auto load = [&](int z) __attribute__((always_inline)) {
                const float *lp;
                if (p0 + 31 < a.l && r0 + 31 < rows) {
                    const T *q = Qp + h0 * a.sq1 + p0 * a.sq2;
#pragma unroll
                    for (int j = 0; j < DPT; ++j)
                        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(q + off_j[j]),
                                                         (__attribute__((address_space(3))) void *)to_lds(sQ[z][wave] + j * 1024), 16, 0, 0);
                    lp = Lp + (int64_t)h0 * a.l + p0 + lq;
                    pn[z] = p0 + lq;
                } else {
#pragma unroll
                    for (int j = 0; j < DPT; ++j) {
                        const int r = min(r0 + row_j[j], rows - 1), h = r / per;
                        const T *q = Qp + h * a.sq1 + (i0 + r - h * per) * a.sq2 + col_j[j];
                        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)q,
                                                         (__attribute__((address_space(3))) void *)to_lds(sQ[z][wave] + j * 1024), 16, 0, 0);
                    }
                    const int r = min(r0 + lq, rows - 1), h = r / per;
                    pn[z] = i0 + r - h * per;
                    lp = Lp + (int64_t)h * a.l + pn[z];
                }
                const float x = *lp;
                ln[z] = r0 + lq < rows ? x : -INFINITY;
                __builtin_amdgcn_sched_barrier(0);
                r0 += STEP;
                p0 += STEP;
                while (r0 < rows && p0 >= a.l) {
                    p0 -= per;
                    ++h0;
                }
            };
            f32x16 sum[KT];
#pragma unroll
            for (int t = 0; t < KT; ++t) sum[t] = f32x16{};
#pragma unroll
            for (int z = 0; z < NS - 1; ++z) load(z);
            for (int rb = mine * 32; rb < rows; rb += NS * STEP) {
#pragma unroll
                for (int z = 0; z < NS; ++z) {
                    if (rb + z * STEP >= rows) break;
                    load((z + NS - 1) % NS);
                    // this turn's rows have landed: only the later turns' loads are younger
                    constexpr int Y = (NS - 1) * (DPT + 1);
                    __builtin_amdgcn_s_waitcnt((Y & 15) | ((Y >> 4) << 14) | (7 << 4) | (15 << 8));
                    __builtin_amdgcn_sched_barrier(0);
                    // (a row that saw nothing, or none: weight 0)
                    float c = ln[z] == -INFINITY ? -INFINITY : -ln[z] * kLog2e;
                    const int last = a.mode == kCausal ? first + pn[z] - k0 : KEYS;       // the row's last key here
                    f32x16 sc[KT];
#pragma unroll
                    for (int kk = 0; kk < KS; ++kk) {
                        const frag qf = as_frag<frag>(*reinterpret_cast<const u32x4 *>(sQ[z][wave] + lq * RB + (((2 * kk + lh) ^ swz(lq)) << 4)));
#pragma unroll
                        for (int t = 0; t < KT; ++t) sc[t] = Mfma<T>::m32(kf[t][kk], qf, kk == 0 ? f32x16{} : sc[t]);
                    }
                    if (__any(last < KEYS - 1)) {
                        // (NaN of the row's lse goes to the scores that it sees)
                        const float bad = c != c ? c : 0.f;
                        c = c != c ? 0.f : c;
#pragma unroll
                        for (int t = 0; t < KT; ++t)
#pragma unroll
                            for (int x = 0; x < 16; ++x)
                                sc[t][x] = 32 * t + 8 * (x >> 2) + 4 * lh + (x & 3) > last ? -INFINITY : sc[t][x] + bad;
                    }
#pragma unroll
                    for (int t = 0; t < KT; ++t)
#pragma unroll
                        for (int x = 0; x < 16; ++x) sum[t][x] += fast_exp2(__builtin_fmaf(sc[t][x], a.scale_log2, c));
                    // (the stage's reads are done before its refill)
                    __builtin_amdgcn_s_waitcnt(0xc07f);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // no DMA is in flight past here
            __builtin_amdgcn_s_waitcnt(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float v = xor_add<16>(group_sum<16>(sum[t][x]));
                    if (lq == 0) s_sum[wave][32 * t + 8 * (x >> 2) + 4 * lh + (x & 3)] = v;
                }
            __syncthreads();
            if (tid < KEYS && k0 + tid < L) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < NWV; ++w) v += s_sum[w][tid];
                if (parts == 1) a.acc[b * a.sa0 + hk * a.sa1 + k0 + tid] += v;
                else a.part_sums[((int64_t)part * a.n * a.hkv + blockIdx.y) * a.spad + k0 + tid] = v;
            }
            __syncthreads();
        }
        if (tile != p || tiles - 1 - p <= p) break;
    }
}

__global__ __launch_bounds__(256) void sum_parts_kernel(CacheAttnArgs a, int parts) {
    const int b = blockIdx.y / a.hkv, hk = blockIdx.y % a.hkv, key = blockIdx.x * 256 + threadIdx.x;
    if (key >= keys_of(a, b)) return;
    float v = 0.f;
    for (int x = 0; x < parts; ++x) v += a.part_sums[((int64_t)x * a.n * a.hkv + blockIdx.y) * a.spad + key];
    a.acc[b * a.sa0 + hk * a.sa1 + key] += v;
}

// ------------------------------------------------------------- host side

struct Plan {
    int hd, rows;          // head dim and rows of a work-group: 16 (cache_attn_kernel) or 128 (cache_rows_kernel)
    int row_groups, splits, pair, head_tiles, sum_here;
    int64_t units;
    int key_groups;        // cache_rows_kernel: groups of 4 waves
    int kt, parts;         // key_weights_kernel: 32-key blocks of a tile, work-groups of a tile
    int64_t weight_groups; // its work-groups of a KV head, 0 without it
    size_t o_bytes, ml_bytes, score_bytes, part_bytes;        // of the workspace
};

// Which kernel.  16-row groups are several work-groups for more rows, each of
// which reads the keys (from L2 behind the first), which fills the GPU soonest;
// 128-row ones read them once and do far less per row.  The 16-row form wins up
// to about 2^25 = (KV heads x 16-row groups x keys x head dim).  Measured around it, us
// with the merge, best split counts, 16 against 128 rows, bf16: head dim 128, 8 KV heads, 256
// rows, 1024 / 2048 / 4096 keys 15.3 / 19.6, 19.7 / 23.3 and 29.7 / 27.4; 32 heads, 64 rows, the
// same keys 15.6 / 18.4, 20.7 / 22.0 and 30.0 / 28.1; 64 heads, 64 rows, 1024 and 4000 keys 17.2 /
// 22.2 and 43.5 / 41.0; 16 heads, 104 rows, 3000 keys 24.7 / 23.7; head dim 64, 32 heads, 256 rows,
// 512 / 1024 / 2048 10.4 / 15.1, 15.1 / 19.2 and 24.3 / 21.8; 8 heads, 32 rows, 256 keys of 128 9.4 /
// 12.3.  f16's two parts: 128 rows 0 to 4 us less.  Rows that fill a quarter of a 128-row group
// cross later: 64 heads, 32 rows, 4000 and 8000 keys of 128 31.2 / 33.3 and 62.5 / 62.2.
//
// How many splits.  About one work-group per CU (of 16-row ones twice that while each
// still has 2048 keys), of at
// least 256 keys: 64 KV heads, 16 rows, 4000 keys of 128: 256 / 512 / 1024 work-groups
// 25.8 / 25.7 / 31.4; 32 rows, 16-row groups, 256 / 512 / 1024 28.9 / 29.5 / 36.2.  Short
// caches are not split, which saves the merge's launch: 8 heads, 32 rows, 640 keys
// of 64 one split 7.7, four 8.6; 1024 keys 9.2 / 8.6; 256 of 128 8.5 / 10.3; 640 12.0 /
// 11.0.
//
// How many key groups.  A 128-row work-group that has a CU for itself takes the keys
// with two groups of 4 waves, unless its keys are few, as the second group's first
// loads and the joining of the sums take their time.  One / two groups, us with the merge,
// at 700, 1000, 1300, 1600, 2000, 2600 and 4000 keys a work-group: bf16, 16 row groups in 16
// splits, 256 rows a head, of 128: 40.3 / 41.5, 47.8 / 47.7, 55.9 / 56.7, 64.0 / 63.3, 78.8 / 76.0, 100 / 94,
// 143 / 136; 104 rows a head: 36.1 / 39.6, 45.6 / 47.2, 56.4 / 58.8, 67.0 / 67.4, 84.0 / 77.8, 105 / 98, 154 /
// 149; 64 row groups in 4 splits, 35.2 / 37.4 to 57.2 / 58.5, 69.7 / 70.2, 90.5 / 87.5, 134 / 129;
// head dim 64, 16 row groups: 27.0 / 26.7, 31.1 / 29.9, 36.1 / 35.1, 41.1 / 38.8 to 83.2 / 75.0; f16
// alike (two groups gain up to 17% at 4000 keys of 64).  So they are equal near 1600 at head
// dim 128 and near 700 at 64, where one group costs 9% at most up to the limit.  With more
// work-groups two of them share a CU: 512 of 4000 keys, one part, 137 / 150.
constexpr int kCUs = 256;
Plan plan_of(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t s, int64_t e, int64_t ev, int mode, bool accum) {
    Plan p{};
    const int64_t w = std::max(e, ev), rows = hq / hkv * l;
    p.hd = w <= 64 ? 64 : w <= 128 ? 128 : 256;
    p.rows = p.hd == 256 || rows <= 16 || n * hkv * cdiv(rows, 16) * s <= ((int64_t)1 << 25) / p.hd ? 16 : 128;
    p.row_groups = (int)cdiv(rows, p.rows);
    // long causal pieces: no row group crosses heads (one that does sees the last
    // row of one head next to the first of another, so every block of it is masked:
    // a 1999-token prompt, 32 / 8 heads of 64: 47 -> 40 us); 7 groups a head waste an
    // eighth of the rows at most
    if (p.rows == 128 && mode == kCausal && l > 7 * 128) {
        p.head_tiles = (int)cdiv(l, 128);
        p.row_groups = (int)(hq / hkv) * p.head_tiles;
    }
    const int64_t groups = n * hkv * p.row_groups, want = p.rows == 16 && cdiv(s * groups, 2 * kCUs) >= 2048 ? 2 * kCUs : kCUs;
    p.splits = s * p.hd <= 640 * 64 ? 1 : (int)std::max<int64_t>(1, std::min(want / std::max<int64_t>(groups, 1), cdiv(s, 256)));
    p.splits = std::min(p.splits, 64);          // (accum_merge_kernel has a lane for each)
    p.units = n * hkv * p.splits;
    p.pair = p.rows == 128 && mode == kCausal && p.splits == 1 && p.row_groups > 1;
    if (p.pair) p.row_groups = (p.row_groups + 1) / 2;
    p.key_groups = p.rows == 128 && p.units * p.row_groups <= kCUs && cdiv(s, p.splits) >= 1536 ? 2 : 1;
    const bool keep = accum && p.rows == 16 && rows <= kScoreRows;
    p.o_bytes = p.splits > 1 ? (size_t)p.splits * n * hq * l * p.hd * 4 : 0;
    p.score_bytes = keep ? (size_t)n * hkv * rows * (cdiv(s, 32) * 32) * 4 : 0;
    // one work-group a KV head: one launch (one token over 600 keys, 8 heads of 64, host
    // and all: 16.3 -> 12.5 us)
    p.sum_here = keep && p.splits == 1 && p.row_groups == 1;
    p.ml_bytes = p.splits > 1 || (keep && !p.sum_here) ? (size_t)p.splits * n * hq * l * 8 : 0;
    // Tiles of 64 keys halve the rows' traffic where there are enough of them, or
    // enough rows to share among the work-groups of a tile; parts: a work-group for
    // every CU, of two turns of its waves at least.  Whole calls, us, 32 keys one part / 32
    // keys parts / 64 keys one part / 64 keys parts, 32 / 8 heads of 64 if not said: a
    // 1999-token prompt 69.0 / 77.3 / 74.4 / 64.7 (f16, run after run: 63.6 / - / - / 66.5), two
    // of them 113.6 / 124 / 94.2 / 106.5, 1000 tokens 42.7 / 41.9 / 49.9 / 43.9, 512 29.8 / 28.9 /
    // 35.6 / 32.3, 128 behind 1920 23.9 / 31.8 / 28.6 / 27.8, 1000 tokens of 14 / 2 heads 47.9 /
    // 38.4 / 58.6 / 42.7; heads of 128, 1999 tokens 104 / 106 / 101 / 92.
    p.kt = p.parts = 1;
    if (accum && !keep && s > 0) {
        const int64_t groups32 = n * hkv * cdiv(cdiv(s, 32), 2);
        if (p.hd <= 128 && (groups32 >= 2 * kCUs || (p.hd == 128 && groups32 >= kCUs && rows >= 4096))) p.kt = 2;
        const int64_t pairs = n * hkv * cdiv(cdiv(s, 32 * p.kt), 2), turns = cdiv(rows, 256);
        p.parts = (int)std::max<int64_t>(1, std::min({(int64_t)8, kCUs / pairs, turns / 2}));
        if (p.parts > 1) p.part_bytes = (size_t)p.parts * n * hkv * (cdiv(s, 32) * 32) * 4;
        p.weight_groups = cdiv(cdiv(s, 32 * p.kt), 2) * p.parts;
    }
    return p;
}

size_t state_bytes(const Plan &p) { return p.o_bytes + p.score_bytes + p.ml_bytes + p.part_bytes; }

template <typename T, int HD>
void launch_weights(const CacheAttnArgs &a, const Plan &p, hipStream_t st) {
    const unsigned heads = (unsigned)(a.n * a.hkv), tiles = (unsigned)cdiv(a.s, 32 * p.kt);
    const dim3 grid((unsigned)p.weight_groups, heads), threads(HD <= 128 ? 512 : 256);
    if constexpr (HD <= 128) {
        if (p.kt == 2) hipLaunchKernelGGL((key_weights_kernel<T, HD, 2>), grid, threads, 0, st, a, (int)tiles, p.parts);
    }
    if (p.kt == 1) hipLaunchKernelGGL((key_weights_kernel<T, HD, 1>), grid, threads, 0, st, a, (int)tiles, p.parts);
    if (p.parts > 1) hipLaunchKernelGGL(sum_parts_kernel, dim3((unsigned)cdiv(a.s, 256), heads), dim3(256), 0, st, a, p.parts);
}

template <typename T, int HD>
int launch_attn(const CacheAttnArgs &a, const Plan &p, hipStream_t st) {
    const dim3 grid((unsigned)(cdiv(p.units, 8) * 8 * p.row_groups));
    if (p.rows == 16) hipLaunchKernelGGL((cache_attn_kernel<T, HD>), grid, dim3(256), 0, st, a);
    else if constexpr (HD <= 128) {
        if (p.key_groups == 2) hipLaunchKernelGGL((cache_rows_kernel<T, HD, 2>), grid, dim3(512), 0, st, a);
        else hipLaunchKernelGGL((cache_rows_kernel<T, HD, 1>), grid, dim3(256), 0, st, a);
    }
    if (a.sum_here) return launch_status();
    if (a.scores) {
        hipLaunchKernelGGL((accum_merge_kernel<T, HD>), dim3((unsigned)cdiv(a.s, 512), (unsigned)(a.n * a.hkv)), dim3(256), 0, st, a);
        return launch_status();
    }
    if (p.splits > 1) {
        const int64_t rows = (int64_t)a.n * a.hq * a.l;
        hipLaunchKernelGGL((cache_merge_kernel<T, HD>), dim3((unsigned)cdiv(rows, 256 / (HD / 4))), dim3(256), 0, st, a);
    }
    if (a.acc)
        launch_weights<T, HD>(a, p, st);
    return launch_status();
}

template <typename T>
int launch_attn_hd(const CacheAttnArgs &a, const Plan &p, hipStream_t st) {
    return p.hd == 64 ? launch_attn<T, 64>(a, p, st) : p.hd == 128 ? launch_attn<T, 128>(a, p, st) : launch_attn<T, 256>(a, p, st);
}

// What both entry points ask of their arguments; KUIOPS_OK if the kernels take them.
int check_attn(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t s, int64_t e, int64_t ev, int dtype, const void *Q,
               const int64_t *sq, const void *K, const int64_t *sk, const void *V, const int64_t *sv, const void *O,
               const int64_t *so, float scale) {
    if (n < 0 || hq < 0 || hkv <= 0 || l < 0 || s < 0 || e <= 0 || ev <= 0 || hq % hkv || !sq || !sk || !sv || !so)
        return KUIOPS_E_INVALID;
    if (n == 0 || hq == 0 || l == 0) return KUIOPS_OK;
    if (!Q || !O || (s > 0 && (!K || !V))) return KUIOPS_E_INVALID;
    if (dtype != KUIOPS_BF16 && dtype != KUIOPS_F16) return KUIOPS_E_UNSUPPORTED;
    if (e % 8 || ev % 8 || e > 256 || ev > 256) return KUIOPS_E_UNSUPPORTED;
    if (!(scale > 0.f) || !(scale * kLog2e < INFINITY)) return KUIOPS_E_UNSUPPORTED;
    if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || (reinterpret_cast<uintptr_t>(O) & 7)) return KUIOPS_E_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (sq[i] % 8 || sk[i] % 8 || sv[i] % 8 || so[i] % 4 || sk[i] < 0 || sv[i] < 0) return KUIOPS_E_UNSUPPORTED;
    // 32-bit indices of rows, keys and work-groups
    if (s >= (1 << 30) || hq / hkv * l >= (1 << 24) || n * hq * l >= ((int64_t)1 << 31) || n * hkv > 65535) return KUIOPS_E_UNSUPPORTED;
    return KUIOPS_OK;
}

// A split's keys are addressed with 31-bit byte offsets from its first one, and a
// launch has fewer than 2^32 threads.
bool plan_fits(const Plan &p, int64_t s, int64_t sk2, int64_t sv2) {
    const int64_t chunk = (cdiv(cdiv(s, 32), (int64_t)p.splits * 4) * 4 + 8) * 32;
    return chunk * std::max(sk2, sv2) * 2 + 1024 < ((int64_t)1 << 31) && cdiv(p.units, 8) * 8 * p.row_groups < ((int64_t)1 << 24) &&
           p.weight_groups * (p.hd <= 128 ? 512 : 256) < ((int64_t)1 << 32);
}

CacheAttnArgs fill_attn(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t s, int64_t e, int64_t ev, const void *Q,
                        const int64_t *sq, const void *K, const int64_t *sk, const void *V, const int64_t *sv, void *O,
                        const int64_t *so, float *lse, float scale, int mode, const int32_t *kv_len, const Plan &p,
                        void *workspace) {
    CacheAttnArgs a{};
    a.n = (int)n; a.hq = (int)hq; a.hkv = (int)hkv; a.l = (int)l; a.e = (int)e; a.ev = (int)ev; a.mode = mode;
    a.s = s;
    a.Q = Q; a.K = K; a.V = V; a.O = O;
    a.sq0 = sq[0]; a.sq1 = sq[1]; a.sq2 = sq[2];
    a.sk0 = sk[0]; a.sk1 = sk[1]; a.sk2 = sk[2];
    a.sv0 = sv[0]; a.sv1 = sv[1]; a.sv2 = sv[2];
    a.so0 = so[0]; a.so1 = so[1]; a.so2 = so[2];
    a.lse = lse;
    a.scale_log2 = scale * kLog2e;
    a.kv_len = kv_len;
    a.splits = p.splits; a.row_groups = p.row_groups; a.pair = p.pair; a.head_tiles = p.head_tiles; a.sum_here = p.sum_here;
    // (o and the scores in multiples of 16 bytes)
    char *ws = reinterpret_cast<char *>(workspace);
    a.ws_o = p.o_bytes ? reinterpret_cast<float *>(ws) : nullptr;
    a.scores = p.score_bytes ? reinterpret_cast<float *>(ws + p.o_bytes) : nullptr;
    a.ws_ml = p.ml_bytes ? reinterpret_cast<float *>(ws + p.o_bytes + p.score_bytes) : nullptr;
    // (behind the row sums, which are multiples of 8 bytes)
    a.part_sums = p.part_bytes ? reinterpret_cast<float *>(ws + p.o_bytes + p.score_bytes + p.ml_bytes) : nullptr;
    a.spad = cdiv(s, 32) * 32;
    return a;
}

}  // namespace

}  // namespace kuiops

using namespace kuiops;

extern "C" size_t kuiops_sdpa_tree_workspace(int64_t n, int64_t hq, int64_t hkv, int64_t t, int64_t s, int64_t e, int64_t ev) {
    if (n <= 0 || hq <= 0 || hkv <= 0 || t <= 0 || s < 0 || e <= 0 || ev <= 0) return 0;
    return state_bytes(plan_of(n, hq, hkv, t, s, e, ev, kTree, false));
}

extern "C" int kuiops_sdpa_tree(int64_t n, int64_t hq, int64_t hkv, int64_t t, int64_t s, int64_t e, int64_t ev, int dtype,
                                const void *Q, const int64_t sq[3], const void *K, const int64_t sk[3], const void *V,
                                const int64_t sv[3], void *O, const int64_t so[3], float *lse, float scale,
                                const int32_t *parent, const int32_t *kv_len, void *workspace, size_t workspace_bytes,
                                void *stream) {
    const int bad = check_attn(n, hq, hkv, t, s, e, ev, dtype, Q, sq, K, sk, V, sv, O, so, scale);
    if (bad) return bad;
    if (n == 0 || hq == 0 || t == 0) return KUIOPS_OK;
    if (!parent || t > s) return KUIOPS_E_INVALID;
    if (t > kMaxTree) return KUIOPS_E_UNSUPPORTED;
    const Plan p = plan_of(n, hq, hkv, t, s, e, ev, kTree, false);
    if (!plan_fits(p, s, sk[2], sv[2])) return KUIOPS_E_UNSUPPORTED;
    const size_t need = state_bytes(p);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KUIOPS_E_WORKSPACE;
    CacheAttnArgs a = fill_attn(n, hq, hkv, t, s, e, ev, Q, sq, K, sk, V, sv, O, so, lse, scale, kTree, kv_len, p, workspace);
    a.parent = parent;
    return dtype == KUIOPS_BF16 ? launch_attn_hd<bf16_t>(a, p, as_stream(stream)) : launch_attn_hd<f16_t>(a, p, as_stream(stream));
}

extern "C" size_t kuiops_sdpa_decode_accum_workspace(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t s, int64_t e,
                                                     int64_t ev) {
    if (n <= 0 || hq <= 0 || hkv <= 0 || l <= 0 || s < 0 || e <= 0 || ev <= 0) return 0;
    return std::max(state_bytes(plan_of(n, hq, hkv, l, s, e, ev, kCausal, true)),
                    state_bytes(plan_of(n, hq, hkv, l, s, e, ev, kFull, true)));
}

extern "C" int kuiops_sdpa_decode_accum(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t s, int64_t e, int64_t ev,
                                        int dtype, const void *Q, const int64_t sq[3], const void *K, const int64_t sk[3],
                                        const void *V, const int64_t sv[3], void *O, const int64_t so[3], float *lse,
                                        float scale, int causal, const int32_t *kv_len, float *acc, const int64_t sa[2],
                                        void *workspace, size_t workspace_bytes, void *stream) {
    const int bad = check_attn(n, hq, hkv, l, s, e, ev, dtype, Q, sq, K, sk, V, sv, O, so, scale);
    if (bad) return bad;
    if (n == 0 || hq == 0 || l == 0) return KUIOPS_OK;
    if (!lse || !sa || (s > 0 && !acc) || (causal && l > s)) return KUIOPS_E_INVALID;
    const Plan p = plan_of(n, hq, hkv, l, s, e, ev, causal ? kCausal : kFull, true);
    if (!plan_fits(p, s, sk[2], sv[2])) return KUIOPS_E_UNSUPPORTED;
    const size_t need = state_bytes(p);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KUIOPS_E_WORKSPACE;
    CacheAttnArgs a = fill_attn(n, hq, hkv, l, s, e, ev, Q, sq, K, sk, V, sv, O, so, lse, scale, causal ? kCausal : kFull,
                                kv_len, p, workspace);
    a.acc = s > 0 ? acc : nullptr;
    a.sa0 = sa[0]; a.sa1 = sa[1];
    return dtype == KUIOPS_BF16 ? launch_attn_hd<bf16_t>(a, p, as_stream(stream)) : launch_attn_hd<f16_t>(a, p, as_stream(stream));
}
