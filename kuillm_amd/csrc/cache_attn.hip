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

#include "common.hpp"

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
__device__ __forceinline__ void dma16_buf(__amdgpu_buffer_rsrc_t r, uint32_t voff, const void *dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)to_lds(dst), 16, (int)voff, 0,
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
    int splits, row_groups;
    float *ws_ml;              // [splits][n * hq * l][2]: maximum (log2 domain), sum
    float *ws_o;               // [splits][n * hq * l][HD]: unnormalised output
    float *acc;                // kuiops_sdpa_decode_accum: per key sums, strides sa0, sa1, 1
    int64_t sa0, sa1;
};

__device__ __forceinline__ int keys_of(const CacheAttnArgs &a, int b) {
    return a.kv_len ? (int)max((int64_t)0, min((int64_t)a.kv_len[b], a.s)) : (int)a.s;
}

// Which nodes each node of the tree sees (itself and its ancestors), as bits,
// by pointer doubling: after round r a node's word holds its 2^r nearest
// ancestors and `up` the next one, so 8 rounds suffice for 256 nodes and a
// shallow tree stops early.  A node is absent if its parent is below -1 or not
// an earlier node, or if an ancestor of it is: it then sees nothing.  Thread i
// has node i.
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

// ------------------------------------------------------------------------
// cache_attn_kernel -- 4 waves, each with key steps of 32 of its own; all have
// the same 16 * RT query rows.
//   S = K Q^T (16x16x32 MFMA): K straight from memory to registers; a lane
//   holds 8 scores of one row per 16-row tile, the row's maximum crosses lanes
//   16 and 32 apart only.  O^T += V^T P^T: V through LDS (DMA), read transposed;
//   the scores' registers are the other operand as they stand, keys numbered
//   in that order.  The probability is the sum of two 16-bit parts, one MFMA
//   each (2^-16 of it is lost in bf16, 2^-21 in f16): with the few rows of
//   this kernel the K / V stream takes the time, not the MFMAs.
// A part that is 0 times an infinite value is NaN, so is a masked NaN: a wave
// whose sums are not finite goes over its keys again, `careful`: values that
// are not finite are then taken out of the tile and multiplied by themselves,
// for the rows that see them.
template <typename T> struct Parts;
template <> struct Parts<bf16_t> {
    // p <= 2^8 between rescales
    static constexpr float kShift = 0.f;
};
template <> struct Parts<f16_t> {
    // p <= 2^15, so that f16's smallest step 2^-24 is 2^-39 of it
    static constexpr float kShift = -7.f;
};
constexpr float kSlack = 8.f;       // a row's maximum may grow by 2^8 before its sums are rescaled

template <typename T, int HD, int RT>
__global__ __launch_bounds__(256) void cache_attn_kernel(CacheAttnArgs a) {
    constexpr int NWV = 4, KB = 32, R = 16 * RT;
    constexpr int RB = HD * 2, VT = KB * RB;          // bytes per V row / wave tile
    constexpr int KK = HD / 32, DT = HD / 16, DV = VT / 1024;
    typedef typename Mfma<T>::frag frag;
    typedef T t8 __attribute__((ext_vector_type(8)));
    __shared__ __attribute__((aligned(1024))) char sV0[NWV * VT], sV1[NWV * VT];
    __shared__ float sm[NWV][R], sl[NWV][R];
    __shared__ TreeBits tb;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, G4 = lane >> 4;

    // The row groups of a (sequence, KV head, split) run on one XCD, whose L2
    // then has the keys for all but the first.
    const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
    const int unit = idx / a.row_groups * 8 + xcd, rg = idx % a.row_groups;
    if (unit >= a.n * a.hkv * a.splits) return;
    const int split = unit % a.splits, bh = unit / a.splits;
    const int b = bh / a.hkv, hk = bh % a.hkv;
    const int G = a.hq / a.hkv, rows_kv = G * a.l, r0 = rg * R;

    const int L = keys_of(a, b);
    const int steps = (L + KB - 1) / KB;
    // a sequence's steps are spread evenly over its splits, whole steps of the work-group
    const int chunk = (steps + a.splits * NWV - 1) / (a.splits * NWV) * NWV * KB;
    const int kbeg = min(L, split * chunk), kend = min(L, kbeg + chunk);
    const int first_node = L - a.l;                    // kTree: key of node 0 (may be below 0)
    const int free_end = a.mode == kFull ? L : a.mode == kCausal ? L - a.l + 1 : first_node;

    if (a.mode == kTree) tree_bits<NWV * 64>(tb, a.parent + (int64_t)b * a.l, a.l);

    const T *Kp = reinterpret_cast<const T *>(a.K) + b * a.sk0 + hk * a.sk1 + (int64_t)kbeg * a.sk2;
    const T *Vp = reinterpret_cast<const T *>(a.V) + b * a.sv0 + hk * a.sv1 + (int64_t)kbeg * a.sv2;
    const uint32_t kbytes = kend > kbeg ? (uint32_t)(((int64_t)(kend - kbeg - 1) * a.sk2 + a.e) * 2) : 0u;
    const uint32_t vbytes = kend > kbeg ? (uint32_t)(((int64_t)(kend - kbeg - 1) * a.sv2 + a.ev) * 2) : 0u;
    const __amdgpu_buffer_rsrc_t rsK = make_rsrc(Kp, kbytes), rsV = make_rsrc(Vp, vbytes);

    // query rows r0 + 16 rt + lr (B operand; rows past the list are 0)
    frag qf[RT][KK];
    bool row_ok[RT];
    int pos[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int rr = r0 + rt * 16 + lr;
        row_ok[rt] = rr < rows_kv;
        const int h = row_ok[rt] ? rr / a.l : 0;
        pos[rt] = row_ok[rt] ? rr % a.l : 0;
        // (an absent node's query is not read: whatever it holds stays out)
        if (a.mode == kTree && row_ok[rt]) row_ok[rt] = (tb.w[pos[rt]][pos[rt] >> 6] >> (pos[rt] & 63)) & 1;
        const T *q = reinterpret_cast<const T *>(a.Q) + b * a.sq0 + (hk * G + h) * a.sq1 + pos[rt] * a.sq2;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int d = kk * 32 + G4 * 8;
            qf[rt][kk] = as_frag<frag>(row_ok[rt] && d < a.e ? *reinterpret_cast<const u32x4 *>(q + d) : u32x4{0, 0, 0, 0});
        }
    }
    auto sees = [&](int rt, int key) __attribute__((always_inline)) -> bool {
        if (!row_ok[rt] || key >= kend) return false;
        if (key < free_end) return true;
        if (a.mode == kCausal) return key <= first_node + pos[rt];
        const int j = key - first_node;
        return (tb.w[pos[rt]][j >> 6] >> (j & 63)) & 1;
    };

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
        const uint32_t kb = on ? (uint32_t)((int64_t)(k0 - kbeg) * a.sk2 * 2) : kOut;
        const uint32_t vb = on ? (uint32_t)((int64_t)(k0 - kbeg) * a.sv2 * 2) : kOut;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                kr[slot][t][kk] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    rsK, (int)((kb | offK[t][kk]) >= kOut ? kOut : kb + offK[t][kk]), 0, 0));
#pragma unroll
        for (int j = 0; j < DV; ++j)
            dma16_buf(rsV, (vb | offV[j]) >= kOut ? kOut : vb + offV[j], sv + wave * VT + j * 1024);
        __builtin_amdgcn_sched_barrier(0);
    };

    f32x4 o[RT][DT];
    float m_used[RT], l_run[RT];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m_used[rt] = -INFINITY;
            l_run[rt] = 0.f;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    clear();
    bool careful = false;
    auto step = [&](int k0, int slot, char *sv) __attribute__((always_inline)) {
        t8 hi[RT], lo[RT];
        float pk[RT][8];
        const bool masked = k0 + KB > min(free_end, kend);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            f32x4 sc[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) sc[t] = Mfma<T>::m16(as_frag<frag>(kr[slot][t][kk]), qf[rt][kk], sc[t]);
            }
            // score (t, i): key k0 + 16 t + 4 G4 + i
            if (masked) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!sees(rt, k0 + 16 * t + 4 * G4 + i)) sc[t][i] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[t][i]);
            mx = xor_max<32>(xor_max<16>(mx)) * a.scale_log2;
            if (__any(mx > m_used[rt] + kSlack)) {
                const float m_new = fmaxf(m_used[rt], mx);
                const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_used[rt] - m_new);
                l_run[rt] *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[rt][t][i] *= alpha;
                m_used[rt] = m_new;
            }
            const float mref = m_used[rt] == -INFINITY ? 0.f : m_used[rt] + Parts<T>::kShift;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = fast_exp2(__builtin_fmaf(sc[t][i], a.scale_log2, -mref));
                    l_run[rt] += p;
                    pk[rt][4 * t + i] = p;
                    const T h = from_f32<T>(p);
                    hi[rt][4 * t + i] = h;
                    lo[rt][4 * t + i] = from_f32<T>(p - to_f32(h));
                }
        }
        // this step's V tile has landed: only the next step's loads are younger
        constexpr int Y = 2 * KK + DV;
        __builtin_amdgcn_s_waitcnt((Y & 15) | ((Y >> 4) << 14) | (7 << 4) | (15 << 8));
        __builtin_amdgcn_sched_barrier(0);
        if (careful) {
            // (d, key) of this lane's outputs: d = 16 dt + 4 G4 + i for row lr
            for (int x = 0; x < 8; ++x)
                for (int g = 0; g < 4; ++g) {
                    const int kr_ = 16 * (x >> 2) + 4 * g + (x & 3);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const int d = dt * 16 + 4 * G4;
                        T *vp = reinterpret_cast<T *>(sv + wave * VT + kr_ * RB + (((d >> 3) ^ vsw(kr_)) << 4) + (d & 4) * 2);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float val = to_f32(vp[i]);
                            const bool odd = !(fabsf(val) < INFINITY);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                float p = pk[rt][0];
#pragma unroll
                                for (int y = 1; y < 8; ++y) p = x == y ? pk[rt][y] : p;
                                p = __shfl(p, g * 16 + lr, 64);
                                if (odd && sees(rt, k0 + kr_)) o[rt][dt][i] += p * val;
                            }
                        }
                    }
                }
            __builtin_amdgcn_s_waitcnt(0xc07f);
            for (int c = lane; c < VT / 2; c += 64) {
                T *vp = reinterpret_cast<T *>(sv + wave * VT) + c;
                if (!(fabsf(to_f32(*vp)) < INFINITY)) *vp = from_f32<T>(0.f);
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const char *vb = sv + wave * VT + offVr[dt];
            const s16x4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)to_lds(vb));
            const s16x4 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)to_lds(vb + 16 * RB));
            const u32x2 h0 = __builtin_bit_cast(u32x2, t0), h1 = __builtin_bit_cast(u32x2, t1);
            const frag vf = as_frag<frag>(u32x4{h0[0], h0[1], h1[0], h1[1]});
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                o[rt][dt] = Mfma<T>::m16(vf, __builtin_bit_cast(frag, hi[rt]), o[rt][dt]);
                o[rt][dt] = Mfma<T>::m16(vf, __builtin_bit_cast(frag, lo[rt]), o[rt][dt]);
            }
        }
    };

    constexpr int KS = NWV * KB;
    for (;;) {
        int k0 = kbeg + wave * KB;
        issue(k0, 0, sV0);
        for (; k0 < kend; k0 += 2 * KS) {
            issue(k0 + KS, 1, sV1);
            step(k0, 0, sV0);
            // (this wave's reads of the tile are done before its refill)
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_sched_barrier(0);
            issue(k0 + 2 * KS, 0, sV0);
            step(k0 + KS, 1, sV1);
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_sched_barrier(0);
        }
        // no DMA is in flight past here
        __builtin_amdgcn_s_waitcnt(0);
        __builtin_amdgcn_sched_barrier(0);
        float z = 0.f;                  // stays 0 if every sum is finite
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) z = __builtin_fmaf(o[rt][t][i], 0.f, z);
        if (careful || !__any(z != 0.f)) break;
        careful = true;
        clear();
    }

    // the waves' sums merge through LDS, 16 rows at a time in the first tiles' place
    constexpr int D4 = HD / 4;
    float (*so)[16][HD] = reinterpret_cast<float (*)[16][HD]>(sV0);
    static_assert(16 * HD * 4 == VT, "a wave's 16 rows take its V tile");
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        // lanes of a row hold disjoint keys: row sums over the lane groups
        const float lsum = xor_add<32>(xor_add<16>(l_run[rt]));
        if (G4 == 0) {
            sm[wave][rt * 16 + lr] = row_ok[rt] ? m_used[rt] + Parts<T>::kShift : -INFINITY;
            sl[wave][rt * 16 + lr] = row_ok[rt] ? lsum : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            *reinterpret_cast<f32x4 *>(&so[wave][lr][dt * 16 + 4 * G4]) = row_ok[rt] ? o[rt][dt] : f32x4{0.f, 0.f, 0.f, 0.f};
        __syncthreads();
        for (int x = tid; x < 16 * D4; x += NWV * 64) {
            const int r = x / D4, d = x % D4 * 4, rr = r0 + rt * 16 + r;
            if (rr >= rows_kv) continue;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < NWV; ++w) mm = fmaxf(mm, sm[w][rt * 16 + r]);
            const float mu = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f;
            f32x4 oo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NWV; ++w) {
                const float wgt = fast_exp2(sm[w][rt * 16 + r] - mu);
                ll = __builtin_fmaf(sl[w][rt * 16 + r], wgt, ll);
                const f32x4 ov = *reinterpret_cast<const f32x4 *>(&so[w][r][d]);
#pragma unroll
                for (int i = 0; i < 4; ++i) oo[i] = __builtin_fmaf(ov[i], wgt, oo[i]);
            }
            const int head = hk * G + rr / a.l, i = rr % a.l;
            const int64_t row = ((int64_t)b * a.hq + head) * a.l + i;
            if (a.splits > 1) {
                const int64_t st = (int64_t)split * a.n * a.hq * a.l + row;
                *reinterpret_cast<f32x4 *>(&a.ws_o[st * HD + d]) = oo;
                if (d == 0) {
                    a.ws_ml[st * 2] = mm;
                    a.ws_ml[st * 2 + 1] = ll;
                }
                continue;
            }
            const float inv = ll != 0.f ? 1.f / ll : 0.f;
            if (d < a.ev) {
                typedef T t4 __attribute__((ext_vector_type(4)));
                t4 w;
#pragma unroll
                for (int y = 0; y < 4; ++y) w[y] = from_f32<T>(oo[y] * inv);
                *reinterpret_cast<t4 *>(reinterpret_cast<T *>(a.O) + b * a.so0 + head * a.so1 + i * a.so2 + d) = w;
            }
            if (a.lse && d == 0) a.lse[row] = ll != 0.f ? (mm + __log2f(ll)) * kLn2 : -INFINITY;
        }
    }
}

// The splits' states of a row, merged in split order (the same bits whatever
// order the work-groups ended in): a thread has 4 columns of a row.
template <typename T, int HD>
__global__ __launch_bounds__(256) void cache_merge_kernel(CacheAttnArgs a) {
    constexpr int D4 = HD / 4;
    const int64_t rows = (int64_t)a.n * a.hq * a.l;
    const int64_t row = (int64_t)blockIdx.x * (256 / D4) + threadIdx.x / D4;
    if (row >= rows) return;
    const int d = threadIdx.x % D4 * 4;
    float mm = -INFINITY;
    for (int z = 0; z < a.splits; ++z) mm = fmaxf(mm, a.ws_ml[(z * rows + row) * 2]);
    const float mu = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    f32x4 oo = {0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < a.splits; ++z) {
        const f32x2 ml = *reinterpret_cast<const f32x2 *>(&a.ws_ml[(z * rows + row) * 2]);
        const f32x4 ov = *reinterpret_cast<const f32x4 *>(&a.ws_o[(z * rows + row) * HD + d]);
        const float wgt = fast_exp2(ml[0] - mu);
        ll = __builtin_fmaf(ml[1], wgt, ll);
#pragma unroll
        for (int i = 0; i < 4; ++i) oo[i] = __builtin_fmaf(ov[i], wgt, oo[i]);
    }
    const int i = (int)(row % a.l), head = (int)(row / a.l % a.hq);
    const int64_t b = row / a.l / a.hq;
    const float inv = ll != 0.f ? 1.f / ll : 0.f;
    if (d < a.ev) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 w;
#pragma unroll
        for (int y = 0; y < 4; ++y) w[y] = from_f32<T>(oo[y] * inv);
        *reinterpret_cast<t4 *>(reinterpret_cast<T *>(a.O) + b * a.so0 + head * a.so1 + i * a.so2 + d) = w;
    }
    if (a.lse && d == 0) a.lse[row] = ll != 0.f ? (mm + __log2f(ll)) * kLn2 : -INFINITY;
}

// key_weights_kernel -- acc[key] += sum over the rows of its KV head of
// exp(scale q k - lse).  A wave keeps 16 keys in registers (A operand) and goes
// over the rows 16 at a time; the rows' sum crosses lanes once, at the end.
template <typename T, int HD>
__global__ __launch_bounds__(256) void key_weights_kernel(CacheAttnArgs a) {
    constexpr int KK = HD / 32;
    typedef typename Mfma<T>::frag frag;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lr = lane & 15, G4 = lane >> 4;
    const int b = blockIdx.y / a.hkv, hk = blockIdx.y % a.hkv;
    const int G = a.hq / a.hkv, rows_kv = G * a.l;
    const int L = keys_of(a, b), first = L - a.l;
    const int k0 = blockIdx.x * 64 + wave * 16;
    if (k0 >= L) return;
    frag kf[KK];
    const bool key_ok = k0 + lr < L;
    const T *kp = reinterpret_cast<const T *>(a.K) + b * a.sk0 + hk * a.sk1 + (int64_t)(k0 + lr) * a.sk2;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        const int d = kk * 32 + G4 * 8;
        kf[kk] = as_frag<frag>(key_ok && d < a.e ? *reinterpret_cast<const u32x4 *>(kp + d) : u32x4{0, 0, 0, 0});
    }
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < rows_kv; r0 += 16) {
        const int rr = r0 + lr;
        const bool ok = rr < rows_kv;
        const int h = ok ? rr / a.l : 0, i = ok ? rr % a.l : 0;
        const T *q = reinterpret_cast<const T *>(a.Q) + b * a.sq0 + (hk * G + h) * a.sq1 + i * a.sq2;
        const float lse = ok ? a.lse[((int64_t)b * a.hq + hk * G + h) * a.l + i] * kLog2e : -INFINITY;
        f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int d = kk * 32 + G4 * 8;
            const frag qf = as_frag<frag>(ok && d < a.e ? *reinterpret_cast<const u32x4 *>(q + d) : u32x4{0, 0, 0, 0});
            sc = Mfma<T>::m16(kf[kk], qf, sc);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int key = k0 + 4 * G4 + x;
            const bool vis = ok && lse != -INFINITY && (a.mode == kFull || key <= first + i);
            sum[x] += vis ? fast_exp2(__builtin_fmaf(sc[x], a.scale_log2, -lse)) : 0.f;
        }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const float t = group_sum<16>(sum[x]);
        const int key = k0 + 4 * G4 + x;
        if (lr == 0 && key < L) a.acc[b * a.sa0 + hk * a.sa1 + key] += t;
    }
}

// ------------------------------------------------------------- host side

constexpr int kGroupsWanted = 512;      // work-groups of a launch: two for each of the 256 CUs
constexpr int kMaxSplits = 64;

struct Plan {
    int hd, rt, row_groups, splits;
    int64_t units;
};

// Rows of a work-group: 16, or 32 where there are more than 16.  Splits: as
// many as fill the GPU, of at least 128 keys (a step of each wave).
Plan plan_of(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t s, int64_t e, int64_t ev) {
    Plan p{};
    const int64_t w = std::max(e, ev), rows = hq / hkv * l;
    p.hd = w <= 64 ? 64 : w <= 128 ? 128 : 256;
    p.rt = rows > 16 && p.hd <= 128 ? 2 : 1;
    p.row_groups = (int)cdiv(rows, 16 * p.rt);
    const int64_t groups = n * hkv * p.row_groups;
    p.splits = (int)std::max<int64_t>(1, std::min({(int64_t)kMaxSplits, kGroupsWanted / std::max<int64_t>(groups, 1), cdiv(s, 128)}));
    p.units = n * hkv * p.splits;
    return p;
}

size_t state_bytes(const Plan &p, int64_t rows) {
    return p.splits > 1 ? (size_t)p.splits * rows * (p.hd + 2) * sizeof(float) + 32 : 0;
}

template <typename T, int HD>
int launch_attn(const CacheAttnArgs &a, const Plan &p, hipStream_t st) {
    const dim3 grid((unsigned)(cdiv(p.units, 8) * 8 * p.row_groups));
    if (p.rt == 1) hipLaunchKernelGGL((cache_attn_kernel<T, HD, 1>), grid, dim3(256), 0, st, a);
    else if constexpr (HD <= 128) hipLaunchKernelGGL((cache_attn_kernel<T, HD, 2>), grid, dim3(256), 0, st, a);
    if (p.splits > 1) {
        const int64_t rows = (int64_t)a.n * a.hq * a.l;
        hipLaunchKernelGGL((cache_merge_kernel<T, HD>), dim3((unsigned)cdiv(rows, 256 / (HD / 4))), dim3(256), 0, st, a);
    }
    if (a.acc)
        hipLaunchKernelGGL((key_weights_kernel<T, HD>), dim3((unsigned)cdiv(a.s, 64), (unsigned)(a.n * a.hkv)), dim3(256),
                           0, st, a);
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
    if (!(scale > 0.f) || !(scale < INFINITY)) return KUIOPS_E_UNSUPPORTED;
    if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || (reinterpret_cast<uintptr_t>(O) & 7)) return KUIOPS_E_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (sq[i] % 8 || sk[i] % 8 || sv[i] % 8 || so[i] % 4 || sk[i] < 0 || sv[i] < 0) return KUIOPS_E_UNSUPPORTED;
    // 32-bit indices of rows, keys and work-groups
    if (s >= (1 << 30) || hq / hkv * l >= (1 << 24) || n * hq * l >= ((int64_t)1 << 31) || n * hkv > 65535) return KUIOPS_E_UNSUPPORTED;
    return KUIOPS_OK;
}

// A split's keys are addressed with 31-bit byte offsets from its first one.
bool split_fits(const Plan &p, int64_t s, int64_t sk2, int64_t sv2) {
    const int64_t chunk = (cdiv(cdiv(s, 32), (int64_t)p.splits * 4) * 4 + 8) * 32;
    return chunk * std::max(sk2, sv2) * 2 + 1024 < ((int64_t)1 << 31);
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
    a.splits = p.splits; a.row_groups = p.row_groups;
    a.ws_o = reinterpret_cast<float *>(workspace);
    a.ws_ml = p.splits > 1 ? a.ws_o + (int64_t)p.splits * n * hq * l * p.hd : nullptr;
    return a;
}

}  // namespace

}  // namespace kuiops

using namespace kuiops;

extern "C" size_t kuiops_sdpa_tree_workspace(int64_t n, int64_t hq, int64_t hkv, int64_t t, int64_t s, int64_t e, int64_t ev) {
    if (n <= 0 || hq <= 0 || hkv <= 0 || t <= 0 || s < 0 || e <= 0 || ev <= 0) return 0;
    return state_bytes(plan_of(n, hq, hkv, t, s, e, ev), n * hq * t);
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
    const Plan p = plan_of(n, hq, hkv, t, s, e, ev);
    if (!split_fits(p, s, sk[2], sv[2])) return KUIOPS_E_UNSUPPORTED;
    const size_t need = state_bytes(p, n * hq * t);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KUIOPS_E_WORKSPACE;
    CacheAttnArgs a = fill_attn(n, hq, hkv, t, s, e, ev, Q, sq, K, sk, V, sv, O, so, lse, scale, kTree, kv_len, p, workspace);
    a.parent = parent;
    return dtype == KUIOPS_BF16 ? launch_attn_hd<bf16_t>(a, p, as_stream(stream)) : launch_attn_hd<f16_t>(a, p, as_stream(stream));
}

extern "C" size_t kuiops_sdpa_decode_accum_workspace(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t s, int64_t e,
                                                     int64_t ev) {
    if (n <= 0 || hq <= 0 || hkv <= 0 || l <= 0 || s < 0 || e <= 0 || ev <= 0) return 0;
    return state_bytes(plan_of(n, hq, hkv, l, s, e, ev), n * hq * l);
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
    const Plan p = plan_of(n, hq, hkv, l, s, e, ev);
    if (!split_fits(p, s, sk[2], sv[2])) return KUIOPS_E_UNSUPPORTED;
    const size_t need = state_bytes(p, n * hq * l);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KUIOPS_E_WORKSPACE;
    CacheAttnArgs a = fill_attn(n, hq, hkv, l, s, e, ev, Q, sq, K, sk, V, sv, O, so, lse, scale, causal ? kCausal : kFull,
                                kv_len, p, workspace);
    a.acc = s > 0 ? acc : nullptr;
    a.sa0 = sa[0]; a.sa1 = sa[1];
    return dtype == KUIOPS_BF16 ? launch_attn_hd<bf16_t>(a, p, as_stream(stream)) : launch_attn_hd<f16_t>(a, p, as_stream(stream));
}
