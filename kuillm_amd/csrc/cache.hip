// What happens to a KV cache besides attention, gfx950:
//
//   kuiops_tree_accept     the branch of a drafted tree that the model agrees with
//   kuiops_kv_tree_commit  its rows moved behind the context
//   kuiops_kv_evict        the cache cut down to the keys that weighed most
//
// All are copies and comparisons: results are exact, ties go to the lowest
// index, and nothing depends on the order in which work-groups run.
#include <algorithm>

#include "common.hpp"

namespace kuiops {

namespace {

constexpr int kMaxTree = 256;                 // nodes of a tree

// ------------------------------------------------------------ tree_accept
// A wave per sequence, 4 nodes per lane.  A node is a candidate if its token is
// the target of its parent; the walk from node 0 takes the lowest candidate
// among the children, a ballot per 64 nodes and step.  Bound by latency, one load
// and the path's length: 2.0 us for a tree of 8 nodes, 3.1 us for 16 of 64.
__global__ __launch_bounds__(64) void tree_accept_kernel(int t, const int64_t *tokens, const int32_t *parent,
                                                         const int64_t *target, int32_t *path, int32_t *count, int64_t *next) {
    constexpr int NW = kMaxTree / 64;
    const int lane = threadIdx.x;
    const int64_t b = blockIdx.x;
    tokens += b * t;
    parent += b * t;
    target += b * t;
    path += b * t;
    __shared__ int64_t s_target[kMaxTree];
    int up[NW], mine[NW];                     // parent of a candidate (else -1); the path's node at this lane's place
    int64_t token[NW];
#pragma unroll
    for (int x = 0; x < NW; ++x) {
        const int i = x * 64 + lane;
        up[x] = mine[x] = -1;
        token[x] = 0;
        if (i < t) {
            up[x] = parent[i];
            token[x] = tokens[i];
            s_target[i] = target[i];
        }
    }
    __syncthreads();
    int at = __shfl(up[0], 0, 64) == -1 ? 0 : -1, last = -1, n = 0;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
        const int i = x * 64 + lane, p = up[x];
        up[x] = i < t && p >= 0 && p < i && token[x] == s_target[p] ? p : -1;
    }
    while (at >= 0) {
#pragma unroll
        for (int x = 0; x < NW; ++x)
            if (n == x * 64 + lane) mine[x] = at;
        ++n;
        last = at;
        at = -1;
#pragma unroll
        for (int x = NW - 1; x >= 0; --x) {
            const uint64_t hits = __ballot(up[x] == last);
            if (hits) at = x * 64 + __builtin_ctzll(hits);
        }
    }
#pragma unroll
    for (int x = 0; x < NW; ++x)
        if (x * 64 + lane < t) path[x * 64 + lane] = mine[x];
    if (lane == 0) {
        count[b] = n;
        next[b] = last >= 0 ? s_target[last] : -1;
    }
}

// --------------------------------------------------------- kv_tree_commit
// A wave has up to 512 bytes of each row of a head's K or V, and all rows of a
// pass over their columns are in its registers before the first is written, so
// any path is right, whichever rows it reads and overwrites.  As many columns a
// pass as 16 registers of 16 bytes hold: all 32 for up to 32 rows.  Bound by
// latency (path, rows, stores, each behind the one before): 16 layers of 8 heads,
// one sequence, heads of 64: 4.2 us; 16 sequences, heads of 128: 7.0 us.
constexpr int kCommitRegs = 16, kCommitWaves = 4;
struct CommitArgs {
    int n, p, t, hkv;
    int64_t cap, units;
    char *K, *V;
    int64_t sk0, sk1, sk2, sv0, sv1, sv2;     // bytes
    int kcols, vcols, kblocks, blocks;        // 16-byte chunks of a row; waves of 32 chunks for K, for both
    const int32_t *path, *kv_len;
    int32_t *len_out;
};
__global__ __launch_bounds__(kCommitWaves * 64) void tree_commit_kernel(CommitArgs a) {
    constexpr int NW = kMaxTree / 64;
    __shared__ int s_path[kCommitWaves][kMaxTree];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = (int64_t)blockIdx.x * kCommitWaves + wave;
    if (unit >= a.units) return;
    const int blk = (int)(unit % a.blocks), head = (int)(unit / a.blocks % a.hkv);
    const int64_t row = unit / a.blocks / a.hkv;
    const int b = (int)(row % a.n);
    const bool is_v = blk >= a.kblocks;
    const int c0 = (blk - (is_v ? a.kblocks : 0)) * 32;
    const int cols = min(32, (is_v ? a.vcols : a.kcols) - c0);
    const int64_t len = a.kv_len[b], base = len - a.t;
    // the path ends at its first entry that is no row of the tree in the cache
    int count = a.p;
#pragma unroll
    for (int x = NW - 1; x >= 0; --x) {
        const int i = x * 64 + lane;
        int v = -1;
        if (i < a.p) v = a.path[(int64_t)b * a.p + i];
        s_path[wave][i] = v;
        const uint64_t bad = __ballot(i < a.p && (v < 0 || v >= a.t || base < 0 || base + max(v, i) >= a.cap));
        if (bad) count = x * 64 + __builtin_ctzll(bad);
    }
    if (unit < (int64_t)a.n * a.hkv * a.blocks && head == 0 && blk == 0 && lane == 0)
        a.len_out[b] = (int)(base < 0 ? len : base + count);
    if (count == 0) return;
    __builtin_amdgcn_s_waitcnt(0xc07f);           // (the wave's own LDS writes)
    char *p = is_v ? a.V + row * a.sv0 + head * a.sv1 : a.K + row * a.sk0 + head * a.sk1;
    const int64_t st = is_v ? a.sv2 : a.sk2;
    p += base * st + c0 * 16;
    int sh = 5;                                   // 2^sh columns a pass
    while ((count << sh) > kCommitRegs * 64) --sh;
    while (sh > 0 && (1 << (sh - 1)) >= cols) --sh;
    for (int cb = 0; cb < cols; cb += 1 << sh) {
        u32x4 r[kCommitRegs];
#pragma unroll
        for (int x = 0; x < kCommitRegs; ++x) {
            const int i = x * 64 + lane, to = i >> sh, c = cb + (i & ((1 << sh) - 1));
            if (to < count && c < cols) r[x] = *reinterpret_cast<const u32x4 *>(p + s_path[wave][to] * st + c * 16);
        }
        __builtin_amdgcn_s_waitcnt(0);            // read before any row is written
        __builtin_amdgcn_sched_barrier(0);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
        for (int x = 0; x < kCommitRegs; ++x) {
            const int i = x * 64 + lane, to = i >> sh, c = cb + (i & ((1 << sh) - 1));
            if (to < count && c < cols && s_path[wave][to] != to) *reinterpret_cast<u32x4 *>(p + to * st + c * 16) = r[x];
        }
    }
}

// --------------------------------------------------------------- kv_evict
// evict_select_kernel, a work-group per (sequence, KV head): the key of a slot
// is its weight's bits in ascending order, or the largest of all for the
// `recent` newest positions.  The budget-th largest key is found 11, 11 and 10
// bits at a time with a histogram in LDS (as many bits as that spread weights,
// which share a few exponents, over enough counters); slots with a larger key are
// kept, and of those with the same key the first ones.  Ranks in slot order then
// pair the freed slots below the budget with the kept ones behind it: as many of
// one as of the other, and the i-th kept row goes to the i-th freed slot.  Sources
// are at or behind the budget and destinations below it, so the moves need no
// order.  Slots of 1024 x IPT keys stay in registers (thread t has t, t + 1024,
// ...); longer caches are read again (from L2) in each of the five passes (newest
// position, three digits, ranks).
// evict_move_kernel moves the rows of K and V (few of them move in the first kernel).
// What bounds them: a few hundred slots, one work-group's latency (576 keys: 8.2 us with
// the move); 64 heads of 8000, select 15 us (13.3 with the slots in L2), of it the
// histograms about half, on 64 of the 256 CUs; the moves, 91 MB read and written in 20 us,
// 4.5 TB/s: row by row they stay 12% below a large copy.
constexpr int kEvictThreads = 1024;
struct EvictArgs {
    int n, hkv, budget, recent;
    int64_t cap;
    const int32_t *kv_len;
    int32_t *len_out;
    const float *acc;
    const int32_t *pos;
    float *acc_out;
    int32_t *pos_out;
    int64_t sa0, sa1, sp0, sp1, sao0, sao1, spo0, spo1;
    int32_t *moves;            // [n * hkv][1 + 2 * budget]: count, destinations, sources
    char *K, *V;
    int64_t sk0, sk1, sk2, sv0, sv1, sv2;     // bytes
    int kcols, vcols;                         // 16-byte chunks of a row
    int move_here;                            // evict_select_kernel moves its head's rows too
};

// Rows first .. of a head's moves, 16 bytes a thread, `step` apart.
__device__ __forceinline__ void move_rows(const EvictArgs &a, int b, int hk, const int32_t *moves, int count, int64_t first, int64_t step) {
    const int cols = a.kcols + a.vcols;
    char *K = a.K + b * a.sk0 + hk * a.sk1, *V = a.V + b * a.sv0 + hk * a.sv1;
    for (int64_t x = first; x < (int64_t)count * cols; x += step) {
        const int i = (int)(x / cols), c = (int)(x % cols);
        const int64_t to = moves[1 + i], from = moves[1 + a.budget + i];
        if (c < a.kcols)
            *reinterpret_cast<u32x4 *>(K + to * a.sk2 + c * 16) = *reinterpret_cast<const u32x4 *>(K + from * a.sk2 + c * 16);
        else
            *reinterpret_cast<u32x4 *>(V + to * a.sv2 + (c - a.kcols) * 16) =
                *reinterpret_cast<const u32x4 *>(V + from * a.sv2 + (c - a.kcols) * 16);
    }
}
__device__ __forceinline__ int new_length(const EvictArgs &a, int b) {
    return min(max(a.kv_len[b], 0), (int)min((int64_t)a.budget, a.cap));
}

__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xfffffffeu;           // NaN ranks above every number
    const uint32_t u = __float_as_uint(w + 0.f);              // (-0 is 0)
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive sums of one value per thread, and their total (all threads).
template <int NT>
__device__ __forceinline__ int block_scan(int v, int *s_wave, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(incl, o, 64);
        incl += lane >= o ? x : 0;
    }
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const int c = s_wave[w];
        before += w < wave ? c : 0;
        total += c;
    }
    __syncthreads();
    return before + incl - v;
}

template <int IPT>        // slots of a thread held in registers; 0: none, any number
__global__ __launch_bounds__(kEvictThreads) void evict_select_kernel(EvictArgs a) {
    constexpr int NT = kEvictThreads, NW = NT / 64, NR = IPT > 0 ? IPT : 1;
    constexpr int kBins = 2048;
    static_assert(IPT * NW < kBins, "the counts take the histogram's place");
    __shared__ int s_wave[NW], s_hist[kBins];
    __shared__ uint16_t s_rank[NW][2];
    __shared__ int s_digit, s_left, s_same;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.x / a.hkv, hk = blockIdx.x % a.hkv, m = a.budget;
    const int L = (int)max((int64_t)0, min((int64_t)a.kv_len[b], a.cap)), cap = (int)a.cap;
    const float *acc = a.acc + b * a.sa0 + hk * a.sa1;
    const int32_t *pos = a.pos + b * a.sp0 + hk * a.sp1;
    float *acc_out = a.acc_out + b * a.sao0 + hk * a.sao1;
    int32_t *pos_out = a.pos_out + b * a.spo0 + hk * a.spo1;
    int32_t *moves = a.moves + (int64_t)blockIdx.x * (1 + 2 * m);
    if (a.move_here && hk == 0 && tid == 0) a.len_out[b] = new_length(a, b);
    if (L <= m) {
        for (int j = tid; j < cap; j += NT) {
            acc_out[j] = j < L ? acc[j] : 0.f;
            pos_out[j] = j < L ? pos[j] : -1;
        }
        if (tid == 0) moves[0] = 0;
        return;
    }
    const int chunks = (L + NT - 1) / NT;
    // this thread's slots
    float ra[NR];
    int32_t rp[NR];
    uint32_t rk[NR];
    int newest = -INT32_MAX;
    if constexpr (IPT > 0) {
#pragma unroll
        for (int c = 0; c < IPT; ++c) {
            const int j = c * NT + tid;
            ra[c] = j < L ? acc[j] : 0.f;
            rp[c] = j < L ? pos[j] : INT32_MIN;
        }
#pragma unroll
        for (int c = 0; c < IPT; ++c) newest = max(newest, rp[c]);
    } else {
        for (int j = tid; j < L; j += NT) newest = max(newest, pos[j]);
    }
    for (int x = tid; x < kBins; x += NT) s_hist[x] = 0;
    newest = -wave_min_i32(-newest);
    if (lane == 0) s_wave[wave] = newest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) newest = max(newest, s_wave[w]);
    const int64_t floor_pos = (int64_t)newest - a.recent;
    auto key_of = [&](float w, int32_t p) -> uint32_t { return p > floor_pos ? 0xffffffffu : weight_key(w); };
    if constexpr (IPT > 0) {
#pragma unroll
        for (int c = 0; c < IPT; ++c) rk[c] = key_of(ra[c], rp[c]);
    }
    // f(slot, key) for this thread's slots, in slot order
    auto each = [&](auto f) {
        if constexpr (IPT > 0) {
#pragma unroll
            for (int c = 0; c < IPT; ++c)
                if (c * NT + tid < L) f(c * NT + tid, rk[c]);
        } else {
            for (int j = tid; j < L; j += NT) f(j, key_of(acc[j], pos[j]));
        }
    };

    uint32_t prefix = 0, mask = 0;
    int need = m, same = 0;                    // of the keys with this prefix, the need-th largest is sought
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        each([&](int, uint32_t k) {
            if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> sh) & ((1 << bits) - 1)], 1);
        });
        __syncthreads();
        // thread t has the two largest counters that are left of it: kBins - 1 - 2 t and the next one below
        const int hi = s_hist[kBins - 1 - 2 * tid], lo = s_hist[kBins - 2 - 2 * tid];
        int total;
        const int above = block_scan<NT>(hi + lo, s_wave, total);
        if (above < need && need <= above + hi + lo) {
            const bool first = need <= above + hi;
            s_digit = kBins - 1 - 2 * tid - (first ? 0 : 1);
            s_left = need - above - (first ? 0 : hi);
            s_same = first ? hi : lo;
        }
        s_hist[kBins - 1 - 2 * tid] = s_hist[kBins - 2 - 2 * tid] = 0;
        __syncthreads();
        prefix |= (uint32_t)s_digit << sh;
        mask |= ((1u << bits) - 1) << sh;
        need = s_left;
        same = s_same;
    }

    const bool ties = need < same;              // some of the equal keys are freed
    const uint64_t below = (1ull << lane) - 1;
    auto place = [&](int j, bool kept, bool hole, int hr, int fr, float w, int32_t p) __attribute__((always_inline)) {
        const bool far = j >= m && kept;
        if (hole) moves[1 + hr] = j;
        if (far) moves[1 + m + fr] = j;
        if (kept && !far) {
            acc_out[j] = w;
            pos_out[j] = p;
        }
    };
    int holes_all = 0;
    if constexpr (IPT > 0) {
        // counts per 1024 slots and wave, in slot order, and one scan of them all
        // (wave 0), first of the equal keys, then of freed (low half) and far slots
        uint32_t *s_count = reinterpret_cast<uint32_t *>(s_hist);
        constexpr int NC = IPT * NW, PER = (NC + 63) / 64;
        auto scan_counts = [&](uint32_t &total) __attribute__((always_inline)) {
            __syncthreads();
            if (wave == 0) {
                uint32_t v[PER], sum = 0;
#pragma unroll
                for (int x = 0; x < PER; ++x) {
                    v[x] = lane * PER + x < NC ? s_count[lane * PER + x] : 0;
                    sum += v[x];
                }
                uint32_t incl = sum;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const uint32_t y = __shfl_up(incl, o, 64);
                    incl += lane >= o ? y : 0;
                }
                uint32_t run = incl - sum;
#pragma unroll
                for (int x = 0; x < PER; ++x) {
                    if (lane * PER + x < NC) s_count[lane * PER + x] = run;
                    run += v[x];
                }
                if (lane == 63) s_count[NC] = run;
            }
            __syncthreads();
            total = s_count[NC];
        };
        uint32_t keeps = 0;                    // of this thread's slots, as bits
        uint32_t total;
        if (ties) {
#pragma unroll
            for (int c = 0; c < IPT; ++c) {
                const uint64_t eqs = __ballot(c * NT + tid < L && rk[c] == prefix);
                if (lane == 0) s_count[c * NW + wave] = (uint32_t)__popcll(eqs);
            }
            scan_counts(total);
        }
#pragma unroll
        for (int c = 0; c < IPT; ++c) {
            const bool in = c * NT + tid < L;
            bool kept = in && rk[c] >= prefix;
            if (ties) {
                const uint64_t eqs = __ballot(in && rk[c] == prefix);
                kept = in && (rk[c] > prefix || (rk[c] == prefix && (int)s_count[c * NW + wave] + __popcll(eqs & below) < need));
            }
            keeps |= kept ? 1u << c : 0u;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < IPT; ++c) {
            const int j = c * NT + tid;
            const bool kept = keeps >> c & 1;
            const uint32_t holes = (uint32_t)__popcll(__ballot(j < m && j < L && !kept)), fars = (uint32_t)__popcll(__ballot(j >= m && kept));
            if (lane == 0) s_count[c * NW + wave] = fars << 16 | holes;
        }
        scan_counts(total);
        holes_all = (int)(total & 0xffffu);
#pragma unroll
        for (int c = 0; c < IPT; ++c) {
            const int j = c * NT + tid;
            const bool kept = keeps >> c & 1, hole = j < m && j < L && !kept;
            const uint64_t hb = __ballot(hole), fb = __ballot(j >= m && kept);
            const uint32_t before = s_count[c * NW + wave];
            place(j, kept, hole, (int)(before & 0xffffu) + __popcll(hb & below), (int)(before >> 16) + __popcll(fb & below), ra[c], rp[c]);
        }
    } else {
        // 1024 slots at a time, with running counts
        int eq0 = 0, hole0 = 0, far0 = 0;
        for (int c = 0; c < chunks; ++c) {
            const int j = c * NT + tid;
            const bool in = j < L;
            const float w = in ? acc[j] : 0.f;
            const int32_t p = in ? pos[j] : 0;
            const uint32_t k = in ? key_of(w, p) : 0;
            const bool eq = in && k == prefix;
            int eqr = 0;
            if (ties) {
                const uint64_t eqs = __ballot(eq);
                if (lane == 0) s_wave[wave] = __popcll(eqs);
                __syncthreads();
                eqr = eq0 + __popcll(eqs & below);
#pragma unroll
                for (int v = 0; v < NW; ++v) {
                    const int x = s_wave[v];
                    eqr += v < wave ? x : 0;
                    eq0 += x;
                }
                // (the barriers below separate these reads from the next writes)
            }
            const bool kept = in && (k > prefix || (eq && eqr < need));
            const bool hole = in && j < m && !kept, far = j >= m && kept;
            const uint64_t hb = __ballot(hole), fb = __ballot(far);
            if (lane == 0) {
                s_rank[wave][0] = (uint16_t)__popcll(hb);
                s_rank[wave][1] = (uint16_t)__popcll(fb);
            }
            __syncthreads();
            int hr = hole0 + __popcll(hb & below), fr = far0 + __popcll(fb & below);
#pragma unroll
            for (int v = 0; v < NW; ++v) {
                const int x = s_rank[v][0], y = s_rank[v][1];
                hr += v < wave ? x : 0;
                fr += v < wave ? y : 0;
                hole0 += x;
                far0 += y;
            }
            __syncthreads();
            place(j, kept, hole, hr, fr, w, p);
        }
        holes_all = hole0;
    }
    if (tid == 0) moves[0] = holes_all;
    __builtin_amdgcn_s_waitcnt(0);
    __threadfence_block();
    __syncthreads();
    for (int i = tid; i < holes_all; i += NT) {
        const int to = moves[1 + i], from = moves[1 + m + i];
        acc_out[to] = acc[from];
        pos_out[to] = pos[from];
    }
    if (a.move_here) move_rows(a, b, hk, moves, holes_all, tid, NT);
    __builtin_amdgcn_s_waitcnt(0);             // (acc_out may be acc: read before it is cleared)
    __syncthreads();
    for (int j = m + tid; j < cap; j += NT) {
        acc_out[j] = 0.f;
        pos_out[j] = -1;
    }
}

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    const int bh = blockIdx.y, b = bh / a.hkv, hk = bh % a.hkv;
    const int32_t *moves = a.moves + (int64_t)bh * (1 + 2 * a.budget);
    if (hk == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.len_out[b] = new_length(a, b);
    move_rows(a, b, hk, moves, moves[0], (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

bool rows_ok(const void *p, const int64_t *st, int64_t bytes) {
    return aligned16(p) && bytes > 0 && bytes % 16 == 0 && st[0] % 16 == 0 && st[1] % 16 == 0 && st[2] % 16 == 0 &&
           st[2] >= bytes && st[0] >= 0 && st[1] >= 0;
}

}  // namespace

}  // namespace kuiops

using namespace kuiops;

extern "C" int kuiops_tree_accept(int64_t n, int64_t t, const int64_t *tokens, const int32_t *parent, const int64_t *target,
                                  int32_t *path, int32_t *count, int64_t *next, void *stream) {
    if (n < 0 || t <= 0) return KUIOPS_E_INVALID;
    if (n == 0) return KUIOPS_OK;
    if (!tokens || !parent || !target || !path || !count || !next) return KUIOPS_E_INVALID;
    if (t > kMaxTree || n >= ((int64_t)1 << 26)) return KUIOPS_E_UNSUPPORTED;
    hipLaunchKernelGGL(tree_accept_kernel, dim3((unsigned)n), dim3(64), 0, as_stream(stream), (int)t, tokens, parent, target,
                       path, count, next);
    return launch_status();
}

extern "C" int kuiops_kv_tree_commit(int64_t batch, int64_t n, int64_t hkv, int64_t cap, int64_t krow, int64_t vrow,
                                     void *K, const int64_t sk[3], void *V, const int64_t sv[3], int64_t p,
                                     const int32_t *path, int64_t t, const int32_t *kv_len, int32_t *len_out, void *stream) {
    if (batch < 0 || n < 0 || hkv < 0 || cap < 0 || p < 0 || t <= 0 || !sk || !sv) return KUIOPS_E_INVALID;
    if (n == 0 || batch == 0) return batch == n ? KUIOPS_OK : KUIOPS_E_INVALID;
    if (batch % n || hkv == 0 || (p > 0 && !path) || !kv_len || !len_out || len_out == kv_len) return KUIOPS_E_INVALID;
    if (cap > 0 && (!K || !V || K == V)) return KUIOPS_E_INVALID;
    if (p > t) return KUIOPS_E_INVALID;
    if (p > kMaxTree || batch > 65535 || hkv > 65535 || cap >= ((int64_t)1 << 31)) return KUIOPS_E_UNSUPPORTED;
    if (!rows_ok(K, sk, krow) || !rows_ok(V, sv, vrow) || krow > (1 << 20) || vrow > (1 << 20)) return KUIOPS_E_UNSUPPORTED;
    CommitArgs a{};
    a.n = (int)n; a.p = (int)p; a.t = (int)std::min<int64_t>(t, INT32_MAX); a.cap = cap;
    a.K = reinterpret_cast<char *>(K); a.V = reinterpret_cast<char *>(V);
    a.sk0 = sk[0]; a.sk1 = sk[1]; a.sk2 = sk[2];
    a.sv0 = sv[0]; a.sv1 = sv[1]; a.sv2 = sv[2];
    a.kcols = (int)(krow / 16); a.vcols = (int)(vrow / 16); a.kblocks = (int)cdiv(a.kcols, 32);
    a.blocks = a.kblocks + (int)cdiv(a.vcols, 32);
    a.hkv = (int)hkv;
    a.units = batch * hkv * a.blocks;
    a.path = path; a.kv_len = kv_len; a.len_out = len_out;
    if (cdiv(a.units, kCommitWaves) >= ((int64_t)1 << 24)) return KUIOPS_E_UNSUPPORTED;
    hipLaunchKernelGGL(tree_commit_kernel, dim3((unsigned)cdiv(a.units, kCommitWaves)), dim3(kCommitWaves * 64), 0,
                       as_stream(stream), a);
    return launch_status();
}

extern "C" size_t kuiops_kv_evict_workspace(int64_t n, int64_t hkv, int64_t budget) {
    if (n <= 0 || hkv <= 0 || budget <= 0) return 0;
    return (size_t)n * hkv * (1 + 2 * budget) * sizeof(int32_t);
}

extern "C" int kuiops_kv_evict(int64_t n, int64_t hkv, int64_t cap, int64_t krow, int64_t vrow, void *K, const int64_t sk[3],
                               void *V, const int64_t sv[3], const float *acc, const int64_t sa[2], const int32_t *pos,
                               const int64_t sp[2], const int32_t *kv_len, int64_t budget, int64_t recent, float *acc_out,
                               const int64_t sao[2], int32_t *pos_out, const int64_t spo[2], int32_t *len_out,
                               void *workspace, size_t workspace_bytes, void *stream) {
    if (n < 0 || hkv < 0 || cap < 0 || budget <= 0 || recent < 0 || recent > budget || !sk || !sv || !sa || !sp || !sao || !spo)
        return KUIOPS_E_INVALID;
    if (n == 0) return KUIOPS_OK;
    if (hkv == 0 || !kv_len || !len_out) return KUIOPS_E_INVALID;
    if (cap > 0 && (!K || !V || !acc || !pos || !acc_out || !pos_out)) return KUIOPS_E_INVALID;
    if (n * hkv > 65535 || cap >= ((int64_t)1 << 30)) return KUIOPS_E_UNSUPPORTED;
    if (!rows_ok(K, sk, krow) || !rows_ok(V, sv, vrow) || krow > (1 << 20) || vrow > (1 << 20)) return KUIOPS_E_UNSUPPORTED;
    // (a budget past the capacity never evicts)
    budget = std::min(budget, std::max<int64_t>(cap, 1));
    recent = std::min(recent, budget);
    if (!workspace || workspace_bytes < kuiops_kv_evict_workspace(n, hkv, budget) || (reinterpret_cast<uintptr_t>(workspace) & 3))
        return KUIOPS_E_WORKSPACE;
    EvictArgs a{};
    a.n = (int)n; a.hkv = (int)hkv; a.budget = (int)budget; a.recent = (int)recent; a.cap = cap;
    a.kv_len = kv_len; a.len_out = len_out; a.acc = acc; a.pos = pos; a.acc_out = acc_out; a.pos_out = pos_out;
    a.sa0 = sa[0]; a.sa1 = sa[1]; a.sp0 = sp[0]; a.sp1 = sp[1];
    a.sao0 = sao[0]; a.sao1 = sao[1]; a.spo0 = spo[0]; a.spo1 = spo[1];
    a.moves = reinterpret_cast<int32_t *>(workspace);
    a.K = reinterpret_cast<char *>(K); a.V = reinterpret_cast<char *>(V);
    a.sk0 = sk[0]; a.sk1 = sk[1]; a.sk2 = sk[2];
    a.sv0 = sv[0]; a.sv1 = sv[1]; a.sv2 = sv[2];
    a.kcols = (int)(krow / 16); a.vcols = (int)(vrow / 16);
    const int64_t most = std::max<int64_t>(0, std::min(budget, cap - budget)) * (a.kcols + a.vcols);
    // Few rows to move: the selecting work-group moves them itself, one launch less
    // (us, two launches / one, graph replays: 8 heads of 64, 512 of 576 keys 9.4 / 7.6, 1792 of 2048
    // 10.9 / 10.2, 1024 of 2048 11.2 / 12.7; 64 heads of 128, 512 of 640 10.3 / 9.2, 512 of 1024 13.0 /
    // 15.2).  Not where len_out is kv_len: a head's work-group that starts late would read
    // the new length of its sequence, so that one needs the second launch.
    a.move_here = len_out != kv_len && most <= 4 * kEvictThreads;
    const int64_t per = std::max<int64_t>(1, cdiv(2048, n * hkv));
    const dim3 grid((unsigned)std::max<int64_t>(1, std::min(per, cdiv(most, 256))), (unsigned)(n * hkv));
    const dim3 heads((unsigned)(n * hkv)), threads(kEvictThreads);
    // (slots of registers as the capacity needs: 8000 slots, 16 against 8 per thread 16.1 / 13.3 us;
    // 2000, 4 against 2 10.9 / 10.0, the same slots over and over; the device lengths may be
    // far below the capacity, which the host cannot see)
    if (cap <= kEvictThreads) hipLaunchKernelGGL((evict_select_kernel<1>), heads, threads, 0, as_stream(stream), a);
    else if (cap <= 2 * kEvictThreads) hipLaunchKernelGGL((evict_select_kernel<2>), heads, threads, 0, as_stream(stream), a);
    else if (cap <= 4 * kEvictThreads) hipLaunchKernelGGL((evict_select_kernel<4>), heads, threads, 0, as_stream(stream), a);
    else if (cap <= 8 * kEvictThreads) hipLaunchKernelGGL((evict_select_kernel<8>), heads, threads, 0, as_stream(stream), a);
    else if (cap <= 16 * kEvictThreads) hipLaunchKernelGGL((evict_select_kernel<16>), heads, threads, 0, as_stream(stream), a);
    else hipLaunchKernelGGL((evict_select_kernel<0>), heads, threads, 0, as_stream(stream), a);
    if (!a.move_here) hipLaunchKernelGGL(evict_move_kernel, grid, dim3(256), 0, as_stream(stream), a);
    return launch_status();
}
