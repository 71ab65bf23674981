// Attention of the newest tokens over a paged KV cache, gfx950.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i)  over the slots j <= L - l + i
//
// of the sequence's L = kv_len[b] ones, as far as its table goes; slot j is row j % page of page
// table[b][j / page].  8-bit pages: k_j = ks_j * K_j and v_j = vs_j * V_j with a scale
// per row.  Rows of the query heads that share a KV head are one list (row = head in
// group * l + position), so K and V are read once for all of them.
#include <algorithm>
#include <type_traits>

#include "paged.hpp"
#include "prob_parts.hpp"

namespace kuiops {

namespace {

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// (the same in all lanes, said so: a size that came out of a vector minimum puts a loop over
// the lanes' descriptors around every load)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void *base, uint32_t bytes) {
    const uint64_t p = reinterpret_cast<uint64_t>(base);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p), hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>((uint64_t)hi << 32 | lo), (short)0,
                                             __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

constexpr float kLn2 = 0.69314718055994530942f, kLog2e = 1.44269504088896340736f;
constexpr uint32_t kOut = 0x80000000u;        // an offset past every descriptor
constexpr int kCounterStride = 16;            // words: a cache line's atomics serialise
constexpr int kTile = 32;                     // slots that a wave takes at once
constexpr int kSwitch = 12, kLeast = 16;      // tiles that going on to another unit takes the time of; of a work-group, at least
constexpr int kWhole = 12, kPiece = 4;        // tiles that are not worth a merge; of a piece, at least
// tiles of a work-group from which on the work is spread evenly; with two units a work-group and more
constexpr int kEven = 16, kEvenMany = 64;

struct PagedArgs {
    PagedCache c;
    int n, hq, l, groups, row_groups;      // groups: work-groups that share the keys evenly
    int launched, G;           // query heads of a KV head
    float share;               // 1 / groups, a little more
    int may_part;              // there are work-groups enough for a piece each
    const void *Q;
    void *O;
    int64_t sq0, sq1, sq2, so0, so1, so2;
    float *lse;                // [n][hq][l], or null
    float scale_log2;          // softmax scale * log2(e), > 0
    const int32_t *kv_len;
    // per work-group a counter that is zero between calls, and for two pieces 16 rows of
    // (maximum in the log2 domain, sum) and of the unnormalised output
    unsigned *counters;
    float *ws_ml, *ws_o;
};

enum PageKind { kSame = 0, kInt8 = 1, kE4M3 = 2 };

// Probabilities as sums of 16-bit parts (Parts): with the few rows of this kernel the K / V
// stream takes the time, not the MFMAs.

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
// Bytes 0, 1 (H = 0) or 2, 3 (H = 1) of w as two bf16 (e4m3: one conversion; two and a
// permute took 77.2 us where this takes 75.0).
template <int PK, int H>
__device__ __forceinline__ uint32_t pair_of(uint32_t w) {
    if constexpr (PK == kE4M3) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, H));
    else return upper_halves(byte_value<PK, 2 * H>(w), byte_value<PK, 2 * H + 1>(w));
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
// AUX: the cache policy, 2 for non-temporal
template <int W, int AUX = 0>
__device__ __forceinline__ typename Words<W>::type load_words(__amdgpu_buffer_rsrc_t r, uint32_t voff) {
    if constexpr (W == 1) return __builtin_amdgcn_raw_buffer_load_b32(r, (int)voff, 0, AUX);
    else if constexpr (W == 2) return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)voff, 0, AUX));
    else return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, 0, AUX));
}
__device__ __forceinline__ uint32_t word(uint32_t v, int) { return v; }
template <typename V> __device__ __forceinline__ uint32_t word(const V &v, int i) { return v[i]; }

// The schedule.  A unit is one sequence's KV head; its slots are tiles of 32.
//   Short caches (`apart`): a work-group has one piece of a unit, the pieces of a unit all of
//   about the same size and a short unit one piece.
//   Long ones: the tiles of all units stand in one list, sequence after sequence, of which a
//   work-group has `per` adjacent places, so the work is even whatever the sequences' lengths;
//   it goes through pieces of one or more units.
// A unit that lies in one work-group is finished there; the pieces of the others are merged
// by the last of its work-groups to arrive.
// Where they cross: a piece that follows another in its work-group costs 5 us (drained loads,
// the waves' merge, the unit's), uneven pieces up to their difference.  Pieces apart / even
// list, us, 8 KV heads of 128, with tiles a work-group if even: 8 sequences of 500 (3) 11.3 / 17.3,
// 5 of 3000 (11) 15.3 / 18.5, 8 of 2000 (12) 18.6 / 17.6, 64 of 600 (28) 25.4 / 31.8, 16 of 2000
// (23) 30.9 / 25.7, 8 of 6000 (35) 43.7 / 32.8, 16 of 4000 (47) 52.0 / 40.0, 64 of 2000 (94) 70.0 / 70.7,
// 32 of 8000 in int8 (141) 100 / 75.8.
struct Piece {
    int b, hk, L;              // the unit, and its sequence's length
    int t0, t1;                // its tiles
    int first, pieces, late;   // the unit's first work-group and number of pieces; `late`: the first
                               // piece is its work-group's last one, not its first
};

// Tiles of a sequence; an empty one has one too, whose rows see nothing.
__device__ __forceinline__ int paged_tiles(int len) { return max(1, (len + kTile - 1) / kTile); }
// The sum over this lane and those before it (lane moves within rows of 16, then the rows'
// last lanes to the rows behind)
template <int CTRL, int ROWS> __device__ __forceinline__ int from_before(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_prefix(int v) {
    v += from_before<0x111, 0xF>(v);
    v += from_before<0x112, 0xF>(v);
    v += from_before<0x114, 0xF>(v);
    v += from_before<0x118, 0xF>(v);
    v += from_before<0x142, 0xA>(v);
    v += from_before<0x143, 0xC>(v);
    return v;
}
// The arguments, read again where they are used: held in scalar registers over the loop they
// would be spilled into vector lanes.
template <typename A> __device__ __forceinline__ const A &late_args() {
    typedef const A __attribute__((address_space(4))) *ptr;
    ptr p = (ptr)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const A *)p;
}

// ------------------------------------------------------------------------
// paged_attn_kernel -- up to 16 query rows of a KV head; the waves take a piece's tiles in
// turn.  Pages are multiples of 16 rows, so 16 slots lie in one page: every load has its
// page's address in scalar registers, and a buffer descriptor that ends with the last row
// that is there, so rows behind it and absent pages read as zeros and nothing is read
// there.  The pages' numbers of 32 turns are fetched at once, a lane each.
//   S = K Q^T (16x16x32 MFMA): K straight to registers, 16 bytes a lane; a lane then holds
//   8 scores of one row, keys 16 t + 4 G + i (G = lane / 16): the row's maximum crosses
//   lanes 16 and 32 apart only.
//   O^T += V^T P^T: the scores' registers are the second operand as they stand.  The first
//   wants 8 keys of a column in a lane: a lane loads HD / 16 adjacent columns of its 8 keys
//   (16 lanes a whole row) and transposes them in registers, so neither product needs LDS.
// A part that is 0 times an infinite value is NaN, so is a masked NaN: a wave whose sums
// are not finite goes over its keys again with the row maxima that it found, value by value
// for the rows that see them.
// What bounds it: the K / V stream (a plain read of as much reaches 5.4 to 6.1 TB/s with the
// launch) and what lies around it: arguments, lengths, page numbers and first keys one after
// another 3 us, the waves' merge 0.9, pieces stored, counted and merged 2.  Kernel alone: 16
// sequences of 2111 to 4000 keys, 32 / 8 heads of 128, bf16 40 us, 5.1 TB/s; 32 of 4085 to
// 8000 in e4m3 75 us, 5.5 TB/s; 60001 keys of one sequence in int8 31 us, 4.1 TB/s; 600 keys of
// one sequence, heads of 64: 8.7 us.  Two tiles in flight a wave took longer, with 214 instead of
// 256 registers, in an earlier form of the loop and in bf16 (16 sequences 45.8 against 44.2 then;
// not tried in 8 bits); so did 8 waves.
template <typename T, int PK, int HD, int NWV, int AUX>
__global__ __launch_bounds__(64 * NWV, 2) void paged_attn_kernel(PagedArgs a) {
    typedef typename std::conditional<PK == kSame, T, bf16_t>::type C;       // the products' type
    typedef typename Mfma<C>::frag frag;
    typedef C c8 __attribute__((ext_vector_type(8)));
    constexpr int KB = kTile, R = 16, NT = 64 * NWV, NP = Parts<C>::N;
    constexpr int B = PK == kSame ? 2 : 1;            // bytes of a cached value
    constexpr int KK = HD / 32, KL = HD * B / 64;     // MFMAs over a key, loads of 16 keys
    constexpr int DT = HD / 16, VW = DT * B / 4;      // columns of V a lane has, in dwords
    constexpr int NQ = PK != kSame && sizeof(T) == 2 && !std::is_same<T, bf16_t>::value ? 2 : 1;
    typedef typename Words<VW>::type vwords;
    constexpr int LD = HD + 4;                        // row stride of the waves' sums in LDS
    __shared__ __attribute__((aligned(16))) float so[NWV][R][LD];
    __shared__ float sm[NWV][R], sl[NWV][R];
    __shared__ int s_last;
    // (one word of each of the arguments' lines: they arrive together, not one after another)
    asm volatile("" ::"s"(a.c.K), "s"(a.c.sv0), "s"(a.c.pages), "s"(a.Q), "s"(a.so1), "s"(a.ws_o));
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, G4 = lane >> 4;

    // the row groups of a work-group's keys run on one XCD, whose L2 then has them for all but
    // the first
    // (what would be divided by 1 mostly is not: 40 instructions one after another)
    const int idx = blockIdx.x >> 3, of = a.row_groups == 1 ? idx : idx / a.row_groups, rg = idx - of * a.row_groups;
    const int me = of * 8 + (blockIdx.x & 7);
    if (me >= a.launched) return;
    const int G = a.G, rows_kv = G * a.l, r0 = rg * R, nrows = min(R, rows_kv - r0);

    // Places in the list (`apart`: pieces) of a sequence's KV head.  A unit begins with kSwitch
    // places that no tile has.
    int per = 0, x0 = 0, before = 0, lens, all = 0;
    auto len_of = [&](int x) __attribute__((always_inline)) { return x < a.n ? paged_len(a.c, a.kv_len, x) : 0; };
    // a lane has the lengths of 64 sequences at a time
    for (x0 = 0; x0 < a.n; x0 += 64) {
        lens = len_of(x0 + lane);
        all += __builtin_amdgcn_readlane(wave_prefix(x0 + lane < a.n ? paged_tiles(lens) : 0), 63);
    }
    all *= a.c.hkv;
    const bool apart = a.may_part && all < (a.n * a.c.hkv < 2 * a.groups ? kEven : kEvenMany) * a.groups;
    if (!apart && me >= a.groups) return;
    // (more than a share of the places, by 2^-20 of it and one: the same in all work-groups)
    per = apart ? max(kPiece, (int)((float)all * a.share) + 1)
                : max(kSwitch + kLeast, (int)((float)(all + a.n * a.c.hkv * kSwitch) * a.share) + 1);
    int cur = apart ? me : me * per;
    auto weight = [&](int len) __attribute__((always_inline)) {
        const int t = paged_tiles(len);
        return !apart ? t + kSwitch : t <= kWhole ? 1 : (t + per - 1) / per;
    };
    const int stop = cur + per;                       // (past the last tile for the last work-group)
    Piece p;
    for (x0 = 0;; x0 += 64) {
        if (x0 >= a.n) return;                        // nothing for this work-group
        if (a.n > 64) lens = len_of(x0 + lane);
        const int here = x0 + lane < a.n ? weight(lens) : 0, upto = wave_prefix(here);
        const uint64_t past = __ballot((before + upto) * a.c.hkv > cur);
        if (past) {
            const int at = __builtin_ctzll(past);
            p.b = x0 + at;
            before += __builtin_amdgcn_readlane(upto - here, at);
            p.pieces = __builtin_amdgcn_readlane(here, at);
            p.L = __builtin_amdgcn_readlane(lens, at);
            break;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    // (in a unit of the sequence: its KV head, and the piece of an `apart` one)
    const int inside = cur - before * a.c.hkv;
    p.hk = p.pieces == 1 ? inside : inside / p.pieces;
    if (apart) {
        const int z = inside - p.hk * p.pieces, tiles = paged_tiles(p.L);
        const int each = p.pieces == 1 ? tiles : tiles / p.pieces, longer = tiles - each * p.pieces;      // the first ones have one more
        p.first = me - z;
        p.late = 0;
        p.t0 = z * each + min(z, longer);
        p.t1 = p.t0 + each + (z < longer ? 1 : 0);
    }
    // the tiles of u among the places cur .. stop - 1
    auto cut_out = [&](Piece &u) __attribute__((always_inline)) {
        const int tiles = paged_tiles(u.L), unit0 = before * a.c.hkv + u.hk * (tiles + kSwitch), tile0 = unit0 + kSwitch;
        u.t0 = max(cur - tile0, 0);
        u.t1 = min(tiles, stop - tile0);
        u.first = tile0 / per;
        u.pieces = (tile0 + tiles - 1) / per - u.first + 1;
        u.late = unit0 > u.first * per;
        cur = tile0 + u.t1;
    };
    if (!apart) cut_out(p);
    // the piece behind u, false if there is none
    auto next_piece = [&](Piece &u) __attribute__((always_inline)) {
        if (cur + kSwitch >= stop) return false;
        if (++u.hk == a.c.hkv) {
            before += paged_tiles(u.L) + kSwitch;
            u.hk = 0;
            if (++u.b == a.n) return false;
            if (u.b == x0 + 64) {
                x0 = u.b;
                lens = len_of(x0 + lane);
            }
            u.L = __builtin_amdgcn_readlane(lens, u.b - x0);
        }
        cut_out(u);
        return true;
    };

    // row r0 + lr of the KV head's list
    const int rr = r0 + lr;
    const bool row_ok = rr < rows_kv;
    const int h = !row_ok ? 0 : a.l == 1 ? rr : rr / a.l, pos = row_ok ? rr - h * a.l : 0;
    uint32_t offK[KL];
#pragma unroll
    for (int j = 0; j < KL; ++j) {
        const int d = (j * 64 + G4 * 16) / B;
        offK[j] = d < a.c.hd ? (uint32_t)((lr * a.c.sk2 + d) * B) : kOut;
    }
    uint32_t offV[4];                                 // rows 4 G4 + i of 16
#pragma unroll
    for (int i = 0; i < 4; ++i) offV[i] = lr * DT < a.c.hd ? (uint32_t)(((4 * G4 + i) * a.c.sv2 + lr * DT) * B) : kOut;

    const uint32_t rowK = (uint32_t)a.c.sk2 * B, rowV = (uint32_t)a.c.sv2 * B;        // (below 2^25)
    constexpr int D4 = HD / 4;

    // Where the 16-slot groups of 32 turns lie, a lane each: the rows that are there, the
    // addresses of the first one's key, value and scales.  The next 32 turns' page numbers
    // are on their way meanwhile.
    auto group_key = [&](const Piece &u, int turn, int g) __attribute__((always_inline)) { return (u.t0 + turn * NWV + wave) * KB + 16 * g; };
    int turn0 = 0;
    struct Entries {
        int entry, row;
    } soon;
    auto fetch = [&](const Piece &u, int from) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rs_t = make_rsrc(a.c.table + u.b * a.c.ld_table, a.c.width * 4);
        const int key = group_key(u, from + (lane >> 1), lane & 1);
        Entries x;
        const int at = paged_entry(key, a.c.page, a.c.div, x.row);
        // (an entry behind the piece is out of the descriptor's reach: nothing is fetched)
        x.entry = __builtin_amdgcn_raw_buffer_load_b32(rs_t, key < min(u.L, u.t1 * KB) ? at * 4 : (int)kOut, 0, 0);
        return x;
    };
    u32x4 qr[KK];
    auto load_q = [&](const Piece &u) __attribute__((always_inline)) {
        const T *q = reinterpret_cast<const T *>(a.Q) + u.b * a.sq0 + (u.hk * G + h) * a.sq1 + pos * a.sq2;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            // (columns in the order of K's loads: 8-bit ones bring 16 columns, for two MFMAs)
            const int d = B == 2 ? kk * 32 + G4 * 8 : (kk >> 1) * 64 + G4 * 16 + (kk & 1) * 8;
            qr[kk] = row_ok && d < a.c.hd ? *reinterpret_cast<const u32x4 *>(q + d) : u32x4{0, 0, 0, 0};
        }
    };
    struct Groups {
        int n;
        uint64_t k, v, ks, vs;
    } now;
    auto locate = [&](const Piece &u, const Entries &x) __attribute__((always_inline)) {
        const int key = group_key(u, turn0 + (lane >> 1), lane & 1), id = paged_id(x.entry, a.c.pages);
        const int64_t page = max(id, 0);
        now.n = paged_rows16(id, key, min(u.L, u.t1 * KB));
        now.k = reinterpret_cast<uint64_t>(a.c.K) + (page * a.c.sk0 + u.hk * a.c.sk1 + x.row * a.c.sk2) * B;
        now.v = reinterpret_cast<uint64_t>(a.c.V) + (page * a.c.sv0 + u.hk * a.c.sv1 + x.row * a.c.sv2) * B;
        if constexpr (PK != kSame) {
            now.ks = reinterpret_cast<uint64_t>(a.c.ks + page * a.c.sks0 + u.hk * a.c.sks1 + x.row);
            now.vs = reinterpret_cast<uint64_t>(a.c.vs + page * a.c.svs0 + u.hk * a.c.svs1 + x.row);
        }
        soon = fetch(u, turn0 + 32);
    };
    auto address = [&](uint64_t x, int from) __attribute__((always_inline)) {
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, from), hi = __builtin_amdgcn_readlane((uint32_t)(x >> 32), from);
        return reinterpret_cast<const char *>((uint64_t)hi << 32 | lo);
    };

    // One tile of keys and of values: a tile's registers are loaded again as soon as its
    // product has read them.
    u32x4 kr[2][KL];
    vwords vr[8];
    f32x4 ks[2], vs[2];
    int there[2];                                     // rows of the two groups that are there
    auto issue_k = [&](int turn) __attribute__((always_inline)) {
        if (turn >= turn0 + 32) {
            turn0 += 32;
            locate(p, soon);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int from = 2 * (turn - turn0) + t;
            const int m = there[t] = __builtin_amdgcn_readlane(now.n, from);
            const __amdgpu_buffer_rsrc_t rk = make_rsrc(address(now.k, from), m ? (m - 1) * rowK + a.c.hd * B : 0u);
#pragma unroll
            for (int j = 0; j < KL; ++j) kr[t][j] = load_words<4, AUX>(rk, offK[j]);
            if constexpr (PK != kSame)
                ks[t] = __builtin_bit_cast(f32x4, load_words<4>(make_rsrc(address(now.ks, from), m * 4), G4 * 16));
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // (behind issue_k of the same turn)
    auto issue_v = [&](int turn) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int from = 2 * (turn - turn0) + t, m = there[t];
            const __amdgpu_buffer_rsrc_t rv = make_rsrc(address(now.v, from), m ? (m - 1) * rowV + a.c.hd * B : 0u);
            if constexpr (PK != kSame)
                vs[t] = __builtin_bit_cast(f32x4, load_words<4>(make_rsrc(address(now.vs, from), m * 4), G4 * 16));
#pragma unroll
            for (int j = 0; j < 4; ++j) vr[4 * t + j] = load_words<VW, AUX>(rv, offV[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    {
        const Entries x = fetch(p, 0);
        load_q(p);
        locate(p, x);
        issue_k(0);
        issue_v(0);
    }
    for (;;) {
    Piece then = p;
    const bool more = !apart && next_piece(then);
    Entries later{};
    if (more) later = fetch(then, 0);
    // (a length may pass its table's end.  Read here, where keys are waited for: 600 slots 8.6 us, as
    // without it; with the lengths above 8.8)
    const int told = max(a.kv_len[p.b], p.L);
    const int free_end = told - a.l + 1;              // slots below are seen by every row
    const int last = told - a.l + pos;                // the row's last slot
    const int mine = (p.t1 - p.t0 - wave + NWV - 1) / NWV;  // turns of this wave
    frag qf[NQ][KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        if constexpr (NQ == 1) qf[0][kk] = as_frag<frag>(qr[kk]);
        else {
            // f16 as two bf16: 8 bits and the 3 behind them
            typedef T t8 __attribute__((ext_vector_type(8)));
            const t8 v = __builtin_bit_cast(t8, qr[kk]);
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

    // scores of a turn, scales of K in them: (t, i) is slot k0 + 16 t + 4 G4 + i; unseen ones -inf
    auto scores = [&](int turn, f32x4 *sc) __attribute__((always_inline)) {
        const int k0 = group_key(p, turn, 0);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                u32x4 kw;
                if constexpr (PK == kSame) kw = kr[t][kk];
                else {
                    const uint32_t w0 = kr[t][kk >> 1][2 * (kk & 1)], w1 = kr[t][kk >> 1][2 * (kk & 1) + 1];
                    kw = u32x4{pair_of<PK, 0>(w0), pair_of<PK, 1>(w0), pair_of<PK, 0>(w1), pair_of<PK, 1>(w1)};
                }
#pragma unroll
                for (int y = 0; y < NQ; ++y) sc[t] = Mfma<C>::m16(as_frag<frag>(kw), qf[y][kk], sc[t]);
            }
            if constexpr (PK != kSame) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[t][i] *= ks[t][i];
            }
        }
        if (k0 + KB > free_end || there[0] + there[1] < KB) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * G4 + i >= there[t] || k0 + 16 * t + 4 * G4 + i > last) sc[t][i] = -INFINITY;
        }
    };

    f32x4 o[DT];                                      // o[c][i]: column (4 G4 + i) * DT + c of row lr
    float m_used = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int c = 0; c < DT; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int turn = 0; turn < mine; ++turn) {
        f32x4 sc[2];
        scores(turn, sc);
        __builtin_amdgcn_sched_barrier(0);
        issue_k(turn + 1);
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
                float w = fast_exp2(__builtin_fmaf(sc[t][i], a.scale_log2, -mref));
                l_run += w;
                if constexpr (PK != kSame) w *= vs[t][i];
                C x[NP];
                Parts<C>::split(w, x);
#pragma unroll
                for (int y = 0; y < NP; ++y) part[y][4 * t + i] = x[y];
            }
#pragma unroll
        for (int c = 0; c < DT; ++c) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (PK == kSame) {
                    const uint32_t lo = word(vr[2 * e], c >> 1), hi = word(vr[2 * e + 1], c >> 1);
                    w[e] = c & 1 ? __builtin_amdgcn_perm(hi, lo, 0x07060302u) : __builtin_amdgcn_perm(hi, lo, 0x05040100u);
                } else {
                    const uint32_t a0 = word(vr[2 * e], c >> 2), a1 = word(vr[2 * e + 1], c >> 2);
                    if constexpr (PK == kInt8) {
                        switch (c & 3) {
                            case 0: w[e] = pair_across<PK, 0>(a0, a1); break;
                            case 1: w[e] = pair_across<PK, 1>(a0, a1); break;
                            case 2: w[e] = pair_across<PK, 2>(a0, a1); break;
                            default: w[e] = pair_across<PK, 3>(a0, a1); break;
                        }
                    } else {
                        // (columns c and c ^ 1 of a key in one conversion)
                        const uint32_t lo = c & 2 ? pair_of<PK, 1>(a0) : pair_of<PK, 0>(a0), hi = c & 2 ? pair_of<PK, 1>(a1) : pair_of<PK, 0>(a1);
                        w[e] = c & 1 ? __builtin_amdgcn_perm(hi, lo, 0x07060302u) : __builtin_amdgcn_perm(hi, lo, 0x05040100u);
                    }
                }
            }
#pragma unroll
            for (int y = 0; y < NP; ++y) o[c] = Mfma<C>::m16(as_frag<frag>(w), __builtin_bit_cast(frag, part[y]), o[c]);
        }
        __builtin_amdgcn_sched_barrier(0);
        issue_v(turn + 1);
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
        locate(p, fetch(p, 0));
        for (int turn = 0; turn < mine; ++turn) {
            issue_k(turn);
            issue_v(turn);
            f32x4 sc[2];
            scores(turn, sc);
            const int k0 = group_key(p, turn, 0);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                float w = fast_exp2(__builtin_fmaf(sc[x >> 2][x & 3], a.scale_log2, -mref));
                if constexpr (PK != kSame) w *= vs[x >> 2][x & 3];
                const int from = 2 * (turn - turn0) + (x >> 2);
                const char *vfirst = address(now.v, from);
                for (int g = 0; g < 4; ++g) {
                    const int at = 4 * g + (x & 3);
                    const float pk = __shfl(w, g * 16 + lr, 64);
                    if (at >= there[x >> 2] || !row_ok || k0 + 16 * (x >> 2) + at > last) continue;
                    const char *vp = vfirst + at * rowV;
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

    // the next piece's query, addresses and (behind the stores below) first keys are on their
    // way while this one is finished
    const Piece u = p;
    if (more) {
        p = then;
        turn0 = 0;
        load_q(p);
        locate(p, later);
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

    const PagedArgs &e = late_args<PagedArgs>();
    auto store_row = [&](int r, int d, f32x4 v, float m, float ls) __attribute__((always_inline)) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        const int hr = e.l == 1 ? r0 + r : (r0 + r) / e.l, head = u.hk * G + hr, i = r0 + r - hr * e.l;
        const float inv = ls != 0.f ? 1.f / ls : 0.f;
        if (d < e.c.hd) {
            t4 w;
#pragma unroll
            for (int y = 0; y < 4; ++y) w[y] = from_f32<T>(v[y] * inv);
            *reinterpret_cast<t4 *>(reinterpret_cast<T *>(e.O) + u.b * e.so0 + head * e.so1 + i * e.so2 + d) = w;
        }
        if (e.lse && d == 0) e.lse[((int64_t)u.b * e.hq + head) * e.l + i] = ls != 0.f ? (m + __log2f(ls)) * kLn2 : -INFINITY;
    };

    // Pieces of a unit that several work-groups have: their states, agent-coherent (sc1), are
    // written through the XCD's L2 and read past it, as the work-group that merges them may
    // run on another XCD.  A work-group has two such pieces at most, its first and its last.
    const bool alone = u.pieces == 1;
    const __amdgpu_buffer_rsrc_t rs_o = make_rsrc(alone ? nullptr : e.ws_o, alone ? 0u : 0x7fffffffu);
    const __amdgpu_buffer_rsrc_t rs_ml = make_rsrc(alone ? nullptr : e.ws_ml, alone ? 0u : 0x7fffffffu);
    // the rows of piece z: its owner's first piece, unless the unit begins behind the owner's first tile
    auto state = [&](int z) __attribute__((always_inline)) {
        return (((u.first + z) * e.row_groups + rg) * 2 + (z == 0 ? u.late : 0)) * R;
    };
    for (int x = tid; x < nrows * D4; x += NT) {
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
        const int at = state(me - u.first) + r;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, oo), rs_o, (at * HD + d) * 4, 0, kSc1Aux);
        if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{mm, ll}), rs_ml, at * 8, 0, kSc1Aux);
    }
    if (!alone) {
        // Every thread waits for its stores' acknowledgements before the barrier that precedes
        // the counter's agent-scope addition.
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0);
    }
    if (more) {
        issue_k(0);
        issue_v(0);
    }
    if (!alone) {
        __syncthreads();
        unsigned *ctr = e.counters + (int64_t)(u.first * e.row_groups + rg) * kCounterStride;
        if (tid == 0) s_last = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(u.pieces - 1);
        __syncthreads();
        if (s_last) {
            // Merged in the pieces' order, the same bits whatever the order of arrival.  A thread
            // has 4 columns of a row; threads to spare share the pieces and join through LDS.
            const int items = nrows * D4, share = max(1, min(NT / items, u.pieces / 2));
            for (int x0 = 0; x0 < items; x0 += NT) {
                const int zg = share > 1 ? tid / items : 0, x = x0 + tid - zg * items;
                const int r = x / D4, d = x % D4 * 4;
                const bool on = x < items && zg < share;
                float m = -INFINITY, ls = 0.f;
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                constexpr int Z = 8;
                for (int z0 = zg; on && z0 < u.pieces; z0 += Z * share) {
                    f32x4 ov[Z];
                    f32x2 ml[Z];
#pragma unroll
                    for (int z = 0; z < Z; ++z) {
                        // (pieces that are not there: past the end of the descriptor, no memory is read)
                        const int y = z0 + z * share, at = state(y) + r;
                        ov[z] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs_o, y < u.pieces ? (at * HD + d) * 4 : (int)kOut, 0, kSc1Aux));
                        ml[z] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rs_ml, y < u.pieces ? at * 8 : (int)kOut, 0, kSc1Aux));
                    }
                    float mx = m;
#pragma unroll
                    for (int z = 0; z < Z; ++z) {
                        if (z0 + z * share >= u.pieces) ml[z][0] = -INFINITY;
                        mx = fmaxf(mx, ml[z][0]);
                    }
                    const float mu = mx == -INFINITY ? 0.f : mx, keep = fast_exp2(m - mu);
                    ls *= keep;
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i] *= keep;
#pragma unroll
                    for (int z = 0; z < Z; ++z) {
                        const float w = fast_exp2(ml[z][0] - mu);
                        ls = __builtin_fmaf(w, ml[z][1], ls);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(w, ov[z][i], acc[i]);
                    }
                    m = mx;
                }
                if (share > 1) {
                    // (the waves' sums there were read before the counter's barrier)
                    float *slots = &so[0][0][0];
                    static_assert(sizeof(so) >= NT * 32, "8 words a thread");
                    *reinterpret_cast<f32x4 *>(slots + tid * 8) = acc;
                    *reinterpret_cast<f32x2 *>(slots + tid * 8 + 4) = f32x2{m, ls};
                    __syncthreads();
                    for (int g = 1; g < share && tid < items; ++g) {
                        const f32x4 ov = *reinterpret_cast<const f32x4 *>(slots + (tid + g * items) * 8);
                        const f32x2 ml = *reinterpret_cast<const f32x2 *>(slots + (tid + g * items) * 8 + 4);
                        const float mx = fmaxf(m, ml[0]), mu = mx == -INFINITY ? 0.f : mx;
                        const float w0 = fast_exp2(m - mu), w1 = fast_exp2(ml[0] - mu);
                        ls = ls * w0 + ml[1] * w1;
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * w0 + ov[i] * w1;
                        m = mx;
                    }
                }
                if (x < items && zg == 0) store_row(r, d, acc, m, ls);
            }
            if (tid == 0) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (!more) break;
    __syncthreads();
    }
}

// ------------------------------------------------------------- host side

struct PagedPlan {
    int row_groups, groups, may_part, launched;
    size_t counter_bytes, ml_bytes, o_bytes;
};

constexpr int kWaves = 4;
// work-groups that share the keys evenly (512, two a CU: 16 sequences of 4000 39.8 -> 42.7 us, 60001
// keys of one in int8 31.4 -> 34.4, 32 of 8000 in e4m3 75.1 -> 77.0), and units that have work-groups
// of their own
constexpr int kMaxGroups = 256;
// The counters' part of a workspace, the same for calls of all sizes
constexpr int kApart = 2048;
constexpr size_t kCounterBytes = (size_t)(kApart + kMaxGroups) * kCounterStride * 4;
static_assert(kCounterBytes == KUIOPS_SDPA_PAGED_ZEROED, "what callers clear");

PagedPlan plan_of(int64_t n, int64_t hq, int64_t hkv, int64_t l, int64_t slots, int64_t hd) {
    PagedPlan p{};
    p.row_groups = (int)cdiv(hq / hkv * l, 16);
    // no more work-groups than full tables have tiles for
    const int64_t tiles = n * hkv * std::max<int64_t>(1, cdiv(slots, kTile));
    p.groups = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxGroups / p.row_groups, tiles));
    p.may_part = n * hkv * p.row_groups <= kApart;
    p.launched = p.groups + (p.may_part ? (int)(n * hkv) : 0);
    // (a single work-group for the keys has every unit whole, as has one tile a unit)
    if (tiles > n * hkv && p.groups > 1) {
        const size_t states = (size_t)p.launched * p.row_groups * 2 * 16;
        p.counter_bytes = kCounterBytes;
        p.ml_bytes = states * 8;
        p.o_bytes = states * (hd <= 64 ? 64 : 128) * 4;
    }
    return p;
}

// Keys and values of pools (or full tables) of this many bytes pass by the caches
// (non-temporal loads); those of smaller ones may be found in the 256 MB of memory-side cache the
// next time: us without / with, 52 MB read 17.7 / 19.5, 119 MB 28.4 / 27.8, 145 MB 33.1 / 31.5, 204
// MB 43.2 / 39.9, 394 MB 74.6 / 66.9.  The lengths are not known here: short contexts whose tables
// could hold more (16 sequences, tables of 32768 slots over a pool of 2 GB) take 15.6 us instead of
// 14.6 for up to 600 slots, 21.6 instead of 19.5 for 1200, 25.8 instead of 25.7 for 2000.
constexpr int64_t kStreamBytes = 120 << 20;

template <typename T, int PK, int AUX>
void launch_paged(const PagedArgs &a, const PagedPlan &p, hipStream_t st) {
    const dim3 grid((unsigned)(cdiv(p.launched, 8) * 8 * p.row_groups));
    if (a.c.hd <= 64) hipLaunchKernelGGL((paged_attn_kernel<T, PK, 64, kWaves, AUX>), grid, dim3(64 * kWaves), 0, st, a);
    else hipLaunchKernelGGL((paged_attn_kernel<T, PK, 128, kWaves, AUX>), grid, dim3(64 * kWaves), 0, st, a);
}
template <typename T, int PK>
void launch_paged(const PagedArgs &a, const PagedPlan &p, hipStream_t st) {
    const int64_t rows = std::min<int64_t>(a.c.pages, (int64_t)a.n * a.c.width) * a.c.page * a.c.hkv;
    if (rows * a.c.hd * 2 * (PK == kSame ? 2 : 1) >= kStreamBytes) launch_paged<T, PK, 2>(a, p, st);
    else launch_paged<T, PK, 0>(a, p, st);
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
    // 32-bit indices of rows and tiles, launches below 2^32 threads
    const int64_t rows = hq / at->hkv * l, slots = at->width * at->page;
    if (l >= (1 << 24) || rows >= (1 << 24) || n * hq * l >= ((int64_t)1 << 31) ||
        n * at->hkv >= (1 << 20) || n * at->hkv * (slots / kTile + 1 + kSwitch) >= ((int64_t)1 << 30))
        return KUIOPS_E_UNSUPPORTED;
    const PagedPlan p = plan_of(n, hq, at->hkv, l, slots, at->hd);
    const size_t need = p.counter_bytes + p.ml_bytes + p.o_bytes;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KUIOPS_E_WORKSPACE;
    a.n = (int)n; a.hq = (int)hq; a.l = (int)l; a.groups = p.groups; a.may_part = p.may_part; a.launched = p.launched; a.G = (int)(hq / at->hkv); a.share = (1.f + 0x1p-20f) / (float)p.groups; a.row_groups = p.row_groups;
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
