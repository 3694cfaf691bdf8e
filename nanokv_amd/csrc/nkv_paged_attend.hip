// nkv_paged_attend.hip -- attention over the paged key/value cache
// (nkv_paged_attend): tokens, causal chunks, frames and trees of drafted tokens.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(z_j - m), z = softmax_scale log2(e)
// q.k, over the keys a query sees, with the running maximum m of a row at most TAU
// behind; l = sum p in fp32.  The scores' products are exact and added in fp32.
//
// What a query does not see does not reach its result, whatever it holds: a masked
// score becomes -inf before the softmax, and values that are not finite (which a zero
// weight would not remove) leave the product and are added apart to the rows that
// see them.
#include "nkv_paged.h"

#include <math.h>

#include <algorithm>
#include <utility>

namespace nkv {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float TAU = 3.0f;           // a row's maximum is moved when it is off by 2^TAU

// The 16-bit types as weights and values.  LIFT: fp16 weights are held 2^12 higher
// (2^(12 + TAU) < 65504), so that they keep all 11 bits down to 2^-26 of the row's
// largest.
template <typename T>
struct Value;
template <>
struct Value<Bf16> {
    static constexpr float LIFT = 0.0f;
    static constexpr uint32_t EXP = 0x7f807f80u, STEP = 0x00800080u, FRAC = 0x007fu;
    static constexpr uint32_t ONE = 0x3f80u, N128 = 0x4300u, N129 = 0x4301u;
};
template <>
struct Value<Fp16> {
    static constexpr float LIFT = 12.0f;
    static constexpr uint32_t EXP = 0x7c007c00u, STEP = 0x04000400u, FRAC = 0x03ffu;
    static constexpr uint32_t ONE = 0x3c00u, N128 = 0x5800u, N129 = 0x5808u;
};

// The high bit of each half of a word that is not finite.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & Value<T>::EXP) + Value<T>::STEP) & 0x80008000u;
}

// A word's two values in two parts: the finite ones (0 in place of the others), and
// what the others are, as numbers whose sums tell them apart: +inf 1, -inf 128, NaN
// 129 (exact in either type).
struct Parts {
    uint32_t finite, kind;
};
template <typename T>
__device__ __forceinline__ Parts part_word(uint32_t w) {
    using V = Value<T>;
    const uint32_t bad = (not_finite<T>(w) >> 15) * 0xffffu;               // whole halves
    const uint32_t nan = (((w & V::FRAC * 0x10001u) + 0x7fff7fffu) >> 15) & 0x10001u;
    const uint32_t down = ((w >> 15) & 0x10001u) | nan;
    return {w & ~bad, (V::ONE * 0x10001u + down * (V::N128 - V::ONE) + nan * (V::N129 - V::N128)) & bad};
}
// What a sum of such numbers (up to 32 of them) adds to a result.
__device__ __forceinline__ float parted(float o, float sum) {
    const int n = (int)sum;
    return o + (n & 127 ? INFINITY : 0.0f) + (n >= 128 ? -INFINITY : 0.0f);
}

// Division by a number known on the host, of numbers below 2^31: with 2^(s - 1) < d <=
// 2^s and mul = floor(2^(31 + s) / d) + 1 the error e = mul d - 2^(31 + s) <= d <= 2^s,
// so that n e < 2^(31 + s) and the product's high bits are the quotient.
struct Divisor {
    uint32_t d, mul, shift;
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};
Divisor divisor(int64_t d) {
    int s = 0;
    while (((int64_t)1 << s) < d) ++s;
    return {(uint32_t)d, s ? (uint32_t)((((unsigned __int128)1 << (31 + s)) / d) + 1) : 0, s ? (uint32_t)s - 1 : 0};
}

typedef int i32x2 __attribute__((ext_vector_type(2)));

struct AttendParams {
    PageTable table;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* length;
    const int32_t* counts;
    const int32_t* parents;
    int64_t parents_sb;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    // partial results of the splits, [H][B * splits][rows]: the output's D sums (in units
    // of 2^(m - LIFT)), and (m, l)
    float* part;
    f32x2* part_ml;
    i32x2* shares;                // [B] a sequence's first slot and splits, or null: all alike
    int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;
    int64_t items;
    Divisor by_G, by_H, by_B, by_groups;
    float scale_log2;
    int B, H, G, D, Q, n, causal, splits, groups, rows;
    int page_d;
    int per_group;                // tile kernel: 32-row blocks of a group
};

// Query row r of key head hk is query t = r / G of query head hk * G + r % G.
struct RowAt {
    int t, head;
    bool there;
};
__device__ __forceinline__ RowAt row_at(const AttendParams& p, int row, int hk) {
    const bool there = row < p.rows;
    const int r = there ? row : 0, t = (int)p.by_G.of(r);
    return {t, hk * p.G + r - t * p.G, there};
}

// The queries of an item: `nq` of its Q rows, the last tokens of `len`.
struct Queries {
    int len, nq, causal, tree;
    // keys that query t < nq sees without a gap from the first on, and any row t
    __device__ __forceinline__ int sees(int t) const {
        return causal ? len - nq + 1 + t : tree ? len - nq : len;
    }
    __device__ __forceinline__ int end(int t) const { return t >= nq ? 0 : sees(t); }
    // the least that any of the queries t0 .. t1 sees so, and the end of all they see
    __device__ __forceinline__ int least(int t0, int t1) const { return t1 >= nq ? 0 : sees(t0); }
    __device__ __forceinline__ int most(int t0, int t1) const {
        return t0 >= nq ? 0 : tree ? len : sees(min(t1, nq - 1));
    }
};
// ---------------------------------------------------------------- trees
// For each of a workgroup's tokens one bit for every token of the draft that it sees:
// its own and those on the way to the root.
constexpr int TREE_WORDS = NKV_PAGED_TREE / 32;

template <int TOKENS>
struct TreeSmem {
    int32_t parents[NKV_PAGED_TREE];
    uint32_t bits[TOKENS][TREE_WORDS];
};

// A workgroup's thread's part of the parents (workgroups have at least as many threads
// as a tree tokens): loaded ahead of all else, and stored where it is needed.
static_assert(NKV_PAGED_TREE <= 256, "a thread for each token");
__device__ __forceinline__ int32_t tree_parent(const AttendParams& p, int b) {
    return p.parents && (int)threadIdx.x < p.Q ? p.parents[b * p.parents_sb + threadIdx.x] : -1;
}

// Tokens t0 .. t0 + count, by all threads of the workgroup.  A way goes to lower tokens
// only, so it ends.
template <int TOKENS>
__device__ __forceinline__ void tree_bits(TreeSmem<TOKENS>& sm, int32_t parent, int nq, int t0, int count) {
    if (threadIdx.x < NKV_PAGED_TREE) sm.parents[threadIdx.x] = parent;
    __syncthreads();
    if ((int)threadIdx.x < count) {
        uint32_t* bits = sm.bits[threadIdx.x];
#pragma unroll
        for (int w = 0; w < TREE_WORDS; ++w) bits[w] = 0;
        const int own = t0 + (int)threadIdx.x;
        for (int a = own < nq ? own : -1; a >= 0;) {
            const int up = sm.parents[a];
            bits[a >> 5] |= 1u << (a & 31);
            a = up < a ? up : -1;
        }
    }
    __syncthreads();
}

// 32 bits from bit `at` on, at > -32; bits below 0 are set (rows before the draft),
// bits past the last are not.
__device__ __forceinline__ uint32_t tree_word(const uint32_t* bits, int at) {
    if (at < 0) return (bits[0] << -at) | ((1u << -at) - 1);
    const int i = at >> 5;
    const uint32_t lo = i < TREE_WORDS ? bits[i] : 0, hi = i + 1 < TREE_WORDS ? bits[i + 1] : 0;
    return (uint32_t)((((uint64_t)hi << 32) | lo) >> (at & 31));
}

// The first n bits.
__device__ __forceinline__ uint32_t low_bits(int n) {
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
}

// ---------------------------------------------------------------- results
// A row's running maximum (log2 units, -inf before the first key) and sum.
struct Stat {
    float m, l;
};
constexpr float NONE = -INFINITY;

// 2^(m - M) of a part whose maximum is m (a part without keys has weight 0).
__device__ __forceinline__ float weight(float m, float M) {
    return m == NONE ? 0.0f : __builtin_amdgcn_exp2f(m - M);
}

// Eight columns of a row's result, o in units of 2^(m - LIFT).
template <typename T>
__device__ __forceinline__ void store_row(const AttendParams& p, int b, int hk, int row, int d,
                                          const Stat& st, const float (&o)[8]) {
    const RowAt at = row_at(p, row, hk);
    if (!at.there || d >= p.D) return;
    constexpr float DOWN = Value<T>::LIFT == 0.0f ? 1.0f : 1.0f / 4096.0f;
    const float f = st.l == 0.0f ? 0.0f : DOWN / st.l;
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = o[k] * f;
    *reinterpret_cast<u32x4*>(p.out + b * p.o_sb + at.t * p.o_st + at.head * p.o_sh + d) =
        u32x4{T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7])};
    if (d == 0 && p.lse)
        p.lse[((int64_t)b * p.H * p.G + at.head) * p.Q + at.t] =
            st.l == 0.0f ? -INFINITY : st.m * LN2 + logf(st.l);  // (NaN for a NaN query)
}
static_assert(Value<Fp16>::LIFT == 12.0f, "store_row's 4,096");

// The same as one split's partial result.
__device__ __forceinline__ void store_partial(const AttendParams& p, int hk, int slot, int row, int d,
                                              const Stat& st, const float (&o)[8]) {
    if (row >= p.rows || d >= p.D) return;
    const int64_t i = ((int64_t)hk * p.B * p.splits + slot) * p.rows + row;
    f32x4* to = reinterpret_cast<f32x4*>(p.part + i * p.D + d);
    to[0] = f32x4{o[0], o[1], o[2], o[3]};
    to[1] = f32x4{o[4], o[5], o[6], o[7]};
    if (d == 0) p.part_ml[i] = f32x2{st.m, st.l};
}

// ---------------------------------------------------------------- shares
// One of a sequence's key splits, which have the slots from `first` on of the B * splits
// that there are; and the sequence's length and queries.
struct Part {
    int b, split, splits, first;
    bool there;
    int len, nq;
};
__device__ __forceinline__ Queries queries_of(const AttendParams& p, const Part& part) {
    return {part.len, part.nq, p.causal, p.parents != nullptr};
}

// Sum over the wave.
__device__ __forceinline__ int wave_sum(int v) {
    uint32_t x = (uint32_t)v;
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = a[0] + a[1];
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = b[0] + b[1];
    x += (uint32_t)__builtin_amdgcn_mov_dpp(x, 0x128, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_mov_dpp(x, 0x141, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_mov_dpp(x, 0x4e, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_mov_dpp(x, 0xb1, 0xf, 0xf, true);
    return __builtin_amdgcn_readfirstlane((int)x);
}

// Where lengths are in device memory, sequences (up to a wave's lanes) share the slots by
// them: a split takes 128 tau keys for the least tau, two at least, with which all fit.  tau
// = sum / (slots - B) and one more always does, as a sequence of t takes at most t / tau + 1.
// Each wave finds this for itself, a sequence to a lane; the merge is told.  (Only where the
// plan has splits to share: calls of 512 workgroups and more have none, and those of more
// than 64 sequences equal ones, so that a long sequence sets the call's time: one of 131,072
// keys and the others of 4,096, 8 heads, 63 sequences 287 us, 64 1,235; 4 heads, 64 167, 65
// 642.)  us with equal
// splits and with these, 8 heads: 16 sequences, 256 rows, one of 32,768 keys and the others
// of 512 478, 87, lengths evenly up to 32,768 541, 395, all alike 663, 666; 32 sequences, 4
// rows, one of 16,384 keys, the others of 256 61, 36; 4 sequences of 4,096 17.3, 18.7.
// With more workgroups than CUs the splits stay equal unless the longest sequence's are
// half as long again: a CU that is done early takes the next (32 sequences, evenly from 6,144
// to 16,384 keys, 4 rows: 251, by length 278).
constexpr int BALANCED = 64, LEAST_SHARE = 2;
__device__ __forceinline__ Part part_of(const AttendParams& p, int slot) {
    const int split = (int)p.by_B.of((uint32_t)slot), own = slot - split * p.B;
    const Part equal{own, split, p.splits, own * p.splits, true, c8_length(p.length, own, p.n),
                     c8_length(p.counts, own, p.Q)};
    if (!p.shares) return equal;
    const int lane = threadIdx.x & 63, slots = p.B * p.splits;
    const bool in = lane < p.B;
    const int len = in ? c8_length(p.length, lane, p.n) : 0, nq = in ? c8_length(p.counts, lane, p.Q) : 0;
    const int t = nq > 0 ? (len + 127) >> 7 : 0, all = wave_sum(t);
    auto splits = [&](int tau) { return in ? max(1, (int)((uint32_t)(t + tau - 1) / (uint32_t)tau)) : 0; };
    int lo = max(LEAST_SHARE, (all + slots - 1) / slots), hi = max(lo, all / (slots - p.B) + 1);
    while (lo < hi) {
        const int tau = (lo + hi) >> 1;
        if (wave_sum(splits(tau)) <= slots) hi = tau;
        else lo = tau + 1;
    }
    const int longest = __builtin_amdgcn_readfirstlane((int)wave_umax((uint32_t)t));
    if (p.items > 256 && 2 * longest < 3 * hi * p.splits) return equal;
    const int mine = splits(hi);
    int end = mine;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        const int x = __shfl_up(end, i);
        end += lane >= i ? x : 0;
    }
    const int past = __popcll(__ballot(in && end <= slot)), b = min(past, p.B - 1);
    const int n = __builtin_amdgcn_readlane(mine, b), first = __builtin_amdgcn_readlane(end, b) - n;
    return {b, slot - first, n, first, past < p.B, __builtin_amdgcn_readlane(len, b),
            __builtin_amdgcn_readlane(nq, b)};
}
__device__ __forceinline__ void tell_merge(const AttendParams& p, const Part& part, int hk, int group) {
    if (p.shares && part.split == 0 && hk == 0 && group == 0 && threadIdx.x == 0)
        p.shares[part.b] = i32x2{part.first, part.splits};
}

// The work of a workgroup: a group of query rows of a unit (slot and head).
// Block i runs on XCD i % 8, and the groups of a unit take consecutive slots of one
// XCD, whose L2 then serves all but the first read of its rows.  Units go to the XCDs
// in turn, so that sequences of unlike lengths spread over them; of the last ones, fewer
// than eight, an XCD takes a run of (unit, group) pairs, so that none has more than its
// eighth (4 heads of 123,539 keys, 529 rows, 252 workgroups: with 33 on some XCDs' 32 CUs
// 340 us, with 32 186; 28 heads of 10,634, 1,292 rows, 504 workgroups 334, 237).
struct Item {
    uint32_t unit;
    int group;
    bool there;
};

// Part `split` of n tiles: an even share, the first ones a tile more.
__device__ __forceinline__ void share_of(const Part& part, int n, int& from, int& to) {
    const int each = (int)((uint32_t)n / (uint32_t)part.splits), more = n - each * part.splits;
    from = part.split * each + min(part.split, more);
    to = from + each + (part.split < more);
}

__device__ __forceinline__ Item item_of(const AttendParams& p) {
    const uint32_t x = blockIdx.x & 7, k = blockIdx.x >> 3, groups = (uint32_t)p.groups;
    const uint32_t units = p.by_groups.of((uint32_t)p.items), whole = units >> 3, u = p.by_groups.of(k);
    if (u < whole) return {u * 8 + x, (int)(k - u * groups), true};
    const uint32_t rest = (units & 7) * groups, each = (rest + 7) >> 3, j = k - whole * groups;
    const uint32_t item = x * each + j, v = p.by_groups.of(item);
    return {whole * 8 + v, (int)(item - v * groups), j < each && item < rest};
}

// ---------------------------------------------------------------- few rows
// W waves of a workgroup share NQ groups of 16 query rows and a range of 32-key tiles;
// each wave walks a run of tiles of its own, and the waves' results are merged in LDS.
// S^T = K Q^T on 16x16x32 MFMAs leaves lane (r, g) = (lane % 16, lane / 16) the scores of
// row r and keys 16 t + 4 g + e, whose weights are then the operand of O^T += V^T P^T
// without leaving the registers.  V's columns 8 r .. 8 r + 7 are a lane's (4 r .. of
// narrow heads), so its transposition is a choice of halves of eight rows' words, read
// straight from memory, whole rows to 16 lanes.  K's operand has a row to each of 16
// lanes: read from memory that is 64 accesses of the vector cache to a load (a CU then
// moves 58 GB/s of a context, eight waves 75 us for 8,192 keys of 8 heads without
// splits), so that K's rows pass through the wave's own LDS buffers (51 us).
// Long calls are bound by memory: two heads of 262,144 keys, 268 MB, 43 us, 6.2 TB/s
// beside a merge of 6; 32 ragged sequences up to 16,384, 1.47 GB, 251 us, 5.9 TB/s.
// Short ones by the start, the loads' latency and the exchange of the waves' rows: 8 heads
// of 4,096 keys, one or two tiles to each wave of 256 workgroups, 16, 32 and 64 rows 6.9, 8.5
// and 11.9 us (64 rows are eight waves' 135 KB through LDS), and a tree 0.3 to 0.8 more.
constexpr int TILE = 32;

// Page numbers of a run of tiles, 64 at a time, a lane each.
struct Pages {
    const int32_t* at;
    int w, first, ids;
    __device__ __forceinline__ void load(int entry) {
        first = entry;
        ids = w ? at[min(entry + (int)(threadIdx.x & 63), w - 1)] : -1;
        // (has arrived where the branch around this ends: a use behind it would wait for all loads)
        asm volatile("" : "+v"(ids));
    }
    // entry `entry` (uniform; never below that of the last call by more than it has)
    __device__ __forceinline__ uint32_t get(int entry) {
        if (entry >= w) return ~0u;
        if (entry - first >= 64) load(entry);
        return (uint32_t)__builtin_amdgcn_readlane(ids, entry - first);
    }
};

// One 16-byte-per-lane copy from 16 rows of a page (their bytes from `rows` on) into LDS,
// the 64 lanes' pieces one after the other, from `further` bytes on for all of them; a
// lane whose offset is NO_ROW brings zeros.  (By the buffer form: behind a global one every
// wait for a load becomes one for all loads.)
constexpr uint32_t NO_ROW = 1u << 30;
__device__ __forceinline__ void copy_rows(const uint16_t* rows, int bytes, uint32_t offset, int further,
                                          void* l) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(rows), 0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, NKV_LDS(l), 16, (int)offset, further, 0, 0);
}

template <int P>
struct KeyLds {
    static constexpr int PITCH = 2 * P, CH = PITCH / 16, ROWS = 1024 / PITCH;   // rows of a copy
    static constexpr int BUF = TILE * PITCH, COPIES = TILE / ROWS;
};

template <int P, int W, int NQ>
struct RowsSmem {
    union {
        unsigned char k[W][2][KeyLds<P>::BUF];
        float o[W][16 * NQ][P + 4];
    };
    TreeSmem<16 * NQ> tree;
    Stat st[W][16 * NQ];
};

template <int KS>
constexpr int width_of() { return KS == 2 ? 64 : 128; }

template <typename T, int KS, int W, int NQ>
__global__ void __launch_bounds__(64 * W) attend_kernel(AttendParams p) {
    constexpr int DB = KS == 2 ? 4 : 8, WORDS = DB / 2, ROWS = 16 * NQ, P = width_of<KS>();
    constexpr bool SPLIT = std::is_same_v<T, Bf16>;
    using x8 = typename T::x8;
    using V = Value<T>;
    using L = KeyLds<P>;
    extern __shared__ __align__(16) unsigned char rows_smem[];
    RowsSmem<P, W, NQ>& sm = *reinterpret_cast<RowsSmem<P, W, NQ>*>(rows_smem);
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Item it = item_of(p);
    if (!it.there) return;
    const int rg = it.group, at_slot = (int)p.by_H.of(it.unit), hk = (int)it.unit - at_slot * p.H;
    const Part part = part_of(p, at_slot);
    if (!part.there) return;
    tell_merge(p, part, hk, rg);
    const int b = part.b;
    const Queries qs = queries_of(p, part);
    const int32_t parent = tree_parent(p, b);
    const int row0 = rg * ROWS;
    // tiles that some row of the group sees, and keys that every row does
    const int t0 = (int)p.by_G.of(row0), t1 = (int)p.by_G.of(min(row0 + ROWS, p.rows) - 1);
    const int last = max(0, qs.most(t0, t1)), first = qs.least(t0, t1);
    const int nt = (last + TILE - 1) / TILE;
    int b0, b1;
    share_of(part, nt, b0, b1);
    x8 qf[NQ][KS];
    int end[NQ];                              // keys that the lane's row sees
    const uint32_t* bits[NQ];                 // and the draft's tokens
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const RowAt mine = row_at(p, row0 + 16 * n + r, hk);
        end[n] = mine.there ? qs.end(mine.t) : 0;
        bits[n] = sm.tree.bits[mine.there ? mine.t - t0 : 0];
        const uint16_t* q = p.q + b * p.q_sb + mine.t * p.q_st + mine.head * p.q_sh;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 32 * s + 8 * g;
            u32x4 w{};
            if (mine.there && d < p.D) w = *reinterpret_cast<const u32x4*>(q + d);
            qf[n][s] = as_x8<x8>(w);
        }
    }
    // this wave's tiles
    const int w0 = b0 + (int)((uint32_t)(wave * (b1 - b0)) / W);
    const int w1 = b0 + (int)((uint32_t)((wave + 1) * (b1 - b0)) / W);
    const int shift = p.table.shift, page_rows = 1 << shift;
    Pages pages{p.table.at + b * p.table.sb, (int)p.table.w, 0, 0};
    // lane offsets into a page's rows of the head (elements): V's rows, and K's in the copies:
    // row lr of each, whose 16-byte slot `slot` holds chunk slot ^ row
    uint32_t koff[L::COPIES], voff[4];
    const int lr = lane / L::CH, slot = lane % L::CH;
#pragma unroll
    for (int e = 0; e < L::COPIES; ++e) {
        const int row = L::ROWS * e + lr, c = slot ^ (row & (L::CH - 1));
        koff[e] = 8 * c < p.D ? 2 * ((row & 15) * p.D + 8 * c) : NO_ROW;
    }
    // K's operands: row r (+ 16 t), chunk 4 s + g
    uint32_t kofs[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) kofs[s] = r * L::PITCH + 16 * ((4 * s + g) ^ (r & (L::CH - 1)));
#pragma unroll
    for (int j = 0; j < 4; ++j) voff[j] = (4 * g + j) * p.D + min(DB * r, p.D - DB);
    const int64_t head = (int64_t)hk * p.page_d;
    // the 16 keys from key on: their element in the pools (page 0's where there is no
    // page, and `there` false)
    auto at16 = [&](int key, bool& there) -> int64_t {
        uint32_t id = pages.get(key >> shift);
        there = id < p.table.pages;
        id = there ? id : 0;
        return (int64_t)id * p.table.page_elems + head + (int64_t)(key & (page_rows - 1)) * p.D;
    };
    // K's rows of a tile go into one of the wave's two buffers by copies of the memory
    // system; V's into registers.  Each is issued a tile ahead, in this order, which the
    // empty asm statements keep: behind a tile's copies there are its eight loads of V.
    uint32_t vr[8][WORDS];
    int64_t at[2];
    bool there[2], next_there[2];
    auto load_k = [&](int tile) {
        unsigned char* to = sm.k[wave][(tile - w0) & 1];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            at[t] = at16(tile * TILE + 16 * t, next_there[t]);
#pragma unroll
            for (int e = t * L::COPIES / 2; e < (t + 1) * L::COPIES / 2; ++e)
                copy_rows(p.k + at[t], 32 * p.D, koff[e], 0, to + 1024 * e);
        }
        asm volatile("" ::: "memory");
    };
    auto load_v = [&]() {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint16_t* from = p.v + at[t] + voff[j];
                if constexpr (DB == 8) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
                    for (int i = 0; i < 4; ++i) vr[4 * t + j][i] = w[i];
                } else {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(from);
                    vr[4 * t + j][0] = w[0];
                    vr[4 * t + j][1] = w[1];
                }
            }
        asm volatile("" ::: "memory");
    };
    f32x4 o[NQ][DB];
    // the largest score before its scale (a difference of scores is exact where it counts,
    // however large they are), and l over the lane's own keys
    Stat st[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        st[n] = {NONE, 0.0f};
#pragma unroll
        for (int i = 0; i < DB; ++i) o[n][i] = f32x4{};
    }
    if (w0 < w1) {
        pages.load(w0 * TILE >> shift);
        load_k(w0);
        load_v();
    }
    // (behind the first loads, which it does not wait for)
    if (qs.tree && b1 * TILE > first) tree_bits(sm.tree, parent, qs.nq, t0, t1 - t0 + 1);
    // (the last tile apart: with a branch around the loads of a tile to come, a wait for this
    // one's would be one for all)
    auto step = [&](int tile, auto more) {
        const int key0 = tile * TILE;
        there[0] = next_there[0], there[1] = next_there[1];
        // K's copies have arrived, V's loads need not have (the build counts the loads behind
        // the copies in the listing, and refuses fewer than eight)
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        const unsigned char* kb = sm.k[wave][(tile - w0) & 1];
        f32x4 s[NQ][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            x8 kr[KS];
#pragma unroll
            for (int i = 0; i < KS; ++i)
                kr[i] = *reinterpret_cast<const x8*>(kb + kofs[i] + 16 * t * L::PITCH);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                s[n][t] = f32x4{};
#pragma unroll
                for (int i = 0; i < KS; ++i) s[n][t] = T::mfma16(kr[i], qf[n][i], s[n][t]);
            }
        }
        // (into the other buffer, which the tile before this one was read from)
        if constexpr (more) load_k(tile + 1);
        if (key0 + TILE > first || !there[0] || !there[1]) {
            const uint32_t paged = (there[0] ? 0xffffu : 0u) | (there[1] ? 0xffff0000u : 0u);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                uint32_t seen = low_bits(end[n] - key0);
                if (qs.tree && end[n] - key0 < 32) seen = tree_word(bits[n], key0 - end[n]);
                seen = (seen & paged) >> (4 * g);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(seen >> (16 * t + e) & 1)) s[n][t][e] = -INFINITY;
            }
        }
        // values that are not finite are kept apart, also from rows that see them all: half
        // a weight may be zero or below it
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < WORDS; ++i) bad |= not_finite<T>(vr[j][i]);
        const bool apart = __any(bad != 0);
        uint32_t ph[NQ][4], pl[NQ][4], ones[NQ][4];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float tm = s[n][0][0];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) tm = fmaxf(tm, s[n][t][e]);
            tm = rows4_max(tm);
            if (apart) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    ones[n][i] = (s[n][i >> 1][2 * (i & 1)] == -INFINITY ? 0u : V::ONE) |
                                 (s[n][i >> 1][2 * (i & 1) + 1] == -INFINITY ? 0u : V::ONE << 16);
            }
            const bool up = (tm - st[n].m) * p.scale_log2 > TAU;
            if (__any(up)) {
                const float m = up ? tm : st[n].m;
                const float alpha = up ? __builtin_amdgcn_exp2f((st[n].m - m) * p.scale_log2) : 1.0f;
                st[n].m = m;
                st[n].l *= alpha;
#pragma unroll
                for (int i = 0; i < DB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][i][e] *= alpha;
            }
            // (nothing seen yet: all scores are -inf, all weights 0)
            const float off = st[n].m == NONE ? 0.0f : st[n].m;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = __builtin_amdgcn_exp2f(fmaf(s[n][i >> 1][2 * (i & 1)] - off, p.scale_log2, V::LIFT));
                const float c =
                    __builtin_amdgcn_exp2f(fmaf(s[n][i >> 1][2 * (i & 1) + 1] - off, p.scale_log2, V::LIFT));
                sum += a + c;
                ph[n][i] = T::pack(a, c);
                // bf16's 8 bits would be as far off as the output's own: what they leave
                // of a weight is a second operand (the products cost nothing beside the
                // read)
                if constexpr (SPLIT)
                    pl[n][i] = T::pack(a - __uint_as_float(ph[n][i] << 16),
                                       c - __uint_as_float(ph[n][i] & 0xffff0000u));
            }
            st[n].l += sum;
        }
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            uint32_t w[4], kind[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = __builtin_amdgcn_perm(vr[2 * j + 1][i >> 1], vr[2 * j][i >> 1],
                                             i & 1 ? 0x07060302u : 0x05040100u);
            if (apart) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const Parts x = part_word<T>(w[j]);
                    w[j] = x.finite, kind[j] = x.kind;
                }
            }
            const x8 vf = as_x8<x8>(u32x4{w[0], w[1], w[2], w[3]});
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                o[n][i] = T::mfma16(vf, as_x8<x8>(u32x4{ph[n][0], ph[n][1], ph[n][2], ph[n][3]}), o[n][i]);
                if constexpr (SPLIT)
                    o[n][i] = T::mfma16(vf, as_x8<x8>(u32x4{pl[n][0], pl[n][1], pl[n][2], pl[n][3]}), o[n][i]);
                if (apart) {
                    const f32x4 sum =
                        T::mfma16(as_x8<x8>(u32x4{kind[0], kind[1], kind[2], kind[3]}),
                                  as_x8<x8>(u32x4{ones[n][0], ones[n][1], ones[n][2], ones[n][3]}), f32x4{});
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][i][e] = parted(o[n][i][e], sum[e]);
                }
            }
        }
        if constexpr (more) load_v();
    };
    for (int tile = w0; tile < w1 - 1; ++tile) step(tile, std::true_type{});
    if (w0 < w1) step(w1 - 1, std::false_type{});
    // merge of the waves: o[n][i][e] is column DB (4 g + e) + i of row 16 n + r
    __syncthreads();  // (the tree's bits are done with)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < DB; i += 4)
                *reinterpret_cast<f32x4*>(&sm.o[wave][16 * n + r][DB * (4 * g + e) + i]) =
                    f32x4{o[n][i][e], o[n][i + 1][e], o[n][i + 2][e], o[n][i + 3][e]};
        st[n].l = rows4_sum(st[n].l);
        st[n].m *= p.scale_log2;
        if (g == 0) sm.st[wave][16 * n + r] = st[n];
    }
    __syncthreads();
    for (int mr = threadIdx.x / 16; mr < ROWS; mr += 4 * W) {
        const int d = (threadIdx.x % 16) * 8;
        if (d >= P) break;
        Stat all{NONE, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w) all.m = fmaxf(all.m, sm.st[w][mr].m);
        float acc[8] = {};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const Stat one = sm.st[w][mr];
            const float f = weight(one.m, all.m);
            all.l += f * one.l;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += f * sm.o[w][mr][d + i];
        }
        // (l is in the weights' units: 2^LIFT too large)
        if constexpr (V::LIFT != 0.0f) all.l *= 1.0f / 4096.0f;
        if (p.splits > 1) store_partial(p, hk, part.first + part.split, row0 + mr, d, all, acc);
        else store_row<T>(p, b, hk, row0 + mr, d, all, acc);
    }
}

// ---------------------------------------------------------------- many rows
// Eight waves of 32 query rows each share every tile of 128 keys.  K and V rows go from
// their pages into LDS as they are, by 1 KB copies of the memory system (wave w those of
// keys 16 w .. 16 w + 15, which lie in one page), into the other of two buffers a
// tile ahead, one barrier a tile.  S^T = K Q^T on 32x32x16 MFMAs puts a query in a lane's
// column (16 of the scores of each 32 keys, the other 16 in lane ^ 32), and its weights
// are then the operand of O^T += V^T P^T without leaving the registers; V^T's operand
// is read from V's rows by the LDS's transposing reads (four keys of a column each).
//
// LDS: row k of a tile at PITCH k; K's 16-byte chunk c at c ^ (k mod chunks), V's 64-byte
// chunk c at c ^ (k mod 4) (narrow rows: c ^ (k / 2 mod 2)), so that neither kind of
// read meets a bank twice (counted: none of wide rows does, those of narrow ones wait 5 %
// of the cycles); the copies' lanes take their chunks from where that is.  Columns past
// D are zeros.
//
// A weight is one number of the cache's type: bf16's 8 bits, rounded to the nearest, make a
// result's error in norm 0.0018 to 0.0022 where its own rounding is 0.0017 (fp16's 11 bits
// 0.0002 to 0.0003).  The other kernel's second bf16 number would add half again to the
// products, which bound this one; sums and statistics are fp32.
//
// 1,560 queries of 24 heads over 12,480 keys, 239 GFLOP, three splits: 261 to 275
// us, 870 to 910 TFLOP/s, and a merge of 11.  The matrix units are busy 36 % of the SIMDs'
// cycles and the vector units 40 %: the softmax runs beside the products too little, and of
// eight waves one has no rows (49 blocks of 32 are seven groups of seven).  16
// sequences of 8,192 keys, 8 heads, 256 rows, 137 GFLOP and 537 MB: 178 us.  The form for
// 128 columns fills the 256 registers of a lane, with six of them in scratch memory.
constexpr int TILE_WAVES = 8, TILE_KEYS = 128;

template <int P>
struct TileLds {
    static constexpr int PITCH = P == 64 ? 128 : 256, CH = PITCH / 16;
    static constexpr int BUF = TILE_KEYS * PITCH, SMEM = 4 * BUF;        // K0 K1 V0 V1
    static constexpr int ROWS = 1024 / PITCH, COPIES = 16 / ROWS;        // rows of a copy, a wave's
    static __device__ __forceinline__ int vswz(int row) { return P == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2; }
};

typedef short i16x4 __attribute__((ext_vector_type(4)));
// (__restrict__: a read that might alias the copies in flight would wait for them all,
// the next tile's among them; this one's are waited for at the barrier.  16 sequences of
// 8,192 keys, 8 heads, 256 rows: 178 us, 188 without it)
__device__ __forceinline__ u32x2 lds_columns(const unsigned char* __restrict__ p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) i16x4*)p));
}

template <typename T, int P>
__global__ void __launch_bounds__(64 * TILE_WAVES) attend_tile_kernel(AttendParams p) {
    constexpr int KS = P / 16, DB = P / 32;
    using x8 = typename T::x8;
    using V = Value<T>;
    using L = TileLds<P>;
    extern __shared__ __align__(16) unsigned char smem[];  // TileLds::SMEM, and the tree's
    TreeSmem<32 * TILE_WAVES>& tree = *reinterpret_cast<TreeSmem<32 * TILE_WAVES>*>(smem + L::SMEM);
    const int lane = threadIdx.x & 63, hf = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Item it = item_of(p);
    if (!it.there) return;
    const int rg = it.group, at_slot = (int)p.by_H.of(it.unit), hk = (int)it.unit - at_slot * p.H;
    const Part part = part_of(p, at_slot);
    if (!part.there) return;
    tell_merge(p, part, hk, rg);
    const int b = part.b;
    const Queries qs = queries_of(p, part);
    const int32_t parent = tree_parent(p, b);
    const int row0 = rg * p.per_group * 32;
    const int rows_end = min(row0 + p.per_group * 32, p.rows);
    // tiles that some row of the group sees
    const int g0 = (int)p.by_G.of(row0), g1 = (int)p.by_G.of(rows_end - 1);
    const int last = max(0, qs.most(g0, g1));
    const int nt = (last + TILE_KEYS - 1) / TILE_KEYS;
    int b0, b1;
    share_of(part, nt, b0, b1);
    const int wrow = row0 + 32 * wave, row = wrow + l32;
    const bool active = wrow < rows_end;
    const RowAt mine = row_at(p, row, hk);
    const int end = mine.there ? qs.end(mine.t) : 0;
    const int t0 = (int)p.by_G.of(wrow), t1 = (int)p.by_G.of(min(wrow + 32, p.rows) - 1);
    const int first = qs.least(t0, t1), wlast = active ? qs.most(t0, t1) : 0;  // of the wave
    x8 qf[KS];
    {
        const uint16_t* q = p.q + b * p.q_sb + mine.t * p.q_st + mine.head * p.q_sh;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * hf;
            u32x4 w{};
            if (active && mine.there && d < p.D) w = *reinterpret_cast<const u32x4*>(q + d);
            qf[s] = as_x8<x8>(w);
        }
    }
    const uint32_t* bits = tree.bits[active && mine.there ? mine.t - g0 : 0];
    // The pages of 64 tiles, a lane each: that of this wave's rows, and a bit for each
    // 16 keys whether theirs is one.
    const int32_t* table = p.table.at + b * p.table.sb;
    const int shift = p.table.shift, w = (int)p.table.w;
    int ids_of = 0;
    uint32_t ids = 0, there = 0;
    auto load_ids = [&](int tile) {
        ids_of = tile;
        there = 0;
#pragma unroll
        for (int i = 0; i < TILE_KEYS / 16; ++i) {
            const int64_t entry = ((int64_t)(tile + lane) * TILE_KEYS + 16 * i) >> shift;
            const uint32_t id = entry < w ? (uint32_t)table[entry] : ~0u;
            there |= id < p.table.pages ? 1u << i : 0u;
            if (i == wave) ids = id;
        }
        ids = ids < p.table.pages ? ids : 0;
    };
    // this lane's part of the wave's copies: row lr of each, 16-byte slot `slot`
    const int lr = lane / L::CH, slot = lane % L::CH;
    uint32_t koff[L::COPIES], voff;
#pragma unroll
    for (int e = 0; e < L::COPIES; ++e) {
        const int r = L::ROWS * e + lr, c = slot ^ (r & (L::CH - 1));
        koff[e] = 8 * c < p.D ? 2 * (r * p.D + 8 * c) : NO_ROW;
    }
    {
        const int c = slot ^ L::vswz(lr);
        voff = 8 * c < p.D ? 2 * (lr * p.D + 8 * c) : NO_ROW;
    }
    const int64_t head = (int64_t)hk * p.page_d;
    const int page_rows = 1 << shift;
    auto issue = [&](int tile) {
        const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)ids, tile - ids_of);
        const int key = tile * TILE_KEYS + 16 * wave, buf = (tile - b0) & 1;
        const int64_t at = (int64_t)id * p.table.page_elems + head + (int64_t)(key & (page_rows - 1)) * p.D;
        unsigned char* kd = smem + buf * L::BUF + 16 * wave * L::PITCH;
        unsigned char* vd = kd + 2 * L::BUF;
#pragma unroll
        for (int e = 0; e < L::COPIES; ++e) copy_rows(p.k + at, 32 * p.D, koff[e], 0, kd + 1024 * e);
#pragma unroll
        for (int e = 0; e < L::COPIES; ++e)
            copy_rows(p.v + at, 32 * p.D, voff, 2 * L::ROWS * e * p.D, vd + 1024 * e);
    };
    // operand offsets in buffer 0: K row l32 (+ 32 j), chunk 2 kk + hf; V rows 4 hf +
    // lane % 16 / 4 (+ 32 j + 16 k, and 8 on), 32 columns i: column 16 (l32 / 16) on.  A
    // group of 16 lanes gets column 4 a + e in lane 4 a' + e, a' = a with its bits
    // swapped: a lane's results are then eight consecutive columns.
    uint32_t kofs[KS], vofs[DB];
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
        kofs[kk] = l32 * L::PITCH + 16 * ((2 * kk + hf) ^ (l32 & (L::CH - 1)));
        asm volatile("" : "+v"(kofs[kk]));
    }
#pragma unroll
    for (int i = 0; i < DB; ++i) {
        const int x = lane & 15, k = 4 * hf + (x >> 2), a = ((x & 1) << 1) | (x >> 1 & 1);
        const int chunk = 4 * i + 2 * (l32 >> 4) + (a >> 1);
        vofs[i] = 2 * L::BUF + k * L::PITCH + 16 * (chunk ^ L::vswz(k)) + 8 * (a & 1);
        asm volatile("" : "+v"(vofs[i]));
    }
    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x16{};
    Stat st{NONE, 0.0f};
    if (b0 < b1) {
        load_ids(b0);
        issue(b0);
    }
    if (qs.tree && b1 * TILE_KEYS > qs.least(g0, g1)) tree_bits(tree, parent, qs.nq, g0, g1 - g0 + 1);
    // Whether some row of the wave does not see some of the 32 keys from k0 on (there: their
    // halves' pages, a bit each), and which of them the lane's row sees.
    auto masked = [&](int k0, uint32_t there) { return k0 + 32 > first || (there & 3) != 3; };
    auto seen_word = [&](int k0, uint32_t there) {
        const uint32_t seen = qs.tree && end - k0 < 32 ? tree_word(bits, k0 - end) : low_bits(end - k0);
        return seen & ((there & 1 ? 0xffffu : 0u) | (there & 2 ? 0xffff0000u : 0u));
    };
    // One 32-key step's softmax and products with the V^T operands vf.
    auto softmax_pv = [&](f32x16& s, const u32x4 (&vf)[2][DB]) {
        float tm = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) tm = fmaxf(tm, s[i]);
        tm = halfwave_max(tm) * p.scale_log2;
        const bool up = tm > st.m + TAU;
        const float m = up ? tm : st.m;
        const float alpha = up ? __builtin_amdgcn_exp2f(st.m - m) : 1.0f;
        st.m = m;
        float c = p.scale_log2, off = (m == NONE ? 0.0f : m) - V::LIFT;
        if (__any(fabsf(off) > 0x1p20f)) {
            // a maximum so large that its own rounding counts: differences of rounded
            // products instead of the product's remainder
            const float ref = m == NONE ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float z = s[i] * c;
                asm("" : "+v"(z));
                s[i] = z - ref;
            }
            c = 1.0f, off = -V::LIFT;
        }
        uint32_t pw[8];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * i], c, -off));
            const float y = __builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], c, -off));
            sum += x + y;
            pw[i] = T::pack(x, y);
        }
        st.l = st.l * alpha + sum;
        __builtin_amdgcn_s_setprio(1);
        if (__any(up)) {
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const x8 pf = as_x8<x8>(u32x4{pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]});
#pragma unroll
            for (int i = 0; i < DB; ++i) o[i] = T::mfma32(as_x8<x8>(vf[k][i]), pf, o[i]);
        }
        __builtin_amdgcn_s_setprio(0);
    };
    // Waves w and w + 4 share a SIMD.  Waves 4-7 run half a step behind waves 0-3: each
    // carries its tile's last step (masked scores in s, V^T operands in vf) across the
    // barrier and finishes it first in the next tile, so that one's softmax runs beside
    // the other's products.
    const bool lag = wave >= TILE_WAVES / 2;
    bool pend = false;
    bool apart = false;                       // values that are not finite were taken out
    f32x16 s;
    x8 kf[KS];
    u32x4 vf[2][DB];
    auto load_k = [&](int j) {
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
            kf[kk] = *reinterpret_cast<const x8*>(smem + kofs[kk] + j * 32 * L::PITCH);
    };
    auto load_v = [&](int j) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < DB; ++i) {
                const u32x2 a = lds_columns(smem + vofs[i] + (32 * j + 16 * k) * L::PITCH);
                const u32x2 c = lds_columns(smem + vofs[i] + (32 * j + 16 * k + 8) * L::PITCH);
                vf[k][i] = u32x4{a[0], a[1], c[0], c[1]};
            }
    };
    auto scores = [&]() {
        __builtin_amdgcn_s_setprio(1);
        s = T::mfma32(kf[0], qf[0], f32x16{});
#pragma unroll
        for (int kk = 1; kk < KS; ++kk) s = T::mfma32(kf[kk], qf[kk], s);
        __builtin_amdgcn_s_setprio(0);
    };
    constexpr int STEPS = TILE_KEYS / 32;
    // (one more turn than tiles, for what the lagging waves carry out of the last)
    for (int tile = b0; tile <= b1; ++tile) {
        // this tile's copies have arrived, and all reads of the other buffer
        wait_vmcnt<0>();
        lds_barrier();
        const uint32_t paged = tile < b1 ? (uint32_t)__builtin_amdgcn_readlane((int)there, tile - ids_of) : 0;
        if (tile + 1 < b1) {
            if (tile + 1 - ids_of >= 64) load_ids(tile + 1);
            issue(tile + 1);
        }
        const int key0 = tile * TILE_KEYS;
        const int nsub = tile == b1 ? 0 : min(max(wlast - key0 + 31, 0) >> 5, STEPS);
        // (an idle wave's reads of the first step stay inside the buffer)
        load_k(0);
        if (pend) {
            softmax_pv(s, vf);
            // the new tile's V^T reads wait for the carried products, so that both sets
            // are never live at once
            __builtin_amdgcn_sched_barrier(0);
        }
        pend = false;
        load_v(0);
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
            if (j >= nsub) break;
            scores();
            if (j + 1 < nsub) load_k(j + 1);
            const int k0 = key0 + 32 * j;
            if (masked(k0, paged >> (2 * j))) {
                const uint32_t seen = seen_word(k0, paged >> (2 * j)) >> (4 * hf);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(seen >> (8 * (i >> 2) + (i & 3)) & 1)) s[i] = -INFINITY;
                uint32_t bad = 0;
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < DB; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) bad |= not_finite<T>(vf[k][i][e]);
                if (__any(bad != 0)) {
                    apart = true;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int i = 0; i < DB; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) vf[k][i][e] = part_word<T>(vf[k][i][e]).finite;
                }
            }
            if (lag && j + 1 == nsub) {
                pend = true;
                break;
            }
            softmax_pv(s, vf);
            if (j + 1 < nsub) load_v(j + 1);
        }
        const int step = (tile - b0) & 1 ? -L::BUF : L::BUF;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            kofs[kk] += step;
            asm volatile("" : "+v"(kofs[kk]));
        }
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            vofs[i] += step;
            asm volatile("" : "+v"(vofs[i]));
        }
    }
    // What was taken out of masked steps goes to the rows that see it, from memory.
    if (apart)
#pragma unroll 1
        for (int k0 = b0 * TILE_KEYS; k0 < min(b1 * TILE_KEYS, wlast); k0 += 32) {
            uint32_t id[2], pages = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int entry = (k0 + 16 * h) >> shift;
                id[h] = entry < w ? (uint32_t)table[entry] : ~0u;
                if (id[h] < p.table.pages) pages |= 1u << h;
                else id[h] = 0;
            }
            if (!masked(k0, pages)) continue;
            const uint32_t seen = seen_word(k0, pages);
#pragma unroll 1
            for (int k = 0; k < 32; ++k) {
                const int64_t at = (int64_t)id[k >> 4] * p.table.page_elems + head +
                                   (int64_t)((k0 + k) & (page_rows - 1)) * p.D;
#pragma unroll
                for (int i = 0; i < DB; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int d = 32 * i + 16 * e + 8 * hf;
                        u32x4 x{};
                        if (d < p.D && seen >> k & 1) x = *reinterpret_cast<const u32x4*>(p.v + at + d);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float y = T::to_f32((uint16_t)(x[j >> 1] >> (16 * (j & 1))));
                            if (!(fabsf(y) < INFINITY)) o[i][8 * e + j] += y;
                        }
                    }
            }
        }
    st.l = halfwave_sum(st.l);
    if constexpr (V::LIFT != 0.0f) st.l *= 1.0f / 4096.0f;
    if (!active) return;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 32 * i + 16 * e + 8 * hf;
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = o[i][8 * e + k];
            if (p.splits > 1) store_partial(p, hk, part.first + part.split, row, d, st, x);
            else store_row<T>(p, b, hk, row, d, st, x);
        }
}

// ---------------------------------------------------------------- splits
// The merge of the splits' partial results: a thread eight columns, SG groups of
// threads share a row's splits and are joined in LDS, and a thread has AHEAD splits'
// loads in flight.  With M the largest m, out = sum(2^(m - M) o) / sum(2^(m - M) l).
// 37,440 rows of three splits, 68 MB: 11 us; few rows of many splits 4 to 6, the chain of a
// launch, loads and the exchange.
constexpr int AHEAD = 4;
template <typename T, int SG>
__global__ void __launch_bounds__(256) merge_kernel(AttendParams p) {
    constexpr int PARTS = 16, ROWS = 256 / (PARTS * SG);
    const int row = blockIdx.x * ROWS + threadIdx.x / (PARTS * SG);
    const int sg = threadIdx.x / PARTS % SG, part = threadIdx.x % PARTS, d = part * 8;
    const int b = blockIdx.z, hk = blockIdx.y;
    const bool in = row < p.rows && d < p.D;
    const i32x2 share = p.shares ? p.shares[b] : i32x2{b * p.splits, p.splits};
    const int splits = share[1];
    const int64_t first = ((int64_t)hk * p.B * p.splits + share[0]) * p.rows + row;
    Stat all{NONE, 0.0f};
    float acc[8] = {};
    if (in) {
        for (int s0 = sg; s0 < splits; s0 += SG * AHEAD) {
            f32x2 ml[AHEAD];
            f32x4 x[AHEAD][2];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int64_t i = first + (int64_t)min(s0 + SG * j, splits - 1) * p.rows;
                ml[j] = p.part_ml[i];
                const f32x4* from = reinterpret_cast<const f32x4*>(p.part + i * p.D + d);
                x[j][0] = from[0];
                x[j][1] = from[1];
            }
            float m = all.m;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (s0 + SG * j < splits) m = fmaxf(m, ml[j][0]);
            const float f = weight(all.m, m);
            all.m = m;
            all.l *= f;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] *= f;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (s0 + SG * j >= splits) break;
                const float w = weight(ml[j][0], m);
                all.l += w * ml[j][1];
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] += w * x[j][k >> 2][k & 3];
            }
        }
    }
    if constexpr (SG > 1) {
        __shared__ float sh[ROWS][SG][PARTS][8];
        __shared__ Stat sst[ROWS][SG];
        const int lr = threadIdx.x / (PARTS * SG);
#pragma unroll
        for (int k = 0; k < 8; ++k) sh[lr][sg][part][k] = acc[k];
        if (part == 0) sst[lr][sg] = all;
        __syncthreads();
        if (sg) return;
        all = {NONE, 0.0f};
#pragma unroll
        for (int s = 0; s < SG; ++s) all.m = fmaxf(all.m, sst[lr][s].m);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
#pragma unroll
        for (int s = 0; s < SG; ++s) {
            const float f = weight(sst[lr][s].m, all.m);
            all.l += f * sst[lr][s].l;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += f * sh[lr][s][part][k];
        }
    }
    if (in) store_row<T>(p, b, hk, row, d, all, acc);
}

// ---------------------------------------------------------------- host
struct Plan {
    bool tile, eight, two;        // the tile kernel; of the other, eight waves, two groups of rows
    int groups, splits, per_group;
    int64_t items, rows;
    size_t part, ml, shares;      // bytes
};

// The tile kernel takes calls of more than TILE_ROWS rows of a key head that have more than
// TILE_WORK (row, key) pairs in all heads, as a workgroup's start costs it about 10 us (us
// with either, rows first; 8 heads of 4,096 keys: 128 rows 19.7, 23.4, 256 rows 25.4,
// 32.2; 16 heads: 128 rows 24.8, 28.0; 32 heads: 128 rows 32.9, 32.0, 256 rows 51, 40; 64
// heads: 64 rows 34, 41, 96 rows 51, 43; 64 heads of 8,192 keys, 128 rows: 99, 79), or
// more than TILE_BLOCKS times 32 rows, which the other kernel would give a workgroup each,
// with three of its four waves idle over few keys (256 heads of 64 keys, 64 rows 8.8, 8.2,
// 128 rows 15.4, 9.4; 184 heads of 16 keys, 2,360 rows 144, 58; 64 heads, 256 rows 8.9,
// 9.5; 128 heads of 512 keys, 128 rows 18.6, 21.4, 256 rows 34, 26).
constexpr int64_t TILE_ROWS = 64, TILE_WORK = 1 << 24, TILE_BLOCKS = 512;

Plan attend_plan(const nkv_paged_attend_args* a) {
    const nkv_paged_cache& c = a->cache;
    Plan pl{};
    pl.rows = a->Q * a->G;
    const int64_t heads = (int64_t)a->B * c.H, tiles = cdiv(a->n, TILE);
    const bool uneven = a->length && a->B > 1;
    pl.splits = 1;
    pl.tile = pl.rows > TILE_ROWS && (heads * cdiv(pl.rows, 32) > TILE_BLOCKS ||
                                      heads * pl.rows > TILE_WORK / std::max<int64_t>(a->n, 1));
    if (pl.tile) {
        // the fewest groups of up to eight 32-row blocks, of even size
        const int64_t qb = cdiv(pl.rows, 32), blocks = cdiv(a->n, 64);
        pl.groups = (int)cdiv(qb, TILE_WAVES);
        pl.per_group = (int)cdiv(qb, pl.groups);
        const int64_t base = heads * pl.groups;
        // splits whose rounds of 256 workgroups take least, in units of the time of 64 keys
        // (2.0 to 2.6 us): a workgroup's start and end cost five, a merge two and its
        // partials' traffic (us with splits that fill half a round, one and two: 64 heads
        // of 8,192 keys, 256 rows 155, 101, 118; 8 heads of 16,384, 512 rows 76, 63, 76;
        // 32 heads of 4,096, 256 rows 48, 40, 75)
        double best = 0.0;
        const int64_t most = std::max<int64_t>(16, cdiv(256, std::max<int64_t>(base, 1)));
        for (int64_t s = 1; s <= most && (s == 1 || blocks >= 4 * s); ++s) {
            const double merge = s == 1 ? 0.0 : 2.0 + (double)heads * pl.rows * s * 2.5e-5;
            const double t = (double)cdiv(base * s, 256) * ((double)blocks / s + 5.0) + merge;
            if (s == 1 || t < best) {
                best = t;
                pl.splits = (int)s;
            }
        }
        pl.items = base * pl.splits;
        return pl;
    }
    // Two groups of 16 rows to a wave where there are more (us with one and two: 8 heads of
    // 4,096 keys, 32 rows 11.3, 12.6, 64 rows 15.3, 14.8; 64 heads, 64 rows 34.2, 33.1).
    pl.two = pl.rows > 32;
    pl.groups = (int)cdiv(pl.rows, pl.two ? 32 : 16);
    const int64_t base = heads * pl.groups, work = base * tiles;
    // Up to 32 tiles no splits: the second launch and its workspace cost more than they save
    // (8 heads of 1,024 keys 10.3 us without, 8.7 with them, but a call takes the host 10.5
    // and 14; of 2,048 keys 16.2 and 7.9).
    if (tiles <= 32) {
        pl.eight = tiles > 8 && (!pl.two || base <= 256);
        pl.items = base;
        return pl;
    }
    // Else one workgroup a CU, as a start and a merge cost more than latency (8 heads of
    // 4,096 keys, 4 rows: 128, 256, 512 workgroups 10.2, 8.7, 10.3 us), of four waves; two a
    // CU in long calls of unlike lengths (8 sequences evenly up to 32,768 keys, 8 heads: 103,
    // 102), and there eight waves where sequences have one or two splits (32 up to 16,384:
    // 228, 218).  Two groups of rows get eight waves and one workgroup a CU at most (four
    // waves with one a CU, with two, eight with one: 8 heads of 4,096 keys, 256 rows 23.0,
    // 23.4, 20.4; 64 of 2,048, 64 rows 23.4, 22.7, 21.7), or four where there are more (12
    // heads of 1,185 keys, 760 rows: eight 36, four 23).
    const int64_t least = std::max<int64_t>(base, 1);
    int64_t splits = 256 / least;
    if (pl.two) {
        pl.eight = base <= 256;
    } else {
        splits = cdiv(uneven && work >= 32768 ? 512 : 256, least);
        pl.eight = uneven && work >= 4096 && splits <= 2;
    }
    pl.splits = (int)std::max<int64_t>(1, std::min(splits, tiles / (pl.eight ? 8 : 4)));
    pl.items = base * pl.splits;
    return pl;
}

// The plan's workspace; in fewer than `limit` bytes fewer splits where those wanted do
// not fit.
void attend_fit(const nkv_paged_attend_args* a, Plan& pl, size_t limit) {
    if (pl.splits == 1) return;
    const size_t rows = (size_t)a->B * a->cache.H * pl.rows;
    const size_t shares = a->length && a->B > 1 && a->B <= BALANCED ? a->B * sizeof(i32x2) : 0;
    const size_t most = limit < shares ? 0 : (limit - shares) / (rows * (sizeof(f32x2) + 4 * a->cache.D));
    if (most < (size_t)pl.splits) {
        pl.items /= pl.splits;
        pl.splits = (int)std::max<size_t>(1, most);
        pl.items *= pl.splits;
        if (pl.splits == 1) return;
    }
    pl.part = rows * pl.splits * 4 * a->cache.D;
    pl.ml = rows * pl.splits * sizeof(f32x2);
    pl.shares = shares;
}

// Also plans the call, for a workspace of that many bytes, where there is something to do
// (pl.items > 0).
int check_attend(const nkv_paged_attend_args* a, Plan& pl, const void* workspace, size_t bytes) {
    NKV_REQUIRE(a, NKV_ERR_INVALID, "args is null");
    const nkv_paged_cache& c = a->cache;
    int rc = paged_check(c, __func__);
    if (rc) return rc;
    if ((rc = paged_table_check(c, a->table, a->table_sb, a->table_w, a->B, __func__))) return rc;
    const PageTable table = page_table(c, a->table, a->table_sb, a->table_w);
    NKV_REQUIRE(a->G >= 1 && a->Q >= 0, NKV_ERR_INVALID, "G must be positive and Q not negative");
    NKV_REQUIRE(a->Q <= INT32_MAX / 2 && (__int128)a->Q * a->G <= INT32_MAX / 2 &&
                    (int64_t)c.H * a->G <= INT32_MAX,
                NKV_ERR_UNSUPPORTED, "too many query rows");
    NKV_REQUIRE(a->n >= 0 && a->n <= std::min<int64_t>(table.cap(), 1 << 30), NKV_ERR_INVALID,
                "n must be in [0, table_w * page] and at most 2^30");
    NKV_REQUIRE(a->softmax_scale > 0.0f && a->softmax_scale < INFINITY, NKV_ERR_INVALID,
                "softmax_scale must be positive and finite");
    NKV_REQUIRE(!a->parents || !a->causal, NKV_ERR_INVALID, "causal and parents exclude each other");
    NKV_REQUIRE(!a->parents || a->Q <= NKV_PAGED_TREE, NKV_ERR_UNSUPPORTED,
                "a tree has at most 256 tokens");
    NKV_REQUIRE(!a->parents || a->parents_sb >= 0, NKV_ERR_INVALID, "parents_sb must not be negative");
    if (a->B == 0 || a->Q == 0) return NKV_OK;
    NKV_REQUIRE(a->q && a->out, NKV_ERR_INVALID, "q and out are required");
    NKV_REQUIRE((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) % 16 == 0 &&
                    (a->q_sb | a->q_st | a->q_sh | a->o_sb | a->o_st | a->o_sh) % 8 == 0,
                NKV_ERR_INVALID, "q and out must be 16-byte aligned with strides divisible by 8");
    NKV_REQUIRE(a->q_sb >= 0 && a->q_st >= 0 && a->q_sh >= 0, NKV_ERR_INVALID,
                "q's strides must not be negative");
    NKV_REQUIRE((int64_t)a->B * c.H * cdiv(a->Q * a->G, 32 * TILE_WAVES) <= 1 << 22, NKV_ERR_UNSUPPORTED,
                "too many query rows");
    pl = attend_plan(a);
    NKV_REQUIRE(pl.items <= 1 << 22, NKV_ERR_UNSUPPORTED, "too many query rows");
    attend_fit(a, pl, bytes);
    NKV_REQUIRE(rows_span(a->o_sb, a->B, a->o_st, a->Q, a->o_sh, (int64_t)c.H * a->G, c.D) > 0,
                NKV_ERR_INVALID, "out's rows overlap");
    // what is written and what is read
    const int64_t heads = (int64_t)c.H * a->G;
    const RowSet q(a->q, 2, c.D, a->q_sb, a->B, a->q_st, a->Q, a->q_sh, heads);
    const RowSet out(a->out, 2, c.D, a->o_sb, a->B, a->o_st, a->Q, a->o_sh, heads);
    const Range in[6] = {{c.k, pool_bytes(c)}, {c.v, pool_bytes(c)},
                         {a->table, table_bytes(a->B, a->table_sb, a->table_w)},
                         {a->length, a->length ? a->B * 4 : 0}, {a->counts, a->counts ? a->B * 4 : 0},
                         {a->parents, a->parents ? table_bytes(a->B, a->parents_sb, a->Q) : 0}};
    const Range lse(a->lse, a->lse ? a->B * heads * a->Q * 4 : 0);
    for (const Range& r : in)
        NKV_REQUIRE(!r.meets(lse) && !rows_meet(out, r), NKV_ERR_INVALID,
                    "out or lse overlaps the cache, table, length, counts or parents");
    NKV_REQUIRE(!rows_meet(out, lse) && !rows_meet(q, lse), NKV_ERR_INVALID,
                "lse overlaps q or out");
    NKV_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0 || pl.part == 0, NKV_ERR_INVALID,
                "workspace must be 16-byte aligned");
    const Range work(workspace, workspace ? pl.part + pl.ml + pl.shares : 0);
    NKV_REQUIRE(!rows_meet(q, work) && !rows_meet(out, work) && !work.meets(lse), NKV_ERR_INVALID,
                "workspace overlaps q, out or lse");
    for (const Range& r : in)
        NKV_REQUIRE(!work.meets(r), NKV_ERR_INVALID,
                    "workspace overlaps the cache, table, length, counts or parents");
    if (a->out == a->q)
        NKV_REQUIRE(a->q_sb == a->o_sb && a->q_st == a->o_st && a->q_sh == a->o_sh, NKV_ERR_INVALID,
                    "out over q must have its strides");
    else
        NKV_REQUIRE(!rows_meet(out, q), NKV_ERR_INVALID, "out overlaps q");
    return NKV_OK;
}

// Blocks of a launch over p.items workgroups in item_of's order.
unsigned item_blocks(const AttendParams& p) { return (unsigned)(8 * cdiv(p.items, 8)); }

template <typename T, int KS, int W, int NQ>
int rows_run(const AttendParams& p, hipStream_t s) {
    constexpr int SMEM = sizeof(RowsSmem<width_of<KS>(), W, NQ>);
    if (SMEM > 65536)
        if (int rc = set_smem(attend_kernel<T, KS, W, NQ>, SMEM)) return rc;
    attend_kernel<T, KS, W, NQ><<<item_blocks(p), 64 * W, SMEM, s>>>(p);
    return NKV_OK;
}

template <typename T, int P>
int tile_run(const AttendParams& p, hipStream_t s) {
    const int smem = TileLds<P>::SMEM + (p.parents ? (int)sizeof(TreeSmem<32 * TILE_WAVES>) : 0);
    if (int rc = set_smem(attend_tile_kernel<T, P>, smem)) return rc;
    attend_tile_kernel<T, P><<<item_blocks(p), 64 * TILE_WAVES, smem, s>>>(p);
    return NKV_OK;
}

template <typename T, int KS>
int attend_run(const AttendParams& p, const Plan& pl, hipStream_t s) {
    if (pl.two) return pl.eight ? rows_run<T, KS, 8, 2>(p, s) : rows_run<T, KS, 4, 2>(p, s);
    return pl.eight ? rows_run<T, KS, 8, 1>(p, s) : rows_run<T, KS, 4, 1>(p, s);
}

template <typename T>
int attend_width(const AttendParams& p, const Plan& pl, hipStream_t s) {
    if (pl.tile)
        return p.D <= 64 ? tile_run<T, 64>(p, s) : p.D <= 96 ? tile_run<T, 96>(p, s) : tile_run<T, 128>(p, s);
    return p.D <= 64 ? attend_run<T, 2>(p, pl, s)
                     : p.D <= 96 ? attend_run<T, 3>(p, pl, s) : attend_run<T, 4>(p, pl, s);
}

// Sixteen groups of threads to a row where there are few rows and splits to share, by the
// mean of the sequences' splits (their number is known on the device only; a sequence may have
// most of a call's, which one thread then reads four at a time) (whole
// calls, us with sixteen and one: 32 rows of 32 splits 8.7, 16.7, of 12 21.3, 24.0; 128
// rows of 8 18.0, 19.2, of 4 46.1, 46.3; 2,048 rows of 16 50.9, 49.7; 37,440 of 3 378, 278).
template <typename T>
void merge_run(const AttendParams& p, hipStream_t s) {
    const bool share = p.splits > 4 && (int64_t)p.B * p.H * p.rows <= 1024;
    const dim3 grid((unsigned)cdiv(p.rows, share ? 1 : 16), (unsigned)p.H, (unsigned)p.B);
    if (share) merge_kernel<T, 16><<<grid, 256, 0, s>>>(p);
    else merge_kernel<T, 1><<<grid, 256, 0, s>>>(p);
}

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" size_t nkv_paged_attend_workspace_size(const nkv_paged_attend_args* a) {
    clear_error();
    Plan pl{};
    if (check_attend(a, pl, nullptr, SIZE_MAX) || pl.items == 0) return 0;
    return pl.part + pl.ml + pl.shares;
}

extern "C" int nkv_paged_attend(void* stream, const nkv_paged_attend_args* a, void* workspace,
                                size_t workspace_bytes) {
    clear_error();
    Plan pl{};
    int rc = check_attend(a, pl, workspace, workspace ? workspace_bytes : 0);
    if (rc || pl.items == 0) return rc;
    const nkv_paged_cache& c = a->cache;
    AttendParams p{};
    p.table = page_table(c, a->table, a->table_sb, a->table_w);
    p.k = (const uint16_t*)c.k;
    p.v = (const uint16_t*)c.v;
    p.length = a->length;
    p.counts = a->counts;
    p.parents = a->parents;
    p.parents_sb = a->parents_sb;
    p.q = (const uint16_t*)a->q;
    p.out = (uint16_t*)a->out;
    p.lse = a->lse;
    p.part = (float*)workspace;
    p.part_ml = (f32x2*)((char*)workspace + pl.part);
    p.q_sb = a->q_sb, p.q_st = a->q_st, p.q_sh = a->q_sh;
    p.o_sb = a->o_sb, p.o_st = a->o_st, p.o_sh = a->o_sh;
    p.items = pl.items;
    // (kept from 0 and infinity: a hidden score of -inf times 0 would be NaN)
    p.scale_log2 = std::clamp(a->softmax_scale * LOG2E, 0x1p-126f, 0x1.fffffep127f);
    p.B = a->B, p.H = c.H, p.G = a->G, p.D = c.D, p.Q = (int)a->Q, p.n = (int)a->n;
    p.causal = a->causal != 0;
    p.splits = pl.splits;
    p.groups = pl.groups;
    p.rows = (int)pl.rows;
    p.page_d = c.page * c.D;
    p.per_group = pl.per_group;
    p.shares = pl.shares ? (i32x2*)((char*)workspace + pl.part + pl.ml) : nullptr;
    p.by_G = divisor(a->G), p.by_H = divisor(c.H), p.by_B = divisor(a->B), p.by_groups = divisor(pl.groups);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    rc = c.dtype == NKV_ROWS_BF16 ? attend_width<Bf16>(p, pl, s) : attend_width<Fp16>(p, pl, s);
    if (rc) return rc;
    NKV_LAUNCH_CHECK();
    if (pl.splits > 1) {
        if (c.dtype == NKV_ROWS_BF16) merge_run<Bf16>(p, s);
        else merge_run<Fp16>(p, s);
        NKV_LAUNCH_CHECK();
    }
    return NKV_OK;
}
