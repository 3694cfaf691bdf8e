// nkv_cache8_attend.hip -- attention over the 8-bit key/value cache and the
// weight its rows receive (nkv_cache8_attend, nkv_cache8_mass).
//
// With k = sk * code per block of 64 rows, a score is (softmax_scale * sk) *
// (q . code), and with v = sv * code the output is sum p * sv * code / sum p:
// neither scale meets a 16-bit operand.  Codes are exact in bf16 and fp16, so
// the scores are those of the dequantised rows with one rounding less.
//
// The weights p * sv of the second product are rounded to fp16 whatever the
// queries' type: with bf16 their rounding is as large as the output's own (2^-9
// relative; over 262,144 keys the output was 0.0026 off in norm where its own
// rounding makes 0.0017).  fp16's range is enough because a row's weights are held
// relative to its own largest one: with m the row's running maximum of z and wm
// that of z + log2 sv, over the keys it sees, and both at most TAU behind,
//   w = 2^(z + log2 sv - wm + LIFT) <= 2^(LIFT + TAU)
// keeps all 11 bits down to 2^-(14 + LIFT) of the largest weight and is a multiple
// of 2^-(24 + LIFT) of it below.  A loud block that a row does not see, or gives no
// weight to, costs the row nothing.  The softmax's sum is 2^(z - m)'s: the same
// exponentials, multiplied back by what separates the two units.
#include "nkv_cache8.h"

#include <math.h>

#include <algorithm>
#include <utility>

namespace nkv {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float TAU = 3.0f;           // a row's maximum is moved when it is off by 2^TAU
constexpr float LIFT = 12.0f;         // 2^(LIFT + TAU) < 65504
constexpr float FLOOR = -0x1p126f;    // a maximum before the first key (finite: no inf - inf)
// A block's weights that lie more than this below the row's largest are taken as
// 2^-QUIET of their 2^(z - m): they are zero in fp16 (2^(LIFT + TAU - QUIET) = 2^-25)
// either way, and stay normal numbers for the sum.
constexpr float QUIET = 40.0f;
// A score's factor softmax_scale * log2 e * sk, kept from 0 and infinity: a hidden
// score of -inf times 0 and a score of 0 times infinity would be NaN.
__device__ __forceinline__ float score_factor(float scale_log2, float sk) {
    return __builtin_amdgcn_fmed3f(scale_log2 * sk, 0x1p-126f, 0x1.fffffep127f);
}
constexpr float SCALE_MIN = 0x1p-100f;  // keeps an unwritten block's scale out of log2(0)

// A row's running statistics (log2 units): the maximum of z and the sum of 2^(z -
// m); the maximum of z + log2 sv and the sum of 2^(z + log2 sv - wm + LIFT), in which
// units the row's output is.
struct alignas(16) Stat {
    float m, l, wm, lw;
};
constexpr Stat NO_KEYS{FLOOR, 0.0f, FLOOR, 0.0f};

struct AttendParams {
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    const int32_t* length;
    const int32_t* counts;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    // partial results of the splits, [B*H][splits][rows]: the output over its sum of
    // weights, and a Stat
    void* part;                   // [..][P] of T::Partial
    Stat* part_st;
    int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;
    int64_t cap, items;
    float scale_log2;
    int B, H, G, D, Q, n, causal, splits, groups, rows;
    int per_group;                // tile kernel: 32-row blocks of a group
};

// The 16 query rows of one group: row r of key head hk is query t = r / G of
// query head hk * G + r % G.
struct RowAt {
    int t, head;
    bool there;
};
__device__ __forceinline__ RowAt row_at(int row, int hk, int G, int Q) {
    const bool there = row < G * Q;
    const int r = there ? row : 0;
    return {r / G, hk * G + r % G, there};
}

// Whether a row's maxima are more than TAU behind a block's, tm and tm + lsv; where
// they are (up), catch_up moves them there and gives what the output is multiplied
// by.  (The tile kernel does it without a branch and scales its output behind the
// exponentials: with both in a branch before them 70 us instead of 63 at width 64.)
__device__ __forceinline__ bool behind(const Stat& st, float tm, float lsv) {
    return tm > st.m + TAU || tm + lsv > st.wm + TAU;
}
__device__ __forceinline__ float catch_up(Stat& st, bool up, float tm, float lsv) {
    const float m = up ? fmaxf(st.m, tm) : st.m, wm = up ? fmaxf(st.wm, tm + lsv) : st.wm;
    const float alpha = __builtin_amdgcn_exp2f(st.wm - wm);
    st.l *= __builtin_amdgcn_exp2f(st.m - m);
    st.lw *= alpha;
    st.m = m;
    st.wm = wm;
    return alpha;
}

// The queries of an item: `nq` of its Q rows, the last tokens of `len`.
struct Queries {
    int len, nq, causal;
    // keys that query t < nq sees, and any row t
    __device__ __forceinline__ int sees(int t) const { return causal ? len - nq + 1 + t : len; }
    __device__ __forceinline__ int end(int t) const { return t >= nq ? 0 : sees(t); }
    // the least and the most that any of the queries t0 .. t1 sees
    __device__ __forceinline__ int least(int t0, int t1) const { return t1 >= nq ? 0 : sees(t0); }
    __device__ __forceinline__ int most(int t0, int t1) const { return t0 >= nq ? 0 : sees(min(t1, nq - 1)); }
};
template <typename Params>
__device__ __forceinline__ Queries queries_of(const Params& p, int b) {
    return {c8_length(p.length, b, p.n), c8_length(p.counts, b, p.Q), p.causal};
}

// The work of a workgroup: a group of query rows of a unit (head and key split).
// Block i runs on XCD i % 8, and the groups of a unit take consecutive slots of
// one XCD, whose L2 then serves all but the first read of its codes.  Units go
// to the XCDs in turn, so that sequences of unlike lengths spread over them
// (whole runs of sequences to an XCD: 150 us against 137 for 32 of them); with
// fewer than UNITS units an XCD takes a run of (unit, group) pairs instead.
constexpr int UNITS = 32;

struct Item {
    uint32_t unit;
    int group;
    bool there;
};

__device__ __forceinline__ Item item_of(const AttendParams& p) {
    const uint32_t x = blockIdx.x & 7, k = blockIdx.x >> 3, groups = (uint32_t)p.groups;
    const uint32_t items = (uint32_t)p.items, units = items / groups;
    if (units >= UNITS) {
        const uint32_t u = k / groups * 8 + x;
        return {u, (int)(k % groups), u < units};
    }
    const uint32_t item = x * ((items + 7) >> 3) + k, u = item / groups;
    return {u, (int)(item - u * groups), item < items && k < (items + 7) >> 3};
}

// Operand step s of a K or Q row covers d = 64 (s / 2) + 16 g + 8 (s % 2) .. + 8
// in lane row group g (lane / 16): the same order on both sides, and one
// 16-byte piece of codes gives two steps.
template <typename T, int P>
__device__ __forceinline__ void load_q(typename T::x8 (&qf)[P / 32], const uint16_t* q, bool there,
                                       int g, int D) {
#pragma unroll
    for (int s = 0; s < P / 32; ++s) {
        const int d = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
        u32x4 w{};
        if (there && d < D) w = *reinterpret_cast<const u32x4*>(q + d);
        qf[s] = as_x8<typename T::x8>(w);
    }
}

// Eight columns of a row's result, o in units of 2^(wm - LIFT).
template <typename T>
__device__ __forceinline__ void store_row(const AttendParams& p, int b, int hk, int row, int d,
                                          const Stat& st, const float (&o)[8]) {
    const RowAt at = row_at(row, hk, p.G, p.Q);
    if (!at.there) return;
    const float f = st.l == 0.0f ? 0.0f : 1.0f / 4096.0f / st.l;
    const float u = __builtin_amdgcn_exp2f(st.wm - st.m);
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = o[k] * f * u;
    if (d < p.D)
        *reinterpret_cast<u32x4*>(p.out + b * p.o_sb + at.t * p.o_st + at.head * p.o_sh + d) =
            u32x4{T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7])};
    if (d == 0 && p.lse)
        p.lse[((int64_t)b * p.H * p.G + at.head) * p.Q + at.t] =
            st.l == 0.0f ? -INFINITY : st.m * LN2 + logf(st.l);  // (NaN for a NaN query)
}
static_assert(LIFT == 12.0f, "store_row's 4,096");

// The same as one split's partial result, the output over its sum of weights (at
// most the largest code): in fp16 for bf16 outputs, where its rounding is an eighth
// of theirs, in fp32 for fp16 ones.
template <typename T, int P>
__device__ __forceinline__ void store_partial(const AttendParams& p, int bh, int split, int row,
                                              int d, const Stat& st, const float (&o)[8]) {
    if (row >= p.rows) return;
    const int64_t i = ((int64_t)bh * p.splits + split) * p.rows + row;
    const float f = st.lw == 0.0f ? 0.0f : 1.0f / st.lw;
    if (d < P) {
        typename T::Partial x;
        x.set(o, f);
        x.store(p.part, i * P + d);
    }
    if (d == 0) p.part_st[i] = st;
}

// W waves of a workgroup share 16 query rows and a range of 64-row blocks; wave
// w takes blocks w, w + W, ... and the waves' results are merged in LDS.  A
// block costs a wave about 500 VALU instructions, most of them conversions of
// codes, so few blocks want all CUs: four waves a workgroup, and eight only
// where there is a block for each of eight waves on every CU (us with four and
// eight, 8 key heads of 4 query heads: 1 x 8,192 rows 10.8, 13.6; 8 x 2,048
// 12.5, 11.6; 32 x 1,024 16.7, 14.0; 32 x 4,096 45.3, 42.2).  Long calls are
// bound by the read of the codes: 32 ragged sequences up to 16,384 rows, 736 MB,
// 125 us, 5.9 TB/s (a kernel that only reads moves 6.5, a copy 5.1); one query over
// 2 heads of 262,144 rows, 134 MB, 25 us.  Loads issued a block ahead changed
// neither, all 24 of a block before its first product cost 4 % (K's eight are in
// flight together, V's behind them).
constexpr int64_t ROWS_EIGHT = 2048;  // blocks in all heads

template <int P, int W, int NQ>
struct RowsSmem {
    float o[W][16 * NQ][P + 4];
    Stat st[W][16 * NQ];
};

// NQ groups of 16 query rows to a wave: with more than 16 rows two, for half the
// reads and conversions of codes.
template <typename T, int FMT, int P, int W, int NQ>
__global__ void __launch_bounds__(64 * W) attend_kernel(AttendParams p) {
    constexpr int STEPS = P / 32, PIECES = P / 64, DB = P / 16, ROWS = 16 * NQ;
    using x8 = typename T::x8;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Item it = item_of(p);
    if (!it.there) return;
    const int rg = it.group, bh = (int)(it.unit / (uint32_t)p.splits);
    const int split = (int)(it.unit - (uint32_t)bh * p.splits), b = bh / p.H, hk = bh - b * p.H;
    const Queries qs = queries_of(p, b);
    const int len = qs.len;
    const int row0 = rg * ROWS;
    // blocks that some row of the group sees, and keys that every row does
    const int t0 = row0 / p.G, t1 = min(row0 + ROWS - 1, p.rows - 1) / p.G;
    const int last = max(0, qs.most(t0, t1)), first = qs.least(t0, t1);
    const int nb = (last + C8_BLOCK - 1) / C8_BLOCK;
    const int b0 = (int)((int64_t)split * nb / p.splits);
    const int b1 = (int)((int64_t)(split + 1) * nb / p.splits);
    x8 qf[NQ][STEPS];
    int end[NQ];                              // keys that the lane's row sees
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const RowAt mine = row_at(row0 + 16 * n + r, hk, p.G, p.Q);
        end[n] = mine.there ? qs.end(mine.t) : 0;
        load_q<T, P>(qf[n], p.q + b * p.q_sb + mine.t * p.q_st + mine.head * p.q_sh, mine.there, g,
                     p.D);
    }
    const uint8_t* kbase = p.k + ((int64_t)bh * p.cap + r) * P + 16 * g;
    const uint8_t* vbase = p.v + ((int64_t)bh * p.cap + 4 * g) * P + DB * r;
    const float* ks = p.ks + (int64_t)bh * (p.cap / C8_BLOCK);
    const float* vs = p.vs + (int64_t)bh * (p.cap / C8_BLOCK);
    f32x4 o[NQ][DB];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < DB; ++i) o[n][i] = f32x4{};
    // the maxima of the lane's row, the sums over its own keys; o holds the sum of
    // the weights times the codes
    Stat st[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) st[n] = NO_KEYS;
    for (int blk = b0 + wave; blk < b1; blk += W) {
        const int64_t key0 = (int64_t)blk * C8_BLOCK;
        u32x4 kr[4][PIECES];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                kr[t][i] = *reinterpret_cast<const u32x4*>(kbase + (key0 + 16 * t) * P + 64 * i);
        // (K's loads before V's: the scores wait for them alone; 30.4 us without the
        // fence for the long call, 29.6 with it)
        __builtin_amdgcn_sched_barrier(0);
        // V: lane (r, g) holds columns DB r .. + DB of the keys that its weights
        // are of: 32 c + 16 a + 4 g + j
        uint32_t vr[2][8][DB / 4];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint8_t* at = vbase + (key0 + 32 * c + 16 * (j >> 2) + (j & 3)) * P;
                if constexpr (DB == 8) {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(at);
                    vr[c][j][0] = w[0];
                    vr[c][j][1] = w[1];
                } else {
                    vr[c][j][0] = *reinterpret_cast<const uint32_t*>(at);
                }
            }
        const float sk = fmaxf(ks[blk], SCALE_MIN), sv = fmaxf(vs[blk], SCALE_MIN);
        f32x4 s[NQ][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[n][t] = f32x4{};
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const x8 a = codes_x8<T, FMT>(kr[t][i][0], kr[t][i][1]);
                const x8 c = codes_x8<T, FMT>(kr[t][i][2], kr[t][i][3]);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    s[n][t] = T::mfma16(a, qf[n][2 * i], s[n][t]);
                    s[n][t] = T::mfma16(c, qf[n][2 * i + 1], s[n][t]);
                }
            }
        }
        if (key0 + C8_BLOCK > first) {
            // scores of unseen keys; s[n][t][e] is of key 16 t + 4 g + e
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int seen = end[n] - (int)key0;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * t + 4 * g + e >= seen) s[n][t][e] = -INFINITY;
            }
            // rows at or past the length may hold NaN codes, which a zero weight
            // does not remove
            const int valid = len - (int)key0;
            if (FMT == NKV_CACHE8_E4M3 && valid < C8_BLOCK) {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (32 * c + 16 * (j >> 2) + 4 * g + (j & 3) >= valid)
#pragma unroll
                            for (int w = 0; w < DB / 4; ++w) vr[c][j][w] = 0;
            }
        }
        const float c = score_factor(p.scale_log2, sk), lsv = __builtin_amdgcn_logf(sv);
        uint32_t pw[NQ][2][4];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float tm = s[n][0][0];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) tm = fmaxf(tm, s[n][t][e]);
            tm = rows4_max(tm) * c;
            const bool up = behind(st[n], tm, lsv);
            if (__any(up)) {
                const float alpha = catch_up(st[n], up, tm, lsv);
#pragma unroll
                for (int i = 0; i < DB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][i][e] *= alpha;
            }
            const float apart = fminf(st[n].wm - lsv - st[n].m, QUIET) - LIFT;
            const float off = st[n].m + apart;
            float lsum = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(fmaf(s[n][t][e], c, -off));
                    lsum += w[e];
                }
                pw[n][t >> 1][2 * (t & 1)] = Fp16::pack(w[0], w[1]);
                pw[n][t >> 1][2 * (t & 1) + 1] = Fp16::pack(w[2], w[3]);
            }
            st[n].l += lsum * __builtin_amdgcn_exp2f(apart);
            st[n].lw += lsum;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int w = 0; w < DB / 4; ++w) {
                uint32_t pairs[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    column_pairs<FMT>(vr[k][2 * j][w], vr[k][2 * j + 1][w], pairs[j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x8 vf =
                        as_x8<f16x8>(u32x4{pairs[0][e], pairs[1][e], pairs[2][e], pairs[3][e]});
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
                        o[n][4 * w + e] = Fp16::mfma16(
                            vf, as_x8<f16x8>(u32x4{pw[n][k][0], pw[n][k][1], pw[n][k][2], pw[n][k][3]}),
                            o[n][4 * w + e]);
                }
            }
    }
    // merge of the waves: o[n][i][e] is column DB (4 g + e) + i of row 16 n + r
    extern __shared__ __align__(16) unsigned char rows_smem[];
    RowsSmem<P, W, NQ>& sm = *reinterpret_cast<RowsSmem<P, W, NQ>*>(rows_smem);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < DB; i += 4)
                *reinterpret_cast<f32x4*>(&sm.o[wave][16 * n + r][DB * (4 * g + e) + i]) =
                    f32x4{o[n][i][e], o[n][i + 1][e], o[n][i + 2][e], o[n][i + 3][e]};
        st[n].l = rows4_sum(st[n].l);
        st[n].lw = rows4_sum(st[n].lw);
        if (g == 0) sm.st[wave][16 * n + r] = st[n];
    }
    __syncthreads();
    if (threadIdx.x >= 16 * ROWS) return;
    for (int mr = threadIdx.x / 16; mr < ROWS; mr += 4 * W) {
        const int d = (threadIdx.x % 16) * 8;
        Stat all = NO_KEYS;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            all.m = fmaxf(all.m, sm.st[w][mr].m);
            all.wm = fmaxf(all.wm, sm.st[w][mr].wm);
        }
        float acc[8] = {};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const Stat one = sm.st[w][mr];
            all.l += __builtin_amdgcn_exp2f(one.m - all.m) * one.l;
            const float f = __builtin_amdgcn_exp2f(one.wm - all.wm);
            all.lw += f * one.lw;
            if (d < P)
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] += f * sm.o[w][mr][d + i];
        }
        const int row = row0 + mr;
        if (p.splits > 1) store_partial<T, P>(p, bh, split, row, d, all, acc);
        else store_row<T>(p, b, hk, row, d, all, acc);
    }
}

// ---------------------------------------------------------------- many rows
// Eight waves of 32 query rows each share every block of 64 keys: the
// workgroup loads its codes into registers a block ahead, converts them once
// and leaves K rows and V columns in LDS as MFMA operands, double-buffered,
// with one barrier a block.  S^T = K Q^T puts a query in a lane's column (16 of
// the scores of each 32 keys, the other 16 in lane ^ 32), and its weights are
// then the operand of O^T += V^T W^T without leaving the registers.
//
// LDS: K row k at 2 P k, its 16-byte chunk c at c ^ (k mod chunks); V^T row of
// column d at 128 R, R = d with bits 2 and 3 swapped (a lane's results are then
// eight consecutive columns), its chunk 4 j + 2 s + h (keys of 32-key half j,
// product s, lane half h) at chunk ^ vsw(R): reads of eight consecutive rows,
// and writes of every fourth row, meet eight different chunks.
//
// 1,560 queries over 12,480 rows of 24 heads: 239 GFLOP in 268 - 286 us over several
// cards, 840 - 890 TFLOP/s (a large bf16 product reaches 1,337).  MFMAs are busy for
// 36 % of the SIMDs' cycles and the other VALU instructions (softmax, conversions,
// addresses) for 53 %, at 2.3 of 2.4 GHz: the two waves a SIMD run them beside each
// other too little.  Orders of the same work (scores a block ahead, operands read
// ahead, one or two chains of products, priorities or none) took 290 - 294 us all;
// without LDS operand reads 15 % less.  Width 64 has half the products for the same
// softmax (31 GFLOP in 62 us: MFMA 19 %, VALU 41 %; sequences of unlike lengths
// leave part of the chip idle) and one workgroup a CU (128 registers, for two,
// spill).
constexpr int TILE_WAVES = 8;

__device__ __forceinline__ int vsw(int R) { return ((R >> 2) ^ ((R & 3) << 1)) & 7; }

template <typename T, int FMT, int P>
struct TileCodes {
    static constexpr int CH = P / 8;                     // chunks of a K row
    static constexpr int K_BYTES = C8_BLOCK * P * 2, V_BYTES = P * C8_BLOCK * 2;
    static constexpr int SMEM = 2 * K_BYTES + 3 * V_BYTES;
    u32x4 k;
    uint32_t v[4];
    float sk, sv;                                        // the block's scales
    // P = 128: every thread brings 16 bytes of K and 4 x 4 bytes of V; P = 64:
    // the first half of the workgroup K, the other V
    static __device__ __forceinline__ bool has_k() { return P == 128 || threadIdx.x < 256; }
    static __device__ __forceinline__ bool has_v() { return P == 128 || threadIdx.x >= 256; }
    static __device__ __forceinline__ int kt() { return threadIdx.x; }
    static __device__ __forceinline__ int vt() { return P == 128 ? threadIdx.x : threadIdx.x - 256; }

    // block blk of a head, whose first row is kb, vb.  The scales come along: a
    // load where they are used would wait for the next block's codes with it.
    __device__ __forceinline__ void load(const uint8_t* kb, const uint8_t* vb, const float* ks,
                                         const float* vs, int blk) {
        const int64_t key0 = (int64_t)blk * C8_BLOCK;
        sk = ks[blk];
        sv = vs[blk];
        if (has_k())
            k = *reinterpret_cast<const u32x4*>(kb + (key0 + kt() / (P / 16)) * P + 16 * (kt() % (P / 16)));
        if (has_v())
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = *reinterpret_cast<const uint32_t*>(vb + (key0 + 4 * (vt() / (P / 4)) + i) * P +
                                                          4 * (vt() % (P / 4)));
    }
    // valid: the block's rows below the length; V rows past it become zero
    // (they may hold NaN, which a zero weight does not remove)
    __device__ __forceinline__ void store(unsigned char* kd, unsigned char* vd, int valid) {
        if (has_k()) {
            const int row = kt() / (P / 16), c = 2 * (kt() % (P / 16)), x = row & (CH - 1);
            unsigned char* at = kd + row * 2 * P;
            *reinterpret_cast<typename T::x8*>(at + 16 * (c ^ x)) = codes_x8<T, FMT>(k[0], k[1]);
            *reinterpret_cast<typename T::x8*>(at + 16 * ((c + 1) ^ x)) = codes_x8<T, FMT>(k[2], k[3]);
        }
        if (has_v()) {
            const int kq = vt() / (P / 4), dq = vt() % (P / 4);
            if (valid < C8_BLOCK)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * kq + i >= valid) v[i] = 0;
            const int R0 = 4 * ((dq & ~3) | ((dq & 1) << 1) | ((dq >> 1) & 1));
            const int q = kq & 7, chunk = 4 * (kq >> 3) + 2 * (q >> 2) + (q & 1), half = (q >> 1) & 1;
            uint32_t lo[4], hi[4];
            column_pairs<FMT>(v[0], v[1], lo);
            column_pairs<FMT>(v[2], v[3], hi);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<u32x2*>(vd + (R0 + c) * 128 + 16 * (chunk ^ vsw(R0 + c)) +
                                          8 * half) = u32x2{lo[c], hi[c]};
        }
    }
};

template <typename T, int FMT, int P>
__global__ void __launch_bounds__(64 * TILE_WAVES) attend_tile_kernel(AttendParams p) {
    constexpr int KS = P / 16, DB = P / 32;
    using x8 = typename T::x8;
    using Codes = TileCodes<T, FMT, P>;
    extern __shared__ __align__(16) unsigned char smem[];  // TileCodes::SMEM
    const int lane = threadIdx.x & 63, hf = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Item it = item_of(p);
    if (!it.there) return;
    const uint32_t BH = (uint32_t)(p.B * p.H);
    const int rg = it.group, split = (int)(it.unit / BH);
    const int bh = (int)(it.unit - split * BH), b = bh / p.H, hk = bh - b * p.H;
    const Queries qs = queries_of(p, b);
    const int len = qs.len;
    const int row0 = rg * p.per_group * 32;
    const int rows_end = min(row0 + p.per_group * 32, p.rows);
    // keys that some row of the group sees
    const int last = max(0, qs.most(row0 / p.G, (rows_end - 1) / p.G));
    const int nb = (last + C8_BLOCK - 1) / C8_BLOCK;
    const int b0 = (int)((int64_t)split * nb / p.splits);
    const int b1 = (int)((int64_t)(split + 1) * nb / p.splits);
    const int wrow = row0 + 32 * wave, row = wrow + l32;
    const bool active = wrow < rows_end;
    const RowAt mine = row_at(row, hk, p.G, p.Q);
    const int end = mine.there ? qs.end(mine.t) : 0;
    const int t0 = wrow / p.G, t1 = (min(wrow + 32, p.rows) - 1) / p.G;
    const int first = qs.least(t0, t1), wlast = qs.most(t0, t1);  // of the wave
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
    const uint8_t* kb = p.k + (int64_t)bh * p.cap * P;
    const uint8_t* vb = p.v + (int64_t)bh * p.cap * P;
    const float* ks = p.ks + (int64_t)bh * (p.cap / C8_BLOCK);
    const float* vs = p.vs + (int64_t)bh * (p.cap / C8_BLOCK);
    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x16{};
    Stat st = NO_KEYS;
    Codes codes;
    float sk = 1.0f, sv = 1.0f;  // scales of the current block
    if (b0 < b1) {
        codes.load(kb, vb, ks, vs, b0);
        codes.store(smem, smem + 2 * Codes::K_BYTES, len - b0 * C8_BLOCK);
        sk = codes.sk, sv = codes.sv;
        codes.load(kb, vb, ks, vs, min(b0 + 1, b1 - 1));
    }
    // the queries have arrived before the loop: a wait for them inside would
    // wait for the codes in flight
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));
    // this lane's operand offsets in the current slots (kept in registers)
    uint32_t kofs[KS], vofs[4];
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
        kofs[kk] = l32 * 2 * P + 16 * ((2 * kk + hf) ^ (l32 & (Codes::CH - 1)));
        asm volatile("" : "+v"(kofs[kk]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        vofs[i] = 2 * Codes::K_BYTES + l32 * 128 + 16 * ((2 * i + hf) ^ vsw(l32));
        asm volatile("" : "+v"(vofs[i]));
    }
    lds_barrier();
    // Waves w and w + 4 share a SIMD.  Waves 4-7 meet a block's barrier before
    // its softmax, waves 0-3 after it, so that one's softmax runs beside the
    // other's products.  At barrier i every wave has stored its part of block
    // i + 1 and is done with K of block i and V of block i - 1: two slots for
    // K and three for V.
    const bool lag = wave >= TILE_WAVES / 2;
    int slot = 0;  // V's
    for (int blk = b0; blk < b1; ++blk) {
        const int key0 = blk * C8_BLOCK, kslot = (blk - b0) & 1;
        const int next = slot == 2 ? 0 : slot + 1;
        const bool work = active && key0 < wlast;
        f32x16 s[2];
        if (work) {
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
                    s[j] = T::mfma32(*reinterpret_cast<const x8*>(smem + kofs[kk] + j * 64 * P), qf[kk],
                                     kk ? s[j] : f32x16{});
            __builtin_amdgcn_s_setprio(0);
        }
        const float c = score_factor(p.scale_log2, fmaxf(sk, SCALE_MIN));
        const float lsv = __builtin_amdgcn_logf(fmaxf(sv, SCALE_MIN));
        // block blk + 1 (behind the last, the last again, for no one)
        codes.store(smem + (kslot ^ 1) * Codes::K_BYTES,
                    smem + 2 * Codes::K_BYTES + next * Codes::V_BYTES,
                    len - min(key0 + C8_BLOCK, (b1 - 1) * C8_BLOCK));
        sk = codes.sk, sv = codes.sv;
        codes.load(kb, vb, ks, vs, min(blk + 2, b1 - 1));
        if (lag) lds_barrier();
        if (work) {
            if (key0 + C8_BLOCK > first) {
                const int seen = end - key0;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (32 * j + 8 * (i >> 2) + 4 * hf + (i & 3) >= seen) s[j][i] = -INFINITY;
            }
            float tm = s[0][0];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) tm = fmaxf(tm, s[j][i]);
            tm = halfwave_max(tm) * c;
            const bool up = behind(st, tm, lsv);
            const float alpha = catch_up(st, up, tm, lsv);
            const float apart = fminf(st.wm - lsv - st.m, QUIET) - LIFT;
            const float off = st.m + apart;
            float lsum = 0.0f;
            uint32_t pw[2][8];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float w0 = __builtin_amdgcn_exp2f(fmaf(s[j][i], c, -off));
                    const float w1 = __builtin_amdgcn_exp2f(fmaf(s[j][i + 1], c, -off));
                    lsum += w0 + w1;
                    pw[j][i >> 1] = Fp16::pack(w0, w1);
                }
            st.l += lsum * __builtin_amdgcn_exp2f(apart);
            st.lw += lsum;
            __builtin_amdgcn_s_setprio(1);
            if (__any(up)) {
#pragma unroll
                for (int i = 0; i < DB; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const f16x8 pf = as_x8<f16x8>(
                        u32x4{pw[j][4 * k], pw[j][4 * k + 1], pw[j][4 * k + 2], pw[j][4 * k + 3]});
#pragma unroll
                    for (int i = 0; i < DB; ++i)
                        o[i] = Fp16::mfma32(
                            *reinterpret_cast<const f16x8*>(smem + vofs[2 * j + k] + i * 4096), pf, o[i]);
                }
            __builtin_amdgcn_s_setprio(0);
        }
        const uint32_t kstep = kslot ? -Codes::K_BYTES : Codes::K_BYTES;
        const uint32_t vstep = slot == 2 ? -2 * Codes::V_BYTES : Codes::V_BYTES;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            kofs[kk] += kstep;
            asm volatile("" : "+v"(kofs[kk]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            vofs[i] += vstep;
            asm volatile("" : "+v"(vofs[i]));
        }
        slot = next;
        if (!lag) lds_barrier();
    }
    st.l = halfwave_sum(st.l);
    st.lw = halfwave_sum(st.lw);
    if (!active) return;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 32 * i + 16 * e + 8 * hf;
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = o[i][8 * e + k];
            if (p.splits > 1) store_partial<T, P>(p, bh, split, row, d, st, x);
            else store_row<T>(p, b, hk, row, d, st, x);
        }
}

// The merge of the splits' partial results: P / 8 threads a row and group of
// splits, eight columns each; with M and W the largest m and wm, out = 2^(W - M - LIFT)
// sum(2^(wm - W) lw o) / sum(2^(m - M) l).
// SG groups share a row's splits and are joined in LDS; a thread has AHEAD
// splits' loads in flight.  37,440 rows of 3 splits (30 MB) 7.8 us, 16 rows of 256
// 4.6 us (309 us with one thread walking all of a row's splits).
template <typename T, int P, int SG, int AHEAD>
__global__ void __launch_bounds__(256) merge_kernel(AttendParams p) {
    constexpr int PARTS = P / 8, ROWS = 256 / (PARTS * SG);
    const int row = blockIdx.x * ROWS + threadIdx.x / (PARTS * SG);
    const int sg = threadIdx.x / PARTS % SG, d = (threadIdx.x % PARTS) * 8;
    const int b = blockIdx.z, hk = blockIdx.y;
    const bool in = row < p.rows;
    const int64_t first = ((int64_t)b * p.H + hk) * p.splits * p.rows + row;
    Stat all = NO_KEYS;
    float acc[8] = {};
    // (a thread without splits, or with those of no keys, adds zeros)
    auto grow = [&](float m, float wm) {
        const float f = __builtin_amdgcn_exp2f(all.wm - wm);
        all.l *= __builtin_amdgcn_exp2f(all.m - m);
        all.m = m;
        all.wm = wm;
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] *= f;
    };
    if (in) {
        for (int s0 = sg; s0 < p.splits; s0 += SG * AHEAD) {
            Stat st[AHEAD];
            typename T::Partial x[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int s = min(s0 + SG * j, p.splits - 1);
                const int64_t i = first + (int64_t)s * p.rows;
                st[j] = p.part_st[i];
                x[j].load(p.part, i * P + d);
                if (s0 + SG * j >= p.splits) st[j] = NO_KEYS;
            }
            float m1 = all.m, w1 = all.wm;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                m1 = fmaxf(m1, st[j].m);
                w1 = fmaxf(w1, st[j].wm);
            }
            grow(m1, w1);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                all.l += __builtin_amdgcn_exp2f(st[j].m - all.m) * st[j].l;
                const float f = __builtin_amdgcn_exp2f(st[j].wm - all.wm) * st[j].lw;
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] += f * x[j][k];
            }
        }
    }
    if constexpr (SG > 1) {
        __shared__ float sh[ROWS][SG][PARTS][8];
        __shared__ float sml[ROWS][SG][3];
        const int lr = threadIdx.x / (PARTS * SG), part = threadIdx.x % PARTS;
#pragma unroll
        for (int k = 0; k < 8; ++k) sh[lr][sg][part][k] = acc[k];
        if (part == 0) {
            sml[lr][sg][0] = all.m;
            sml[lr][sg][1] = all.l;
            sml[lr][sg][2] = all.wm;
        }
        __syncthreads();
        if (sg) return;
#pragma unroll
        for (int s = 0; s < SG; ++s) {
            all.m = fmaxf(all.m, sml[lr][s][0]);
            all.wm = fmaxf(all.wm, sml[lr][s][2]);
        }
        all.l = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
#pragma unroll
        for (int s = 0; s < SG; ++s) {
            all.l += __builtin_amdgcn_exp2f(sml[lr][s][0] - all.m) * sml[lr][s][1];
            const float f = __builtin_amdgcn_exp2f(sml[lr][s][2] - all.wm);
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += f * sh[lr][s][part][k];
        }
    }
    if (in) store_row<T>(p, b, hk, row, d, all, acc);
}

// ---------------------------------------------------------------- mass
struct MassParams {
    const uint8_t* k;
    const float* ks;
    const int32_t* length;
    const int32_t* counts;
    const uint16_t* q;
    const float* lse;
    const float* mass;
    float* out;
    float* part;                  // [splits][B*H][n64] sums of the row splits
    int64_t q_sb, q_st, q_sh;
    int64_t cap, n64;             // n64: n in whole blocks
    float scale_log2;
    int B, H, G, D, Q, n, causal, rows, splits, blocks, per;
};

// Sums over lanes of many values at once: each step adds two half-sized sets of
// partial sums across lanes, a lane keeping the set that one bit of its number
// names, until lane r of 16 (32) has the sum of v[r].  The exchanges are DPP and
// permlane moves in the VALU; through LDS (__shfl_xor) they took 10 us of a
// 25 us call over 8 ragged sequences.
template <int CTRL>
__device__ __forceinline__ float dpp_from(float x) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, true));
}

template <int H, int CTRL>
__device__ __forceinline__ void reduce_step(float* v, bool upper) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
        const float give = upper ? v[i] : v[i + H], keep = upper ? v[i + H] : v[i];
        v[i] = keep + dpp_from<CTRL>(give);
    }
}

// over the 16 lanes of a row: partners l ^ 8, l ^ 7, l ^ 2, l ^ 1
__device__ __forceinline__ float reduce16(float* v, int r) {
    reduce_step<8, 0x128>(v, r & 8);   // row_ror:8
    reduce_step<4, 0x141>(v, r & 4);   // row_half_mirror
    reduce_step<2, 0x4e>(v, r & 2);    // quad_perm:[2,3,0,1]
    reduce_step<1, 0xb1>(v, r & 1);    // quad_perm:[1,0,3,2]
    return v[0];
}

// over the 32 lanes of a half wave: the swap leaves one value's two rows in the
// even row of the pair and the other's in the odd one
__device__ __forceinline__ float reduce32(float* v, int l32) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]),
                                                        __float_as_uint(v[i + 16]), false, false);
        v[i] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
    return reduce16(v, l32 & 15);
}

// The result of one block's row i: the sum goes to this split's partial sums, or
// with one split on top of the mass.
__device__ __forceinline__ void mass_store(const MassParams& p, int bh, int64_t row, int len,
                                           int split, float x) {
    const int64_t at = (int64_t)bh * p.cap + row;
    if (p.splits > 1) {
        if (row < len) p.part[((int64_t)split * p.B * p.H + bh) * p.n64 + row] = x;
    } else if (row < len) {
        p.out[at] = p.mass[at] + x;
    } else if (p.out != p.mass) {
        p.out[at] = p.mass[at];
    }
}

// Waves from which on a wave takes several blocks (8 ragged sequences of 8 heads
// up to 8,192 rows: 15.6 us with one block a wave, 14.6, 12.6 and 17.1 with
// 4,096, 2,048 and 1,024 waves).
constexpr int64_t MASS_WAVES = 2048;

// Few query rows: a wave holds a block of 64 cached rows (four tiles of 16 keys)
// and takes the groups of 16 query rows in turn; the sums over queries stay in
// registers until the block's end.  Bound by the read of K.  A wave has p.per
// blocks, 4 apart, the next one's codes loaded behind the last use of this one's.
template <typename T, int FMT, int P>
__global__ void __launch_bounds__(256) mass_kernel(MassParams p) {
    constexpr int STEPS = P / 32, PIECES = P / 64;
    using x8 = typename T::x8;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bh = blockIdx.y, b = bh / p.H, hk = bh - b * p.H;
    const Queries qs = queries_of(p, b);
    const int len = qs.len;
    // the row whose sum this lane ends up with, of tile r / 4
    const int mykey = 16 * (r >> 2) + 4 * g + (r & 3);
    const int64_t head = (int64_t)bh * p.cap;
    const float* ks = p.ks + (int64_t)bh * (p.cap / C8_BLOCK);
    const int groups = max(1, (qs.nq * p.G + 15) / 16);
    x8 qf[STEPS];
    float z;
    int end;
    auto load_group = [&](int rg) {
        const RowAt mine = row_at(rg * 16 + r, hk, p.G, qs.nq);
        end = mine.there ? qs.sees(mine.t) : 0;
        load_q<T, P>(qf, p.q + b * p.q_sb + mine.t * p.q_st + mine.head * p.q_sh, mine.there, g, p.D);
        z = mine.there ? p.lse[((int64_t)b * p.H * p.G + mine.head) * p.Q + mine.t] : -INFINITY;
    };
    int blk = blockIdx.x * 4 * p.per + wave;
    const int blk1 = min(p.blocks, (int)(blockIdx.x + 1) * 4 * p.per);
    const int seen = (len + C8_BLOCK - 1) / C8_BLOCK;   // blocks below the length
    u32x4 kr[4][PIECES];
    float sk, before;
    auto load_block = [&](int k) {
        const int64_t at = head + (int64_t)k * C8_BLOCK;
        before = p.mass[at + mykey];
        sk = ks[k];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                kr[t][i] = *reinterpret_cast<const u32x4*>(p.k + (at + 16 * t + r) * P + 64 * i + 16 * g);
    };
    if (blk < min(blk1, seen)) {
        load_block(blk);
        if (groups == 1) load_group(0);
    }
    for (; blk < min(blk1, seen); blk += 4) {
        const int key0 = blk * C8_BLOCK;
        const float c = score_factor(p.scale_log2, fmaxf(sk, SCALE_MIN));
        // the first group with a row that sees the block's first key
        int rg = 0;
        if (p.causal)
            rg = (int)min((int64_t)max(0, key0 - (len - qs.nq)) * p.G / 16, (int64_t)groups - 1);
        f32x4 sum[4] = {};
        for (;;) {
            if (groups > 1) load_group(rg);
            const bool adds = fabsf(z) < INFINITY;      // (a NaN query's lse is NaN)
            const float off = adds ? z * LOG2E : 0.0f;
            const int seen_to = adds ? end : 0;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                f32x4 s{};
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    s = T::mfma16(codes_x8<T, FMT>(kr[t][i][0], kr[t][i][1]), qf[2 * i], s);
                    s = T::mfma16(codes_x8<T, FMT>(kr[t][i][2], kr[t][i][3]), qf[2 * i + 1], s);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(s[e], c, -off));
                    sum[t][e] += key0 + 16 * t + 4 * g + e < seen_to ? w : 0.0f;
                }
            }
            if (++rg >= groups) break;
        }
        const float first = before;
        if (blk + 4 < min(blk1, seen)) load_block(blk + 4);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = sum[i >> 2][i & 3];
        const float x = reduce16(v, r);
        const int64_t at = head + key0 + mykey;
        if (key0 + mykey < len) p.out[at] = first + x;
        else if (p.out != p.mass) p.out[at] = first;
    }
    if (p.out != p.mass)
        for (; blk < blk1; blk += 4) {
            const int64_t at = head + (int64_t)blk * C8_BLOCK + mykey;
            p.out[at] = p.mass[at];
        }
}

// Many query rows: four waves hold a block of 64 cached rows each (two tiles of
// 32 keys) and share the queries, 64 rows a step, through LDS (double-buffered,
// loaded into registers a step ahead, one barrier a step): read by every wave
// from the cache, they would take all of its bandwidth.  Rows are split over
// workgroups where there are few blocks of keys.  1,560 queries over 12,480 rows
// of 24 heads: 120 GFLOP in 150 us, 800 TFLOP/s, with MFMAs busy for 33 % of the
// SIMDs' cycles and the other VALU instructions (exponentials and sums) for 50 %, two
// waves a SIMD (scores held a step ahead to run the two together spill: 258 us).
constexpr int MT_ROWS = 64;

template <typename T, int P>
struct MassRows {
    static constexpr int CH = P / 8, PER = CH / 4;      // chunks of a row, a thread's
    u32x4 q[PER];
    float off;
    int end;
    // rows row0 .. + 64: thread t brings chunks t % 4 + 4 i of row t / 4
    __device__ __forceinline__ void load(const MassParams& p, const Queries& qs, int b, int hk, int row0) {
        const int part = threadIdx.x & 3;
        const RowAt at = row_at(row0 + (threadIdx.x >> 2), hk, p.G, qs.nq);
        const uint16_t* src = p.q + b * p.q_sb + at.t * p.q_st + at.head * p.q_sh;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int d = 8 * (part + 4 * i);
            q[i] = u32x4{};
            if (at.there && d < p.D) q[i] = *reinterpret_cast<const u32x4*>(src + d);
        }
        off = at.there ? p.lse[((int64_t)b * p.H * p.G + at.head) * p.Q + at.t] : -INFINITY;
        end = qs.sees(at.t);
    }
    // a row whose lse is not finite becomes zeros with weight 2^-inf
    __device__ __forceinline__ void store(unsigned char* buf, float* offs, int* ends) {
        const int row = threadIdx.x >> 2, part = threadIdx.x & 3;
        const bool adds = fabsf(off) < INFINITY;
        if (!adds)
#pragma unroll
            for (int i = 0; i < PER; ++i) q[i] = u32x4{};
#pragma unroll
        for (int i = 0; i < PER; ++i)
            *reinterpret_cast<u32x4*>(buf + row * 2 * P + 16 * ((part + 4 * i) ^ (row & (CH - 1)))) = q[i];
        if (part == 0) {
            offs[row] = adds ? off * LOG2E : INFINITY;
            ends[row] = end;
        }
    }
};

template <typename T, int FMT, int P>
__global__ void __launch_bounds__(256, 2) mass_tile_kernel(MassParams p) {
    constexpr int KS = P / 16, CH = P / 8;
    using x8 = typename T::x8;
    __shared__ __align__(16) unsigned char smem[2][MT_ROWS * P * 2];
    __shared__ float offs[2][MT_ROWS];
    __shared__ int ends[2][MT_ROWS];
    const int lane = threadIdx.x & 63, hf = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bh = blockIdx.y, b = bh / p.H, hk = bh % p.H, split = blockIdx.z;
    const Queries qs = queries_of(p, b);
    const int len = qs.len;
    const int first_key = blockIdx.x * 4 * C8_BLOCK;    // of the workgroup
    const int blk = blockIdx.x * 4 + wave, key0 = blk * C8_BLOCK;
    if (first_key >= len) {
        if (blk < p.blocks) mass_store(p, bh, (int64_t)key0 + lane, len, split, 0.0f);
        return;
    }
    const int64_t kblk = min(blk, (len - 1) / C8_BLOCK);  // a block that is there
    x8 kf[2][KS];
    {
        const uint8_t* src = p.k + ((int64_t)bh * p.cap + kblk * C8_BLOCK + l32) * P + 16 * hf;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(src + 32 * t * P + 32 * i);
                kf[t][2 * i] = codes_x8<T, FMT>(w[0], w[1]);
                kf[t][2 * i + 1] = codes_x8<T, FMT>(w[2], w[3]);
            }
    }
    const float c =
        score_factor(p.scale_log2, fmaxf(p.ks[(int64_t)bh * (p.cap / C8_BLOCK) + kblk], SCALE_MIN));
    f32x16 sum[2] = {};
    // steps with a row that sees the workgroup's first key, this split's share
    const int steps = (qs.nq * p.G + MT_ROWS - 1) / MT_ROWS;
    int s0 = 0;
    if (p.causal) s0 = min((int64_t)steps, (int64_t)max(0, first_key - (len - qs.nq)) * p.G / MT_ROWS);
    const int st0 = s0 + (int)((int64_t)split * (steps - s0) / p.splits);
    const int st1 = s0 + (int)((int64_t)(split + 1) * (steps - s0) / p.splits);
    if (st0 < st1) {
        MassRows<T, P> rows;
        rows.load(p, qs, b, hk, st0 * MT_ROWS);
        rows.store(smem[0], offs[0], ends[0]);
        rows.load(p, qs, b, hk, min(st0 + 1, st1 - 1) * MT_ROWS);
        uint32_t qofs[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s)
            qofs[s] = l32 * 2 * P + 16 * ((4 * (s >> 1) + 2 * hf + (s & 1)) ^ (l32 & (CH - 1)));
        lds_barrier();
        for (int st = st0; st < st1; ++st) {
            const int cur = (st - st0) & 1;
            // what the step's first row sees
            const int first = qs.sees(st * MT_ROWS / p.G);
            const bool masked = key0 + C8_BLOCK > first;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                f32x16 s[2];
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const x8 qf = *reinterpret_cast<const x8*>(&smem[cur][qofs[i] + u * 64 * P]);
                    s[0] = T::mfma32(kf[0][i], qf, i ? s[0] : f32x16{});
                    s[1] = T::mfma32(kf[1][i], qf, i ? s[1] : f32x16{});
                }
                const float off = offs[cur][32 * u + l32];
                if (masked) {
                    const int seen = ends[cur][32 * u + l32] - key0;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float w = __builtin_amdgcn_exp2f(fmaf(s[t][e], c, -off));
                            sum[t][e] += 32 * t + 8 * (e >> 2) + 4 * hf + (e & 3) < seen ? w : 0.0f;
                        }
                } else {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            sum[t][e] += __builtin_amdgcn_exp2f(fmaf(s[t][e], c, -off));
                }
            }
            rows.store(smem[cur ^ 1], offs[cur ^ 1], ends[cur ^ 1]);
            rows.load(p, qs, b, hk, min(st + 2, st1 - 1) * MT_ROWS);
            lds_barrier();
        }
    }
    if (blk >= p.blocks) return;
    // value i is sum[i / 16][i % 16], of key 32 (i / 16) + 8 (i % 16 / 4) + 4 hf +
    // i % 4; lane l32 ends up with value l32
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = sum[i >> 4][i & 15];
    const float x = reduce32(v, l32);
    const int e = l32 & 15;
    mass_store(p, bh, (int64_t)key0 + 32 * (l32 >> 4) + 8 * (e >> 2) + 4 * hf + (e & 3), len, split, x);
}

// Joins the row splits' partial sums, in their order.  (With n = 0 it copies mass to
// out: the weight of no queries.)
__global__ void __launch_bounds__(256) mass_join_kernel(MassParams p) {
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int bh = blockIdx.y;
    if (row >= (int64_t)p.blocks * C8_BLOCK) return;
    const int len = c8_length(p.length, bh / p.H, p.n);
    const int64_t at = (int64_t)bh * p.cap + row;
    if (row >= len) {
        if (p.out != p.mass) p.out[at] = p.mass[at];
        return;
    }
    float x = 0.0f;
    for (int s = 0; s < p.splits; ++s) x += p.part[((int64_t)s * p.B * p.H + bh) * p.n64 + row];
    p.out[at] = p.mass[at] + x;
}

// ---------------------------------------------------------------- host
int check_query(const nkv_cache8& c, int G, int dtype, int64_t Q, int64_t n, float scale,
                const void* q, int64_t sb, int64_t st, int64_t sh, const char* who) {
    auto bad = [&](int code, const char* what) {
        set_error(std::string(who) + ": " + what);
        return code;
    };
    int rc = cache8_check(&c, who);
    if (rc) return rc;
    if (G < 1 || Q < 0) return bad(NKV_ERR_INVALID, "G must be positive and Q not negative");
    if (Q * G > INT32_MAX / 2 || Q > INT32_MAX / 2 || (int64_t)c.H * G > INT32_MAX)
        return bad(NKV_ERR_UNSUPPORTED, "too many query rows");
    if (dtype != NKV_ROWS_BF16 && dtype != NKV_ROWS_FP16)
        return bad(NKV_ERR_INVALID, "queries must be bf16 or fp16");
    if (c.H > 65535 || c.B > 65535) return bad(NKV_ERR_UNSUPPORTED, "too many heads or items");
    if (n < 0 || n > c.cap) return bad(NKV_ERR_INVALID, "n must be in [0, cap]");
    if (!(scale > 0.0f) || !(scale < INFINITY))
        return bad(NKV_ERR_INVALID, "softmax_scale must be positive and finite");
    if (c.B == 0 || Q == 0) return NKV_OK;
    if (!q) return bad(NKV_ERR_INVALID, "q is required");
    if (reinterpret_cast<uintptr_t>(q) % 16 || (sb | st | sh) % 8)
        return bad(NKV_ERR_INVALID, "q must be 16-byte aligned with strides divisible by 8");
    return NKV_OK;
}

struct Plan {
    bool tile, eight, two;        // the tile kernel; of the other, eight waves, two groups of rows
    int groups, splits, per_group;
    int64_t items, rows;
    size_t part, ml;              // bytes
};

// Up to this many rows of a key head, the kernel of 16-row groups; above it the
// tile kernel (us with either: 24 x 8 heads of 1,024 rows 27.8, 30.5 at 64 query
// rows and 40.2, 32.3 at 96; 8 heads of 4,096 rows 12.9, 18.0 and 18.5, 18.9).
constexpr int64_t TILE_ROWS = 64;
// Two groups to a wave from this many (group, block) pairs on (us with one and
// two: 1,024 pairs 11.5, 13.2; 2,048 12.9, 14.7; 8,192 24.0, 21.1; 12,288 30.7,
// 27.8).
constexpr int64_t ROWS_TWO = 4096;

Plan attend_plan(const nkv_cache8_attend_args* a) {
    const nkv_cache8& c = a->cache;
    Plan pl{};
    pl.rows = a->Q * a->G;
    const int64_t heads = (int64_t)c.B * c.H, blocks = cdiv(a->n, C8_BLOCK);
    pl.splits = 1;
    pl.tile = pl.rows > TILE_ROWS;
    if (pl.tile) {
        // the fewest groups of up to eight 32-row blocks, of even size
        const int64_t qb = cdiv(pl.rows, 32);
        pl.groups = (int)cdiv(qb, TILE_WAVES);
        pl.per_group = (int)cdiv(qb, pl.groups);
        const int64_t base = heads * pl.groups;
        // splits whose rounds of 256 workgroups take least, in units of a
        // block's time; a workgroup's start and end cost some blocks, and a
        // merge its partials' traffic
        double best = 0.0;
        const int64_t most = std::max<int64_t>(16, cdiv(256, std::max<int64_t>(base, 1)));
        for (int64_t s = 1; s <= most && (s == 1 || blocks >= 4 * s); ++s) {
            const double merge = s == 1 ? 0.0 : 4.0 + (double)heads * pl.rows * s * 2e-4;
            const double t = (double)cdiv(base * s, 256) * ((double)blocks / s + 6.0) + merge;
            if (s == 1 || t < best) {
                best = t;
                pl.splits = (int)s;
            }
        }
        pl.items = base * pl.splits;
    } else {
        // eight waves a CU in either width, and a block of keys for each; twice
        // the workgroups where sequences have lengths of their own, so that CUs
        // with short ones take more (32 ragged sequences up to 16,384: 151 us
        // with 256 workgroups, 137 with 512)
        pl.two = pl.rows > 16 && heads * cdiv(pl.rows, 16) * blocks >= ROWS_TWO;
        pl.groups = (int)cdiv(pl.rows, pl.two ? 32 : 16);
        const int64_t base = heads * pl.groups;
        pl.eight = base * blocks >= ROWS_EIGHT;
        const int64_t slots = pl.eight && !a->length ? 256 : 512, waves = pl.eight ? 8 : 4;
        if (base > 0 && base < slots)
            pl.splits = (int)std::max<int64_t>(1, std::min(cdiv(slots, base), blocks / waves));
        pl.items = base * pl.splits;
    }
    return pl;
}

// The plan's workspace; in fewer than `limit` bytes fewer splits where those wanted do
// not fit.
void attend_fit(const nkv_cache8_attend_args* a, Plan& pl, size_t limit) {
    if (pl.splits == 1) return;
    const size_t part = c8_pitch(a->cache.D) * (a->dtype == NKV_ROWS_FP16 ? 4 : 2);
    const size_t rows = (size_t)a->cache.B * a->cache.H * pl.rows;
    const size_t most = limit / (rows * (sizeof(Stat) + part));
    if (most < (size_t)pl.splits) {
        pl.items /= pl.splits;
        pl.splits = (int)std::max<size_t>(1, most);
        pl.items *= pl.splits;
        if (pl.splits == 1) return;
    }
    pl.ml = rows * pl.splits * sizeof(Stat);
    pl.part = rows * pl.splits * part;
}

// Also plans the call where there is something to do (pl.items > 0).
int check_attend(const nkv_cache8_attend_args* a, Plan& pl) {
    NKV_REQUIRE(a, NKV_ERR_INVALID, "args is null");
    int rc = check_query(a->cache, a->G, a->dtype, a->Q, a->n, a->softmax_scale, a->q, a->q_sb,
                         a->q_st, a->q_sh, __func__);
    if (rc || a->cache.B == 0 || a->Q == 0) return rc;
    NKV_REQUIRE(a->out, NKV_ERR_INVALID, "out is required");
    NKV_REQUIRE(reinterpret_cast<uintptr_t>(a->out) % 16 == 0 && (a->o_sb | a->o_st | a->o_sh) % 8 == 0,
                NKV_ERR_INVALID, "out must be 16-byte aligned with strides divisible by 8");
    // a launch has fewer than 2^32 threads
    pl = attend_plan(a);
    NKV_REQUIRE(pl.items <= 1 << 22, NKV_ERR_UNSUPPORTED, "too many query rows");
    // every row of out lies past the end of those of the smaller strides
    std::pair<int64_t, int64_t> dims[3] = {
        {a->o_sb, a->cache.B}, {a->o_st, a->Q}, {a->o_sh, (int64_t)a->cache.H * a->G}};
    std::sort(dims, dims + 3);
    __int128 end = a->cache.D;
    for (const auto& [stride, count] : dims) {
        if (count == 1) continue;
        NKV_REQUIRE(stride >= end, NKV_ERR_INVALID, "out's rows overlap");
        end += (__int128)stride * (count - 1);
    }
    // what is written and what is read; an out with gaps may have anything in them
    const nkv_cache8& c = a->cache;
    const int64_t heads = (int64_t)c.B * c.H, codes = heads * c.cap * c8_pitch(c.D);
    const int64_t rows = heads * a->G * a->Q;
    const Range in[6] = {{c.k, codes}, {c.v, codes}, {c.k_scale, heads * c.cap / 16},
                         {c.v_scale, heads * c.cap / 16}, {a->length, a->length ? c.B * 4 : 0},
                         {a->counts, a->counts ? c.B * 4 : 0}};
    const Range lse(a->lse, a->lse ? rows * 4 : 0), out(a->out, end == rows * c.D ? rows * c.D * 2 : 0);
    for (const Range& r : in)
        NKV_REQUIRE(!r.meets(lse) && !r.meets(out), NKV_ERR_INVALID,
                    "out or lse overlaps the cache, length or counts");
    NKV_REQUIRE(!lse.meets(out), NKV_ERR_INVALID, "lse overlaps out");
    return NKV_OK;
}

// Blocks of a launch over p.items workgroups in item_of's order.
unsigned item_blocks(const AttendParams& p) {
    const int64_t units = p.items / p.groups;
    return (unsigned)(units >= UNITS ? 8 * cdiv(units, 8) * p.groups : 8 * cdiv(p.items, 8));
}

template <typename T, int FMT, int P, int W, int NQ>
int attend_rows_run(const AttendParams& p, hipStream_t s) {
    constexpr int SMEM = sizeof(RowsSmem<P, W, NQ>);
    if (SMEM > 65536)
        if (int rc = set_smem(attend_kernel<T, FMT, P, W, NQ>, SMEM)) return rc;
    attend_kernel<T, FMT, P, W, NQ><<<item_blocks(p), 64 * W, SMEM, s>>>(p);
    return NKV_OK;
}

template <typename T, int FMT, int P>
int attend_run(const AttendParams& p, const Plan& pl, hipStream_t s) {
    if (pl.tile) {
        constexpr int SMEM = TileCodes<T, FMT, P>::SMEM;
        if (int rc = set_smem(attend_tile_kernel<T, FMT, P>, SMEM)) return rc;
        attend_tile_kernel<T, FMT, P>
            <<<item_blocks(p), 64 * TILE_WAVES, SMEM, s>>>(p);
        return NKV_OK;
    }
    if (pl.two)
        return pl.eight ? attend_rows_run<T, FMT, P, 8, 2>(p, s) : attend_rows_run<T, FMT, P, 4, 2>(p, s);
    return pl.eight ? attend_rows_run<T, FMT, P, 8, 1>(p, s) : attend_rows_run<T, FMT, P, 4, 1>(p, s);
}

template <typename T, int P>
void merge_run(const AttendParams& p, hipStream_t s) {
    constexpr int PARTS = P / 8;
    auto grid = [&](int sg) {
        return dim3((unsigned)cdiv(p.rows, 256 / (PARTS * sg)), (unsigned)p.H, (unsigned)p.B);
    };
    if (p.splits > 8) merge_kernel<T, P, 16, 8><<<grid(16), 256, 0, s>>>(p);
    else if (p.splits > 4) merge_kernel<T, P, 1, 8><<<grid(1), 256, 0, s>>>(p);
    else if (p.splits > 2) merge_kernel<T, P, 1, 4><<<grid(1), 256, 0, s>>>(p);
    else merge_kernel<T, P, 1, 2><<<grid(1), 256, 0, s>>>(p);
}

template <typename T, int FMT, int P>
void mass_run(const MassParams& p, bool tile, hipStream_t s) {
    const dim3 grid((unsigned)cdiv(p.blocks, 4 * p.per), (unsigned)(p.B * p.H), (unsigned)p.splits);
    if (tile) mass_tile_kernel<T, FMT, P><<<grid, 256, 0, s>>>(p);
    else mass_kernel<T, FMT, P><<<grid, 256, 0, s>>>(p);
}

// f.template operator()<T, FMT, P>() of a call's types and pitch.
template <typename F>
void dispatch(int dtype, int format, int D, F f) {
    const bool wide = c8_pitch(D) == 128, e4m3 = format == NKV_CACHE8_E4M3;
    if (dtype == NKV_ROWS_BF16) {
        if (e4m3) wide ? f(Bf16{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 128>{})
                       : f(Bf16{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 64>{});
        else wide ? f(Bf16{}, std::integral_constant<int, 0>{}, std::integral_constant<int, 128>{})
                  : f(Bf16{}, std::integral_constant<int, 0>{}, std::integral_constant<int, 64>{});
    } else {
        if (e4m3) wide ? f(Fp16{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 128>{})
                       : f(Fp16{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 64>{});
        else wide ? f(Fp16{}, std::integral_constant<int, 0>{}, std::integral_constant<int, 128>{})
                  : f(Fp16{}, std::integral_constant<int, 0>{}, std::integral_constant<int, 64>{});
    }
}
static_assert(NKV_CACHE8_INT8 == 0 && NKV_CACHE8_E4M3 == 1, "dispatch");
static_assert(sizeof(Stat) == 16 && alignof(Stat) == 16, "partials");

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" size_t nkv_cache8_attend_workspace_size(const nkv_cache8_attend_args* a) {
    clear_error();
    Plan pl{};
    if (check_attend(a, pl) || pl.items == 0) return 0;
    attend_fit(a, pl, SIZE_MAX);
    return pl.part + pl.ml;
}

extern "C" int nkv_cache8_attend(void* stream, const nkv_cache8_attend_args* a, void* workspace,
                                 size_t workspace_bytes) {
    clear_error();
    Plan pl{};
    int rc = check_attend(a, pl);
    if (rc || pl.items == 0) return rc;
    const nkv_cache8& c = a->cache;
    attend_fit(a, pl, workspace ? workspace_bytes : 0);
    NKV_REQUIRE(pl.part == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, NKV_ERR_INVALID,
                "workspace must be 16-byte aligned");
    AttendParams p{};
    p.k = (const uint8_t*)c.k;
    p.v = (const uint8_t*)c.v;
    p.ks = c.k_scale;
    p.vs = c.v_scale;
    p.length = a->length;
    p.counts = a->counts;
    p.q = (const uint16_t*)a->q;
    p.out = (uint16_t*)a->out;
    p.lse = a->lse;
    p.part_st = (Stat*)workspace;
    p.part = (char*)workspace + pl.ml;
    p.q_sb = a->q_sb, p.q_st = a->q_st, p.q_sh = a->q_sh;
    p.o_sb = a->o_sb, p.o_st = a->o_st, p.o_sh = a->o_sh;
    p.cap = c.cap;
    p.items = pl.items;
    p.scale_log2 = std::min(a->softmax_scale * LOG2E, 0x1.fffffep127f);
    p.B = c.B, p.H = c.H, p.G = a->G, p.D = c.D, p.Q = (int)a->Q, p.n = (int)a->n;
    p.causal = a->causal != 0;
    p.splits = pl.splits;
    p.groups = pl.groups;
    p.rows = (int)pl.rows;
    p.per_group = pl.per_group;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    dispatch(a->dtype, c.format, c.D, [&](auto t, auto f, auto w) {
        rc = attend_run<decltype(t), decltype(f)::value, decltype(w)::value>(p, pl, s);
    });
    if (rc) return rc;
    NKV_LAUNCH_CHECK();
    if (pl.splits > 1) {
        const bool wide = c8_pitch(c.D) == 128, bf16 = a->dtype == NKV_ROWS_BF16;
        if (wide && bf16) merge_run<Bf16, 128>(p, s);
        else if (wide) merge_run<Fp16, 128>(p, s);
        else if (bf16) merge_run<Bf16, 64>(p, s);
        else merge_run<Fp16, 64>(p, s);
        NKV_LAUNCH_CHECK();
    }
    return NKV_OK;
}

namespace nkv {
namespace {
int check_mass(const nkv_cache8_mass_args* a) {
    NKV_REQUIRE(a, NKV_ERR_INVALID, "args is null");
    int rc = check_query(a->cache, a->G, a->dtype, a->Q, a->n, a->softmax_scale, a->q, a->q_sb,
                         a->q_st, a->q_sh, __func__);
    if (rc || a->cache.B == 0) return rc;
    NKV_REQUIRE(a->mass && a->out && (a->Q == 0 || a->lse), NKV_ERR_INVALID,
                "lse, mass and out are required");
    const int64_t bytes = (int64_t)a->cache.B * a->cache.H * a->cache.cap * 4;
    const uintptr_t m = reinterpret_cast<uintptr_t>(a->mass), o = reinterpret_cast<uintptr_t>(a->out);
    NKV_REQUIRE(m == o || m >= o + bytes || o >= m + bytes, NKV_ERR_INVALID,
                "out must be mass itself or not overlap it");
    const nkv_cache8& c = a->cache;
    const int64_t heads = (int64_t)c.B * c.H;
    NKV_REQUIRE(heads <= 65535, NKV_ERR_UNSUPPORTED, "too many heads");
    const Range in[5] = {{c.k, heads * c.cap * c8_pitch(c.D)}, {c.k_scale, heads * c.cap / 16},
                         {a->lse, heads * a->G * a->Q * 4}, {a->length, a->length ? c.B * 4 : 0},
                         {a->counts, a->counts ? c.B * 4 : 0}};
    for (const Range& r : in)
        NKV_REQUIRE(!r.meets({a->out, bytes}), NKV_ERR_INVALID,
                    "out overlaps the cache's keys, lse, length or counts");
    return NKV_OK;
}

// Up to this many rows of a key head each wave reads its queries itself; above,
// they pass through LDS (us with either: 24 x 8 heads of 2,048 rows 20.4, 20.8 at
// 32 query rows and 24.4, 20.8 at 48; 8 heads of 4,096 rows 4.5, 5.7 at 32 and
// 6.0, 5.8 at 64).
constexpr int64_t MASS_FEW = 32;

struct MassPlan {
    bool tile;
    int splits;
    int64_t n64;
    size_t bytes;
};

// Row splits: only where the blocks of keys fill less than two workgroups a CU,
// each with at least four steps (1,176 workgroups of 25 steps took 176 us
// whole, 190 in three splits).
MassPlan mass_plan(const nkv_cache8_mass_args* a, size_t limit = SIZE_MAX) {
    MassPlan pl{};
    const int64_t rows = a->Q * a->G, heads = (int64_t)a->cache.B * a->cache.H;
    pl.n64 = cdiv(a->n, C8_BLOCK) * C8_BLOCK;
    pl.tile = rows > MASS_FEW;
    pl.splits = 1;
    const int64_t base = heads * cdiv(pl.n64, 4 * C8_BLOCK), steps = cdiv(rows, MT_ROWS);
    if (pl.tile && base > 0 && base < 512)
        pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(512, base), steps / 4, 64}));
    const size_t split = (size_t)heads * pl.n64 * sizeof(float);
    if (pl.splits > 1 && limit / split < (size_t)pl.splits)
        pl.splits = (int)std::max<size_t>(1, limit / split);
    if (pl.splits > 1) pl.bytes = pl.splits * split;
    return pl;
}
}  // namespace
}  // namespace nkv

extern "C" size_t nkv_cache8_mass_workspace_size(const nkv_cache8_mass_args* a) {
    clear_error();
    if (check_mass(a) || a->cache.B == 0) return 0;
    return mass_plan(a).bytes;
}

extern "C" int nkv_cache8_mass(void* stream, const nkv_cache8_mass_args* a, void* workspace,
                               size_t workspace_bytes) {
    clear_error();
    int rc = check_mass(a);
    if (rc || a->cache.B == 0) return rc;
    const nkv_cache8& c = a->cache;
    const MassPlan pl = mass_plan(a, workspace ? workspace_bytes : 0);
    NKV_REQUIRE(pl.bytes == 0 || reinterpret_cast<uintptr_t>(workspace) % 4 == 0, NKV_ERR_INVALID,
                "workspace must be 4-byte aligned");
    MassParams p{};
    p.k = (const uint8_t*)c.k;
    p.ks = c.k_scale;
    p.length = a->length;
    p.counts = a->counts;
    p.q = (const uint16_t*)a->q;
    p.lse = a->lse;
    p.mass = a->mass;
    p.out = a->out;
    p.q_sb = a->q_sb, p.q_st = a->q_st, p.q_sh = a->q_sh;
    p.cap = c.cap;
    p.scale_log2 = std::min(a->softmax_scale * LOG2E, 0x1.fffffep127f);
    p.B = c.B, p.H = c.H, p.G = a->G, p.D = c.D, p.Q = (int)a->Q, p.n = (int)a->n;
    p.causal = a->causal != 0;
    p.rows = (int)(a->Q * a->G);
    p.splits = pl.splits;
    p.n64 = pl.n64;
    p.part = (float*)workspace;
    // in place, blocks past n have nothing to do
    p.blocks = (int)(p.out == p.mass ? cdiv(a->n, C8_BLOCK) : c.cap / C8_BLOCK);
    if (p.blocks == 0) return NKV_OK;
    const dim3 join((unsigned)cdiv((int64_t)p.blocks * C8_BLOCK, 256), (unsigned)(c.B * c.H));
    if (a->Q == 0) {  // the kernels take a row at least
        if (p.out == p.mass) return NKV_OK;
        p.n = 0;
        p.length = nullptr;
        mass_join_kernel<<<join, 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(p);
        NKV_LAUNCH_CHECK();
        return NKV_OK;
    }
    p.per = pl.tile ? 1 : (int)std::min<int64_t>(8, std::max<int64_t>(1, (int64_t)c.B * c.H * p.blocks / MASS_WAVES));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    dispatch(a->dtype, c.format, c.D, [&](auto t, auto f, auto w) {
        mass_run<decltype(t), decltype(f)::value, decltype(w)::value>(p, pl.tile, s);
    });
    NKV_LAUNCH_CHECK();
    if (pl.splits > 1) {
        mass_join_kernel<<<join, 256, 0, s>>>(p);
        NKV_LAUNCH_CHECK();
    }
    return NKV_OK;
}
