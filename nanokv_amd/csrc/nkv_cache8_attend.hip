// nkv_cache8_attend.hip -- attention over the 8-bit key/value cache and the
// weight its rows receive (nkv_cache8_attend, nkv_cache8_mass).
//
// With k = sk * code per block of 64 rows, a score is (softmax_scale * sk) *
// (q . code), and with v = sv * code the output is sum p * sv * code / sum p:
// neither scale meets a 16-bit operand.  Codes are exact in bf16 and fp16, so
// the scores are those of the dequantised rows with one rounding less.
#include "nkv_cache8.h"

#include <math.h>

#include <algorithm>

namespace nkv {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float TAU = 8.0f;           // a row's maximum is moved when it is off by 2^TAU
constexpr float SCALE_MIN = 0x1p-100f;  // keeps an unwritten block's scale out of log2(0)

struct AttendParams {
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    const int32_t* length;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    float* part;                  // [item][16 rows][P] fp32 unnormalised outputs
    float* part_ml;               // [item][16 rows][2] running maximum (log2) and sum
    int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;
    int64_t cap, items;
    float scale_log2;
    int B, H, G, D, Q, n, causal, splits, groups;
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

// Four waves of a workgroup share 16 query rows and a range of 64-row blocks;
// wave w takes blocks w, w + 4, ... and the waves' results are merged in LDS.
template <typename T, int FMT, int P>
__global__ void __launch_bounds__(256) attend_kernel(AttendParams p) {
    constexpr int STEPS = P / 32, PIECES = P / 64, DB = P / 16;
    using x8 = typename T::x8;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = blockIdx.x;
    const int rg = (int)(item % p.groups);
    const int64_t rest = item / p.groups;
    const int split = (int)(rest % p.splits);
    const int bh = (int)(rest / p.splits), b = bh / p.H, hk = bh % p.H;
    const int len = c8_length(p.length, b, p.n);
    const int row0 = rg * 16;
    const RowAt mine = row_at(row0 + r, hk, p.G, p.Q);
    const int end = !mine.there ? 0 : p.causal ? len - p.Q + 1 + mine.t : len;
    // blocks that the group's last row sees
    const int last_t = min(row0 + 15, p.G * p.Q - 1) / p.G;
    const int last = max(0, p.causal ? len - p.Q + 1 + last_t : len);
    const int first = p.causal ? len - p.Q + 1 + row0 / p.G : len;  // what its first row sees
    const int nb = (last + C8_BLOCK - 1) / C8_BLOCK;
    const int b0 = (int)((int64_t)split * nb / p.splits);
    const int b1 = (int)((int64_t)(split + 1) * nb / p.splits);
    x8 qf[STEPS];
    load_q<T, P>(qf, p.q + b * p.q_sb + mine.t * p.q_st + mine.head * p.q_sh, mine.there, g, p.D);
    const uint8_t* kbase = p.k + ((int64_t)bh * p.cap + r) * P + 16 * g;
    const uint8_t* vbase = p.v + ((int64_t)bh * p.cap + 4 * g) * P + DB * r;
    const float* ks = p.ks + (int64_t)bh * (p.cap / C8_BLOCK);
    const float* vs = p.vs + (int64_t)bh * (p.cap / C8_BLOCK);
    f32x4 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x4{};
    // m: the row's maximum (log2 units), l: its sum of 2^(z - m) over this
    // lane's keys; o holds sum of 2^(z - m) * sv * code in units of 2^unit
    float m = -INFINITY, l = 0.0f, unit = -INFINITY;
    for (int blk = b0 + wave; blk < b1; blk += 4) {
        const int64_t key0 = (int64_t)blk * C8_BLOCK;
        u32x4 kr[4][PIECES];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                kr[t][i] = *reinterpret_cast<const u32x4*>(kbase + (key0 + 16 * t) * P + 64 * i);
        // V: lane (r, g) holds columns DB r .. + DB of the keys that its
        // probabilities are of: 32 c + 16 a + 4 g + j
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
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4{};
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                s[t] = T::mfma16(codes_x8<T, FMT>(kr[t][i][0], kr[t][i][1]), qf[2 * i], s[t]);
                s[t] = T::mfma16(codes_x8<T, FMT>(kr[t][i][2], kr[t][i][3]), qf[2 * i + 1], s[t]);
            }
        }
        if (key0 + C8_BLOCK > first) {
            // scores of unseen keys; s[t][e] is of key 16 t + 4 g + e
            const int seen = end - (int)key0;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (16 * t + 4 * g + e >= seen) s[t][e] = -INFINITY;
            // rows at or past the length may hold NaN codes, which a zero
            // probability does not remove
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
        const float c = p.scale_log2 * sk, lsv = __builtin_amdgcn_logf(sv);
        if (lsv > unit) {
            const float f = __builtin_amdgcn_exp2f(unit - lsv);
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] *= f;
            unit = lsv;
        }
        float tm = s[0][0];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) tm = fmaxf(tm, s[t][e]);
        tm = rows4_max(tm) * c;
        const bool up = tm > m + TAU;
        const float mn = up ? tm : m;
        const float alpha = up ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
        m = mn;
        const float off = (mn == -INFINITY ? 0.0f : mn) + (unit - lsv);
        float lsum = 0.0f;
        uint32_t pw[2][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = __builtin_amdgcn_exp2f(fmaf(s[t][e], c, -off));
                lsum += w[e];
            }
            pw[t >> 1][2 * (t & 1)] = T::pack(w[0], w[1]);
            pw[t >> 1][2 * (t & 1) + 1] = T::pack(w[2], w[3]);
        }
        l = l * alpha + lsum * __builtin_amdgcn_exp2f(unit - lsv);
        if (__any(up)) {
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] *= alpha;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const x8 pf = as_x8<x8>(u32x4{pw[k][0], pw[k][1], pw[k][2], pw[k][3]});
#pragma unroll
            for (int w = 0; w < DB / 4; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f32x2 a[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[j] = code_pair<FMT>(vr[k][j][w], h);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const x8 vf = as_x8<x8>(u32x4{T::pack(a[0][e], a[1][e]), T::pack(a[2][e], a[3][e]),
                                                      T::pack(a[4][e], a[5][e]), T::pack(a[6][e], a[7][e])});
                        o[4 * w + 2 * h + e] = T::mfma16(vf, pf, o[4 * w + 2 * h + e]);
                    }
                }
        }
    }
    l = rows4_sum(l);
    // merge of the four waves: o[i][e] is column DB (4 g + e) + i of row r
    __shared__ float so[4][16][P + 4];
    __shared__ float sml[4][16][2];
    const float f = unit == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(unit);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < DB; i += 4)
            *reinterpret_cast<f32x4*>(&so[wave][r][DB * (4 * g + e) + i]) =
                f32x4{o[i][e] * f, o[i + 1][e] * f, o[i + 2][e] * f, o[i + 3][e] * f};
    if (g == 0) {
        sml[wave][r][0] = m;
        sml[wave][r][1] = l;
    }
    __syncthreads();
    const int mr = threadIdx.x / 16, d = (threadIdx.x % 16) * 8;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sml[w][mr][0]);
    float L = 0.0f, acc[8] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float mw = sml[w][mr][0];
        const float a = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - M);
        L += a * sml[w][mr][1];
        if (d < P)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += a * so[w][mr][d + i];
    }
    if (p.splits > 1) {
        const int64_t at = item * 16 + mr;
        if (d < P) {
            f32x4* dst = reinterpret_cast<f32x4*>(p.part + at * P + d);
            dst[0] = f32x4{acc[0], acc[1], acc[2], acc[3]};
            dst[1] = f32x4{acc[4], acc[5], acc[6], acc[7]};
        }
        if (d == 0) {
            p.part_ml[2 * at] = M;
            p.part_ml[2 * at + 1] = L;
        }
        return;
    }
    const RowAt ro = row_at(row0 + mr, hk, p.G, p.Q);
    if (!ro.there) return;
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    if (d < p.D)
        *reinterpret_cast<u32x4*>(p.out + b * p.o_sb + ro.t * p.o_st + ro.head * p.o_sh + d) =
            u32x4{T::pack(acc[0] * inv, acc[1] * inv), T::pack(acc[2] * inv, acc[3] * inv),
                  T::pack(acc[4] * inv, acc[5] * inv), T::pack(acc[6] * inv, acc[7] * inv)};
    if (d == 0 && p.lse)
        p.lse[((int64_t)b * p.H * p.G + ro.head) * p.Q + ro.t] =
            L > 0.0f ? M * LN2 + logf(L) : -INFINITY;
}

// The merge of the splits' partial results: 16 threads a row, eight columns
// each; out = sum 2^(m - M) o / sum 2^(m - M) l.
template <typename T, int P>
__global__ void __launch_bounds__(256) merge_kernel(AttendParams p) {
    const int64_t rows = (int64_t)p.groups * 16;
    const int64_t at = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    const int d = (threadIdx.x % 16) * 8;
    const int64_t bh = at / rows;
    if (bh >= (int64_t)p.B * p.H) return;
    const int row = (int)(at % rows), b = (int)(bh / p.H), hk = (int)(bh % p.H);
    const RowAt ro = row_at(row, hk, p.G, p.Q);
    if (!ro.there) return;
    const int64_t step = (int64_t)p.groups * 16;
    const int64_t first = bh * p.splits * step + row;
    float M = -INFINITY;
    for (int s = 0; s < p.splits; ++s) M = fmaxf(M, p.part_ml[2 * (first + s * step)]);
    float L = 0.0f, acc[8] = {};
    for (int s = 0; s < p.splits; ++s) {
        const int64_t i = first + s * step;
        const float mw = p.part_ml[2 * i];
        if (mw == -INFINITY) continue;
        const float a = __builtin_amdgcn_exp2f(mw - M);
        L += a * p.part_ml[2 * i + 1];
        if (d < P) {
            const f32x4* src = reinterpret_cast<const f32x4*>(p.part + i * P + d);
            const f32x4 x = src[0], y = src[1];
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] += a * x[k], acc[4 + k] += a * y[k];
        }
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    if (d < p.D)
        *reinterpret_cast<u32x4*>(p.out + b * p.o_sb + ro.t * p.o_st + ro.head * p.o_sh + d) =
            u32x4{T::pack(acc[0] * inv, acc[1] * inv), T::pack(acc[2] * inv, acc[3] * inv),
                  T::pack(acc[4] * inv, acc[5] * inv), T::pack(acc[6] * inv, acc[7] * inv)};
    if (d == 0 && p.lse)
        p.lse[((int64_t)b * p.H * p.G + ro.head) * p.Q + ro.t] =
            L > 0.0f ? M * LN2 + logf(L) : -INFINITY;
}

// ---------------------------------------------------------------- mass
struct MassParams {
    const uint8_t* k;
    const float* ks;
    const int32_t* length;
    const uint16_t* q;
    const float* lse;
    const float* mass;
    float* out;
    int64_t q_sb, q_st, q_sh;
    int64_t cap;
    float scale_log2;
    int B, H, G, D, Q, n, causal, groups;
};

// One workgroup per block of 64 cached rows and head: the waves hold the
// block's codes as operands and take the groups of 16 query rows in turn; the
// sums over rows stay in registers and are joined in LDS in a fixed order.
template <typename T, int FMT, int P>
__global__ void __launch_bounds__(256) mass_kernel(MassParams p) {
    constexpr int STEPS = P / 32, PIECES = P / 64;
    using x8 = typename T::x8;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blk = blockIdx.x, bh = blockIdx.y, b = bh / p.H, hk = bh % p.H;
    const int len = c8_length(p.length, b, p.n);
    const int64_t key0 = (int64_t)blk * C8_BLOCK;
    const int64_t at = (int64_t)bh * p.cap + key0;
    if (key0 >= len) {
        if (p.out != p.mass && threadIdx.x < C8_BLOCK)
            p.out[at + threadIdx.x] = p.mass[at + threadIdx.x];
        return;
    }
    x8 kf[4][STEPS];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(p.k + (at + 16 * t + r) * P + 64 * i + 16 * g);
            kf[t][2 * i] = codes_x8<T, FMT>(w[0], w[1]);
            kf[t][2 * i + 1] = codes_x8<T, FMT>(w[2], w[3]);
        }
    const float c = p.scale_log2 * fmaxf(p.ks[(int64_t)bh * (p.cap / C8_BLOCK) + blk], SCALE_MIN);
    f32x4 sum[4] = {};
    // the first group with a row that sees the block's first key
    int rg0 = 0;
    if (p.causal) rg0 = max(0, (int)key0 - (len - p.Q)) * p.G / 16;
    for (int rg = rg0 + wave; rg < p.groups; rg += 4) {
        const RowAt mine = row_at(rg * 16 + r, hk, p.G, p.Q);
        const int seen = (!mine.there ? 0 : p.causal ? len - p.Q + 1 + mine.t : len) - (int)key0;
        x8 qf[STEPS];
        load_q<T, P>(qf, p.q + b * p.q_sb + mine.t * p.q_st + mine.head * p.q_sh, mine.there, g, p.D);
        float off = INFINITY;
        if (mine.there) {
            const float z = p.lse[((int64_t)b * p.H * p.G + mine.head) * p.Q + mine.t];
            off = z == -INFINITY ? INFINITY : z * LOG2E;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 s{};
#pragma unroll
            for (int i = 0; i < STEPS; ++i) s = T::mfma16(kf[t][i], qf[i], s);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[e], c, -off));
                sum[t][e] += 16 * t + 4 * g + e < seen ? w : 0.0f;
            }
        }
    }
    __shared__ float part[4][C8_BLOCK];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = sum[t][e];
#pragma unroll
            for (int k = 1; k < 16; k <<= 1) x += __shfl_xor(x, k);
            if (r == 0) part[wave][16 * t + 4 * g + e] = x;
        }
    __syncthreads();
    const int i = threadIdx.x;
    if (i < C8_BLOCK && (key0 + i < len || p.out != p.mass)) {
        float x = p.mass[at + i];
        if (key0 + i < len) x += (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]);
        p.out[at + i] = x;
    }
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
    int groups, splits;
    int64_t items;
    size_t part, ml;              // bytes
};

// Key splits: enough workgroups to fill the chip, each with at least four
// blocks of keys (one a wave).
Plan attend_plan(const nkv_cache8_attend_args* a) {
    const nkv_cache8& c = a->cache;
    Plan pl{};
    pl.groups = (int)cdiv(a->Q * a->G, 16);
    const int64_t base = (int64_t)c.B * c.H * pl.groups;
    const int64_t blocks = cdiv(a->n, C8_BLOCK);
    pl.splits = 1;
    if (base > 0 && base < 1024)
        pl.splits = (int)std::max<int64_t>(1, std::min(cdiv(1024, base), blocks / 4));
    pl.items = base * pl.splits;
    if (pl.splits > 1) {
        pl.part = (size_t)pl.items * 16 * c8_pitch(c.D) * 4;
        pl.ml = (size_t)pl.items * 16 * 8;
    }
    return pl;
}

int check_attend(const nkv_cache8_attend_args* a) {
    NKV_REQUIRE(a, NKV_ERR_INVALID, "args is null");
    int rc = check_query(a->cache, a->G, a->dtype, a->Q, a->n, a->softmax_scale, a->q, a->q_sb,
                         a->q_st, a->q_sh, __func__);
    if (rc || a->cache.B == 0 || a->Q == 0) return rc;
    NKV_REQUIRE(a->out, NKV_ERR_INVALID, "out is required");
    NKV_REQUIRE(reinterpret_cast<uintptr_t>(a->out) % 16 == 0 && (a->o_sb | a->o_st | a->o_sh) % 8 == 0,
                NKV_ERR_INVALID, "out must be 16-byte aligned with strides divisible by 8");
    NKV_REQUIRE(attend_plan(a).items <= INT32_MAX, NKV_ERR_UNSUPPORTED, "too many query rows");
    return NKV_OK;
}

template <typename T, int FMT, int P>
void attend_run(const AttendParams& p, hipStream_t s) {
    attend_kernel<T, FMT, P><<<(unsigned)p.items, 256, 0, s>>>(p);
}

template <typename T, int FMT, int P>
void mass_run(const MassParams& p, hipStream_t s) {
    // in place, blocks past n have nothing to do
    const int64_t blocks = p.out == p.mass ? cdiv(p.n, C8_BLOCK) : p.cap / C8_BLOCK;
    if (!blocks) return;
    const dim3 grid((unsigned)blocks, (unsigned)(p.B * p.H));
    mass_kernel<T, FMT, P><<<grid, 256, 0, s>>>(p);
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

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" size_t nkv_cache8_attend_workspace_size(const nkv_cache8_attend_args* a) {
    clear_error();
    if (check_attend(a) || a->cache.B == 0 || a->Q == 0) return 0;
    const Plan pl = attend_plan(a);
    return pl.part + pl.ml;
}

extern "C" int nkv_cache8_attend(void* stream, const nkv_cache8_attend_args* a, void* workspace,
                                 size_t workspace_bytes) {
    clear_error();
    int rc = check_attend(a);
    if (rc || a->cache.B == 0 || a->Q == 0) return rc;
    const nkv_cache8& c = a->cache;
    const Plan pl = attend_plan(a);
    NKV_REQUIRE(pl.part == 0 || (workspace && workspace_bytes >= pl.part + pl.ml),
                NKV_ERR_WORKSPACE, "workspace missing or too small");
    NKV_REQUIRE(pl.part == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, NKV_ERR_INVALID,
                "workspace must be 16-byte aligned");
    AttendParams p{};
    p.k = (const uint8_t*)c.k;
    p.v = (const uint8_t*)c.v;
    p.ks = c.k_scale;
    p.vs = c.v_scale;
    p.length = a->length;
    p.q = (const uint16_t*)a->q;
    p.out = (uint16_t*)a->out;
    p.lse = a->lse;
    p.part = (float*)workspace;
    p.part_ml = (float*)((char*)workspace + pl.part);
    p.q_sb = a->q_sb, p.q_st = a->q_st, p.q_sh = a->q_sh;
    p.o_sb = a->o_sb, p.o_st = a->o_st, p.o_sh = a->o_sh;
    p.cap = c.cap;
    p.items = pl.items;
    p.scale_log2 = a->softmax_scale * LOG2E;
    p.B = c.B, p.H = c.H, p.G = a->G, p.D = c.D, p.Q = (int)a->Q, p.n = (int)a->n;
    p.causal = a->causal != 0;
    p.splits = pl.splits;
    p.groups = pl.groups;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    dispatch(a->dtype, c.format, c.D, [&](auto t, auto f, auto w) {
        attend_run<decltype(t), decltype(f)::value, decltype(w)::value>(p, s);
    });
    NKV_LAUNCH_CHECK();
    if (pl.splits > 1) {
        const int64_t blocks = (int64_t)c.B * c.H * pl.groups;
        const bool wide = c8_pitch(c.D) == 128, bf16 = a->dtype == NKV_ROWS_BF16;
        if (wide && bf16) merge_kernel<Bf16, 128><<<(unsigned)blocks, 256, 0, s>>>(p);
        else if (wide) merge_kernel<Fp16, 128><<<(unsigned)blocks, 256, 0, s>>>(p);
        else if (bf16) merge_kernel<Bf16, 64><<<(unsigned)blocks, 256, 0, s>>>(p);
        else merge_kernel<Fp16, 64><<<(unsigned)blocks, 256, 0, s>>>(p);
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
    NKV_REQUIRE((int64_t)a->cache.B * a->cache.H <= 65535, NKV_ERR_UNSUPPORTED, "too many heads");
    return NKV_OK;
}
}  // namespace
}  // namespace nkv

extern "C" size_t nkv_cache8_mass_workspace_size(const nkv_cache8_mass_args* a) {
    clear_error();
    check_mass(a);
    return 0;
}

extern "C" int nkv_cache8_mass(void* stream, const nkv_cache8_mass_args* a, void* workspace,
                               size_t workspace_bytes) {
    clear_error();
    int rc = check_mass(a);
    if (rc || a->cache.B == 0) return rc;
    const nkv_cache8& c = a->cache;
    MassParams p{};
    p.k = (const uint8_t*)c.k;
    p.ks = c.k_scale;
    p.length = a->length;
    p.q = (const uint16_t*)a->q;
    p.lse = a->lse;
    p.mass = a->mass;
    p.out = a->out;
    p.q_sb = a->q_sb, p.q_st = a->q_st, p.q_sh = a->q_sh;
    p.cap = c.cap;
    p.scale_log2 = a->softmax_scale * LOG2E;
    p.B = c.B, p.H = c.H, p.G = a->G, p.D = c.D, p.Q = (int)a->Q, p.n = (int)a->n;
    p.causal = a->causal != 0;
    p.groups = (int)cdiv(a->Q * a->G, 16);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    dispatch(a->dtype, c.format, c.D, [&](auto t, auto f, auto w) {
        mass_run<decltype(t), decltype(f)::value, decltype(w)::value>(p, s);
    });
    NKV_LAUNCH_CHECK();
    return NKV_OK;
}
