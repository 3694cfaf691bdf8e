// nkv_cache8.hip -- the 8-bit key/value cache: writing rows into it and
// evicting rows from it (nkv_cache8_write, nkv_cache8_evict).
//
// Compiled without fp contraction: codes are a function of their inputs to the
// last bit (IEEE division by the scale, one rounding to the code).
#include "nkv_cache8.h"

#include <math.h>

#include <algorithm>

namespace nkv {

int cache8_check(const nkv_cache8* c, const char* who) {
    auto bad = [&](int code, const char* what) {
        set_error(std::string(who) + ": " + what);
        return code;
    };
    if (c->B < 0 || c->H < 1 || c->D < 1) return bad(NKV_ERR_INVALID, "cache needs B >= 0, H >= 1, D >= 1");
    if (c->D % 8 || c->D > 128)
        return bad(NKV_ERR_UNSUPPORTED, "head width must be a multiple of 8, at most 128");
    if (c->format != NKV_CACHE8_INT8 && c->format != NKV_CACHE8_E4M3)
        return bad(NKV_ERR_INVALID, "unknown cache format");
    if (c->cap < C8_BLOCK || c->cap % C8_BLOCK || c->cap > (1 << 29))
        return bad(NKV_ERR_INVALID, "cap must be a positive multiple of 64, at most 2^29");
    if ((int64_t)c->B * c->H > 1 << 21) return bad(NKV_ERR_UNSUPPORTED, "too many heads");
    if (c->B == 0) return NKV_OK;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale)
        return bad(NKV_ERR_INVALID, "cache codes and scales are required");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16)
        return bad(NKV_ERR_INVALID, "cache codes must be 16-byte aligned");
    return NKV_OK;
}

namespace {

// ---------------------------------------------------------------- write
struct WriteParams {
    uint8_t* codes[2];            // K, V
    float* scale[2];
    const void* x[2];
    int64_t sb[2], st[2], sh[2];
    const int32_t* start_dev;
    const int32_t* counts;
    int64_t cap;
    int64_t start;
    int64_t T;
    int B, H, D;
};

// Eight consecutive elements of a row as they come.
template <int DTYPE>
struct Piece {
    static constexpr int W = DTYPE == NKV_ROWS_FP32 ? 8 : 4;
    // the least bit pattern of a magnitude that is not finite
    static constexpr uint32_t INF =
        DTYPE == NKV_ROWS_FP32 ? 0x7f800000u : DTYPE == NKV_ROWS_BF16 ? 0x7f80u : 0x7c00u;
    uint32_t w[W];
    __device__ __forceinline__ void load(const void* x, int64_t at) {
        const u32x4* p = reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(x) +
                                                        at * (W / 2));
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const u32x4 v = p[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[4 * i + k] = v[k];
        }
    }
    // magnitudes as integers order as the magnitudes do, NaN above infinity
    __device__ __forceinline__ void largest(uint32_t& m) const {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (DTYPE == NKV_ROWS_FP32) {
                m = max(m, w[i] & 0x7fffffffu);
            } else {
                typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                m = __builtin_bit_cast(
                    uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                        __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu)));
            }
        }
    }
    static __device__ __forceinline__ float from(uint32_t bits) {
        if constexpr (DTYPE == NKV_ROWS_FP32) return __uint_as_float(bits);
        else if constexpr (DTYPE == NKV_ROWS_BF16) return bf16_bits_to_f32((uint16_t)bits);
        else return f16_bits_to_f32((uint16_t)bits);
    }
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (DTYPE == NKV_ROWS_FP32) return __uint_as_float(w[e]);
        else if constexpr (DTYPE == NKV_ROWS_BF16)
            return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        else return f16_bits_to_f32((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
    }
};

// The largest of a workgroup's values, in every thread.
__device__ __forceinline__ uint32_t block_umax(uint32_t x) {
    __shared__ uint32_t part[4];
    x = wave_umax(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = max(max(part[0], part[1]), max(part[2], part[3]));
    __syncthreads();
    return x;
}

// One workgroup per (block of 64 rows, head, K or V, item): the block's new
// rows are read once into registers, eight elements a thread and piece, their
// amplitude is reduced, and the codes are written.  Bound by HBM: three bytes
// move per bf16 element (four prompts of 8,191 x 8 heads, 201 MB: 32 us where the
// last call's cache is still on the chip's side, 41 us, 4.9 TB/s, where it is
// not; a copy moves 5.2 TB/s), small calls by their one chain of load, reduction
// and store (a frame of 1,560 x 24 heads, 29 MB: 7.5 us).  Blocks that hold a
// value that is not finite take a slower path of the same results.
template <int DTYPE, int FMT, int P>
__global__ void __launch_bounds__(256) write_kernel(WriteParams p) {
    constexpr int CH = P / 8, STEP = 256 / CH, N = C8_BLOCK / STEP;
    constexpr float TOP = Fmt8<FMT>::TOP;
    using X = Piece<DTYPE>;
    const int kv = blockIdx.z & 1, b = blockIdx.z >> 1, h = blockIdx.y;
    const int64_t start =
        p.start_dev ? min(max((int64_t)p.start_dev[b], (int64_t)0), p.cap) : p.start;
    const int64_t count = p.counts ? min(max((int64_t)p.counts[b], (int64_t)0), p.T) : p.T;
    const int64_t end = min(start + count, p.cap);
    const int64_t blk = start / C8_BLOCK + blockIdx.x;
    const int64_t row0 = blk * C8_BLOCK;               // the block's first row
    if (row0 >= end || start >= end) return;
    const int64_t bh = (int64_t)b * p.H + h;
    uint8_t* codes = p.codes[kv] + (bh * p.cap + row0) * P;
    float* scale = p.scale[kv] + bh * (p.cap / C8_BLOCK) + blk;
    const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
    const int lo = (int)max(start - row0, (int64_t)0), hi = (int)min(end - row0, (int64_t)C8_BLOCK);
    X x[N];
    const int64_t src = b * p.sb[kv] + (row0 - start) * p.st[kv] + h * p.sh[kv] + 8 * c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + STEP * i;
        x[i] = X{};
        if (r >= lo && r < hi && 8 * c < p.D) x[i].load(p.x[kv], src + r * p.st[kv]);
    }
    const float s0 = lo > 0 ? *scale : 0.0f;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i].largest(m);
    if constexpr (DTYPE != NKV_ROWS_FP32) m = max(m & 0xffffu, m >> 16);
    m = block_umax(m);
    const bool finite = m < X::INF;
    float top = X::from(m);
    if (!finite) {  // the largest finite value
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = fabsf(x[i][e]);
                t = fmaxf(t, a < INFINITY ? a : 0.0f);
            }
        top = __uint_as_float(block_umax(__float_as_uint(t)));
    }
    float s = fmaxf(top, C8_TINY) / TOP;
    if (lo > 0) {
        if (s0 >= s) {
            s = s0;
        } else {
            const float ratio = s0 / s;
            for (int r = r0; r < lo; r += STEP) {
                u32x2* at = reinterpret_cast<u32x2*>(codes + r * P + 8 * c);
                u32x2 w = *at;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const f32x2 a = code_pair<FMT>(w[k], 0), d = code_pair<FMT>(w[k], 1);
                    w[k] = to_codes<FMT>(a[0] * ratio, a[1] * ratio, d[0] * ratio, d[1] * ratio);
                }
                *at = w;
            }
        }
    }
    const float y = 1.0f / s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + STEP * i;
        if (r < lo || r >= hi) continue;
        float q[8];
        u32x2 w;
        if (finite) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[e] = div_by(x[i][e], s, y);
                // (-0, whose remainder is +0; e4m3 keeps its sign)
                if constexpr (FMT == NKV_CACHE8_E4M3) q[e] = copysignf(q[e], x[i][e]);
            }
            w[0] = to_codes_fast<FMT>(q[0], q[1], q[2], q[3]);
            w[1] = to_codes_fast<FMT>(q[4], q[5], q[6], q[7]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = x[i][e] / s;
            w[0] = to_codes<FMT>(q[0], q[1], q[2], q[3]);
            w[1] = to_codes<FMT>(q[4], q[5], q[6], q[7]);
        }
        *reinterpret_cast<u32x2*>(codes + r * P + 8 * c) = w;
    }
    if (threadIdx.x == 0) *scale = s;  // read by every thread before block_umax
}

template <int DTYPE>
void write_launch(const WriteParams& p, int format, dim3 grid, hipStream_t s) {
    const bool wide = c8_pitch(p.D) == 128;
    if (format == NKV_CACHE8_INT8) {
        if (wide) write_kernel<DTYPE, NKV_CACHE8_INT8, 128><<<grid, 256, 0, s>>>(p);
        else write_kernel<DTYPE, NKV_CACHE8_INT8, 64><<<grid, 256, 0, s>>>(p);
    } else {
        if (wide) write_kernel<DTYPE, NKV_CACHE8_E4M3, 128><<<grid, 256, 0, s>>>(p);
        else write_kernel<DTYPE, NKV_CACHE8_E4M3, 64><<<grid, 256, 0, s>>>(p);
    }
}

// ---------------------------------------------------------------- evict
struct EvictParams {
    const uint8_t* codes[2];
    const float* scale[2];
    uint8_t* out[2];
    float* out_scale[2];
    const float* mass;
    float* out_mass;
    int32_t* rows;
    int32_t* out_length;
    const int32_t* length;
    int64_t cap, out_cap;
    int B, H, n, keep, sink, recent;
    void* work;                   // part_kernel: the states, then the counts
    int parts, part_rows;
};

// A mass as an integer that orders as the masses do: NaN above all, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    uint32_t u = __float_as_uint(x);
    if (u == 0x80000000u) u = 0;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The rows an eviction keeps of a head: the key of the last of them is found
// digit by digit (11, 11 and 10 bits, counts in LDS); then every wave lists the
// kept rows of its own contiguous part in order, behind those of the waves
// before it, rows equal to the last key from the lowest up.
constexpr int SEL_WAVES = 16, SEL_THREADS = 64 * SEL_WAVES;
constexpr int SEL_BINS = 2048, SEL_SLOTS = SEL_BINS + SEL_BINS / 32;

__device__ __forceinline__ constexpr int digit_shift(int pass) {
    return pass == 0 ? 21 : pass == 1 ? 10 : 0;
}
__device__ __forceinline__ constexpr uint32_t digit_top(int pass) {
    return pass == 2 ? 1023u : 2047u;
}

// digit d is counted at d + d / 32: lane l reads the 32 from 33 (63 - l) on
// in find_digit, without bank conflicts
__device__ __forceinline__ constexpr uint32_t bin(uint32_t d) { return d + (d >> 5); }

__device__ __forceinline__ void count_digit(uint32_t* hist, int lane, bool count, uint32_t d) {
    if (__ballot(count) == ~0ull) {  // one add where the whole wave has one digit (equal masses)
        const uint32_t d0 = __builtin_amdgcn_readfirstlane(d);
        if (__ballot(d == d0) == ~0ull) {
            if (lane == 0) atomicAdd(&hist[bin(d0)], 64u);
            return;
        }
    }
    if (count) atomicAdd(&hist[bin(d)], 1u);
}

// Sums over lanes 0 .. l: within the rows of 16, then from row to row (DPP).
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return x;
}

// The digit at which the count from above reaches `left`, found by every wave
// for itself: lane l has the 32 digits below 2048 - 32 l.  `left` becomes what
// is left at that digit.
__device__ __forceinline__ uint32_t find_digit(const uint32_t* hist, int lane, uint32_t& left) {
    uint32_t h[32], mine = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        h[i] = hist[33 * (63 - lane) + i];
        mine += h[i];
    }
    const uint32_t through = wave_scan(mine);
    const int l0 = __builtin_ctzll(__ballot(through >= left));
    uint32_t above = through - mine, passed = 32, over = above;
#pragma unroll
    for (int i = 31; i >= 0; --i) {
        above += h[i];
        if (above < left) {                             // the digit lies below this one
            passed = i;
            over = above;
        }
    }
    left -= (uint32_t)__builtin_amdgcn_readlane(over, l0);
    return (uint32_t)__builtin_amdgcn_readlane(SEL_BINS - 32 * (lane + 1) + passed - 1, l0);
}

// The key of row i: its mass's, which is at least that of -infinity, or for a
// row kept in any case 0, for one past the end 1.
struct Chosen {
    int lo, hi, n;                // the rows lo .. hi are chosen from
};
constexpr uint32_t FIXED = 0, PAST = 1;
__device__ __forceinline__ uint32_t row_key(const Chosen& r, float x, int i) {
    return i >= r.lo && i < r.hi ? order_key(x) : i < r.n ? FIXED : PAST;
}

// Lists the kept rows of a workgroup's part, in order, behind `bk` kept and `bt`
// tied rows before it: `left` of all rows whose key is `prefix`, and all above
// it.  each(f) calls f(key, row) for the keys of this wave's part.
template <typename Each>
__device__ __forceinline__ void list_rows(Each each, uint32_t prefix, uint32_t left, uint32_t want,
                                          uint32_t bk, uint32_t bt, int wave, int lane,
                                          int32_t* rows) {
    __shared__ uint32_t kept[SEL_WAVES], tied[SEL_WAVES];
    const uint32_t floor_key = want > 0 ? prefix : 0xffffffffu;
    uint32_t nk = 0, nt = 0;
    auto marks = [&](uint32_t k, uint64_t& a, uint64_t& t) {
        a = __ballot(k > floor_key || k == FIXED);
        t = __ballot(k == prefix);
    };
    each([&](uint32_t k, int) {
        uint64_t a, t;
        marks(k, a, t);
        nk += (uint32_t)__popcll(a);
        nt += (uint32_t)__popcll(t);
    });
    if (lane == 0) {
        kept[wave] = nk;
        tied[wave] = nt;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SEL_WAVES; ++w) {
        bk += w < wave ? kept[w] : 0;
        bt += w < wave ? tied[w] : 0;
    }
    each([&](uint32_t k, int i) {
        uint64_t a, t;
        marks(k, a, t);
        const uint32_t ra = bk + __builtin_amdgcn_mbcnt_hi((uint32_t)(a >> 32),
                                                           __builtin_amdgcn_mbcnt_lo((uint32_t)a, 0));
        if (t == 0) {
            if ((a >> lane) & 1) rows[ra + min(bt, left)] = i;
        } else {
            const uint32_t rt = bt + __builtin_amdgcn_mbcnt_hi(
                                         (uint32_t)(t >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)t, 0));
            if (((a >> lane) & 1) || (((t >> lane) & 1) && rt < left)) rows[ra + min(rt, left)] = i;
        }
        bk += (uint32_t)__popcll(a);
        bt += (uint32_t)__popcll(t);
    });
}

// Up to SEL_LDS rows: one workgroup a head, whose keys stay in LDS (one read of
// the masses, one launch).  It is bound by its CU's instruction issue: 64 heads
// of 32,768 rows 26.5 us, of which the first digit with the read takes 10, the
// others 5 each and the two passes of the list 7; 8 heads of 2,048 rows 9.6 us,
// a chain of barriers.
constexpr int SEL_LDS = 32768;
constexpr int SEL_AHEAD = 4;            // keys of a lane in flight from LDS

__global__ void __launch_bounds__(SEL_THREADS) select_kernel(EvictParams p) {
    const int b = blockIdx.x / p.H;
    const int64_t bh = blockIdx.x;
    const int n = c8_length(p.length, b, p.n);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int32_t* rows = p.rows + bh * p.keep;
    if (blockIdx.x % p.H == 0 && tid == 0) p.out_length[b] = min(n, p.keep);
    if (n <= p.keep) {
        for (int i = tid; i < p.keep; i += SEL_THREADS) rows[i] = i < n ? i : -1;
        return;
    }
    const float* mass = p.mass + bh * p.cap;
    const Chosen range{p.sink, n - p.recent, n};
    const uint32_t want = p.keep - p.sink - p.recent;
    // this wave's part: `steps` times 64 rows from `part` on
    const int steps = (n + SEL_THREADS - 1) / SEL_THREADS;
    const int part = wave * steps * 64;
    extern __shared__ __align__(16) uint32_t held[];    // the keys in row order
    __shared__ uint32_t hist[3][SEL_SLOTS];  // one a pass: no wave waits to reuse it
    // f(key, row) over the part in order, SEL_AHEAD keys in flight
    auto each = [&](auto f) {
        for (int j0 = 0; j0 < steps; j0 += SEL_AHEAD) {
            uint32_t k[SEL_AHEAD];
            const int i0 = part + 64 * j0 + lane;
#pragma unroll
            for (int j = 0; j < SEL_AHEAD; ++j)
                k[j] = held[i0 + 64 * j];  // (up to SEL_AHEAD steps past the end)
#pragma unroll
            for (int j = 0; j < SEL_AHEAD; ++j) {
                if (j0 + j >= steps) break;
                f(k[j], i0 + 64 * j);
            }
        }
    };
    uint32_t prefix = 0, left = want, mask = 0;
    for (int i = tid; i < 3 * SEL_SLOTS; i += SEL_THREADS) hist[0][i] = 0;
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = digit_shift(pass);
        const uint32_t top = digit_top(pass);
        if (pass == 0) {
            // four rows a thread and load, every load of the workgroup in flight
            constexpr int PER = SEL_LDS / (4 * SEL_THREADS);
            f32x4 x[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = 4 * (tid + SEL_THREADS * j);
                if (i < n) x[j] = *reinterpret_cast<const f32x4*>(mass + i);
            }
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = 4 * (tid + SEL_THREADS * j);
                if (4 * SEL_THREADS * j >= n) break;
                u32x4 k;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    k[e] = row_key(range, x[j][e], i + e);
                    count_digit(hist[0], lane, k[e] > PAST, k[e] >> shift);
                }
                if (i < steps * SEL_THREADS) *reinterpret_cast<u32x4*>(held + i) = k;
            }
        } else {
            each([&](uint32_t k, int) {
                count_digit(hist[pass], lane, (k & mask) == prefix, (k >> shift) & top);
            });
        }
        __syncthreads();
        prefix |= find_digit(hist[pass], lane, left) << shift;
        mask |= top << shift;
    }
    list_rows(each, prefix, left, want, 0, 0, wave, lane, rows);
}

// Longer heads: parts of PART_ROWS rows or more, at most PARTS of them, each one
// workgroup's.  A launch counts one digit over every part and stores the counts;
// the next adds up its head's parts (every workgroup for itself, no atomics in
// memory, nothing to clear), finds the digit and with it how many rows the parts
// before its own keep; the fourth lists.  Bound by the chain of four launches (4.9,
// 7.9, 7.8 and 10.5 us for one head of 131,072 rows; masses loaded ahead of the
// sums change nothing there and cost 10 % of a full chip's).  Whole evictions of
// width 64, a quarter kept: that head 34 us, where one workgroup that read the
// masses five times took 141; one of 1,000,000 rows 73; 64 heads of 65,536 rows 118
// (146 with one workgroup a head; at width 128, with twice the codes to move, 157).
// At SEL_LDS rows and below the chain costs more than it spreads (8 heads of 32,768
// rows: 34.7 us against select_kernel's 32.3, 64 heads: 65.6 against 60.8, 8 heads
// of 16,384: 30.8 against 21.4).  Parts of 4,096 rows add up twice the counts (64
// heads of 65,536 rows: 143 us), of 16,384 lengthen the chain (one head of 131,072:
// 39), and 128 parts a head instead of 64 add up more (one head of 1,000,000 rows, an
// earlier measure: 78 us against 65).
constexpr int PART_ROWS = 8192, PARTS = 64;

int part_rows(int64_t n) {
    const int64_t rows = std::max<int64_t>(PART_ROWS, (n + PARTS - 1) / PARTS);
    return (int)((rows + 4 * SEL_THREADS - 1) / (4 * SEL_THREADS) * (4 * SEL_THREADS));
}

// A part's counts of two passes (a launch reads one and writes the other) and what
// its workgroup knows after them.
struct PartState {
    uint32_t prefix, left, kept, pad;
};
constexpr size_t PART_BYTES = 2 * SEL_BINS * sizeof(uint32_t) + sizeof(PartState);

template <int PASS>
__global__ void __launch_bounds__(SEL_THREADS) part_kernel(EvictParams p) {
    const int64_t bh = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts, b = (int)(bh / p.H);
    const int n = c8_length(p.length, b, p.n);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int32_t* rows = p.rows + bh * p.keep;
    if (PASS == 0 && part == 0 && tid == 0 && bh % p.H == 0) p.out_length[b] = min(n, p.keep);
    if (n <= p.keep) {
        if (PASS == 0)
            for (int i = part * SEL_THREADS + tid; i < p.keep; i += p.parts * SEL_THREADS)
                rows[i] = i < n ? i : -1;
        return;
    }
    const int first = part * p.part_rows;
    if (first >= n) return;
    const int last = min(first + p.part_rows, n), active = (n + p.part_rows - 1) / p.part_rows;
    const float* mass = p.mass + bh * p.cap;
    const Chosen range{p.sink, n - p.recent, n};
    const uint32_t want = p.keep - p.sink - p.recent;
    const int64_t all = (int64_t)p.B * p.H * p.parts;
    PartState* state = reinterpret_cast<PartState*>(p.work) + blockIdx.x;
    uint32_t* counts = reinterpret_cast<uint32_t*>(reinterpret_cast<PartState*>(p.work) + all);
    auto counts_of = [&](int pass, int w) {
        return counts + ((pass & 1) * all + bh * p.parts + w) * SEL_BINS;
    };
    __shared__ uint32_t hist[SEL_SLOTS], total[SEL_SLOTS], sums[SEL_WAVES], tie;
    for (int i = tid; i < SEL_SLOTS; i += SEL_THREADS) hist[i] = 0;
    uint32_t prefix = 0, mask = 0, tied = 0;
    PartState st{0, want, 0, 0};
    if constexpr (PASS > 0) {
        if constexpr (PASS > 1) st = *state;
        // digits 2 tid and 2 tid + 1 of all parts, and of those before this one
        u32x2 s{}, e{};
#pragma unroll 8
        for (int w = 0; w < active; ++w) {
            const u32x2 x = reinterpret_cast<const u32x2*>(counts_of(PASS - 1, w))[tid];
            s += x;
            if (w < part) e += x;
        }
        total[bin(2 * tid)] = s[0];
        total[bin(2 * tid + 1)] = s[1];
        __syncthreads();
        const uint32_t d = find_digit(total, lane, st.left);
        const uint32_t over = (2u * tid > d ? e[0] : 0) + (2u * tid + 1 > d ? e[1] : 0);
        if (tid == (int)(d >> 1)) tie = e[d & 1];
        const uint32_t sum = wave_scan(over);
        if (lane == 63) sums[wave] = sum;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SEL_WAVES; ++w) st.kept += sums[w];
        tied = tie;
        prefix = st.prefix |= d << digit_shift(PASS - 1);
        if (PASS < 3 && tid == 0) *state = st;
        mask = PASS == 1 ? 0xffe00000u : 0xfffffc00u;
    } else {
        __syncthreads();
    }
    if constexpr (PASS < 3) {
        for (int i0 = first + 4 * tid; i0 < first + p.part_rows; i0 += PART_ROWS) {
            f32x4 x[PART_ROWS / (4 * SEL_THREADS)];
#pragma unroll
            for (int j = 0; j < PART_ROWS / (4 * SEL_THREADS); ++j) {
                const int i = i0 + 4 * SEL_THREADS * j;
                x[j] = f32x4{};
                if (i < last) x[j] = *reinterpret_cast<const f32x4*>(mass + i);
            }
#pragma unroll
            for (int j = 0; j < PART_ROWS / (4 * SEL_THREADS); ++j) {
                const int i = i0 + 4 * SEL_THREADS * j;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // (rows of the next part, where this one's end inside the step, do not count)
                    const uint32_t k = i < last ? row_key(range, x[j][e], i + e) : PAST;
                    count_digit(hist, lane, PASS == 0 ? k > PAST : (k & mask) == prefix,
                                (k >> digit_shift(PASS)) & digit_top(PASS));
                }
            }
        }
        __syncthreads();
        const u32x2 mine{hist[bin(2 * tid)], hist[bin(2 * tid + 1)]};
        reinterpret_cast<u32x2*>(counts_of(PASS, part))[tid] = mine;
    } else {
        const int steps = (last - first + SEL_THREADS - 1) / SEL_THREADS;
        const int begin = first + wave * steps * 64;
        constexpr int AHEAD = 8;
        auto each = [&](auto f) {
            for (int j0 = 0; j0 < steps; j0 += AHEAD) {
                float x[AHEAD];
                const int i0 = begin + 64 * j0 + lane;
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) x[j] = mass[min(i0 + 64 * j, n - 1)];
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    if (j0 + j >= steps) break;
                    const int i = i0 + 64 * j;
                    f(i < last ? row_key(range, x[j], i) : PAST, i);
                }
            }
        };
        const uint32_t fixed = min(first, range.lo) + max(first - range.hi, 0);
        list_rows(each, prefix, st.left, want, fixed + st.kept, tied, wave, lane, rows);
    }
}

// One workgroup per (block of 64 kept rows, head, K or V, item): gathers the
// rows' codes onto the largest of their scales.  Bound by HBM: 64 heads of 8,192
// kept rows, 236 MB, in 47 us, 5.0 TB/s (a copy moves 5.2).
template <int FMT, int P>
__global__ void __launch_bounds__(256) compact_kernel(EvictParams p) {
    constexpr int CH = P / 8, STEP = 256 / CH, N = C8_BLOCK / STEP;
    const int kv = blockIdx.z & 1, b = blockIdx.z >> 1, h = blockIdx.y;
    const int left = min(c8_length(p.length, b, p.n), p.keep);
    const int row0 = blockIdx.x * C8_BLOCK;
    if (row0 >= left) return;
    const int hi = min(left - row0, C8_BLOCK);
    const int64_t bh = (int64_t)b * p.H + h;
    __shared__ int src[C8_BLOCK];
    __shared__ float from[C8_BLOCK];
    __shared__ float top;
    if (threadIdx.x < 64) {
        const int r = threadIdx.x;
        int at = 0;
        float s = 0.0f;
        if (r < hi) {
            at = p.rows[bh * p.keep + row0 + r];
            s = p.scale[kv][bh * (p.cap / C8_BLOCK) + at / C8_BLOCK];
            if (kv == 0) p.out_mass[bh * p.out_cap + row0 + r] = p.mass[bh * p.cap + at];
        }
        src[r] = at;
        from[r] = s;
        const float m = __uint_as_float(wave_umax(__float_as_uint(s)));  // (not negative)
        if (r == 0) {
            top = m;
            p.out_scale[kv][bh * (p.out_cap / C8_BLOCK) + blockIdx.x] = m;
        }
    }
    __syncthreads();
    const uint8_t* codes = p.codes[kv] + bh * p.cap * P;
    uint8_t* out = p.out[kv] + (bh * p.out_cap + row0) * P;
    const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
    const float s = top;
    u32x2 w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + STEP * i;
        if (r < hi) w[i] = *reinterpret_cast<const u32x2*>(codes + (int64_t)src[r] * P + 8 * c);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + STEP * i;
        if (r >= hi) continue;
        const float s0 = from[r];
        if (s0 != s) {
            const float ratio = s0 / s;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f32x2 a = code_pair<FMT>(w[i][k], 0), d = code_pair<FMT>(w[i][k], 1);
                w[i][k] = to_codes<FMT>(a[0] * ratio, a[1] * ratio, d[0] * ratio, d[1] * ratio);
            }
        }
        *reinterpret_cast<u32x2*>(out + r * P + 8 * c) = w[i];
    }
}

int evict_parts(int64_t n) { return (int)cdiv(n, part_rows(n)); }

int check_evict(const nkv_cache8_evict_args* a) {
    NKV_REQUIRE(a, NKV_ERR_INVALID, "args is null");
    int rc = cache8_check(&a->cache, __func__);
    if (rc) return rc;
    rc = cache8_check(&a->out, __func__);
    if (rc) return rc;
    const nkv_cache8 &c = a->cache, &o = a->out;
    NKV_REQUIRE(c.B == o.B && c.H == o.H && c.D == o.D && c.format == o.format, NKV_ERR_INVALID,
                "out must be a cache of the same items, heads, width and format");
    NKV_REQUIRE(a->n >= 0 && a->n <= c.cap, NKV_ERR_INVALID, "n must be in [0, cap]");
    NKV_REQUIRE(a->keep >= 1 && a->keep <= o.cap, NKV_ERR_INVALID, "keep must be in [1, out.cap]");
    NKV_REQUIRE(a->sink >= 0 && a->recent >= 0 && a->sink <= a->keep && a->recent <= a->keep - a->sink,
                NKV_ERR_INVALID, "sink + recent must be at most keep");
    NKV_REQUIRE(c.H <= 65535 && c.B <= 32767, NKV_ERR_UNSUPPORTED, "too many heads or items");
    if (c.B == 0) return NKV_OK;
    NKV_REQUIRE(a->mass && a->out_mass && a->rows && a->out_length, NKV_ERR_INVALID,
                "mass, out_mass, rows and out_length are required");
    NKV_REQUIRE(reinterpret_cast<uintptr_t>(a->mass) % 16 == 0, NKV_ERR_INVALID,
                "mass must be 16-byte aligned");
    const int64_t heads = (int64_t)c.B * c.H, P = c8_pitch(c.D);
    const Range in[6] = {{c.k, heads * c.cap * P}, {c.v, heads * c.cap * P},
                         {c.k_scale, heads * c.cap / 16}, {c.v_scale, heads * c.cap / 16},
                         {a->mass, heads * c.cap * 4}, {a->length, a->length ? c.B * 4 : 0}};
    const Range out[7] = {{o.k, heads * o.cap * P}, {o.v, heads * o.cap * P},
                          {o.k_scale, heads * o.cap / 16}, {o.v_scale, heads * o.cap / 16},
                          {a->out_mass, heads * o.cap * 4}, {a->rows, heads * a->keep * 4},
                          {a->out_length, c.B * 4}};
    for (int i = 0; i < 7; ++i) {
        for (const Range& r : in)
            NKV_REQUIRE(!out[i].meets(r), NKV_ERR_INVALID,
                        "the outputs overlap the cache, mass or length");
        for (int j = 0; j < i; ++j)
            NKV_REQUIRE(!out[i].meets(out[j]), NKV_ERR_INVALID, "the outputs overlap each other");
    }
    NKV_REQUIRE(a->n <= SEL_LDS || heads * evict_parts(a->n) < 1 << 22, NKV_ERR_UNSUPPORTED,
                "too many heads of this length");
    return NKV_OK;
}

size_t evict_bytes(const nkv_cache8_evict_args* a) {
    if (a->n <= SEL_LDS) return 0;
    return (size_t)a->cache.B * a->cache.H * evict_parts(a->n) * PART_BYTES;
}

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" int nkv_cache8_write(void* stream, const nkv_cache8_write_args* a) {
    clear_error();
    NKV_REQUIRE(a, NKV_ERR_INVALID, "args is null");
    int rc = cache8_check(&a->cache, __func__);
    if (rc) return rc;
    const nkv_cache8& c = a->cache;
    NKV_REQUIRE(a->T >= 0 && a->T <= INT32_MAX, NKV_ERR_INVALID, "T must be in [0, 2^31)");
    NKV_REQUIRE(a->dtype >= NKV_ROWS_BF16 && a->dtype <= NKV_ROWS_FP32, NKV_ERR_INVALID,
                "unknown row dtype");
    if (!a->start_dev)
        NKV_REQUIRE(a->start >= 0 && a->start <= c.cap && (a->counts || a->T <= c.cap - a->start),
                    NKV_ERR_INVALID, "rows start .. start + T must lie in [0, cap]");
    NKV_REQUIRE(c.H <= 65535 && c.B <= 32767, NKV_ERR_UNSUPPORTED, "too many heads or items");
    if (c.B == 0 || a->T == 0) return NKV_OK;
    NKV_REQUIRE(a->k && a->v, NKV_ERR_INVALID, "k and v are required");
    NKV_REQUIRE((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) % 16 == 0 &&
                    (a->k_sb | a->k_st | a->k_sh | a->v_sb | a->v_st | a->v_sh) % 8 == 0,
                NKV_ERR_INVALID, "k and v must be 16-byte aligned with strides divisible by 8");
    const int64_t heads = (int64_t)c.B * c.H, bytes = heads * c.cap * c8_pitch(c.D);
    const Range out[4] = {{c.k, bytes}, {c.v, bytes}, {c.k_scale, heads * c.cap / 16},
                          {c.v_scale, heads * c.cap / 16}};
    for (int i = 1; i < 4; ++i)
        for (int j = 0; j < i; ++j)
            NKV_REQUIRE(!out[i].meets(out[j]), NKV_ERR_INVALID,
                        "the cache's codes and scales overlap each other");
    for (const Range& r : out)
        NKV_REQUIRE(!r.meets({a->start_dev, a->start_dev ? c.B * 4 : 0}) &&
                        !r.meets({a->counts, a->counts ? c.B * 4 : 0}),
                    NKV_ERR_INVALID, "the cache overlaps start_dev or counts");
    WriteParams p{{(uint8_t*)c.k, (uint8_t*)c.v}, {c.k_scale, c.v_scale}, {a->k, a->v},
                  {a->k_sb, a->v_sb}, {a->k_st, a->v_st}, {a->k_sh, a->v_sh},
                  a->start_dev, a->counts, c.cap, a->start, a->T, c.B, c.H, c.D};
    // blocks that rows start .. start + T may touch, start anywhere in a block
    int64_t blocks = (std::min<int64_t>(a->T, c.cap) + C8_BLOCK - 2) / C8_BLOCK + 1;
    if (!a->start_dev)
        blocks = cdiv(std::min<int64_t>(a->start + a->T, c.cap), C8_BLOCK) - a->start / C8_BLOCK;
    if (blocks <= 0) return NKV_OK;
    const dim3 grid((unsigned)blocks, (unsigned)c.H, (unsigned)(2 * c.B));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (a->dtype == NKV_ROWS_BF16) write_launch<NKV_ROWS_BF16>(p, c.format, grid, s);
    else if (a->dtype == NKV_ROWS_FP16) write_launch<NKV_ROWS_FP16>(p, c.format, grid, s);
    else write_launch<NKV_ROWS_FP32>(p, c.format, grid, s);
    NKV_LAUNCH_CHECK();
    return NKV_OK;
}

extern "C" size_t nkv_cache8_evict_workspace_size(const nkv_cache8_evict_args* a) {
    clear_error();
    return check_evict(a) == NKV_OK ? evict_bytes(a) : 0;
}

extern "C" int nkv_cache8_evict(void* stream, const nkv_cache8_evict_args* a, void* workspace,
                                size_t workspace_bytes) {
    clear_error();
    int rc = check_evict(a);
    if (rc) return rc;
    const nkv_cache8 &c = a->cache, &o = a->out;
    if (c.B == 0) return NKV_OK;
    const size_t need = evict_bytes(a);
    NKV_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), NKV_ERR_WORKSPACE,
                "workspace is smaller than nkv_cache8_evict_workspace_size");
    NKV_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, NKV_ERR_INVALID,
                "workspace must be 16-byte aligned");
    EvictParams p{{(const uint8_t*)c.k, (const uint8_t*)c.v}, {c.k_scale, c.v_scale},
                  {(uint8_t*)o.k, (uint8_t*)o.v}, {o.k_scale, o.v_scale}, a->mass, a->out_mass,
                  a->rows, a->out_length, a->length, c.cap, o.cap, c.B, c.H, (int)a->n,
                  (int)a->keep, (int)a->sink, (int)a->recent, workspace, 0, 0};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (need == 0) {
        // whole steps of every wave, and the reads ahead of the last one
        const size_t smem = (size_t)(cdiv(a->n, SEL_THREADS) * SEL_THREADS + 64 * SEL_AHEAD) * 4;
        if ((rc = set_smem(select_kernel, smem))) return rc;
        select_kernel<<<(unsigned)(c.B * c.H), SEL_THREADS, smem, s>>>(p);
    } else {
        p.part_rows = part_rows(a->n);
        p.parts = evict_parts(a->n);
        const unsigned grid = (unsigned)(c.B * c.H * p.parts);
        part_kernel<0><<<grid, SEL_THREADS, 0, s>>>(p);
        part_kernel<1><<<grid, SEL_THREADS, 0, s>>>(p);
        part_kernel<2><<<grid, SEL_THREADS, 0, s>>>(p);
        part_kernel<3><<<grid, SEL_THREADS, 0, s>>>(p);
    }
    NKV_LAUNCH_CHECK();
    const int64_t blocks = cdiv(std::min(a->keep, a->n), C8_BLOCK);
    if (blocks) {
        const dim3 grid((unsigned)blocks, (unsigned)c.H, (unsigned)(2 * c.B));
        const bool wide = c8_pitch(c.D) == 128;
        if (c.format == NKV_CACHE8_INT8) {
            if (wide) compact_kernel<NKV_CACHE8_INT8, 128><<<grid, 256, 0, s>>>(p);
            else compact_kernel<NKV_CACHE8_INT8, 64><<<grid, 256, 0, s>>>(p);
        } else {
            if (wide) compact_kernel<NKV_CACHE8_E4M3, 128><<<grid, 256, 0, s>>>(p);
            else compact_kernel<NKV_CACHE8_E4M3, 64><<<grid, 256, 0, s>>>(p);
        }
        NKV_LAUNCH_CHECK();
    }
    return NKV_OK;
}
