// nkv_paged.hip -- writes of the paged key/value cache: the append of new rows with
// their rotation (nkv_paged_append) and the commit of a draft's accepted rows
// (nkv_paged_commit).
#include "nkv_paged.h"

#include <algorithm>
#include <utility>

namespace nkv {
namespace {

// ---------------------------------------------------------------- append
struct RowsAt {
    const void* p;
    int64_t sb, st, sh;
};

struct AppendParams {
    PageTable table;
    uint16_t* pool_k;
    uint16_t* pool_v;
    RowsAt k, v, q;
    uint16_t* out;
    int64_t o_sb, o_st, o_sh;
    const float* freqs;
    const int32_t* positions;
    int64_t pos_sb, start;
    const int32_t* start_dev;
    const int32_t* counts;
    uint32_t B, T, units, slots;  // 16-column units of a row, threads that share a token's rows
    int H, Hq, D, rot, interleaved, page_d;
};

// Eight values of a row of the cache's type or fp32.
struct Eight {
    float x[8];
};
template <typename T, bool F32>
__device__ __forceinline__ Eight load8(const void* p, int64_t at) {
    Eight e;
    if constexpr (F32) {
        const f32x4* s = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + at);
        const f32x4 a = s[0], b = s[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) e.x[i] = a[i], e.x[4 + i] = b[i];
    } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) e.x[i] = T::to_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
    }
    return e;
}
template <typename T>
__device__ __forceinline__ void store8(uint16_t* p, const Eight& e) {
    *reinterpret_cast<u32x4*>(p) = u32x4{T::pack(e.x[0], e.x[1]), T::pack(e.x[2], e.x[3]),
                                         T::pack(e.x[4], e.x[5]), T::pack(e.x[6], e.x[7])};
}

// The cosine and sine of position * freq.  In turns and in 64 bits, where whole turns
// drop out exactly; the rest, at most half a turn, is within 2^-25 of a turn in 32.
__device__ __forceinline__ void turn(double position, float freq, float& c, float& s) {
    constexpr double PER_TURN = 0.15915494309189535;   // 1 / 2 pi
    double t = position * ((double)freq * PER_TURN);
    t -= rint(t);
    sincospif(2.0f * (float)t, &s, &c);
}

// A thread takes one 16-column unit of a token's rows slot, slot + slots, .. (queries,
// keys, values in turn): two 8-column chunks, the two that a rotation of halves
// couples or two neighbours, so that the unit's eight angles are formed once for all of
// them.  Bound by memory: 32,764 tokens of 48 heads' rows, 0.8 GB, 150 to 157 us, 5.1 to
// 5.3 TB/s; 1,560 of 72 heads' 57 MB 13.6 us, where launch and angles show.
template <typename T, bool F32>
__global__ void __launch_bounds__(256) append_kernel(AppendParams p) {
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    const uint32_t unit = g % p.units, rest = g / p.units;
    const uint32_t slot = rest % p.slots, token = rest / p.slots;
    if (token >= p.B * p.T) return;
    const int b = (int)(token / p.T), t = (int)(token - (uint32_t)b * p.T);
    if (t >= c8_length(p.counts, b, (int)p.T)) return;
    const int64_t row = paged_start(p.start_dev, b, p.start, p.table.cap()) + t;
    const int64_t dst = page_row(p.table, b, row, p.D);
    // the unit's chunks, and the first frequency of each
    const int chunks = p.D / 8, turned = p.rot / 8, half = p.rot / 16;
    int ca, cb;
    bool halves = false;
    if (!p.interleaved && (int)unit < half) {
        ca = (int)unit;
        cb = ca + half;
        halves = true;
    } else {
        ca = p.interleaved ? 2 * (int)unit : turned + 2 * ((int)unit - half);
        cb = ca + 1;
    }
    const bool has_b = cb < chunks;
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.0f, s[i] = 0.0f;
    const bool turns_a = halves || (p.interleaved && ca < turned);
    const bool turns_b = halves || (p.interleaved && cb < turned);
    if (turns_a && (int)slot < p.Hq + p.H) {
        const double at = p.positions ? p.positions[b * p.pos_sb + t] : row;
        const float* f = p.freqs + (halves ? 8 * ca : 4 * ca);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < 4 || halves || turns_b) turn(at, f[i], c[i], s[i]);
    }
    for (int r = (int)slot; r < p.Hq + 2 * p.H; r += (int)p.slots) {
        const int kind = r < p.Hq ? 0 : r < p.Hq + p.H ? 1 : 2;
        const int head = r - (kind == 0 ? 0 : kind == 1 ? p.Hq : p.Hq + p.H);
        if (kind && dst < 0) break;  // (queries come first)
        const RowsAt& src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
        const int64_t at = b * src.sb + t * src.st + head * src.sh;
        uint16_t* to = kind == 0 ? p.out + b * p.o_sb + t * p.o_st + head * p.o_sh
                                 : (kind == 1 ? p.pool_k : p.pool_v) + dst + (int64_t)head * p.page_d;
        Eight x = load8<T, F32>(src.p, at + 8 * ca), y{};
        if (has_b) y = load8<T, F32>(src.p, at + 8 * cb);
        if (kind < 2 && halves) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = x.x[i], w = y.x[i];
                x.x[i] = u * c[i] - w * s[i];
                y.x[i] = w * c[i] + u * s[i];
            }
        } else if (kind < 2 && turns_a) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float u = x.x[2 * i], w = x.x[2 * i + 1];
                x.x[2 * i] = u * c[i] - w * s[i];
                x.x[2 * i + 1] = w * c[i] + u * s[i];
                if (turns_b) {
                    u = y.x[2 * i], w = y.x[2 * i + 1];
                    y.x[2 * i] = u * c[4 + i] - w * s[4 + i];
                    y.x[2 * i + 1] = w * c[4 + i] + u * s[4 + i];
                }
            }
        }
        store8<T>(to + 8 * ca, x);
        if (has_b) store8<T>(to + 8 * cb, y);
    }
}

// ---------------------------------------------------------------- commit

struct CommitParams {
    PageTable table;
    const int32_t* rows;
    int64_t rows_sb, start;
    const int32_t* start_dev;
    const int32_t* counts;
    int32_t* out_length;
    int H, D, M, B, page_d;
    uint16_t* pool[NKV_PAGED_CACHES][2];
};

// A workgroup moves one head's rows of one sequence in one cache, all of which it holds
// in registers before it writes any: thread t has 16 bytes of rows t / 16 + 16 i.  Bound by
// its chain of loads (row, two table entries, the row's bytes) and the launch: 5 rows of 8
// sequences in 16 caches of 8 heads, 10 MB both ways, 3.2 us; so all caches in one launch.
template <int ROUNDS>
__global__ void __launch_bounds__(256) commit_kernel(CommitParams p) {
    const int b = blockIdx.y, h = blockIdx.x, chunk = threadIdx.x & 15;
    const int n = c8_length(p.counts, b, p.M);
    const int64_t start = paged_start(p.start_dev, b, p.start, p.table.cap());
    if (p.out_length && h == 0 && blockIdx.z == 0 && threadIdx.x == 0)
        p.out_length[b] = (int32_t)min(start + n, (int64_t)INT32_MAX);
    u32x4 x[ROUNDS][2];
    int64_t to[ROUNDS];
    uint16_t* const pk = p.pool[blockIdx.z][0];
    uint16_t* const pv = p.pool[blockIdx.z][1];
    const int64_t mine = (int64_t)h * p.page_d + 8 * chunk;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int j = threadIdx.x / 16 + 16 * i;
        to[i] = -1;
        if (j < n && 8 * chunk < p.D) {
            const int64_t row = p.rows[b * p.rows_sb + j];
            const int64_t from = row < 0 ? -1 : page_row(p.table, b, start + row, p.D);
            const int64_t dst = page_row(p.table, b, start + j, p.D);
            if (row != j && from >= 0 && dst >= 0) {
                to[i] = dst + mine;
                x[i][0] = *reinterpret_cast<const u32x4*>(pk + from + mine);
                x[i][1] = *reinterpret_cast<const u32x4*>(pv + from + mine);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i)
        if (to[i] >= 0) {
            *reinterpret_cast<u32x4*>(pk + to[i]) = x[i][0];
            *reinterpret_cast<u32x4*>(pv + to[i]) = x[i][1];
        }
}

// ---------------------------------------------------------------- host
int fail(const char* who, int code, const char* what) {
    set_error(std::string(who) + ": " + what);
    return code;
}

int check_start(int64_t start, const int32_t* start_dev, const int32_t* counts, int64_t rows,
                int64_t cap, const char* who) {
    if (start_dev) return NKV_OK;
    if (start < 0 || start > std::min<int64_t>(cap, INT32_MAX) || (!counts && rows > cap - start))
        return fail(who, NKV_ERR_INVALID, "rows from start on must lie in the table");
    return NKV_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

int paged_check(const nkv_paged_cache& c, const char* who) {
    if (c.dtype != NKV_ROWS_BF16 && c.dtype != NKV_ROWS_FP16)
        return fail(who, NKV_ERR_INVALID, "the cache must be bf16 or fp16");
    if (c.D < 1 || c.H < 1) return fail(who, NKV_ERR_INVALID, "D >= 1 and H >= 1 are required");
    if (c.D % 8 || c.D > 128)
        return fail(who, NKV_ERR_UNSUPPORTED, "D must be a multiple of 8, at most 128");
    if (c.page < 16 || c.page > 1024 || (c.page & (c.page - 1)))
        return fail(who, NKV_ERR_UNSUPPORTED, "page must be a power of two in [16, 1024]");
    if (c.pages < 1 || c.pages > INT32_MAX)
        return fail(who, NKV_ERR_INVALID, "pages must be in [1, 2^31)");
    if ((int64_t)c.H * c.page * c.D > 1 << 29 || c.H > 65535)
        return fail(who, NKV_ERR_UNSUPPORTED, "too many heads");
    if (!c.k || !c.v || !aligned16(c.k) || !aligned16(c.v))
        return fail(who, NKV_ERR_INVALID, "k and v are required and 16-byte aligned");
    return NKV_OK;
}

int paged_table_check(const nkv_paged_cache& c, const int32_t* table, int64_t sb, int64_t w, int B,
                      const char* who) {
    if (B < 0 || w < 0 || w > INT32_MAX)
        return fail(who, NKV_ERR_INVALID, "B >= 0 and table_w in [0, 2^31) are required");
    if (B > 65535) return fail(who, NKV_ERR_UNSUPPORTED, "too many sequences");
    if (sb < 0 || sb > INT64_MAX / 4 / 65536) return fail(who, NKV_ERR_INVALID, "table_sb out of range");
    if (B > 0 && w > 0 && !table) return fail(who, NKV_ERR_INVALID, "table is required");
    return NKV_OK;
}

PageTable page_table(const nkv_paged_cache& c, const int32_t* table, int64_t sb, int64_t w) {
    return {table, sb, w, (uint32_t)c.pages, __builtin_ctz((unsigned)c.page), (int64_t)c.H * c.page * c.D};
}

int64_t rows_span(int64_t s0, int64_t n0, int64_t s1, int64_t n1, int64_t s2, int64_t n2, int D) {
    std::pair<int64_t, int64_t> dims[3] = {{s0, n0}, {s1, n1}, {s2, n2}};
    std::sort(dims, dims + 3);
    __int128 end = D;
    for (const auto& [stride, count] : dims) {
        if (count == 1) continue;
        if (stride < end) return -1;
        end += (__int128)stride * (count - 1);
    }
    return end > INT64_MAX / 8 ? -1 : (int64_t)end;
}

RowSet::RowSet(const void* p, int es, int D, int64_t s0, int64_t n0, int64_t s1, int64_t n1,
               int64_t s2, int64_t n2) {
    if (!p) return;
    at = reinterpret_cast<uintptr_t>(p);
    span = bytes = (int64_t)D * es;
    const int64_t s[3] = {s0, s1, s2}, n[3] = {n0, n1, n2};
    // (a dimension of stride 0 is the same rows again)
    for (int i = 0; i < 3; ++i)
        if (s[i] > 0 && n[i] > 1) {
            dims[i].stride = std::min(s[i], INT64_MAX / 8) * es;
            dims[i].count = n[i];
            span += (__int128)dims[i].stride * (n[i] - 1);
        }
}

namespace {

struct Steps {
    __int128 stride, count;
};

// A set's dimensions in descending order of their strides.
struct Nest {
    Steps d[3];
    int n = 0;
    bool apart = true, packed;             // no two rows overlap; no gaps either
    explicit Nest(const RowSet& r) {
        __int128 rows = 1, span = r.bytes;
        for (const auto& x : r.dims)
            if (x.count > 1) d[n++] = {x.stride, x.count};
        std::sort(d, d + n, [](const Steps& a, const Steps& b) { return a.stride > b.stride; });
        for (int i = n - 1; i >= 0; --i) {
            apart = apart && d[i].stride >= span;
            span += d[i].stride * (d[i].count - 1);
            rows *= d[i].count;
        }
        packed = apart && span == rows * r.bytes;
    }
};

// Whether one of the rows of `bytes` bytes at `at` + multiples of n strides (descending)
// meets [lo, hi).  Of a dimension's parts only those that reach over an end of it are looked
// into: a part inside it holds a row.
bool steps_meet(const Steps* d, int n, __int128 at, __int128 bytes, __int128 lo, __int128 hi) {
    if (n == 0) return at < hi && at + bytes > lo;
    __int128 part = bytes;
    for (int i = 1; i < n; ++i) part += d[i].stride * (d[i].count - 1);
    const __int128 s = d[0].stride, before = lo - part - at;
    if (hi <= at) return false;
    const __int128 first = before < 0 ? 0 : before / s + 1, last = std::min((hi - 1 - at) / s, d[0].count - 1);
    for (__int128 i = first; i <= last; ++i) {
        const __int128 x = at + i * s;
        if ((x >= lo && x + part <= hi) || steps_meet(d + 1, n - 1, x, bytes, lo, hi)) return true;
    }
    return false;
}

}  // namespace

bool rows_meet(const RowSet& a, const RowSet& b) {
    const __int128 ax = a.at, by = b.at;
    if (a.bytes == 0 || b.bytes == 0 || ax >= by + b.span || by >= ax + a.span) return false;
    const Nest x(a), y(b);
    if (!x.apart || !y.apart) return true;
    if (x.packed) return steps_meet(y.d, y.n, by, b.bytes, ax, ax + a.span);
    if (y.packed) return steps_meet(x.d, x.n, ax, a.bytes, by, by + b.span);
    // like strides: the distances between a row of each are steps of the same strides
    Steps d[3];
    int n = 0;
    __int128 at = ax - by;
    for (int i = 0; i < 3; ++i) {
        const auto &p = a.dims[i], &q = b.dims[i];
        if (p.count > 1 && q.count > 1 && p.stride != q.stride) return false;
        const __int128 stride = p.count > 1 ? p.stride : q.stride;
        at -= stride * (q.count - 1);
        if (p.count > 1 || q.count > 1) d[n++] = {stride, (__int128)p.count + q.count - 1};
    }
    std::sort(d, d + n, [](const Steps& l, const Steps& r) { return l.stride > r.stride; });
    return steps_meet(d, n, at, 1, 1 - (__int128)a.bytes, b.bytes);
}

namespace {

template <typename T>
void append_run(const AppendParams& p, bool f32, unsigned grid, hipStream_t s) {
    if (f32) append_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else append_kernel<T, false><<<grid, 256, 0, s>>>(p);
}

// Threads that share a token's rows: as many as there are rows in small calls, above
// them a third (us with one, two, three, four and eight rows a thread: 512 tokens of 48
// heads' rows of 128 6.1, 6.0, 6.2, 6.8, 9.0; 1,024 9.0, 7.5, 7.3, 8.2, 11.5; 1,560 of 72
// 16.3, 13.8, 13.6, 14.0, 14.9; 32,764 of 48 238, 170, 157, 157, 162).
uint32_t append_slots(int64_t tokens, int units, int rows) {
    const int64_t per = std::clamp<int64_t>(tokens * units * rows >> 17, 1, 3);
    return (uint32_t)cdiv(rows, per);
}

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" int nkv_paged_append(void* stream, const nkv_paged_append_args* a) {
    clear_error();
    NKV_REQUIRE(a, NKV_ERR_INVALID, "args is null");
    const nkv_paged_cache& c = a->cache;
    int rc = paged_check(c, __func__);
    if (rc) return rc;
    if ((rc = paged_table_check(c, a->table, a->table_sb, a->table_w, a->B, __func__))) return rc;
    NKV_REQUIRE(a->T >= 0 && a->T <= INT32_MAX, NKV_ERR_INVALID, "T must be in [0, 2^31)");
    NKV_REQUIRE(a->dtype == c.dtype || a->dtype == NKV_ROWS_FP32, NKV_ERR_INVALID,
                "rows must have the cache's type or be fp32");
    const PageTable table = page_table(c, a->table, a->table_sb, a->table_w);
    if ((rc = check_start(a->start, a->start_dev, a->counts, a->T, table.cap(), __func__))) return rc;
    NKV_REQUIRE(!a->q || (a->q_out && a->Hq >= 1), NKV_ERR_INVALID, "q needs q_out and Hq >= 1");
    NKV_REQUIRE(a->q || !a->q_out, NKV_ERR_INVALID, "q_out needs q");
    NKV_REQUIRE(a->freqs || !a->q, NKV_ERR_INVALID, "q without freqs has nothing to be done");
    NKV_REQUIRE(a->freqs || !a->positions, NKV_ERR_INVALID, "positions need freqs");
    if (a->freqs) {
        NKV_REQUIRE(a->rot >= 2 && a->rot <= c.D, NKV_ERR_INVALID, "rot must be in [2, D]");
        NKV_REQUIRE(a->rot % (a->interleaved ? 8 : 16) == 0, NKV_ERR_UNSUPPORTED,
                    "rot must be a multiple of 16, of 8 where interleaved");
        NKV_REQUIRE(!a->positions || a->pos_sb >= 0, NKV_ERR_INVALID, "pos_sb must not be negative");
    }
    if (a->B == 0 || a->T == 0) return NKV_OK;
    const int Hq = a->q ? a->Hq : 0;
    NKV_REQUIRE(Hq <= 1 << 20 && (int64_t)a->B * a->T <= 1 << 26, NKV_ERR_UNSUPPORTED, "too many rows");
    NKV_REQUIRE(a->k && a->v, NKV_ERR_INVALID, "k and v are required");
    NKV_REQUIRE(aligned16(a->k) && aligned16(a->v) && aligned16(a->q) && aligned16(a->q_out) &&
                    (a->k_sb | a->k_st | a->k_sh | a->v_sb | a->v_st | a->v_sh) % 8 == 0 &&
                    (Hq == 0 || (a->q_sb | a->q_st | a->q_sh | a->o_sb | a->o_st | a->o_sh) % 8 == 0),
                NKV_ERR_INVALID, "rows must be 16-byte aligned with strides divisible by 8");
    NKV_REQUIRE(a->k_sb >= 0 && a->k_st >= 0 && a->k_sh >= 0 && a->v_sb >= 0 && a->v_st >= 0 &&
                    a->v_sh >= 0 && (Hq == 0 || (a->q_sb >= 0 && a->q_st >= 0 && a->q_sh >= 0)),
                NKV_ERR_INVALID, "strides must not be negative");
    // what is written, the pools and q_out, and what is read
    if (Hq) {
        NKV_REQUIRE(rows_span(a->o_sb, a->B, a->o_st, a->T, a->o_sh, Hq, c.D) > 0, NKV_ERR_INVALID,
                    "q_out's rows overlap");
        NKV_REQUIRE(a->q_out != a->k && a->q_out != a->v, NKV_ERR_INVALID, "q_out overlaps the rows");
        if (a->q_out == a->q)
            NKV_REQUIRE(a->dtype == c.dtype && a->q_sb == a->o_sb && a->q_st == a->o_st && a->q_sh == a->o_sh,
                        NKV_ERR_INVALID, "q_out over q must have its type and strides");
    }
    const int es = a->dtype == NKV_ROWS_FP32 ? 4 : 2;
    const RowSet k(a->k, es, c.D, a->k_sb, a->B, a->k_st, a->T, a->k_sh, c.H);
    const RowSet v(a->v, es, c.D, a->v_sb, a->B, a->v_st, a->T, a->v_sh, c.H);
    const RowSet q(a->q, es, c.D, a->q_sb, a->B, a->q_st, a->T, a->q_sh, Hq);
    const RowSet q_out(a->q_out, 2, c.D, a->o_sb, a->B, a->o_st, a->T, a->o_sh, Hq);
    const Range pools[2] = {{c.k, pool_bytes(c)}, {c.v, pool_bytes(c)}};
    const Range small[5] = {{a->table, table_bytes(a->B, a->table_sb, a->table_w)},
                            {a->start_dev, a->start_dev ? a->B * 4 : 0},
                            {a->counts, a->counts ? a->B * 4 : 0},
                            {a->freqs, a->freqs ? a->rot * 2 : 0},
                            {a->positions, a->positions ? table_bytes(a->B, a->pos_sb, a->T) : 0}};
    NKV_REQUIRE(!pools[0].meets(pools[1]), NKV_ERR_INVALID, "the pools overlap each other");
    for (const Range& r : pools) {
        NKV_REQUIRE(!rows_meet(r, k) && !rows_meet(r, v) && !rows_meet(r, q) && !rows_meet(r, q_out),
                    NKV_ERR_INVALID, "the pools overlap the rows");
        for (const Range& x : small)
            NKV_REQUIRE(!r.meets(x), NKV_ERR_INVALID,
                        "the pools overlap the table, start_dev, counts, freqs or positions");
    }
    for (const Range& x : small)
        NKV_REQUIRE(!rows_meet(q_out, x), NKV_ERR_INVALID,
                    "q_out overlaps the table, start_dev, counts, freqs or positions");
    NKV_REQUIRE(!rows_meet(q_out, k) && !rows_meet(q_out, v) && (a->q_out == a->q || !rows_meet(q_out, q)),
                NKV_ERR_INVALID, "q_out overlaps the rows");
    AppendParams p{};
    p.table = table;
    p.pool_k = (uint16_t*)c.k;
    p.pool_v = (uint16_t*)c.v;
    p.k = {a->k, a->k_sb, a->k_st, a->k_sh};
    p.v = {a->v, a->v_sb, a->v_st, a->v_sh};
    p.q = {a->q, a->q_sb, a->q_st, a->q_sh};
    p.out = (uint16_t*)a->q_out;
    p.o_sb = a->o_sb, p.o_st = a->o_st, p.o_sh = a->o_sh;
    p.freqs = a->freqs;
    p.positions = a->positions;
    p.pos_sb = a->pos_sb;
    p.start = a->start;
    p.start_dev = a->start_dev;
    p.counts = a->counts;
    p.B = (uint32_t)a->B, p.T = (uint32_t)a->T;
    p.H = c.H, p.Hq = Hq, p.D = c.D;
    p.rot = a->freqs ? a->rot : 0;
    p.interleaved = a->interleaved != 0;
    p.page_d = c.page * c.D;
    p.units = (uint32_t)cdiv(c.D, 16);
    p.slots = append_slots((int64_t)a->B * a->T, (int)p.units, Hq + 2 * c.H);
    const int64_t threads = (int64_t)a->B * a->T * p.units * p.slots;
    NKV_REQUIRE(threads <= (int64_t)1 << 31, NKV_ERR_UNSUPPORTED, "too many rows");
    const unsigned grid = (unsigned)cdiv(threads, 256);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const bool f32 = a->dtype == NKV_ROWS_FP32;
    if (c.dtype == NKV_ROWS_BF16) append_run<Bf16>(p, f32, grid, s);
    else append_run<Fp16>(p, f32, grid, s);
    NKV_LAUNCH_CHECK();
    return NKV_OK;
}

extern "C" int nkv_paged_commit(void* stream, const nkv_paged_commit_args* a) {
    clear_error();
    NKV_REQUIRE(a, NKV_ERR_INVALID, "args is null");
    NKV_REQUIRE(a->pools && a->n_caches >= 1, NKV_ERR_INVALID, "a cache is required");
    NKV_REQUIRE(a->n_caches <= NKV_PAGED_CACHES, NKV_ERR_UNSUPPORTED, "at most 64 caches a call");
    const int n = (int)a->n_caches;
    nkv_paged_cache c = a->cache;
    int rc = NKV_OK;
    for (int i = 0; i < n; ++i) {
        c.k = a->pools[2 * i], c.v = a->pools[2 * i + 1];
        if ((rc = paged_check(c, __func__))) return rc;
    }
    if ((rc = paged_table_check(c, a->table, a->table_sb, a->table_w, a->B, __func__))) return rc;
    const PageTable table = page_table(c, a->table, a->table_sb, a->table_w);
    NKV_REQUIRE(a->M >= 0, NKV_ERR_INVALID, "M must not be negative");
    NKV_REQUIRE(a->M <= NKV_PAGED_COMMIT, NKV_ERR_UNSUPPORTED, "M must be at most 256");
    NKV_REQUIRE(a->rows_sb >= 0 && (a->M == 0 || a->B == 0 || a->rows), NKV_ERR_INVALID,
                "rows is required, rows_sb must not be negative");
    if ((rc = check_start(a->start, a->start_dev, a->counts, a->M, table.cap(), __func__))) return rc;
    if (a->B == 0 || (a->M == 0 && !a->out_length)) return NKV_OK;
    // every pool against every other: sorted, neighbours must not meet
    uintptr_t sorted[2 * NKV_PAGED_CACHES];
    for (int i = 0; i < 2 * n; ++i) sorted[i] = reinterpret_cast<uintptr_t>(a->pools[i]);
    std::sort(sorted, sorted + 2 * n);
    const uintptr_t bytes = (uintptr_t)pool_bytes(c);
    for (int i = 1; i < 2 * n; ++i)
        NKV_REQUIRE(sorted[i] - sorted[i - 1] >= bytes, NKV_ERR_INVALID, "pools overlap");
    const Range small[5] = {{a->table, table_bytes(a->B, a->table_sb, a->table_w)},
                            {a->rows, a->M ? table_bytes(a->B, a->rows_sb, a->M) : 0},
                            {a->start_dev, a->start_dev ? a->B * 4 : 0},
                            {a->counts, a->counts ? a->B * 4 : 0},
                            {a->out_length, a->out_length ? a->B * 4 : 0}};
    for (int i = 0; i < 2 * n; ++i)
        for (const Range& r : small)
            NKV_REQUIRE(!r.meets({reinterpret_cast<const void*>(sorted[i]), (int64_t)bytes}),
                        NKV_ERR_INVALID, "the pools overlap the table, rows, start_dev, counts or out_length");
    for (int i = 0; i < 4; ++i)
        NKV_REQUIRE(!small[4].meets(small[i]), NKV_ERR_INVALID,
                    "out_length overlaps the table, rows, start_dev or counts");
    CommitParams p{};
    p.table = table;
    p.rows = a->rows;
    p.rows_sb = a->rows_sb;
    p.start = a->start;
    p.start_dev = a->start_dev;
    p.counts = a->counts;
    p.out_length = a->out_length;
    p.H = c.H, p.D = c.D, p.M = a->M, p.B = a->B;
    p.page_d = c.page * c.D;
    for (int i = 0; i < 2 * n; ++i) p.pool[i / 2][i % 2] = (uint16_t*)a->pools[i];
    const dim3 grid((unsigned)c.H, (unsigned)a->B, (unsigned)n);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    // (up to 64 rows with fewer registers: 8 sequences' 40 rows in 8 caches 5.3 us, 5.6)
    if (a->M <= 64) commit_kernel<4><<<grid, 256, 0, s>>>(p);
    else commit_kernel<16><<<grid, 256, 0, s>>>(p);
    NKV_LAUNCH_CHECK();
    return NKV_OK;
}
