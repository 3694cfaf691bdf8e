// nkv_cache8.h -- types and conversions shared by the kernels of the 8-bit
// key/value cache (nkv_cache8.hip, nkv_cache8_attend.hip).
//
// A cache holds, per batch item and key head, `cap` rows of 8-bit codes at a
// pitch of P = 64 or 128 bytes (the head width D rounded up, the columns past
// D zero) and one fp32 scale for each block of 64 rows: value = code * scale.
#pragma once

#include "nkv_common.h"

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

namespace nkv {

constexpr int C8_BLOCK = 64;                   // rows that share a scale
constexpr float C8_TINY = 0x1p-64f;            // the least amplitude a scale stands for

__host__ __device__ constexpr int c8_pitch(int D) { return D <= 64 ? 64 : 128; }

template <int FMT>
struct Fmt8 {
    static constexpr float TOP = FMT == NKV_CACHE8_INT8 ? 127.0f : 448.0f;
};

// Four values, already divided by their scale, as four codes: to the nearest,
// ties to even, clamped to the largest code; NaN gives the zero code, so that
// a cache never holds anything but finite numbers.
template <int FMT>
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
    float x[4] = {a, b, c, d};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = x[i] == x[i] ? x[i] : 0.0f;
        x[i] = fminf(fmaxf(x[i], -Fmt8<FMT>::TOP), Fmt8<FMT>::TOP);
    }
    if constexpr (FMT == NKV_CACHE8_INT8) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)rintf(x[i]) & 0xffu) << (8 * i);
        return w;
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
    }
}

// The values of codes 2 h and 2 h + 1 of a word (exact).
template <int FMT>
__device__ __forceinline__ f32x2 code_pair(uint32_t w, int h) {
    if constexpr (FMT == NKV_CACHE8_INT8) {
        return f32x2{(float)(int8_t)(w >> (16 * h)), (float)(int8_t)(w >> (16 * h + 8))};
    } else {
        return h ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true)
                 : __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    }
}

// x / s with y = 1 / s rounded to the nearest, itself rounded to the nearest:
// x y corrected twice by its exact remainder (the second correction of a result
// within one step rounds as the division does; Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor").  Five
// instructions, where the compiler's division takes ten.  Quotients below 2^-60,
// where a remainder may underflow, give the zero code either way; -0 gives +0.
__device__ __forceinline__ float div_by(float x, float s, float y) {
    float q = x * y;
    q = fmaf(fmaf(-q, s, x), y, q);
    return fmaf(fmaf(-q, s, x), y, q);
}

// to_codes of values that are known to be finite and within the largest code.
template <int FMT>
__device__ __forceinline__ uint32_t to_codes_fast(float a, float b, float c, float d) {
    if constexpr (FMT == NKV_CACHE8_INT8) {
        // 1.5 * 2^23 + x: the sum's rounding is the rounding to a whole number,
        // and its low byte is the code
        constexpr float BIG = 12582912.0f;
        const uint32_t x = __float_as_uint(a + BIG), y = __float_as_uint(b + BIG);
        const uint32_t z = __float_as_uint(c + BIG), w = __float_as_uint(d + BIG);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0c0c0400u),
                                     __builtin_amdgcn_perm(y, x, 0x0c0c0400u), 0x05040100u);
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    }
}

// max over a wave, in the VALU: the four 16-lane rows first, then lanes l ^ 8,
// l ^ 7, l ^ 2 and l ^ 1 of a row
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(b[0], b[1]);
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp(x, 0x128, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp(x, 0x141, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp(x, 0x4e, 0xf, 0xf, true));
    return max(x, (uint32_t)__builtin_amdgcn_mov_dpp(x, 0xb1, 0xf, 0xf, true));
}

// Eight values of a key split's partial result, in fp16 or in fp32.
struct Partial16 {
    u32x4 w;
    __device__ __forceinline__ void load(const void* p, int64_t at) {
        w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p) + at);
    }
    __device__ __forceinline__ void store(void* p, int64_t at) const {
        *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p) + at) = w;
    }
    __device__ __forceinline__ void set(const float (&o)[8], float f);
    __device__ __forceinline__ float operator[](int k) const {
        return f16_bits_to_f32((uint16_t)(w[k >> 1] >> (16 * (k & 1))));
    }
};

struct Partial32 {
    f32x4 a, b;
    __device__ __forceinline__ void load(const void* p, int64_t at) {
        const f32x4* q = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + at);
        a = q[0];
        b = q[1];
    }
    __device__ __forceinline__ void store(void* p, int64_t at) const {
        f32x4* q = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + at);
        q[0] = a;
        q[1] = b;
    }
    __device__ __forceinline__ void set(const float (&o)[8], float f) {
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = o[k] * f, b[k] = o[4 + k] * f;
    }
    __device__ __forceinline__ float operator[](int k) const { return k < 4 ? a[k] : b[k - 4]; }
};

// The 16-bit types of queries and outputs.  Both hold every code exactly, so
// scores are formed in the queries' own type.
struct Bf16 {
    using x8 = bf16x8;
    using Partial = Partial16;
    static __device__ __forceinline__ float to_f32(uint16_t b) { return bf16_bits_to_f32(b); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
    // e4m3 codes 2 h and 2 h + 1 of a word
    template <int h>
    static __device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, h));
    }
    static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

struct Fp16 {
    using x8 = f16x8;
    using Partial = Partial32;
    static __device__ __forceinline__ float to_f32(uint16_t b) { return f16_bits_to_f32(b); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        f16x2 v;
        v[0] = (_Float16)a;
        v[1] = (_Float16)b;
        uint32_t u;
        __builtin_memcpy(&u, &v, 4);
        return u;
    }
    template <int h>
    static __device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, h));
    }
    static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

__device__ __forceinline__ void Partial16::set(const float (&o)[8], float f) {
    w = u32x4{Fp16::pack(o[0] * f, o[1] * f), Fp16::pack(o[2] * f, o[3] * f),
              Fp16::pack(o[4] * f, o[5] * f), Fp16::pack(o[6] * f, o[7] * f)};
}

template <typename X8>
__device__ __forceinline__ X8 as_x8(u32x4 v) {
    X8 r;
    __builtin_memcpy(&r, &v, 16);
    return r;
}

// Eight consecutive codes as an MFMA operand of type T.
template <typename T, int FMT>
__device__ __forceinline__ typename T::x8 codes_x8(uint32_t lo, uint32_t hi) {
    if constexpr (FMT == NKV_CACHE8_E4M3)
        return as_x8<typename T::x8>(u32x4{T::template e4m3_pair<0>(lo), T::template e4m3_pair<1>(lo),
                                           T::template e4m3_pair<0>(hi), T::template e4m3_pair<1>(hi)});
    const f32x2 a = code_pair<FMT>(lo, 0), b = code_pair<FMT>(lo, 1);
    const f32x2 c = code_pair<FMT>(hi, 0), d = code_pair<FMT>(hi, 1);
    return as_x8<typename T::x8>(
        u32x4{T::pack(a[0], a[1]), T::pack(b[0], b[1]), T::pack(c[0], c[1]), T::pack(d[0], d[1])});
}

// Four columns of two rows' codes (one word each) as fp16 pairs (row a, row b) of
// each column.  int8: a code + 128 in the low byte of the half 0x6400 is 1,152 +
// code; two byte permutations and one packed subtraction, where converting and
// packing one code at a time takes half as many instructions again.
template <int FMT>
__device__ __forceinline__ void column_pairs(uint32_t a, uint32_t b, uint32_t (&out)[4]) {
    if constexpr (FMT == NKV_CACHE8_INT8) {
        a ^= 0x80808080u;
        b ^= 0x80808080u;
        const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u);  // a0 b0 a1 b1
        const uint32_t hi = __builtin_amdgcn_perm(b, a, 0x07030602u);  // a2 b2 a3 b3
        const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t x = __builtin_amdgcn_perm(0x64646464u, c < 2 ? lo : hi,
                                                     c & 1 ? 0x04030402u : 0x04010400u);
            out[c] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - bias);
        }
    } else {
        const f32x2 a0 = code_pair<FMT>(a, 0), a1 = code_pair<FMT>(a, 1);
        const f32x2 b0 = code_pair<FMT>(b, 0), b1 = code_pair<FMT>(b, 1);
        out[0] = Fp16::pack(a0[0], b0[0]);
        out[1] = Fp16::pack(a0[1], b0[1]);
        out[2] = Fp16::pack(a1[0], b1[0]);
        out[3] = Fp16::pack(a1[1], b1[1]);
    }
}

// Sequence length of batch item b: its own entry clamped to [0, n], or n.
__device__ __forceinline__ int c8_length(const int32_t* length, int b, int n) {
    return length ? min(max(length[b], 0), n) : n;
}

// max / sum over the four 16-lane rows of a wave (lanes l, l ^ 16, l ^ 32,
// l ^ 48): v_permlane16_swap exchanges odd rows of one copy with even rows of
// the other, so the pair holds both rows' values in either order.
__device__ __forceinline__ float rows4_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    return halfwave_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

__device__ __forceinline__ float rows4_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    return halfwave_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Bytes of an array of a call, for tests of overlap (host; none where `bytes` is 0).
struct Range {
    uintptr_t lo, hi;
    Range(const void* p, int64_t bytes)
        : lo(reinterpret_cast<uintptr_t>(p)), hi(reinterpret_cast<uintptr_t>(p) + (uintptr_t)bytes) {}
    bool meets(const Range& o) const { return lo < o.hi && o.lo < hi; }
};

// Validates a cache and its shapes (host).
int cache8_check(const nkv_cache8* c, const char* who);

}  // namespace nkv
