// What the latent-attention kernels share: MFMA forms and packing for the two
// activation types, transposed LDS reads and the conversion of 8-bit values.
#pragma once

#include <hip/hip_runtime.h>

#include "kda_common.h"

namespace kda {
namespace mla {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float kLog2E = 1.4426950408889634f;
// A maximum that no score has been compared with yet: no score is below it, and it is
// finite, so that a row whose keys are all masked (scores of -inf) has
// exp2(-inf - max) = 0 terms and not a NaN.
constexpr float kNoMax = -0x1.fffffep127f;
// A fused s c - reference keeps what rounding took from the reference itself, up to
// 2^-24 of it; for references past this (the rest is 2^-8 here) the product is rounded
// first, as the reference was, so that the largest score's weight is 1 at any magnitude.
constexpr float kFar = 0x1p16f;
__device__ __forceinline__ bool far_from_zero(float reference) {
    return fabsf(reference) > kFar && fabsf(reference) < -kNoMax;
}

// A row's weights are formed as 2^(s' - reference), s' its scores times log2(e), and go into
// the value product in the activation type.  In bf16 the reference is the largest score.  In
// fp16, whose values end at 2^-14 (2^-24 with fewer and fewer bits), it is 2^15 below it: a
// weight keeps its 11 bits down to 2^-29 of the largest and something of itself down to 2^-39.
// Without that room a token that takes nearly all of a row's weight and has zeros in its
// values takes the others' share with it (18 nats above 4096 others: 95 % of the output lost).
// Beyond 2^20, where the difference of 15 is rounded, there is none.
template <typename T>
__device__ __forceinline__ float reference(float largest) {
    if constexpr (Elem<T>::code == KDA_DTYPE_F16) return fabsf(largest) < 0x1p20f ? largest - 15.f : largest;
    else return largest;
}

template <typename T> struct Act;
template <> struct Act<_Float16> {
    // 16x16 tile, depth 32: lane l has row/column l % 16 and the k slots 8 (l / 16) on;
    // the result's rows 4 (l / 16) + j of column l % 16.
    static __device__ __forceinline__ f4 mma16(uint4 a, uint4 b, f4 c) {
        return mfma16x16x32(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c);
    }
    // 32x32 tile, depth 16: lane l has row/column l % 32 and the k slots 8 (l / 32)
    // on; the result's rows 8 (j / 4) + 4 (l / 32) + j % 4 of column l % 32.
    static __device__ __forceinline__ f16v mma32(uint4 a, uint4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, h2));
    }
    // two e4m3 values of a word (its low or high half), exactly
    template <bool HI>
    static __device__ __forceinline__ uint32_t from8(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
    }
};
template <> struct Act<bf16_t> {
    static __device__ __forceinline__ f4 mma16(uint4 a, uint4 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0,
                                                       0);
    }
    static __device__ __forceinline__ f16v mma32(uint4 a, uint4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0,
                                                       0);
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) { return bf16_pair(lo, hi); }
    template <bool HI>
    static __device__ __forceinline__ uint32_t from8(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
    }
};

// Eight e4m3 values in the activation type.
template <typename T>
__device__ __forceinline__ uint4 widen8(uint32_t lo, uint32_t hi) {
    return uint4{Act<T>::template from8<false>(lo), Act<T>::template from8<true>(lo),
                 Act<T>::template from8<false>(hi), Act<T>::template from8<true>(hi)};
}

// Four 16-bit values of one column from a row-major LDS tile: within 16 lanes,
// lane i gets rows 0..3 of column i where lane 4 r + c points at row r,
// columns 4 c on.
__device__ __forceinline__ uint2 read_tr(const void* p) {
    typedef __attribute__((address_space(3))) s4* lds_s4;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (lds_s4)(reinterpret_cast<const s4*>(p))));
}

// Eight 8-bit values of one column: within 16 lanes, lane i gets rows 0..7 of
// column i where lane 2 r + c points at row r, columns 8 c on.
__device__ __forceinline__ uint2 read_tr8(const void* p) {
    typedef int i2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i2* lds_i2;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2)(reinterpret_cast<const i2*>(p))));
}

// Four neighbouring outputs, and where `low` is there what rounding took from each.
template <typename T>
__device__ __forceinline__ void store_out(T* out, T* low, f4 x) {
    const uint2 r{Act<T>::pair(x[0], x[1]), Act<T>::pair(x[2], x[3])};
    *reinterpret_cast<uint2*>(out) = r;
    if (low) {
        T e[4];
        __builtin_memcpy(e, &r, 8);
        *reinterpret_cast<uint2*>(low) = uint2{Act<T>::pair(x[0] - Elem<T>::ld(&e[0]), x[1] - Elem<T>::ld(&e[1])),
                                               Act<T>::pair(x[2] - Elem<T>::ld(&e[2]), x[3] - Elem<T>::ld(&e[3]))};
    }
}

// log2 of a row's sum of exp(s) from its reference and the sum against it, with what rounding takes
// from it (+inf for a row without keys).
__device__ __forceinline__ void store_lse(float* lse, float* low, int64_t row, float top, float sum) {
    const float rest = __builtin_amdgcn_logf(sum), x = sum == 0.f ? INFINITY : top + rest;
    lse[row] = x;
    if (low) low[row] = sum == 0.f ? 0.f : fabsf(top) > fabsf(rest) ? (top - x) + rest : (rest - x) + top;
}

// Largest x over the four lanes that share l & 15.
__device__ __forceinline__ float lanegroup4_max(float x) {
    {
        const unsigned u = __float_as_uint(x);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    {
        const unsigned u = __float_as_uint(x);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return x;
}
// The sum and the largest x over the two lanes that share l & 31.
__device__ __forceinline__ float half_sum(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float half_max(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Tokens of sequence b: lengths[b] clamped to [0, S], or S.
__device__ __forceinline__ int tokens(const int32_t* lengths, int64_t b, int64_t S) {
    const int n = lengths ? lengths[b] : static_cast<int>(S);
    return max(0, min(n, static_cast<int>(S)));
}

// Position of sequence b's first query: starts[b] clamped to [-T, S], beyond which no query sees a key, or S - T.
__device__ __forceinline__ int first_position(const int32_t* starts, int64_t b, int64_t S, int64_t T) {
    return starts ? max(-static_cast<int>(T), min(starts[b], static_cast<int>(S))) : static_cast<int>(S - T);
}

}  // namespace mla
}  // namespace kda
