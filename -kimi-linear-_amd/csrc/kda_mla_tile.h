// Tiles of rows moved from memory to LDS for the expanded latent attention.
#pragma once

#include "kda_mla.h"

namespace kda {
namespace mla {

// ROWS rows of C channels (16 bits each) moved by NT threads, 16 bytes each, to
// LDS rows of PITCH elements.  The loads go through a buffer descriptor that
// ends with the last row there is: rows past it read as zeros, without a
// branch or a clamp, so that the loads of a tile stay in flight together.
template <typename T, int ROWS, int C, int NT, int PITCH>
struct Rows {
    static constexpr int kPieces = ROWS * C / 8;
    static constexpr int kPer = (kPieces + NT - 1) / NT;
    static_assert(kPieces % NT == 0 || kPieces < NT, "whole rounds, or less than one");
    uint32_t from[kPer];
    uint4 r[kPer];

    // Threads past a round that is less than whole move its first pieces once more.
    static __device__ __forceinline__ int piece(int i) { return (threadIdx.x + i * NT) % kPieces; }

    __device__ __forceinline__ void start(int64_t stride) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int c = piece(i);
            from[i] = static_cast<uint32_t>(c / (C / 8)) * static_cast<uint32_t>(stride * 2) + c % (C / 8) * 16;
        }
    }
    // Rows first.. of base, of which there are `rows` in all.
    __device__ __forceinline__ void fetch(const T* base, int64_t stride, int first, int rows) {
        const int n = min(rows - first, ROWS);
        const uint32_t bytes = n > 0 ? static_cast<uint32_t>(n - 1) * static_cast<uint32_t>(stride * 2) + 2 * C : 0u;
        const auto rsrc = make_rsrc_uniform(base + static_cast<int64_t>(first) * stride, bytes);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            r[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, static_cast<int>(from[i]), 0, 0));
    }
    __device__ __forceinline__ void put(T* lds) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int c = piece(i);
            *reinterpret_cast<uint4*>(lds + c / (C / 8) * PITCH + c % (C / 8) * 8) = r[i];
        }
    }
};
template <typename T, int ROWS, int NT, int PITCH>
struct Rows<T, ROWS, 0, NT, PITCH> {
    __device__ __forceinline__ void start(int64_t) {}
    __device__ __forceinline__ void fetch(const T*, int64_t, int, int) {}
    __device__ __forceinline__ void put(T*) const {}
};

// What rounding two values to the activation type leaves of them, rounded.
__device__ __forceinline__ uint32_t rest(float x, float y, _Float16) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 r = __builtin_bit_cast(h2, Act<_Float16>::pair(x, y));
    return Act<_Float16>::pair(x - static_cast<float>(r[0]), y - static_cast<float>(r[1]));
}
__device__ __forceinline__ uint32_t rest(float x, float y, bf16_t) {
    const uint32_t r = Act<bf16_t>::pair(x, y);
    return Act<bf16_t>::pair(x - __uint_as_float(r << 16), y - __uint_as_float(r & 0xffff0000u));
}
// Whether the expanded form's p and ds go into the products with what their rounding
// leaves: of few values one rounding may be most of an output's error, and there is
// time for it (bf16: two tokens dk 2.9e-3 off, 33 tokens 2.6e-3, by its own rounding 1.6e-3
// and 1.7e-3, which it comes down to).  Of many the roundings average out to 2.4e-3.
// By the tensors' sizes: the lengths are on the device, and other variants' registers are
// full.  (So are these: the backward's at 128 channels spill 10 to 36, in kernels of 10 to 13 us.)
inline bool few(const kda_mla_expanded_args& a) { return a.S <= 32 || (a.S <= 128 && a.B * a.H <= 64); }

// Loads issued before this stay before it: the compiler otherwise sinks a
// prefetch past the products it is to overlap, down to its first use.
__device__ __forceinline__ void issued() { asm volatile("" ::: "memory"); }

// A tile of keys and values: [KEYS][D + 8] keys, the head's channels and the
// position channels side by side, then [KEYS][V + VPAD] values.
template <typename T, int N, int P, int NT, int KEYS, int VPAD>
struct KvTile {
    static constexpr int D = N + P, V = N;
    static constexpr int kK = D + 8, kV = V + VPAD;               // LDS rows, elements
    static constexpr int kBuf = KEYS * (kK + kV);                 // elements of one buffer
    Rows<T, KEYS, N, NT, kK> k;
    Rows<T, KEYS, P, NT, kK> pe;
    Rows<T, KEYS, V, NT, kV> v;
    const T *kp, *pp, *vp;

    __device__ __forceinline__ KvTile(const kda_mla_expanded_args& a, int64_t b, int64_t h) {
        kp = static_cast<const T*>(a.k) + b * a.k_stride[0] + h * a.k_stride[2];
        pp = static_cast<const T*>(a.k_pe) + b * a.k_pe_stride[0];
        vp = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2];
        k.start(a.k_stride[1]);
        pe.start(a.k_pe_stride[1]);
        v.start(a.v_stride[1]);
    }
    __device__ __forceinline__ void fetch(const kda_mla_expanded_args& a, int j0, int keys) {
        k.fetch(kp, a.k_stride[1], j0, keys);
        pe.fetch(pp, a.k_pe_stride[1], j0, keys);
        v.fetch(vp, a.v_stride[1], j0, keys);
        issued();
    }
    __device__ __forceinline__ void put_keys(T* buf) const {
        k.put(buf);
        pe.put(buf + N);
    }
    __device__ __forceinline__ void put_values(T* buf) const { v.put(buf + KEYS * kK); }
    __device__ __forceinline__ void put(T* buf) const {
        put_keys(buf);
        put_values(buf);
    }
};

}  // namespace mla
}  // namespace kda
