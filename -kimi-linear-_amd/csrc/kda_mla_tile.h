// The key and value tiles of the expanded latent attention's kernels.
#pragma once

#include "kda_mla.h"

namespace kda {
namespace mla {

constexpr int kTile = 64;             // keys a tile

// A tile of keys and values moved from memory to LDS by a workgroup of NT
// threads: [kTile][D + 8] keys, the head's channels and the position channels
// side by side, then [kTile][V + VPAD] values.
template <typename T, int N, int P, int NT, int VPAD>
struct KvTile {
    static constexpr int D = N + P, V = N;
    static constexpr int kK = D + 8, kV = V + VPAD;               // LDS rows, elements
    static constexpr int kBuf = kTile * (kK + kV);                // elements of one buffer
    static constexpr int kChunks = kTile * (D + V) / 8;           // 16-byte pieces of a tile
    static constexpr int kPer = (kChunks + NT - 1) / NT;

    // Piece c of a tile: first the head's keys, then the position parts, then the values.
    static __device__ __forceinline__ void fetch(const kda_mla_expanded_args& a, const T* k, const T* pe, const T* v,
                                                 int j0, int keys, uint4 (&r)[kPer]) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int c = threadIdx.x + i * NT;
            if (kChunks % NT != 0 && c >= kChunks) break;
            // rows past the last repeat it: their scores are masked
            if (c < kTile * N / 8) {
                const int row = min(c / (N / 8), keys - 1 - j0);
                r[i] = *reinterpret_cast<const uint4*>(k + (j0 + row) * a.k_stride[1] + c % (N / 8) * 8);
            } else if (P > 0 && c < kTile * D / 8) {
                const int d = c - kTile * N / 8, row = min(d / (P > 0 ? P / 8 : 1), keys - 1 - j0);
                r[i] = *reinterpret_cast<const uint4*>(pe + (j0 + row) * a.k_pe_stride[1] + d % (P > 0 ? P / 8 : 1) * 8);
            } else {
                const int d = c - kTile * D / 8, row = min(d / (V / 8), keys - 1 - j0);
                r[i] = *reinterpret_cast<const uint4*>(v + (j0 + row) * a.v_stride[1] + d % (V / 8) * 8);
            }
        }
    }
    static __device__ __forceinline__ void put(T* buf, const uint4 (&r)[kPer]) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int c = threadIdx.x + i * NT;
            if (kChunks % NT != 0 && c >= kChunks) break;
            int at;
            if (c < kTile * N / 8) {
                at = c / (N / 8) * kK + c % (N / 8) * 8;
            } else if (P > 0 && c < kTile * D / 8) {
                const int d = c - kTile * N / 8;
                at = d / (P > 0 ? P / 8 : 1) * kK + N + d % (P > 0 ? P / 8 : 1) * 8;
            } else {
                const int d = c - kTile * D / 8;
                at = kTile * kK + d / (V / 8) * kV + d % (V / 8) * 8;
            }
            *reinterpret_cast<uint4*>(buf + at) = r[i];
        }
    }
};

}  // namespace mla
}  // namespace kda
