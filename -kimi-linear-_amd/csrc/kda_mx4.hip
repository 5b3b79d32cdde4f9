// Matrices in 4 bits: y = x W^T, and rows to that form and back.
//
//   W_nk = v_nk 2^e_n,k/32,   v e2m1 (two a byte, the lower half first), e + 127 a byte.
//
// W's 16 rows are the matrix product's A operand, 16 rows of x the B operand, so a lane
// ends up with four neighbouring outputs of one row.  A lane's 16 bytes of W are one
// group of 32; the group's power is an operand of the conversions that widen it, so it costs
// nothing, and in bf16 the product is exact.
#include <hip/hip_runtime.h>

#include "kda_launch.h"
#include "kda_mla.h"

namespace kda {
namespace {

using mla::Act;
using mla::landed;
using mla::to_lds;

// b's lower half (16 lanes: even ones) in place of a's upper (odd) and the other way round.
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
}
__device__ __forceinline__ uint32_t word(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }

// landed<N>(), which the compiler takes into account: what came before those it does not wait for again.
template <int N>
__device__ __forceinline__ void known_landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0xf70);
    asm volatile("" ::: "memory");
}

// The scales of four chunks, a lane group a chunk's, handed around: e[j] of chunk j.
__device__ __forceinline__ void hand_around(uint32_t held, uint32_t (&e)[4]) {
    e[0] = e[2] = held;
    swap32(e[0], e[2]);
    e[1] = e[0];
    e[3] = e[2];
    swap16(e[0], e[1]);
    swap16(e[2], e[3]);
}

// What goes to four neighbouring outputs n.. of a row beside the product, asked for ahead of it.
template <typename T>
struct Beside {
    T bias[4], res[4];
    __device__ __forceinline__ void load(const kda_mx4_linear_args& a, int64_t row, int64_t n) {
        if (row >= a.M || n >= a.N) return;
        const int count = static_cast<int>(min(a.N - n, static_cast<int64_t>(4)));
        if (a.bias) four(static_cast<const T*>(a.bias) + n, count, bias);
        if (a.residual) four(static_cast<const T*>(a.residual) + row * a.residual_stride + n, count, res);
    }
    static __device__ __forceinline__ void four(const T* p, int count, T (&out)[4]) {
        if (count == 4 && reinterpret_cast<uintptr_t>(p) % 8 == 0) {
            const uint2 raw = *reinterpret_cast<const uint2*>(p);
            __builtin_memcpy(out, &raw, 8);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = p[min(j, count - 1)];
        }
    }
};
// Four outputs: bias, rounding, residual.
template <typename T>
__device__ __forceinline__ uint2 outputs(const kda_mx4_linear_args& a, f4 r, const Beside<T>& s) {
    T out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float v = r[j];
        if (a.bias) v += Elem<T>::ld(&s.bias[j]);
        if (a.residual) v = Elem<T>::ld(&s.res[j]) + round_elem<T>(v);
        Elem<T>::st(&out[j], v);
    }
    uint2 raw;
    __builtin_memcpy(&raw, out, 8);
    return raw;
}
// To their place, n.. of a row.
template <typename T>
__device__ __forceinline__ void put(const kda_mx4_linear_args& a, int64_t row, int64_t n, f4 r, const Beside<T>& s) {
    if (row >= a.M || n >= a.N) return;
    T* y = static_cast<T*>(a.y) + row * a.N + n;
    const uint2 raw = outputs<T>(a, r, s);
    if (a.N % 4 == 0) {          // (y is 8-byte aligned)
        *reinterpret_cast<uint2*>(y) = raw;
    } else {
        T out[4];
        __builtin_memcpy(out, &raw, 8);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < a.N) y[j] = out[j];
    }
}

// ---- few outputs ------------------------------------------------------------
// Grid (ceil(N / (16 NT)), ceil(M / (16 MT))), 64 SPLIT threads.  MT 16-row tiles of x, NT of
// W; the waves take chunks of 128 channels in turn, and their sums meet in LDS.
//
// Bound by the way to memory.  Five things carry it.  Four chunks' scales are one load, a lane
// group a chunk's, handed around in registers: a load for each chunk took as long as W's own (one
// row by 28672 x 8192 41 us, without any scales 29).  x goes through LDS, a buffer a wave, where
// a row's 256 bytes come as one piece; read as operands they come as 64 from each of
// sixteen rows (53 rows by 6160 x 4096 18.9 us, this way 12.3).  W and the scales come
// through descriptors that end with the workgroup's rows, so that what does not exist is an
// offset past the end, which reads as zero without a branch and asks memory for nothing.  A chunk's
// loads are under way while the one before is used, W's a chunk earlier still (the one row 35.2 ->
// 34.2 us).  And neighbouring waves have neighbouring chunks, which share W's lines of 128 bytes
// and make 2 KB pieces of x's rows (with two or four chunks on end a wave 34.2, in turn 31.3; the 53 rows 11.7).
//
// x's 16-byte piece c of row r lies at c turned by r, so that sixteen rows' pieces are in
// different banks.  A lane has the same group of x and W, channels 32 lg + 8 i of a chunk in step
// i.  Rows of x past the last leave what LDS holds, in columns of the product that go nowhere.
template <typename T, int MT, int NT, int SPLIT, bool WORDS>
__global__ __launch_bounds__(64 * SPLIT) void rows_kernel(kda_mx4_linear_args a) {
    constexpr int kTiles = NT * MT, kOwn = (kTiles + SPLIT - 1) / SPLIT, kNone = 0x7f000000;
    constexpr int kLoads = 4 * MT;                           // of a chunk of x, four rows each
    __shared__ __align__(16) char buf[SPLIT][1024 * (kLoads > kTiles ? kLoads : kTiles)];
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT), m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
    const int groups = static_cast<int>(a.K / 32), chunks = (groups + 3) / 4;
    const uint32_t rows = static_cast<uint32_t>(min(a.N - n0, static_cast<int64_t>(16 * NT)));
    const auto w = make_rsrc(static_cast<const uint8_t*>(a.w) + n0 * groups * 16, rows * groups * 16);
    const auto scale = make_rsrc(static_cast<const uint8_t*>(a.w_scale) + n0 * groups, rows * groups);
    int w_at[NT], e_at[NT], x_at[kLoads];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        e_at[t] = (16 * t + ln) * groups;
        w_at[t] = 16 * (e_at[t] + lg);
    }
    const int last = static_cast<int>(min(a.M - 1 - m0, static_cast<int64_t>(16 * MT - 1)));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = 4 * i + lg;
        x_at[i] = min(r, last) * static_cast<int>(a.x_stride) * 2 + 16 * (ln ^ (r & 15));
    }
    const T* xb = static_cast<const T*>(a.x) + m0 * a.x_stride;
    char* mine = buf[wave];
    const auto load_x = [&](int c) {
        if (4 * c + 4 <= groups) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (4 * i <= last) to_lds(xb + 128 * c, x_at[i], mine + 1024 * i);
        } else {                                             // pieces past the last are read as it
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                if (4 * i > last) continue;
                const int piece = ln ^ ((4 * i + lg) & 15);
                to_lds(xb + 128 * c, x_at[i] - 16 * max(piece - (4 * (groups - 4 * c) - 1), 0), mine + 1024 * i);
            }
        }
    };
    const auto load_w = [&](int c, uint4 (&p)[NT]) {
        const bool there = 4 * c + lg < groups;
#pragma unroll
        for (int t = 0; t < NT; ++t)
            p[t] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(w, there ? w_at[t] + 64 * c : kNone, 0, 0));
    };
    const auto load_scales = [&](int c, uint32_t (&e)[NT]) {
        const int g = 4 * (c + SPLIT * lg);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (WORDS) {
                e[t] = __builtin_amdgcn_raw_buffer_load_b32(scale, g < groups ? e_at[t] + g : kNone, 0, 0);
            } else {
                e[t] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    e[t] |= static_cast<uint32_t>(
                        __builtin_amdgcn_raw_buffer_load_b8(scale, g + i < groups ? e_at[t] + g + i : kNone, 0, 0)) << (8 * i);
            }
        }
    };
    f4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = f4{0.f, 0.f, 0.f, 0.f};
    // tile i's outputs of this lane, i one of the wave's in the end
    const auto row = [&](int i) { return m0 + 16 * (i % MT) + ln; };
    const auto col = [&](int i) { return n0 + 16 * (i / MT) + 4 * lg; };
    Beside<T> beside[kOwn];
#pragma unroll
    for (int o = 0; o < kOwn; ++o)
        if (wave + o * SPLIT < kTiles) beside[o].load(a, row(wave + o * SPLIT), col(wave + o * SPLIT));

    // Under way at the top of a chunk: its W and x, then the next chunk's W.  As soon as x is in registers its
    // buffer takes the next chunk's, as soon as W's words are used their registers take the chunk's after that.
    uint32_t next[NT];
    uint4 p[2][NT];
    load_scales(wave, next);
    load_w(wave, p[0]);
    if (wave < chunks) load_x(wave);
    load_w(wave + SPLIT, p[1]);
    for (int c0 = wave; c0 < chunks; c0 += 4 * SPLIT) {
        uint32_t e[NT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + j * SPLIT;
            if (c >= chunks) break;
            uint4 x[4][MT];
            known_landed<NT>();
            if (j == 0) {
#pragma unroll
                for (int t = 0; t < NT; ++t) hand_around(next[t], e[t]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    x[i][m] = *reinterpret_cast<const uint4*>(mine + 4096 * m + 256 * ln + 16 * ((4 * lg + i) ^ ln));
            if (4 * c + 4 > groups && 4 * c + lg >= groups) {    // (W's are zero already)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int m = 0; m < MT; ++m) x[i][m] = uint4{0, 0, 0, 0};
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the chunk has been read: the next may lie there
            const int after = c + SPLIT;
            if (j == 0) load_scales(c0 + 4 * SPLIT, next);
            if (after < chunks) load_x(after);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float pw = __uint_as_float((e[t][j] >> (8 * lg) & 255u) << 23);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 wide = mla::widen4<T>(word(p[j % 2][t], i), pw);
#pragma unroll
                    for (int m = 0; m < MT; ++m) acc[t][m] = Act<T>::mma16(wide, x[i][m], acc[t][m]);
                }
            }
            load_w(c + 2 * SPLIT, p[j % 2]);
        }
    }
    landed<0>();                                                 // (the scales asked for last)
    f4* part = reinterpret_cast<f4*>(buf);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTiles; ++i) part[(wave * kTiles + i) * 64 + lane] = acc[i / MT][i % MT];
    __syncthreads();
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
        const int i = wave + o * SPLIT;
        if (i >= kTiles) break;
        f4 r = part[i * 64 + lane];
#pragma unroll
        for (int v = 1; v < SPLIT; ++v) {
            const f4 q = part[(v * kTiles + i) * 64 + lane];
#pragma unroll
            for (int k = 0; k < 4; ++k) r[k] += q[k];
        }
        put<T>(a, row(i), col(i), r, beside[o]);
    }
}

// ---- many outputs -----------------------------------------------------------
// 64 WM rows of x and 16 NT WN of W a workgroup, 64 and 16 NT a wave.  Both go to LDS 128
// channels at a time, asynchronously, STAGES buffers.  x's 16-byte piece c of row r lies at c
// turned by r, W's by bits of r, so that sixteen rows' pieces are in different banks; W is widened
// after it is read.  A lane has the same group of x and W, channels 32 lg + 8 i of a chunk in step i.
//
// Bound by the matrix cores and what stands beside them: at 8192^3 (1.22 PFLOP/s) 711 us
// without the loads, 643 without the barriers too, 631 without the conversions and LDS reads
// as well; over 2048 channels a tile's way in and out is about a fifth of it.  So the W rows of
// a wave's tiles are dealt in fours, which gives a lane 8 NT bytes of a row of outputs on end
// (4000 rows by 6144 x 2048 107 -> 101 us).
constexpr int kChunk = 128;

template <typename T, int WM, int WN, int NT, int STAGES, bool WORDS>
struct Tile {
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves, kM = 64 * WM, kN = 16 * NT * WN;
    static constexpr int kX = kM * 2 * kChunk, kW = kN * kChunk / 2;             // bytes of a stage
    static constexpr int kBytes = STAGES * (kX + kW), kAcross = WN;
    static constexpr int kXLoads = kX / 1024 / kWaves, kWLoads = kW / 1024 / kWaves;
    static_assert(kXLoads * kWaves * 1024 == kX && kWLoads * kWaves * 1024 == kW, "whole loads, as many each wave");
    // Row r of tile t is W's 4 NT (r / 4) + 4 t + r % 4 of the wave's, so that a lane's outputs of one row of x, four a
    // tile, lie on end.
    static __device__ __forceinline__ int w_row(int t, int r) { return 4 * NT * (r >> 2) + 4 * t + (r & 3); }
    // What W's row r turns its pieces by: the sixteen rows of a read are in different banks.
    static __device__ __forceinline__ int turn(int r) { return r / (4 * NT) & 3; }
};

// A tile's outputs where rows of y begin at no multiple of 8 bytes: gathered in LDS, and written from there a row's pairs on
// end.  (3483 rows by 7693 x 224 in the largest tile 56 us, with a store for each of a lane's values 98; a width of 7696
// 38.  In the one that it gets 45 and 32.)
template <typename T, typename K, int NT>
__device__ __forceinline__ void through_lds(const kda_mx4_linear_args& a, const f4 (&acc)[NT][4], T* tile, int64_t m0, int64_t n0,
                                            int rows, int cols) {
    constexpr int kStride = K::kN + 4, kPairs = K::kN / 2 + 1;
    static_assert(K::kM * kStride * 2 <= K::kBytes, "the tile fits where its operands were");
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4, wave = threadIdx.x >> 6;
    const int row = 64 * (wave / K::kAcross) + ln, col = 16 * NT * (wave % K::kAcross) + 4 * NT * lg;
    __syncthreads();                                     // all waves have read their last operands
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        T bias[4] = {};
        if (a.bias && col + 4 * t < cols) Beside<T>::four(static_cast<const T*>(a.bias) + n0 + col + 4 * t, min(cols - col - 4 * t, 4), bias);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            T out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) Elem<T>::st(&out[j], a.bias ? acc[t][m][j] + Elem<T>::ld(&bias[j]) : acc[t][m][j]);
            __builtin_memcpy(tile + (row + 16 * m) * kStride + col + 4 * t, out, 8);
        }
    }
    __syncthreads();
    constexpr int kAtOnce = 8;                           // read before any is written
    T* y = static_cast<T*>(a.y) + m0 * a.N + n0;
    const T* res = static_cast<const T*>(a.residual) + (a.residual ? m0 * a.residual_stride + n0 : 0);
    const uint32_t odd = a.N & 1, base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(y) >> 1 & 1);
    for (int i0 = threadIdx.x; i0 < rows * kPairs; i0 += kAtOnce * K::kThreads) {
        T out[kAtOnce][2];
        int row_of[kAtOnce], col_of[kAtOnce];            // c: a multiple of 4 bytes in y, from -1 on
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int i = i0 + u * K::kThreads, r = i / kPairs, c = 2 * (i - r * kPairs) - static_cast<int>((base + r * odd) & 1);
            row_of[u] = min(r, K::kM - 1);
            col_of[u] = r < rows ? c : cols;
            const T* from = tile + row_of[u] * kStride;
            out[u][0] = from[max(c, 0)];
            out[u][1] = from[c + 1];
        }
        if (a.residual) {
            T held[kAtOnce][2];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const T* from = res + row_of[u] * a.residual_stride;
                if (col_of[u] >= 0 && col_of[u] < cols) held[u][0] = from[col_of[u]];
                if (col_of[u] + 1 < cols) held[u][1] = from[col_of[u] + 1];
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                for (int j = 0; j < 2; ++j) Elem<T>::st(&out[u][j], Elem<T>::ld(&held[u][j]) + Elem<T>::ld(&out[u][j]));
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            T* to = y + row_of[u] * a.N;
            const int c = col_of[u];
            if (c >= 0 && c + 1 < cols) {
                uint32_t raw;
                __builtin_memcpy(&raw, out[u], 4);
                *reinterpret_cast<uint32_t*>(to + c) = raw;
            } else if (c >= 0 && c < cols) {
                to[c] = out[u][0];
            } else if (c + 1 < cols) {
                to[c + 1] = out[u][1];
            }
        }
    }
}

template <typename T, int WM, int WN, int NT, int STAGES, bool WORDS>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(kda_mx4_linear_args a) {
    using K = Tile<T, WM, WN, NT, STAGES, WORDS>;
    __shared__ __align__(16) char buf[STAGES][K::kX + K::kW];
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * K::kN, m0 = static_cast<int64_t>(blockIdx.y) * K::kM;
    const int groups = static_cast<int>(a.K / 32), chunks = (groups + 3) / 4;
    const int last_m = static_cast<int>(min(a.M - 1 - m0, static_cast<int64_t>(K::kM - 1)));
    const int last_n = static_cast<int>(min(a.N - 1 - n0, static_cast<int64_t>(K::kN - 1)));
    const T* xb = static_cast<const T*>(a.x) + m0 * a.x_stride;
    const uint8_t* wb = static_cast<const uint8_t*>(a.w) + n0 * groups * 16;
    const uint8_t* scale[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
        scale[t] = static_cast<const uint8_t*>(a.w_scale) + min(n0 + 16 * NT * wn + K::w_row(t, ln), a.N - 1) * groups;
    // a lane's rows of a stage, and its piece of each: constant from chunk to chunk
    int x_at[K::kXLoads], w_at[K::kWLoads];
#pragma unroll
    for (int i = 0; i < K::kXLoads; ++i) {               // four rows a load
        const int r = 4 * (K::kXLoads * wave + i) + lg;
        x_at[i] = min(r, last_m) * static_cast<int>(a.x_stride) * 2 + 16 * (ln ^ (r & 15));
    }
#pragma unroll
    for (int i = 0; i < K::kWLoads; ++i) {               // sixteen
        const int r = 16 * (K::kWLoads * wave + i) + (lane >> 2);
        w_at[i] = 16 * (min(r, last_n) * groups + ((lane & 3) ^ K::turn(r)));
    }
    const auto load = [&](int c, char* stage) {
        char* xs = stage + 1024 * K::kXLoads * wave;
        char* ws = stage + K::kX + 1024 * K::kWLoads * wave;
        if (4 * c + 4 <= groups) {
#pragma unroll
            for (int i = 0; i < K::kXLoads; ++i) to_lds(xb + kChunk * static_cast<int64_t>(c), x_at[i], xs + 1024 * i);
#pragma unroll
            for (int i = 0; i < K::kWLoads; ++i) to_lds(wb + 64 * static_cast<int64_t>(c), w_at[i], ws + 1024 * i);
        } else {                                         // pieces past the last are read as it
            const int held = groups - 4 * c;
#pragma unroll
            for (int i = 0; i < K::kXLoads; ++i) {
                const int piece = ln ^ ((4 * (K::kXLoads * wave + i) + lg) & 15);
                to_lds(xb + kChunk * static_cast<int64_t>(c), x_at[i] - 16 * max(piece - (4 * held - 1), 0), xs + 1024 * i);
            }
#pragma unroll
            for (int i = 0; i < K::kWLoads; ++i) {
                const int piece = (lane & 3) ^ K::turn(16 * (K::kWLoads * wave + i) + (lane >> 2));
                to_lds(wb + 64 * static_cast<int64_t>(c), w_at[i] - 16 * max(piece - (held - 1), 0), ws + 1024 * i);
            }
        }
    };
    // the scales of four chunks from c on: a lane group a chunk's
    const auto load_scales = [&](int c, uint32_t (&e)[NT]) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (WORDS) {
                e[t] = *reinterpret_cast<const uint32_t*>(scale[t] + min(4 * (c + lg), groups - 4));
            } else {
                e[t] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) e[t] |= static_cast<uint32_t>(scale[t][min(4 * (c + lg) + i, groups - 1)]) << (8 * i);
            }
        }
    };
    f4 acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[t][m] = f4{0.f, 0.f, 0.f, 0.f};
    uint32_t next[NT];
    load_scales(0, next);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) load(min(i, chunks - 1), buf[i]);
    int at = 0;                                          // the stage of chunk c
    for (int c0 = 0; c0 < chunks; c0 += 4) {
        uint32_t e[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) hand_around(next[t], e[t]);
        load_scales(min(c0 + 4, chunks - 1), next);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + j;
            if (c >= chunks) break;
            // chunk c is there, in every wave; the stage of chunk c - 1 is free
            landed<(STAGES - 2) * (K::kXLoads + K::kWLoads)>();
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            load(min(c + STAGES - 1, chunks - 1), buf[at == 0 ? STAGES - 1 : at - 1]);
            const char* xs = buf[at] + (64 * wm + ln) * (2 * kChunk);
            const char* ws = buf[at] + K::kX + (16 * NT * wn + K::w_row(0, ln)) * (kChunk / 2) + 16 * (lg ^ (ln >> 2));
            uint4 p[NT], x[4][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) p[t] = *reinterpret_cast<const uint4*>(ws + 4 * t * (kChunk / 2));
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    x[i][m] = *reinterpret_cast<const uint4*>(xs + 16 * m * (2 * kChunk) + 16 * ((4 * lg + i) ^ ln));
            asm volatile("" ::: "memory");              // all asked for before the first product
            float power[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) power[t] = __uint_as_float((e[t][j] >> (8 * lg) & 255u) << 23);
            if (4 * c + 4 > groups && 4 * c + lg >= groups) {       // no channels of the lane's: zero, on both sides
#pragma unroll
                for (int t = 0; t < NT; ++t) p[t] = uint4{0, 0, 0, 0}, power[t] = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int m = 0; m < 4; ++m) x[i][m] = uint4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint4 wide = mla::widen4<T>(word(p[t], i), power[t]);
#pragma unroll
                    for (int m = 0; m < 4; ++m) acc[t][m] = Act<T>::mma16(wide, x[i][m], acc[t][m]);
                }
            at = at + 1 == STAGES ? 0 : at + 1;
        }
    }
    landed<0>();                                         // no load is under way when the workgroup's LDS goes to another
    if (a.N % 4 != 0) {
        through_lds<T, K>(a, acc, reinterpret_cast<T*>(buf), m0, n0, last_m + 1, last_n + 1);
        return;
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const int64_t row = m0 + 64 * wm + 16 * m + ln, n = n0 + 16 * NT * wn + 4 * NT * lg;
        Beside<T> beside[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) beside[t].load(a, row, n + 4 * t);
        if (NT % 2 == 0 && a.N % 8 == 0 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0) {
            if (row >= a.M) continue;
#pragma unroll
            for (int t = 0; t + 1 < NT; t += 2) {
                if (n + 4 * t >= a.N) break;
                const uint2 lo = outputs<T>(a, acc[t][m], beside[t]), hi = outputs<T>(a, acc[t + 1][m], beside[t + 1]);
                *reinterpret_cast<uint4*>(static_cast<T*>(a.y) + row * a.N + n + 4 * t) = uint4{lo.x, lo.y, hi.x, hi.y};
            }
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t) put<T>(a, row, n + 4 * t, acc[t][m], beside[t]);
        }
    }
}

template <typename T, int MT, int NT, int SPLIT>
void launch_rows(const kda_mx4_linear_args& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((a.N + 16 * NT - 1) / (16 * NT)), static_cast<unsigned>((a.M + 16 * MT - 1) / (16 * MT)));
    if (a.K % 128 == 0 && reinterpret_cast<uintptr_t>(a.w_scale) % 4 == 0)
        rows_kernel<T, MT, NT, SPLIT, true><<<grid, 64 * SPLIT, 0, stream>>>(a);
    else
        rows_kernel<T, MT, NT, SPLIT, false><<<grid, 64 * SPLIT, 0, stream>>>(a);
}

template <typename T, int WM, int WN, int NT, int STAGES>
void launch_tile(const kda_mx4_linear_args& a, hipStream_t stream) {
    using K = Tile<T, WM, WN, NT, STAGES, true>;
    const dim3 grid(static_cast<unsigned>((a.N + K::kN - 1) / K::kN), static_cast<unsigned>((a.M + K::kM - 1) / K::kM));
    if (a.K % 128 == 0 && reinterpret_cast<uintptr_t>(a.w_scale) % 4 == 0)
        tile_kernel<T, WM, WN, NT, STAGES, true><<<grid, K::kThreads, 0, stream>>>(a);
    else
        tile_kernel<T, WM, WN, NT, STAGES, false><<<grid, K::kThreads, 0, stream>>>(a);
}

// The smallest tiles of outputs that are at most a workgroup a CU, since a workgroup's way to its
// first product is most of a small call, and larger ones of larger calls, whose operands come
// less often.  us in a graph of 24 over weights that rotate through 600 MB, fp16 (M, N, K):
//   M x N of a tile     16x16  16x32  16x64
//   1, 2048, 2048         3.6    4.3    5.8
//   1, 8192, 8192        11.1   11.1   16.0
//   16, 6144, 2048        5.4    4.8    6.2
//   16, 28672, 8192      49.5   42.2   37.4      (one row 32.9, 31.4, 30.9)
// Up to four rows of x are one load a chunk, so small tiles cost little: the smallest as long as all workgroups are
// under way at once (three a CU), then up to two a CU.
//   1, 11008, 4096        8.2    9.2   10.1      (four rows 8.5, 9.8, 10.2, eight 10.3, 10.7, 10.6)
//   1, 12288, 2048        6.1    6.6    6.8
//   1, 14336, 4096       10.8    9.4   10.2
//   4, 14336, 2048        7.5    6.9    7.0
//   4, 32768, 4096       21.1   19.5   17.6
//                       32x32  32x64  64x32  64x64  64x128  128x128
//   32, 2048, 2048        5.5    7.2    6.0    8.6
//   32, 28672, 8192      54.0   43.6   64.3   53.6    55.5
//   53, 6160, 4096       13.8   12.8   11.8   16.3    28.3
//   64, 28672, 8192      78.9   73.7   74.3   56.7    57.4
//   128, 6144, 2048      12.0   11.7   13.2   10.3    16.3     27.7
//   128, 16384, 4096     48.4   38.7   43.7   35.3    29.3     51.9
// 64x128 with eight waves of 64x16, and with four of 64x32, and 128x128 with four of 64x64 (fp16):
//   300, 6144, 2048      17.7   18.7   28.4
//   1250, 6144, 2048            43.3   39.2
//   1400, 6144, 2048            46.0   55.7
//   2000, 6144, 2048            59.8   60.8
//   2560, 6144, 2048            72.3   68.1
//   2700, 6144, 2048            78.0   81.6
//   4000, 6144, 2048     132   106.5   99.5     (the library's product of 16-bit operands 98)
//   4200, 6144, 2048           111.5  112.3
//   5000, 4096, 4096           167.6  159.4
//   1000, 8192, 8192           148.4  127.8
//   8192, 8192, 8192    1238    1021    949     (771)
//   12000, 7696, 1024          236.0  231.1
//   12000, 7696, 448           147.6  153.0
//   7000, 7696, 224             61.7   67.7
// The largest, two a CU, are faster where their rounds of 512 are full to 5/6 or more (480 and 512 tiles, 960, 1280, 1536; not
// 528, 768, 1056 and 1584) and a tile is deep enough for its way in and out; bf16 is within 5 %.
constexpr int64_t kDeep = 1024;
template <typename T>
int launch_linear(const kda_mx4_linear_args& a, hipStream_t stream) {
    const auto tiles = [&](int64_t m, int64_t n) { return ((a.M + m - 1) / m) * ((a.N + n - 1) / n); };
    constexpr int64_t kCus = 256;
    if (a.M <= 16) {
        const bool few = a.M <= 4;
        if (tiles(16, 16) <= kCus) launch_rows<T, 1, 1, 8>(a, stream);
        else if (tiles(16, 32) <= kCus) launch_rows<T, 1, 2, 8>(a, stream);
        else if (few && tiles(16, 16) <= 3 * kCus) launch_rows<T, 1, 1, 8>(a, stream);
        else if (few && tiles(16, 32) <= 2 * kCus) launch_rows<T, 1, 2, 8>(a, stream);
        else launch_rows<T, 1, 4, 4>(a, stream);
    } else if (tiles(32, 32) <= kCus) {
        launch_rows<T, 2, 2, 8>(a, stream);
    } else if (a.M <= 32) {
        launch_rows<T, 2, 4, 4>(a, stream);
    } else if (tiles(64, 32) <= kCus) {
        launch_rows<T, 4, 2, 8>(a, stream);
    } else if (tiles(64, 64) <= kCus) {
        launch_rows<T, 4, 4, 8>(a, stream);
    } else if (tiles(64, 128) <= kCus) {
        launch_tile<T, 1, 8, 1, 3>(a, stream);
    } else {
        const int64_t large = tiles(128, 128), round = 2 * kCus, rounds = (large + round - 1) / round;
        if (a.K >= kDeep && 6 * large >= 5 * round * rounds) launch_tile<T, 2, 2, 4, 2>(a, stream);
        else launch_tile<T, 1, 4, 2, 2>(a, stream);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

// ---- conversions ------------------------------------------------------------
// Bound by HBM: each value is read once and written once.  A lane takes eight
// values, four lanes a group.
constexpr uint32_t kLeast = 1;                   // 2^-126

__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
    x = max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0xb1, 0xf, 0xf, false)));   // quad_perm 1 0 3 2
    return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x4e, 0xf, 0xf, false)));   // 2 3 0 1
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    constexpr int kWords = sizeof(T) / 2;
    uint4 raw[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    T e[8];
    __builtin_memcpy(e, raw, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::ld(&e[i]);
}

// Where eight values lie: rows one stride apart.
__device__ __forceinline__ int64_t value_at(const kda_mx4_convert_args& a, uint32_t i) {
    const uint32_t per = static_cast<uint32_t>(a.K / 8), row = i / per;
    return row * a.value_stride + 8 * static_cast<int64_t>(i - row * per);
}

template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(kda_mx4_convert_args a, uint32_t units) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= units) return;                      // (whole groups: units are a multiple of 4)
    float x[8];
    load8(static_cast<const T*>(a.values) + value_at(a, i), x);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    const uint32_t e = mla::group_exponent(quad_max(top), kLeast);
    static_cast<uint32_t*>(a.data)[i] = mla::narrow4(x, e);
    if (i % 4 == 0) static_cast<uint8_t*>(a.scale)[i / 4] = static_cast<uint8_t>(e);
}

template <typename T>
__global__ __launch_bounds__(256) void dequantize_kernel(kda_mx4_convert_args a, uint32_t units) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= units) return;
    const uint32_t raw = static_cast<const uint32_t*>(a.data)[i], e = static_cast<const uint8_t*>(a.scale)[i / 4];
    *reinterpret_cast<uint4*>(static_cast<T*>(a.values) + value_at(a, i)) = mla::widen4<T>(raw, __uint_as_float(e << 23));
}

}  // namespace

int mx4_linear_launch(const kda_mx4_linear_args& a, hipStream_t stream) {
    // rows in pieces that a grid's second dimension (65535) reaches with the smallest tiles of many rows
    constexpr int64_t kMost = int64_t{65535} * 64;
    for (int64_t m = 0; m < a.M; m += kMost) {
        kda_mx4_linear_args p = a;
        p.M = min(a.M - m, kMost);
        p.x = static_cast<const char*>(a.x) + 2 * m * a.x_stride;
        p.y = static_cast<char*>(a.y) + 2 * m * a.N;
        if (a.residual) p.residual = static_cast<const char*>(a.residual) + 2 * m * a.residual_stride;
        const int status = a.dtype == KDA_DTYPE_F16 ? launch_linear<_Float16>(p, stream) : launch_linear<bf16_t>(p, stream);
        if (status != KDA_OK) return status;
    }
    return KDA_OK;
}

int mx4_quantize_launch(const kda_mx4_convert_args& a, hipStream_t stream) {
    const uint32_t units = static_cast<uint32_t>(a.N * a.K / 8);
    const dim3 grid(units / 256 + (units % 256 != 0));
    if (a.dtype == KDA_DTYPE_F32) quantize_kernel<float><<<grid, 256, 0, stream>>>(a, units);
    else if (a.dtype == KDA_DTYPE_F16) quantize_kernel<_Float16><<<grid, 256, 0, stream>>>(a, units);
    else quantize_kernel<bf16_t><<<grid, 256, 0, stream>>>(a, units);
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

int mx4_dequantize_launch(const kda_mx4_convert_args& a, hipStream_t stream) {
    const uint32_t units = static_cast<uint32_t>(a.N * a.K / 8);
    const dim3 grid(units / 256 + (units % 256 != 0));
    if (a.dtype == KDA_DTYPE_F16) dequantize_kernel<_Float16><<<grid, 256, 0, stream>>>(a, units);
    else dequantize_kernel<bf16_t><<<grid, 256, 0, stream>>>(a, units);
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

}  // namespace kda
