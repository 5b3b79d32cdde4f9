// Matrices in 4 bits: y = x W^T, and rows to that form and back.
//
//   W_nk = v_nk 2^e_n,k/32,   v e2m1 (two a byte, the lower half first), e + 127 a byte.
//
// A lane's 16 bytes are one group of 32, so a group's power is one operand of the
// conversions that widen it (four a step of the matrix product, exact in bf16), and the four
// products that a piece feeds take x's channels in the order that the piece has them:
// lane group lg has channels 32 lg + 8 i of each 128 in step i.  W's 16 rows are the
// product's A operand, 16 rows of x the B operand, so a lane ends up with four neighbouring
// outputs of one row.
#include <hip/hip_runtime.h>

#include "kda_launch.h"
#include "kda_mla.h"

namespace kda {
namespace {

using mla::Act;

// A lane's share of 128 channels of one 16-row tile of W: its piece and the piece's power.
struct Piece {
    uint4 w;
    float power;
};
__device__ __forceinline__ Piece load_piece(const uint8_t* w, const uint8_t* scale, int64_t group) {
    return Piece{*reinterpret_cast<const uint4*>(w + 16 * group), __uint_as_float(static_cast<uint32_t>(scale[group]) << 23)};
}
template <typename T>
__device__ __forceinline__ uint4 widen(const Piece& p, int i) {
    return mla::widen4<T>(i == 0 ? p.w.x : i == 1 ? p.w.y : i == 2 ? p.w.z : p.w.w, p.power);
}

// Four neighbouring outputs n.. of one row: bias, rounding, residual.
template <typename T>
__device__ __forceinline__ void put(const kda_mx4_linear_args& a, int64_t row, int64_t n, f4 r) {
    if (row >= a.M || n >= a.N) return;
    T* y = static_cast<T*>(a.y) + row * a.N + n;
    const T* res = static_cast<const T*>(a.residual) + row * a.residual_stride + n;
    const T* bias = static_cast<const T*>(a.bias) + n;
    const int count = static_cast<int>(min(a.N - n, static_cast<int64_t>(4)));
    T out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j >= count) break;
        float v = r[j];
        if (a.bias) v += Elem<T>::ld(bias + j);
        if (a.residual) v = Elem<T>::ld(res + j) + round_elem<T>(v);
        Elem<T>::st(&out[j], v);
    }
    if (a.N % 4 == 0) {          // (y is 8-byte aligned)
        uint2 raw;
        __builtin_memcpy(&raw, out, 8);
        *reinterpret_cast<uint2*>(y) = raw;
    } else {
        for (int j = 0; j < count; ++j) y[j] = out[j];
    }
}

// ---- few rows of x ----------------------------------------------------------
// Grid ceil(N / (16 NT)), 64 SPLIT threads.  MT 16-row tiles of x, NT of W; the
// waves take the chunks of 128 channels in turn.
template <typename T, int MT, int NT, int SPLIT>
__global__ __launch_bounds__(64 * SPLIT) void few_kernel(kda_mx4_linear_args a) {
    constexpr int kDepth = MT == 1 ? 4 : (MT == 2 ? 2 : 1);       // chunks whose loads are in flight together
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, lg = lane >> 4;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT);
    const int groups = static_cast<int>(a.K / 32), chunks = (groups + 3) / 4;
    const uint8_t *w[NT], *scale[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = min(n0 + 16 * t + ln, a.N - 1) * groups;
        w[t] = static_cast<const uint8_t*>(a.w) + 16 * n;
        scale[t] = static_cast<const uint8_t*>(a.w_scale) + n;
    }
    const T* x[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
        x[m] = static_cast<const T*>(a.x) + min(static_cast<int64_t>(16 * m + ln), a.M - 1) * a.x_stride;
    f4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = f4{0.f, 0.f, 0.f, 0.f};
    for (int c0 = wave; c0 < chunks; c0 += SPLIT * kDepth) {
        Piece p[kDepth][NT];
        uint4 xr[kDepth][MT][4];
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            const int g = min(4 * (c0 + SPLIT * d) + lg, groups - 1);     // (past the last group it is read again)
#pragma unroll
            for (int t = 0; t < NT; ++t) p[d][t] = load_piece(w[t], scale[t], g);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) xr[d][m][i] = *reinterpret_cast<const uint4*>(x[m] + 32 * g + 8 * i);
        }
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            const int c = c0 + SPLIT * d;
            if (c >= chunks) break;
            if (4 * c + lg >= groups) {                                   // counts as zero, on both sides
#pragma unroll
                for (int t = 0; t < NT; ++t) p[d][t].w = uint4{0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) xr[d][m][i] = uint4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint4 wide = widen<T>(p[d][t], i);
#pragma unroll
                    for (int m = 0; m < MT; ++m) acc[t][m] = Act<T>::mma16(wide, xr[d][m][i], acc[t][m]);
                }
        }
    }
    constexpr int kTiles = NT * MT;
    __shared__ f4 part[SPLIT == 1 ? 1 : SPLIT * kTiles * 64];
    if constexpr (SPLIT > 1) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) part[(wave * kTiles + i) * 64 + lane] = acc[i / MT][i % MT];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
        if (SPLIT > 1 && i % SPLIT != wave) continue;
        f4 r = acc[i / MT][i % MT];
        if constexpr (SPLIT > 1) {
            r = part[i * 64 + lane];
#pragma unroll
            for (int v = 1; v < SPLIT; ++v) {
                const f4 p = part[(v * kTiles + i) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] += p[j];
            }
        }
        put<T>(a, 16 * (i % MT) + ln, n0 + 16 * (i / MT) + 4 * lg, r);
    }
}

// ---- many rows of x ---------------------------------------------------------
// 128 rows of x and 128 of W a workgroup, 64 and 64 a wave.  x goes to LDS 128 channels
// at a time, two buffers; its 16-byte piece c of row r lies at c turned by r, so that
// sixteen rows' pieces are in different banks.  W goes to registers as it is, the next
// chunk's under way, and is widened there.
constexpr int kTile = 128, kChunk = 128;

__device__ __forceinline__ uint32_t lds_address(void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)(p)));
}
__device__ __forceinline__ void to_lds(const void* base, int offset, char* lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds_address(lds)), "v"(offset), "s"(base)
                 : "memory");
}

template <typename T>
__global__ __launch_bounds__(256, 2) void many_kernel(kda_mx4_linear_args a) {
    __shared__ __align__(16) char buf[2][kTile * kChunk * 2];
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave & 1, wm = wave >> 1;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kTile, m0 = static_cast<int64_t>(blockIdx.y) * kTile;
    const int groups = static_cast<int>(a.K / 32), chunks = (groups + 3) / 4;
    const int last = static_cast<int>(min(a.M - 1 - m0, static_cast<int64_t>(kTile - 1)));
    const T* xb = static_cast<const T*>(a.x) + m0 * a.x_stride;
    const uint8_t *w[4], *scale[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int64_t n = min(n0 + 64 * wn + 16 * t + ln, a.N - 1) * groups;
        w[t] = static_cast<const uint8_t*>(a.w) + 16 * n;
        scale[t] = static_cast<const uint8_t*>(a.w_scale) + n;
    }
    const int pieces = 4 * groups;               // of 8 channels, in a row of x
    const auto load_x = [&](int c, char* to) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {            // four rows a load
            const int r = 32 * wave + 4 * i + lg;
            const int piece = min(16 * c + (ln ^ (r & 15)), pieces - 1);
            to_lds(xb, (min(r, last) * static_cast<int>(a.x_stride) + 8 * piece) * 2, to + (32 * wave + 4 * i) * (2 * kChunk));
        }
    };
    const auto load_w = [&](int c, Piece (&p)[4]) {
        const int g = min(4 * c + lg, groups - 1);
#pragma unroll
        for (int t = 0; t < 4; ++t) p[t] = load_piece(w[t], scale[t], g);
    };
    f4 acc[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[t][m] = f4{0.f, 0.f, 0.f, 0.f};
    Piece p[4], next[4];
    load_w(0, p);
    load_x(0, buf[0]);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int c = 0; c < chunks; ++c) {
        if (c + 1 < chunks) {
            load_w(c + 1, next);
            load_x(c + 1, buf[(c + 1) & 1]);
        }
        const char* from = buf[c & 1] + (64 * wm + ln) * (2 * kChunk);
        const bool past = 4 * c + lg >= groups;          // no channels of the lane's: zero, on both sides
        if (past) {
#pragma unroll
            for (int t = 0; t < 4; ++t) p[t].w = uint4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 x[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                x[m] = *reinterpret_cast<const uint4*>(from + 16 * m * (2 * kChunk) + 16 * ((4 * lg + i) ^ ln));
                if (past) x[m] = uint4{0, 0, 0, 0};
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint4 wide = widen<T>(p[t], i);
#pragma unroll
                for (int m = 0; m < 4; ++m) acc[t][m] = Act<T>::mma16(wide, x[m], acc[t][m]);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 4; ++t) p[t] = next[t];
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m)
            put<T>(a, m0 + 64 * wm + 16 * m + ln, n0 + 64 * wn + 16 * t + 4 * lg, acc[t][m]);
}

template <typename T, int MT, int NT>
void launch_few(const kda_mx4_linear_args& a, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>((a.N + 16 * NT - 1) / (16 * NT));
    const int64_t chunks = (a.K + 127) / 128;
    if (chunks >= 16) few_kernel<T, MT, NT, 8><<<grid, 512, 0, stream>>>(a);
    else if (chunks >= 4) few_kernel<T, MT, NT, 4><<<grid, 256, 0, stream>>>(a);
    else few_kernel<T, MT, NT, 1><<<grid, 64, 0, stream>>>(a);
}

template <typename T>
int launch_linear(const kda_mx4_linear_args& a, hipStream_t stream) {
    if (a.M > 64) {
        const dim3 grid(static_cast<unsigned>((a.N + kTile - 1) / kTile), static_cast<unsigned>((a.M + kTile - 1) / kTile));
        many_kernel<T><<<grid, 256, 0, stream>>>(a);
    } else if (a.M > 32) {
        launch_few<T, 4, 2>(a, stream);
    } else if (a.M > 16) {
        launch_few<T, 2, 2>(a, stream);
    } else if (a.N > 8192) {
        launch_few<T, 1, 2>(a, stream);
    } else {
        launch_few<T, 1, 1>(a, stream);
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
    return a.dtype == KDA_DTYPE_F16 ? launch_linear<_Float16>(a, stream) : launch_linear<bf16_t>(a, stream);
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
