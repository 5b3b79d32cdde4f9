// Rows written into a latent cache, and an 8-bit cache read back.
//
// A cache row is a token's latent (R channels) and its position channels (P).
// Both kernels touch each row once.  To write, a wave takes a row, a lane eight
// channels of the latent (R <= 512) and, the first P / 8 lanes, eight of the
// position part, so the norm's sum and the two largest magnitudes are wave
// reductions in registers.  To read back, a lane takes sixteen channels, and the
// lanes run on from one row into the next.  Bound by HBM for long calls and by the
// launch for a decode step's few rows: 64 rows of 576 in 8 bits 4 us, 6000 in 16
// bits 5.2 us (2.9 TB/s), reading 32768 back 11.6 us (4.9 TB/s).
#include <hip/hip_runtime.h>

#include "kda_launch.h"
#include "kda_mla.h"

namespace kda {
namespace {

constexpr int kRows = 4;          // rows (waves) a workgroup
constexpr float kE4m3Max = 448.f;
constexpr float kMinScale = 0x1p-60f;   // a row of zeros quantises to zeros, and 1 / scale stays finite

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    T e[8];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::ld(&e[i]);
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const f4 lo = *reinterpret_cast<const f4*>(p), hi = *reinterpret_cast<const f4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = lo[i], x[4 + i] = hi[i];
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    using A = mla::Act<T>;
    return uint4{A::pair(x[0], x[1]), A::pair(x[2], x[3]), A::pair(x[4], x[5]), A::pair(x[6], x[7])};
}

// The scale of a part whose eight channels of this lane are x (`has`: it has
// any), NaN where one of the part's values is not finite.
__device__ __forceinline__ float part_scale(const float (&x)[8], bool has) {
    float m = 0.f;
    bool bad = false;
    if (has) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m = fmaxf(m, fabsf(x[i]));
            bad |= !(fabsf(x[i]) < INFINITY);
        }
    }
    m = wave_max(m);
    return __any(bad) ? __builtin_nanf("") : fmaxf(m / kE4m3Max, kMinScale);
}

// x / scale to the nearest e4m3 value.  The quotient is the exactly rounded one
// (a product with 1 / scale alone would round some ties to the other side): from
// the rounded reciprocal r, q = x r, then q + (x - q scale) r, whose remainder an
// fma gives exactly (Markstein's theorem: r is 1 / scale correctly rounded, and q
// within a unit).  Three operations a value; the division's own sequence took 10.7
// us for 8192 rows of 576, three times their bytes.
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float scale) {
    const float r = 1.f / scale;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = x[i] * r;
        y[i] = __builtin_amdgcn_fmed3f(fmaf(fmaf(-q, scale, x[i]), r, q), -kE4m3Max, kE4m3Max);
    }
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    return uint2{static_cast<uint32_t>(lo), static_cast<uint32_t>(hi)};
}

template <typename T, bool F8>
__global__ __launch_bounds__(64 * kRows) void append_kernel(kda_mla_append_args a) {
    const int lane = threadIdx.x & 63;
    const uint32_t T_ = static_cast<uint32_t>(a.T), row = blockIdx.x * kRows + (threadIdx.x >> 6);
    if (row >= static_cast<uint32_t>(a.B) * T_) return;
    const int64_t b = row / T_, t = row - static_cast<uint32_t>(b) * T_;
    const int R = static_cast<int>(a.R), P = static_cast<int>(a.P);
    const bool lat = 8 * lane < R, pos = 8 * lane < P;
    const T* xr = static_cast<const T*>(a.x) + b * a.x_stride[0] + t * a.x_stride[1];
    float x[8], p[8], w[8];
    // everything is asked for before anything is waited for
    const int64_t held = a.lengths[b], count = a.counts ? a.counts[b] : a.T;
    if (lat) load8(xr + 8 * lane, x);
    if (pos) load8(xr + R + 8 * lane, p);
    if (lat && a.norm_weight) {
        if (a.norm_f32) load8(static_cast<const float*>(a.norm_weight) + 8 * lane, w);
        else load8(static_cast<const T*>(a.norm_weight) + 8 * lane, w);
    }
    const int64_t at = held + t;
    if (t >= count || held < 0 || at >= a.S) return;
    if (a.norm_weight) {
        float ss = 0.f;
        if (lat) {
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
        }
        const float rstd = __builtin_amdgcn_rsqf(wave_sum(ss) * (1.f / static_cast<float>(R)) + a.eps);   // R a power of two
        if (lat) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * rstd * w[i];
        }
    }
    if constexpr (F8) {
        uint8_t* out = static_cast<uint8_t*>(a.cache) + b * a.cache_stride[0] + at * a.cache_stride[1];
        const float s0 = part_scale(x, lat), s1 = P ? part_scale(p, pos) : 1.f;
        if (lat) *reinterpret_cast<uint2*>(out + 8 * lane) = quantise8(x, s0);
        if (pos) *reinterpret_cast<uint2*>(out + R + 8 * lane) = quantise8(p, s1);
        if (lane == 0)
            *reinterpret_cast<float2*>(a.cache_scale + b * a.scale_stride[0] + at * a.scale_stride[1]) = float2{s0, s1};
    } else {
        T* out = static_cast<T*>(a.cache) + b * a.cache_stride[0] + at * a.cache_stride[1];
        if (lat) *reinterpret_cast<uint4*>(out + 8 * lane) = pack8<T>(x);
        if (pos) *reinterpret_cast<uint4*>(out + R + 8 * lane) = pack8<T>(p);
    }
}

// 16 channels a lane: 16 bytes read, 32 written.
template <typename T>
__global__ __launch_bounds__(256) void read_kernel(kda_mla_read_args a) {
    const int per = static_cast<int>(a.R + a.P) / 16;       // lanes a row
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = i / per;
    if (row >= a.B * a.S) return;
    const int c = 16 * static_cast<int>(i - row * per);
    const int64_t b = row / a.S, j = row - b * a.S;
    uint4 out[2] = {};
    if (j < mla::tokens(a.lengths, b, a.S)) {
        const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.cache) +
                                                          b * a.cache_stride[0] + j * a.cache_stride[1] + c);
        const float s = a.cache_scale[b * a.scale_stride[0] + j * a.scale_stride[1] + (c < a.R ? 0 : 1)];
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        float x[2][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            typedef float f2 __attribute__((ext_vector_type(2)));
            const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[k], true);
            float* y = &x[k / 2][4 * (k % 2)];
            y[0] = lo[0] * s; y[1] = lo[1] * s; y[2] = hi[0] * s; y[3] = hi[1] * s;
        }
        out[0] = pack8<T>(x[0]);
        out[1] = pack8<T>(x[1]);
    }
    uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * (a.R + a.P) + c);
    to[0] = out[0];
    to[1] = out[1];
}

}  // namespace

int mla_append_launch(const kda_mla_append_args& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((a.B * a.T + kRows - 1) / kRows));
    const bool f8 = a.cache_dtype == KDA_DTYPE_E4M3;
    if (a.x_dtype == KDA_DTYPE_F16) {
        if (f8) append_kernel<_Float16, true><<<grid, 64 * kRows, 0, stream>>>(a);
        else append_kernel<_Float16, false><<<grid, 64 * kRows, 0, stream>>>(a);
    } else {
        if (f8) append_kernel<bf16_t, true><<<grid, 64 * kRows, 0, stream>>>(a);
        else append_kernel<bf16_t, false><<<grid, 64 * kRows, 0, stream>>>(a);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

int mla_read_launch(const kda_mla_read_args& a, hipStream_t stream) {
    const int64_t lanes = a.B * a.S * ((a.R + a.P) / 16);
    const dim3 grid(static_cast<unsigned>((lanes + 255) / 256));
    if (a.out_dtype == KDA_DTYPE_F16) read_kernel<_Float16><<<grid, 256, 0, stream>>>(a);
    else read_kernel<bf16_t><<<grid, 256, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

}  // namespace kda
