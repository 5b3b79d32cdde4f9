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

// Dword i of lane group lg to dword lg of lane group i.
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
}
__device__ __forceinline__ uint4 turned(uint4 w) {
    swap32(w.x, w.z);
    swap32(w.y, w.w);
    swap16(w.x, w.y);
    swap16(w.z, w.w);
    return w;
}
__device__ __forceinline__ uint32_t word(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
__device__ __forceinline__ float power(uint32_t bytes, int i) { return __uint_as_float((bytes >> (8 * i) & 255u) << 23); }

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
// The outputs: bias, rounding, residual.
template <typename T>
__device__ __forceinline__ void put(const kda_mx4_linear_args& a, int64_t row, int64_t n, f4 r, const Beside<T>& s) {
    if (row >= a.M || n >= a.N) return;
    T* y = static_cast<T*>(a.y) + row * a.N + n;
    T out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float v = r[j];
        if (a.bias) v += Elem<T>::ld(&s.bias[j]);
        if (a.residual) v = Elem<T>::ld(&s.res[j]) + round_elem<T>(v);
        Elem<T>::st(&out[j], v);
    }
    if (a.N % 4 == 0) {          // (y is 8-byte aligned)
        uint2 raw;
        __builtin_memcpy(&raw, out, 8);
        *reinterpret_cast<uint2*>(y) = raw;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < a.N) y[j] = out[j];
    }
}

// ---- few rows of x ----------------------------------------------------------
// Grid ceil(N / (16 NT)), 64 SPLIT threads.  MT 16-row tiles of x, NT of W; the
// waves take the spans of four chunks of 128 channels in turn, D chunks at a time, the
// next D under way.  A span's scales are one load, a lane group a chunk's, and are handed
// around in registers: a load for each chunk took as long as the weight's own
// (28672 x 8192 from HBM, one row: 41 us, without any scales 29).
// All loads go through descriptors that end with the workgroup's rows: what does not exist
// (rows, groups past K, chunks past a wave's last) is an offset past the end, which reads as
// zero without a branch, and asks memory for nothing.
template <typename T, int MT, int NT, int SPLIT, int D, bool WORDS>
struct Few {
    static constexpr int kNone = 0x7f000000;         // past every descriptor's end
    static constexpr int kSpan = 4;
    __amdgpu_buffer_rsrc_t w, scale, x;
    int w_at[NT], e_at[NT], x_at[MT];                // the lane's rows, in bytes
    int groups, lg;
    f4 acc[NT][MT];

    struct Set {
        uint4 p[D][NT], x[D][MT][4];
    };
    struct Scales {
        uint32_t e[NT];                              // of the span's chunk lg
    };
    __device__ __forceinline__ void load(Scales& s, int c) const {
        const int g = 4 * (c + lg);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (WORDS) {
                s.e[t] = __builtin_amdgcn_raw_buffer_load_b32(scale, g < groups ? e_at[t] + g : kNone, 0, 0);
            } else {
                s.e[t] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s.e[t] |= static_cast<uint32_t>(
                        __builtin_amdgcn_raw_buffer_load_b8(scale, g + i < groups ? e_at[t] + g + i : kNone, 0, 0)) << (8 * i);
            }
        }
    }
    __device__ __forceinline__ void load(Set& s, int c0) const {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int g = 4 * (c0 + d);
            const bool mine = g + lg < groups;
#pragma unroll
            for (int t = 0; t < NT; ++t)
                s.p[d][t] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(w, mine ? w_at[t] + 16 * g : kNone, 0, 0));
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s.x[d][m][i] = __builtin_bit_cast(
                        uint4, __builtin_amdgcn_raw_buffer_load_b128(x, x_at[m], g + i < groups ? 64 * (g + i) : kNone, 0));
        }
    }
    // Chunks j.. of a span, e[j][t] their scales.
    __device__ __forceinline__ void add(Set& s, const uint32_t (&e)[kSpan][NT], int j) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
#pragma unroll
            for (int t = 0; t < NT; ++t) s.p[d][t] = turned(s.p[d][t]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint4 wide = mla::widen4<T>(word(s.p[d][t], i), power(e[j + d][t], i));
#pragma unroll
                    for (int m = 0; m < MT; ++m) acc[t][m] = Act<T>::mma16(wide, s.x[d][m][i], acc[t][m]);
                }
        }
    }
};

template <typename T, int MT, int NT, int SPLIT, int D, bool WORDS>
__global__ __launch_bounds__(64 * SPLIT) void few_kernel(kda_mx4_linear_args a) {
    using F = Few<T, MT, NT, SPLIT, D, WORDS>;
    constexpr int kTiles = NT * MT, kOwn = (kTiles + SPLIT - 1) / SPLIT;
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT);
    F f;
    f.groups = static_cast<int>(a.K / 32);
    f.lg = lg;
    const uint32_t rows = static_cast<uint32_t>(min(a.N - n0, static_cast<int64_t>(16 * NT)));
    f.w = make_rsrc(static_cast<const uint8_t*>(a.w) + n0 * f.groups * 16, rows * f.groups * 16);
    f.scale = make_rsrc(static_cast<const uint8_t*>(a.w_scale) + n0 * f.groups, rows * f.groups);
    f.x = make_rsrc(a.x, static_cast<uint32_t>(2 * ((a.M - 1) * a.x_stride + a.K)));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        f.e_at[t] = (16 * t + ln) * f.groups;
        f.w_at[t] = 16 * (f.e_at[t] + lg);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
        f.x_at[m] = 16 * m + ln < a.M ? 2 * (16 * m + ln) * static_cast<int>(a.x_stride) + 16 * lg : F::kNone;
    typename F::Set s[2];
    typename F::Scales next;
    const int chunks = (f.groups + 3) / 4;
    f.load(next, F::kSpan * wave);
    f.load(s[0], F::kSpan * wave);
    // tile i's outputs of this lane, i one of the wave's in the end
    const auto row = [&](int i) { return static_cast<int64_t>(16 * (i % MT) + ln); };
    const auto col = [&](int i) { return n0 + 16 * (i / MT) + 4 * lg; };
    Beside<T> beside[kOwn];
#pragma unroll
    for (int o = 0; o < kOwn; ++o)
        if (wave + o * SPLIT < kTiles) beside[o].load(a, row(wave + o * SPLIT), col(wave + o * SPLIT));
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) f.acc[t][m] = f4{0.f, 0.f, 0.f, 0.f};
    for (int c = F::kSpan * wave; c < chunks; c += F::kSpan * SPLIT) {
        uint32_t e[F::kSpan][NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            e[0][t] = e[2][t] = next.e[t];
            swap32(e[0][t], e[2][t]);
            e[1][t] = e[0][t];
            e[3][t] = e[2][t];
            swap16(e[0][t], e[1][t]);
            swap16(e[2][t], e[3][t]);
        }
        f.load(next, c + F::kSpan * SPLIT);
#pragma unroll
        for (int j = 0; j < F::kSpan; j += D) {
            const bool more = j + D < F::kSpan;
            f.load(s[(j / D + 1) & 1], more ? c + j + D : c + F::kSpan * SPLIT);
            f.add(s[(j / D) & 1], e, j);
        }
    }

    __shared__ f4 part[SPLIT == 1 ? 1 : SPLIT * kTiles * 64];
    if constexpr (SPLIT > 1) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) part[(wave * kTiles + i) * 64 + lane] = f.acc[i / MT][i % MT];
        __syncthreads();
    }
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
        const int i = wave + o * SPLIT;
        if (i >= kTiles) break;
        f4 r;
        if constexpr (SPLIT == 1) {
            r = f.acc[o / MT][o % MT];
        } else {
            r = part[i * 64 + lane];
#pragma unroll
            for (int v = 1; v < SPLIT; ++v) {
                const f4 p = part[(v * kTiles + i) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] += p[j];
            }
        }
        put<T>(a, row(i), col(i), r, beside[o]);
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
    const auto load_w = [&](int c, uint4 (&p)[4], uint32_t (&e)[4]) {
        const int g = min(4 * c + lg, groups - 1);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            p[t] = *reinterpret_cast<const uint4*>(w[t] + 16 * g);
            e[t] = scale[t][g];
        }
    };
    f4 acc[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[t][m] = f4{0.f, 0.f, 0.f, 0.f};
    uint4 p[4], next[4];
    uint32_t e[4], next_e[4];
    load_w(0, p, e);
    load_x(0, buf[0]);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int c = 0; c < chunks; ++c) {
        if (c + 1 < chunks) {
            load_w(c + 1, next, next_e);
            load_x(c + 1, buf[(c + 1) & 1]);
        }
        const char* from = buf[c & 1] + (64 * wm + ln) * (2 * kChunk);
        const bool past = 4 * c + lg >= groups;          // no channels of the lane's: zero, on both sides
        if (past) {
#pragma unroll
            for (int t = 0; t < 4; ++t) p[t] = uint4{0, 0, 0, 0};
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
                const uint4 wide = mla::widen4<T>(word(p[t], i), power(e[t], 0));
#pragma unroll
                for (int m = 0; m < 4; ++m) acc[t][m] = Act<T>::mma16(wide, x[m], acc[t][m]);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 4; ++t) p[t] = next[t], e[t] = next_e[t];
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int64_t row = m0 + 64 * wm + 16 * m + ln, n = n0 + 64 * wn + 16 * t + 4 * lg;
            Beside<T> beside;
            beside.load(a, row, n);
            put<T>(a, row, n, acc[t][m], beside);
        }
}

#include <cstdlib>
static int tune(const char* n, int d) { const char* s = getenv(n); return s ? atoi(s) : d; }
template <typename T, int MT, int NT, int SPLIT, int D>
void launch_few(const kda_mx4_linear_args& a, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>((a.N + 16 * NT - 1) / (16 * NT));
    if (a.K % 128 == 0 && reinterpret_cast<uintptr_t>(a.w_scale) % 4 == 0)
        few_kernel<T, MT, NT, SPLIT, D, true><<<grid, 64 * SPLIT, 0, stream>>>(a);
    else
        few_kernel<T, MT, NT, SPLIT, D, false><<<grid, 64 * SPLIT, 0, stream>>>(a);
}
template <typename T, int MT, int NT, int SPLIT>
void launch_d(const kda_mx4_linear_args& a, hipStream_t stream) {
    const int d = tune("TD", MT == 1 ? 2 : 1);
    if (d == 1 || MT == 4) launch_few<T, MT, NT, SPLIT, 1>(a, stream);
    else launch_few<T, MT, NT, SPLIT, MT == 4 ? 1 : 2>(a, stream);
}
template <typename T, int MT, int NT>
void launch_split(const kda_mx4_linear_args& a, hipStream_t stream) {
    const int64_t spans = (a.K + 511) / 512;
    const int sp = tune("TS", spans >= 8 ? 8 : spans >= 3 ? 4 : spans);
    if (sp == 8) launch_d<T, MT, NT, 8>(a, stream);
    else if (sp == 4) launch_d<T, MT, NT, 4>(a, stream);
    else if (sp == 2) launch_d<T, MT, NT, 2>(a, stream);
    else launch_d<T, MT, NT, 1>(a, stream);
}

template <typename T>
int launch_linear(const kda_mx4_linear_args& a, hipStream_t stream) {
    const int nt = tune("TN", a.N > 8192 ? 2 : 1);
    if (a.M > 64) {
        const dim3 grid(static_cast<unsigned>((a.N + kTile - 1) / kTile), static_cast<unsigned>((a.M + kTile - 1) / kTile));
        many_kernel<T><<<grid, 256, 0, stream>>>(a);
    } else if (a.M > 32) {
        if (nt == 1) launch_split<T, 4, 1>(a, stream);
        else if (nt == 2) launch_split<T, 4, 2>(a, stream);
        else launch_split<T, 4, 4>(a, stream);
    } else if (a.M > 16) {
        if (nt == 1) launch_split<T, 2, 1>(a, stream);
        else if (nt == 2) launch_split<T, 2, 2>(a, stream);
        else launch_split<T, 2, 4>(a, stream);
    } else {
        if (nt == 1) launch_split<T, 1, 1>(a, stream);
        else if (nt == 2) launch_split<T, 1, 2>(a, stream);
        else launch_split<T, 1, 4>(a, stream);
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
