// Latent attention in its expanded form, forward: causal attention whose keys
// are a head's own N channels and P position channels that all heads share.
//
//   s_tj = scale q_t . [k_j | k_pe_j],  o_t = sum_j 2^(s'_tj - M_t) v_j / sum_j 2^(s'_tj - M_t),
//   s' = s log2(e),  M a running maximum (in fp16 less 15).
//
// Bound by the matrix cores: 2 (N + P + V) flops a visible pair.  At 128 + 64
// channels, bf16, H=16: 1110 TFLOP/s at T=16384, 920 for T=2048 over 16384 keys,
// 850 at B=4 T=2048 (a large product reaches 1200); one prompt of 1000 tokens
// takes 21 us (23 in fp16), the longest tile's eight steps in a row.  A wave has 32
// query rows; a workgroup's waves share 64-key tiles of K, K_pe and V in LDS,
// two buffers, the next tile's loads in flight through the current one's
// products.  The scores are formed transposed (keys x rows, 32x32x16), so a
// lane has 32 scores of one row: the row's maximum and sum are its own
// registers and one exchange with the other half of the wave, and the scores,
// rounded, are the second operand of the value product O^T = V^T P^T as they
// lie, in an order of the keys that the transposed reads of V follow.  O^T's
// columns are rows again, so a new maximum rescales a lane's own registers;
// in bf16 it does so only when the maximum has grown by more than 2^8 (P stays
// below 2^8); fp16 has its room below the maximum (reference) and 2^0.75 above.
//
// Few rows over many keys: several workgroups share the keys of a query tile,
// each leaves its sums in the workspace, and a second kernel joins them.
//
// LDS rows are padded so that sixteen rows' 16-byte pieces (K) and the four
// rows of a transposed read (V) fall into different banks.
#include <hip/hip_runtime.h>

#include "kda_launch.h"
#include "kda_mla.h"
#include "kda_mla_tile.h"

namespace kda {
namespace {

using namespace mla;

// log2 of how far a maximum may lag: in fp16 what there is between 2^15 and its largest value
template <typename T> constexpr float kLazy = Elem<T>::code == KDA_DTYPE_F16 ? 0.75f : 8.f;

// The workspace of shared keys: every row's parts, [rows][splits][V] sums and
// their (maximum, denominator).
struct Parts {
    float* o;
    float2* stat;
    __host__ __device__ Parts(void* p, int64_t rows, int splits, int64_t V)
        : o(static_cast<float*>(p)), stat(reinterpret_cast<float2*>(o + rows * splits * V)) {}
};

// A workgroup: RW waves of 32 query rows, times KW waves that share the keys
// of each: of a step's KW KEYS keys, wave group g takes the g-th KEYS.  BUFS
// buffers of a step's tiles; with one, the next step's keys are put where this
// one's were while its values are still in use, and the values during the next
// scores (T=1000 H=16 22.2 -> 21.5 us against both at the step's end).
// Grid: (query tiles, longest first) x (batch, head) with the latter inner, so
// that a head's tiles share an XCD's L2 where B H is a multiple of eight.
// SPLIT: `splits` workgroups a query tile, its steps shared out evenly.
// FEW: p goes into the value product with what its rounding leaves.
template <typename T, int N, int P, int RW, int KW, int KEYS, int BUFS, bool SPLIT, bool FEW>
__global__ __launch_bounds__(64 * RW * KW, RW * KW == 8 ? 2 : 1) void expanded_kernel(kda_mla_expanded_args a,
                                                                                     int qtiles, int splits) {
    constexpr int kStep = KW * KEYS, kRows = 32 * RW, kU = KEYS / 32;
    using F = KvTile<T, N, P, 64 * RW * KW, kStep, 32>;
    constexpr int D = F::D, V = F::V;
    constexpr int kJoin = KW == 1 ? 0 : RW * (KW / 2) * (32 * V + 64) * 4;        // bytes
    constexpr int kBytes = BUFS * F::kBuf * 2 > kJoin ? BUFS * F::kBuf * 2 : kJoin;
    __shared__ __align__(16) char raw[kBytes];
    T* smem = reinterpret_cast<T*>(raw);
    const int64_t bhs = a.B * a.H, unit = SPLIT ? blockIdx.x / splits : blockIdx.x;
    const int part = SPLIT ? static_cast<int>(blockIdx.x - unit * splits) : 0;
    const int64_t bh = unit % bhs, b = bh / a.H, h = bh - b * a.H;
    const int tile_at = qtiles - 1 - static_cast<int>(unit / bhs), t0 = tile_at * kRows;
    const int lane = threadIdx.x & 63, lq = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = wave % RW, group = wave / RW;
    const int len = tokens(a.lengths, b, a.S), nq = static_cast<int>(a.T);
    const int start = first_position(a.starts, b, a.S, a.T);
    const int exist = max(0, min(nq, len - start));              // queries that exist
    const int w0 = t0 + 32 * row, t = w0 + lq;
    const bool live = t < exist;
    const int limit = live ? start + t : -1;                      // last key this lane's row sees
    const int wlast = w0 < exist ? start + min(w0 + 31, exist - 1) : -1;       // and the last of the wave's
    const int wall = w0 + 32 <= exist ? start + w0 : -1;          // keys up to this one every row sees
    const int seen = t0 < exist ? start + min(t0 + kRows, exist) : 0;           // keys that the tile's rows see
    int first = 0, keys = seen;                                   // and the workgroup's
    if constexpr (SPLIT) {
        const int steps = (seen + kStep - 1) / kStep;
        first = static_cast<int>(static_cast<int64_t>(part) * steps / splits) * kStep;
        keys = min(static_cast<int>(static_cast<int64_t>(part + 1) * steps / splits) * kStep, seen);
    }
    const float c = a.scale * kLog2E;

    f16v o[V / 32];
#pragma unroll
    for (int i = 0; i < V / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float top = kNoMax, sum = 0.f;
    bool far = false;                                             // some row's top is far from zero

    if (keys > first) {
        uint4 q[D / 16];
        const T* qr = static_cast<const T*>(a.q) + b * a.q_stride[0] + min(max(t, -start), exist - 1) * a.q_stride[1] +
                      h * a.q_stride[2] + 8 * half;
        F tile(a, b, h);
        tile.fetch(a, first, keys);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) q[k] = *reinterpret_cast<const uint4*>(qr + 16 * k);
        if constexpr (BUFS == 2) tile.put(smem);
        else tile.put_keys(smem);
        __syncthreads();
        int cur = 0;
        for (int j0 = first; j0 < keys; j0 += kStep) {
            if constexpr (BUFS == 1) tile.put_values(smem);
            tile.fetch(a, j0 + kStep, keys);
            const T* buf = smem + cur * F::kBuf;
            const int jw = j0 + KEYS * group;                     // the wave's first key
            f16v s[kU];
            if (jw <= wlast) {
                const T* kt = buf + (KEYS * group + lq) * F::kK + 8 * half;
#pragma unroll
                for (int u = 0; u < kU; ++u) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[u][e] = 0.f;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        s[u] = Act<T>::mma32(*reinterpret_cast<const uint4*>(kt + 32 * u * F::kK + 16 * k), q[k], s[u]);
                }
            }
            if constexpr (BUFS == 1) __syncthreads();     // the values are there, and the keys read
            if (jw <= wlast) {
                if (jw + KEYS - 1 > wall) {
#pragma unroll
                    for (int u = 0; u < kU; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (jw + 32 * u + 8 * (e / 4) + 4 * half + e % 4 > limit) s[u][e] = -INFINITY;
                }
                float mx = s[0][0];
#pragma unroll
                for (int u = 0; u < kU; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[u][e]);
                mx = reference<T>(half_max(mx) * c);
                if (__any(mx > top + kLazy<T>)) {
                    const float now = fmaxf(top, mx), alpha = __builtin_amdgcn_exp2f(top - now);
                    top = now;
                    far = __any(far_from_zero(top));
                    sum *= alpha;
#pragma unroll
                    for (int i = 0; i < V / 32; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
                }
                float m = c;
                if (far) {
#pragma unroll
                    for (int u = 0; u < kU; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[u][e] *= c;
                    m = 1.f;
                }
                uint4 p[2 * kU], left[FEW ? 2 * kU : 1];
#pragma unroll
                for (int u = 0; u < 2 * kU; ++u) {
                    uint32_t w[4], l[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = __builtin_amdgcn_exp2f(fmaf(s[u / 2][8 * (u % 2) + 2 * e], m, -top));
                        const float y = __builtin_amdgcn_exp2f(fmaf(s[u / 2][8 * (u % 2) + 2 * e + 1], m, -top));
                        sum += x;
                        sum += y;
                        w[e] = Act<T>::pair(x, y);
                        if constexpr (FEW) l[e] = rest(x, y, T{});
                    }
                    if constexpr (FEW) left[u] = uint4{l[0], l[1], l[2], l[3]};
                    p[u] = uint4{w[0], w[1], w[2], w[3]};
                }
                const T* vt = buf + kStep * F::kK + (KEYS * group + 4 * half + ((lane & 15) >> 2)) * F::kV +
                              16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
                for (int u = 0; u < 2 * kU; ++u)
#pragma unroll
                    for (int i = 0; i < V / 32; ++i) {
                        const uint2 v0 = read_tr(vt + 16 * u * F::kV + 32 * i);
                        const uint2 v1 = read_tr(vt + (16 * u + 8) * F::kV + 32 * i);
                        o[i] = Act<T>::mma32(uint4{v0.x, v0.y, v1.x, v1.y}, p[u], o[i]);
                        if constexpr (FEW) o[i] = Act<T>::mma32(uint4{v0.x, v0.y, v1.x, v1.y}, left[u], o[i]);
                    }
            }
            if constexpr (BUFS == 2) {
                cur ^= 1;
                tile.put(smem + cur * F::kBuf);
                __syncthreads();
            } else {
                tile.put_keys(smem);
                __syncthreads();
            }
        }
    }
    // the key groups' sums, half of them onto the other half at a time
#pragma unroll
    for (int n = KW / 2; n > 0; n /= 2) {
        f4* part = reinterpret_cast<f4*>(raw);
        const int slot = (group % n) * RW + row;                  // of n RW
        f4* mine = part + slot * (V / 32) * 4 * 64 + lane;
        float2* stat = reinterpret_cast<float2*>(part + n * RW * (V / 32) * 4 * 64) + slot * 64 + lane;
        if (group >= n && group < 2 * n) {
#pragma unroll
            for (int i = 0; i < V / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mine[(4 * i + e) * 64] = f4{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]};
            *stat = float2{top, sum};
        }
        __syncthreads();
        if (group < n) {
            const float2 x = *stat;
            const float now = fmaxf(top, x.x), f0 = __builtin_amdgcn_exp2f(top - now), f1 = __builtin_amdgcn_exp2f(x.x - now);
            top = now;
            sum = sum * f0 + x.y * f1;
#pragma unroll
            for (int i = 0; i < V / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f4 y = mine[(4 * i + e) * 64];
#pragma unroll
                    for (int d = 0; d < 4; ++d) o[i][4 * e + d] = o[i][4 * e + d] * f0 + y[d] * f1;
                }
        }
        __syncthreads();
    }
    if (group != 0 || t >= nq) return;
    sum = half_sum(sum);
    if constexpr (SPLIT) {
        const Parts parts(a.workspace, bhs * a.T, splits, V);
        const int64_t at = (bh * a.T + t) * splits + part;
        if (half == 0) parts.stat[at] = float2{top, sum};
        if (sum != 0.f) {            // (or not a number); a part without keys is not read
#pragma unroll
            for (int i = 0; i < V / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<f4*>(parts.o + at * V + 32 * i + 8 * e + 4 * half) =
                        f4{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]};
        }
        return;
    }
    const float norm = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t to = ((b * a.T + t) * a.H + h) * V + 4 * half;
    T* out = static_cast<T*>(a.o) + to;
    T* low = a.o_low ? static_cast<T*>(a.o_low) + to : nullptr;
#pragma unroll
    for (int i = 0; i < V / 32; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            store_out(out + 32 * i + 8 * e, low ? low + 32 * i + 8 * e : nullptr,
                      f4{o[i][4 * e] * norm, o[i][4 * e + 1] * norm, o[i][4 * e + 2] * norm, o[i][4 * e + 3] * norm});
    if (a.lse && half == 0) store_lse(a.lse, a.lse_low, (b * a.H + h) * a.T + t, top, sum);
}

// The parts of a row joined in order: V / 4 lanes a row.
template <typename T, int V>
__global__ __launch_bounds__(256) void join_kernel(kda_mla_expanded_args a, int splits) {
    constexpr int kLanes = V / 4;
    const int64_t rows = a.B * a.H * a.T, row = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
    if (row >= rows) return;
    const int ch = 4 * (threadIdx.x % kLanes);
    const Parts parts(a.workspace, rows, splits, V);
    const float2* stat = parts.stat + row * splits;
    const float* from = parts.o + row * splits * V + ch;
    float top = kNoMax, sum = 0.f;
    for (int i = 0; i < splits; ++i) top = fmaxf(top, stat[i].x);
    f4 r{};
    for (int i = 0; i < splits; ++i) {
        const float2 x = stat[i];
        if (x.y == 0.f) continue;
        const float w = __builtin_amdgcn_exp2f(x.x - top);
        const f4 y = *reinterpret_cast<const f4*>(from + static_cast<int64_t>(i) * V);
        sum = fmaf(w, x.y, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = fmaf(w, y[e], r[e]);
    }
    const float norm = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t bh = row / a.T, t = row - bh * a.T, b = bh / a.H, h = bh - b * a.H;
    const int64_t to = ((b * a.T + t) * a.H + h) * V + ch;
    store_out(static_cast<T*>(a.o) + to, a.o_low ? static_cast<T*>(a.o_low) + to : nullptr,
              f4{r[0] * norm, r[1] * norm, r[2] * norm, r[3] * norm});
    if (a.lse && ch == 0) store_lse(a.lse, a.lse_low, row, top, sum);
}

// Workgroups that share the keys of a query tile of 64 rows: where there are too
// few tiles for the CUs, as many as fill them with at least 512 keys each, or below
// 2048 keys, where that would leave three or fewer, 256 (up to seven).  us at H=16, parts
// of 512 / 256: T=64 S=1024 17.4 / 15.9, S=4096 23.5 / 27.1.  Between 1280 and 2047 keys
// parts of 256 / four of them, T=1 S=1280 14.5 / 15.7, S=1792 15.7 / 17.3, S=2047 17.2 /
// 17.2, but T=64 S=2047 21.2 / 20.2 and T=128 S=1792 21.6 / 20.9.
int splits_of(int64_t B, int64_t T, int64_t S, int64_t H) {
    const int64_t tiles = B * H * ((T + 63) / 64);
    if (tiles == 0 || tiles > 128 || S < 1024) return 1;
    const int64_t most = S >= 2048 ? S / 512 : S / 256, fill = 256 / tiles;
    return static_cast<int>(most < fill ? most : fill);
}

template <typename T, int N, int P, int RW, int KW, int KEYS, int BUFS, bool SPLIT = false, bool FEW = false>
int launch_as(const kda_mla_expanded_args& a, hipStream_t stream, int splits = 1) {
    const int64_t qtiles = (a.T + 32 * RW - 1) / (32 * RW);
    expanded_kernel<T, N, P, RW, KW, KEYS, BUFS, SPLIT, FEW>
        <<<static_cast<unsigned>(qtiles * a.B * a.H * splits), 64 * RW * KW, 0, stream>>>(a, static_cast<int>(qtiles), splits);
    if constexpr (SPLIT) {
        constexpr int rows = 256 / (N / 4);
        join_kernel<T, N><<<static_cast<unsigned>((a.B * a.H * a.T + rows - 1) / rows), 256, 0, stream>>>(a, splits);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

template <typename T, int N, int P>
int launch(const kda_mla_expanded_args& a, hipStream_t stream) {
    // Eight waves a workgroup, as many of them on rows of their own as leave every
    // CU a workgroup; of 256 rows two where the tiles differ (few keys before the
    // first query), so that a long one is not alone at the end: us, 256 / 128 rows,
    // B=1 T=4096 H=16 132 / 105.  128 / 64 rows, at 128 channels: T=2048 46 / 44, T=3000
    // 66 / 88, B=2 T=1200 31 / 44, B=4 T=512 18 / 23.  At 64 channels two workgroups
    // of either fit a CU, and 64 rows share it better: T=2800 48 / 39.
    if (few(a)) return launch_as<T, N, P, 2, 4, 32, 1, false, true>(a, stream);
    const int64_t heads = a.B * a.H, least = a.S >= 2 * a.T ? 256 : 512;
    if (heads * ((a.T + 255) / 256) >= least) return launch_as<T, N, P, 8, 1, 64, 2>(a, stream);
    if (heads * ((a.T + 127) / 128) >= (N == 128 ? 256 : least)) return launch_as<T, N, P, 4, 2, 32, 2>(a, stream);
    const int splits = splits_of(a.B, a.T, a.S, a.H);
    if (splits > 1) return launch_as<T, N, P, 2, 4, 32, 1, true>(a, stream, splits);
    return launch_as<T, N, P, 2, 4, 32, 1>(a, stream);
}

template <typename T>
int launch_dims(const kda_mla_expanded_args& a, hipStream_t stream) {
    switch (a.N + a.P) {
        case 192: return launch<T, 128, 64>(a, stream);
        case 160: return launch<T, 128, 32>(a, stream);
        case 128: return a.N == 128 ? launch<T, 128, 0>(a, stream) : launch<T, 64, 64>(a, stream);
        case 96: return launch<T, 64, 32>(a, stream);
        default: return launch<T, 64, 0>(a, stream);
    }
}

}  // namespace

int64_t mla_expanded_workspace_bytes(int64_t B, int64_t T, int64_t S, int64_t H, int64_t V) {
    const int splits = splits_of(B, T, S, H);
    return splits > 1 ? B * H * T * splits * (V * 4 + 8) : 0;
}

int mla_expanded_launch(const kda_mla_expanded_args& a, hipStream_t stream) {
    return a.dtype == KDA_DTYPE_F16 ? launch_dims<_Float16>(a, stream) : launch_dims<bf16_t>(a, stream);
}

}  // namespace kda
