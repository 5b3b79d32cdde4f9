// Latent attention in its absorbed form: a few query rows a sequence against
// the cache itself, whose rows are keys and (their first R channels) values.
//
//   s_mj = scale q_m . c_j,   o_m = sum_j 2^(s'_mj - M_m) c_j[0:R] / sum_j 2^(s'_mj - M_m),
//   s' = s log2(e),  M a running maximum.
//
// Bound by reading the cache: 16 heads of one token make 2 (2R + P) 16 flops of
// each row's 2 (R + P) bytes, 30 a byte.  So each row is read from memory once,
// straight into the registers that the score product takes it from (lane: one
// key, eight neighbouring channels), and from there written to LDS, from where
// the value product reads it transposed.  The scores come as keys x rows, whose
// accumulator layout is the value product's operand layout up to an order of
// the keys, which the transposed reads follow: P never leaves its registers.
//
// The four waves of a workgroup each take 32-key tiles of their own, with a
// softmax of their own: nothing in the loop waits for another wave.  They meet
// in LDS once a sequence, in a fixed order.
//
// The tiles of all sequences are one list that the workgroups share evenly,
// whatever the lengths (a decode batch's differ): a workgroup's share may
// begin and end inside a sequence, and what it has of one that others share
// goes to the workspace, to be joined by a second kernel.
//
// In 8 bits a value is widened to the activation type exactly; a key's scale
// multiplies its score, and enters the value product through the exponent,
// 2^(s' + log2 scale - M), so that P keeps its full precision in 16 bits at any
// scale.  M is then the largest of the sums, and the terms of the softmax's
// denominator are divided by the scale again.
#include <hip/hip_runtime.h>

#include "kda_launch.h"
#include "kda_mla.h"

namespace kda {
namespace {

using namespace mla;

constexpr int kTile = 32;         // keys of a wave's tile
constexpr int kWaves = 4;
constexpr int kRowTile = 16;      // query rows of a workgroup

// Workspace: for every slot (a workgroup's part of a row tile's sequence) the
// rows' sums, [16][R] fp32, and their (maximum, denominator); for every row tile
// the first and last workgroup that has a part of it.
struct Workspace {
    float* o;
    float2* ml;
    int2* span;
};
__host__ __device__ inline int64_t slots(int64_t groups, int64_t tiles) { return groups + tiles; }
__host__ __device__ inline Workspace carve(void* p, int64_t n_slots, int64_t R) {
    Workspace w;
    w.o = static_cast<float*>(p);
    w.ml = reinterpret_cast<float2*>(w.o + n_slots * kRowTile * R);
    w.span = reinterpret_cast<int2*>(w.ml + n_slots * kRowTile);
    return w;
}

template <typename T, bool F8, int R, int P>
struct Kernel {
    static constexpr int D = R + P;
    static constexpr int kLat = R / 32, kPos = P / 32;          // depth steps of the score product
    static constexpr int kStride = R + 16;                      // LDS row, elements
    static constexpr int kArea = kTile * kStride * 2;           // bytes of a wave's tile
    static constexpr int kOTiles = R / 16;
    static_assert(kArea >= kOTiles * 64 * 16, "a wave's sums fit its tile's place");

    // A tile's rows as loaded: lane (ln, lg) has row 16 s + ln.  16 bits: step k
    // is channels 32 k + 8 lg on.  8 bits: 16 channels 64 k + 16 lg on serve two
    // steps of the latent part, and the position part comes in 8-byte pieces.
    struct Rows {
        uint4 lat[2][F8 ? kLat / 2 : kLat];
        uint4 pos[2][F8 || kPos == 0 ? 1 : kPos];
        uint2 pos8[2][F8 && kPos ? kPos : 1];
        float2 scale[2][4];
    };

    static __device__ __forceinline__ void load(const kda_mla_absorbed_args& a, int64_t b, int tile, int len, int ln,
                                                int lg, Rows& r) {
        const int es = F8 ? 1 : 2;
        const char* base = static_cast<const char*>(a.cache) + b * a.cache_stride[0] * es;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            // rows past the last repeat it: their scores are masked
            const int j = min(tile * kTile + 16 * s + ln, len - 1);
            const char* row = base + j * a.cache_stride[1] * es + 16 * lg;
#pragma unroll
            for (int k = 0; k < (F8 ? kLat / 2 : kLat); ++k) r.lat[s][k] = *reinterpret_cast<const uint4*>(row + 64 * k);
            if constexpr (kPos > 0 && !F8) {
#pragma unroll
                for (int k = 0; k < kPos; ++k) r.pos[s][k] = *reinterpret_cast<const uint4*>(row + 2 * R + 64 * k);
            }
            if constexpr (F8) {
                if constexpr (kPos > 0) {
#pragma unroll
                    for (int k = 0; k < kPos; ++k)
                        r.pos8[s][k] = *reinterpret_cast<const uint2*>(row + R - 8 * lg + 32 * k);
                }
                const float* sc = a.cache_scale + b * a.scale_stride[0];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = min(tile * kTile + 16 * s + 4 * lg + i, len - 1);
                    r.scale[s][i] = *reinterpret_cast<const float2*>(sc + key * a.scale_stride[1]);
                }
            }
        }
    }

    // The rows' q, as the score product's second operand in the same order of channels.
    static __device__ __forceinline__ void load_q(const T* q, int lg, uint4 (&f)[kLat + kPos]) {
#pragma unroll
        for (int k = 0; k < kLat; ++k) {
            const int c = F8 ? 64 * (k / 2) + 16 * lg + 8 * (k % 2) : 32 * k + 8 * lg;
            f[k] = *reinterpret_cast<const uint4*>(q + c);
        }
#pragma unroll
        for (int k = 0; k < kPos; ++k) f[kLat + k] = *reinterpret_cast<const uint4*>(q + R + 32 * k + 8 * lg);
    }

    // Scores of a tile (keys 16 s + 4 lg + i of row ln), times scale log2(e), plus
    // log2 of the key's scale in 8 bits; the latent part goes to LDS on the way.
    static __device__ __forceinline__ void scores(const Rows& r, const uint4 (&q)[kLat + kPos], float c, T* lds, int ln,
                                                  int lg, f4 (&s)[2], float (&inv)[2][4]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f4 acc{}, pos{};
            T* row = lds + (16 * h + ln) * kStride;
            if constexpr (F8) {
#pragma unroll
                for (int k = 0; k < kLat / 2; ++k) {
                    const uint4 w = r.lat[h][k];
                    const uint4 lo = widen8<T>(w.x, w.y), hi = widen8<T>(w.z, w.w);
                    acc = Act<T>::mma16(lo, q[2 * k], acc);
                    acc = Act<T>::mma16(hi, q[2 * k + 1], acc);
                    uint4* to = reinterpret_cast<uint4*>(row + 64 * k + 16 * lg);
                    to[0] = lo;
                    to[1] = hi;
                }
#pragma unroll
                for (int k = 0; k < kPos; ++k)
                    pos = Act<T>::mma16(widen8<T>(r.pos8[h][k].x, r.pos8[h][k].y), q[kLat + k], pos);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 sc = r.scale[h][i];
                    s[h][i] = fmaf(acc[i] * sc.x + pos[i] * sc.y, c, __builtin_amdgcn_logf(sc.x));
                    inv[h][i] = __builtin_amdgcn_rcpf(sc.x);
                }
            } else {
#pragma unroll
                for (int k = 0; k < kLat; ++k) {
                    acc = Act<T>::mma16(r.lat[h][k], q[k], acc);
                    *reinterpret_cast<uint4*>(row + 32 * k + 8 * lg) = r.lat[h][k];
                }
#pragma unroll
                for (int k = 0; k < kPos; ++k) acc = Act<T>::mma16(r.pos[h][k], q[kLat + k], acc);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][i] = acc[i] * c;
            }
        }
    }

    // One row tile's part of tiles [lo, hi) of sequence b; the whole of it if
    // `whole`, else into the workspace's slot.
    static __device__ __forceinline__ void segment(const kda_mla_absorbed_args& a, char* smem, int64_t b, int rt, int len,
                                                   int lo, int hi, bool whole, const Workspace& ws, int64_t slot) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, lg = lane >> 4;
        const int rows = static_cast<int>(a.T * a.H), H = static_cast<int>(a.H);
        const int m = rt * kRowTile + ln, mc = min(m, rows - 1), t = mc / H, h = mc - t * H;
        const int limit = len - static_cast<int>(a.T) + t;       // last key this lane's row sees
        const float c = a.scale * kLog2E;
        T* lds = reinterpret_cast<T*>(smem + wave * kArea);

        Rows cur;
        int tile = lo + wave;
        if (tile < hi) load(a, b, tile, len, ln, lg, cur);
        uint4 q[kLat + kPos];
        load_q(static_cast<const T*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + h * a.q_stride[2], lg, q);

        f4 o[kOTiles];
#pragma unroll
        for (int i = 0; i < kOTiles; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
        float top = kNoMax, sum = 0.f;
        const int tr_row = 4 * lg + (ln >> 2), tr_col = 4 * (ln & 3);

        for (; tile < hi; tile += kWaves) {
            f4 s[2];
            float inv[2][4];
            scores(cur, q, c, lds, ln, lg, s, inv);
            if (tile + kWaves < hi) load(a, b, tile + kWaves, len, ln, lg, cur);
            const int j0 = tile * kTile + 4 * lg;
            if (tile * kTile + kTile > len - static_cast<int>(a.T)) {
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (j0 + 16 * g + i > limit) s[g][i] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                             fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            mx = fmaxf(top, lanegroup4_max(mx));
            const float alpha = __builtin_amdgcn_exp2f(top - mx);
            top = mx;
            float p[2][4], part = 0.f;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[g][i] = __builtin_amdgcn_exp2f(s[g][i] - mx);
                    part = F8 ? fmaf(p[g][i], inv[g][i], part) : part + p[g][i];
                }
            sum = fmaf(sum, alpha, part);
            const uint4 pf{Act<T>::pair(p[0][0], p[0][1]), Act<T>::pair(p[0][2], p[0][3]),
                           Act<T>::pair(p[1][0], p[1][1]), Act<T>::pair(p[1][2], p[1][3])};
            if (__any(alpha != 1.f)) {
#pragma unroll
                for (int i = 0; i < kOTiles; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][e] *= alpha;
            }
            const T* v = lds + tr_row * kStride + tr_col;
#pragma unroll
            for (int i = 0; i < kOTiles; ++i) {
                const uint2 v0 = read_tr(v + 16 * i), v1 = read_tr(v + 16 * kStride + 16 * i);
                o[i] = Act<T>::mma16(uint4{v0.x, v0.y, v1.x, v1.y}, pf, o[i]);
            }
        }
        sum = lanegroup4_sum(sum);

        // the four waves' sums, on the largest maximum of each row
        __shared__ float2 ml[kWaves][kRowTile];
        __syncthreads();             // an earlier segment's readers are done
        if (lg == 0) ml[wave][ln] = float2{top, sum};
        __syncthreads();
        float big = ml[0][ln].x, den = 0.f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) big = fmaxf(big, ml[w][ln].x);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) den += ml[w][ln].y * __builtin_amdgcn_exp2f(ml[w][ln].x - big);
        const float mine = __builtin_amdgcn_exp2f(top - big);
        f4* area = reinterpret_cast<f4*>(smem + wave * kArea);
#pragma unroll
        for (int i = 0; i < kOTiles; ++i) area[i * 64 + lane] = f4{o[i][0] * mine, o[i][1] * mine, o[i][2] * mine,
                                                                    o[i][3] * mine};
        __syncthreads();
        const float norm = den == 0.f ? 0.f : 1.f / den;
        for (int i = wave; i < kOTiles; i += kWaves) {
            f4 r = reinterpret_cast<const f4*>(smem)[i * 64 + lane];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) {
                const f4 x = reinterpret_cast<const f4*>(smem + w * kArea)[i * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] += x[e];
            }
            if (whole) {
                if (m < rows)
                    *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + (b * rows + m) * R + 16 * i + 4 * lg) =
                        uint2{Act<T>::pair(r[0] * norm, r[1] * norm), Act<T>::pair(r[2] * norm, r[3] * norm)};
            } else {
                *reinterpret_cast<f4*>(ws.o + (slot * kRowTile + ln) * R + 16 * i + 4 * lg) = r;
            }
        }
        if (!whole && wave == 0 && lg == 0) ws.ml[slot * kRowTile + ln] = float2{big, den};
    }
};

__device__ __forceinline__ int tiles_of(const kda_mla_absorbed_args& a, int64_t v, int64_t nv, int rts) {
    return v < nv ? (tokens(a.lengths, v / rts, a.S) + kTile - 1) / kTile : 0;
}
__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}

// Grid: one workgroup for each row tile of each sequence.
template <typename T, bool F8, int R, int P>
__global__ __launch_bounds__(64 * kWaves, 1) void absorbed_kernel(kda_mla_absorbed_args a, int rts) {
    using K = Kernel<T, F8, R, P>;
    __shared__ __align__(16) char smem[kWaves * K::kArea];
    const int64_t b = blockIdx.x / rts;
    const int len = tokens(a.lengths, b, a.S);
    K::segment(a, smem, b, static_cast<int>(blockIdx.x - b * rts), len, 0, (len + kTile - 1) / kTile, true, Workspace{},
               0);
}

// Grid: any number of workgroups, each with its share of all tiles.
template <typename T, bool F8, int R, int P>
__global__ __launch_bounds__(64 * kWaves, 1) void absorbed_shared_kernel(kda_mla_absorbed_args a, int rts) {
    using K = Kernel<T, F8, R, P>;
    __shared__ __align__(16) char smem[kWaves * K::kArea];
    const int lane = threadIdx.x & 63;
    const int64_t nv = a.B * rts;
    const Workspace ws = carve(a.workspace, slots(gridDim.x, nv), R);
    int64_t total = 0;
    for (int64_t v = 0; v < nv; v += 64) total += __shfl(wave_scan(tiles_of(a, v + lane, nv, rts), lane), 63);
    const int64_t share = (total + gridDim.x - 1) / gridDim.x;
    const int64_t from = blockIdx.x * share, to = min(from + share, total);
    if (from >= to) return;
    int64_t before = 0;              // tiles of the row tiles before this chunk's
    for (int64_t v0 = 0; v0 < nv && before < to; v0 += 64) {
        const int n = tiles_of(a, v0 + lane, nv, rts);
        const int end = wave_scan(n, lane);
        const int chunk = __shfl(end, 63);
        const int64_t mine = before + end - n;       // this lane's first tile in the list
        uint64_t todo = __ballot(n > 0 && mine < to && mine + n > from);
        while (todo) {
            const int i = __builtin_ctzll(todo);
            todo &= todo - 1;
            const int tiles = __builtin_amdgcn_readlane(n, i);
            const int64_t first = before + __builtin_amdgcn_readlane(end, i) - tiles, v = v0 + i, b = v / rts;
            const int lo = static_cast<int>(max(from - first, static_cast<int64_t>(0)));
            const int hi = static_cast<int>(min(to - first, static_cast<int64_t>(tiles)));
            K::segment(a, smem, b, static_cast<int>(v - b * rts), tokens(a.lengths, b, a.S), lo, hi,
                       lo == 0 && hi == tiles, ws, blockIdx.x + v);
            if (threadIdx.x == 0) {
                if (lo == 0) ws.span[v].x = static_cast<int>(blockIdx.x);
                if (hi == tiles) ws.span[v].y = static_cast<int>(blockIdx.x);
            }
        }
        before += chunk;
    }
}

// The parts of one row's sequence joined: grid (row tiles, 16, R / 64), sixteen
// lanes on 64 channels and sixteen groups of them on every sixteenth part, whose
// sums meet in LDS, in an order that the lengths alone decide.
constexpr int kJoinGroups = 16;
template <typename T>
__global__ __launch_bounds__(16 * kJoinGroups) void join_kernel(kda_mla_absorbed_args a, int rts, int groups) {
    const int64_t v = blockIdx.x, b = v / rts, nv = a.B * rts;
    const int rows = static_cast<int>(a.T * a.H), m = static_cast<int>(v - b * rts) * kRowTile + blockIdx.y;
    if (m >= rows) return;
    const int c = 64 * blockIdx.z + 4 * (threadIdx.x & 15), group = threadIdx.x >> 4;
    const Workspace ws = carve(a.workspace, slots(groups, nv), a.R);
    const int2 span = tokens(a.lengths, b, a.S) > 0 ? ws.span[v] : int2{0, -1};
    if (span.x == span.y) return;                // one workgroup had it all, and wrote the result
    const float2* ml = ws.ml + v * kRowTile + blockIdx.y;
    const float* o = ws.o + (v * kRowTile + blockIdx.y) * a.R + c;
    float top = kNoMax, den = 0.f;
    f4 r{};
    for (int g = span.x + group; g <= span.y; g += kJoinGroups) {
        const float2 x = ml[g * kRowTile];
        const f4 y = *reinterpret_cast<const f4*>(o + static_cast<int64_t>(g) * kRowTile * a.R);
        const float now = fmaxf(top, x.x), f0 = __builtin_amdgcn_exp2f(top - now);
        const float f1 = x.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x.x - now);
        top = now;
        den = den * f0 + x.y * f1;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = r[e] * f0 + y[e] * f1;
    }
    __shared__ f4 sums[kJoinGroups][16];
    __shared__ float2 stats[kJoinGroups];
    sums[group][threadIdx.x & 15] = r;
    if ((threadIdx.x & 15) == 0) stats[group] = float2{top, den};
    __syncthreads();
    if (group != 0) return;
    const int n = min(kJoinGroups, span.y - span.x + 1);
    for (int g = 0; g < n; ++g) top = fmaxf(top, stats[g].x);
    den = 0.f;
    r = f4{};
    for (int g = 0; g < n; ++g) {
        const float w = __builtin_amdgcn_exp2f(stats[g].x - top);
        den = fmaf(w, stats[g].y, den);
        const f4 y = sums[g][threadIdx.x];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = fmaf(w, y[e], r[e]);
    }
    const float norm = den == 0.f ? 0.f : 1.f / den;
    *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + (b * rows + m) * a.R + c) =
        uint2{Act<T>::pair(r[0] * norm, r[1] * norm), Act<T>::pair(r[2] * norm, r[3] * norm)};
}

int row_tiles(int64_t T, int64_t H) { return static_cast<int>((T * H + kRowTile - 1) / kRowTile); }

constexpr int64_t kGroups = 256;      // workgroups of the shared form: one a CU
// Whether the tiles are shared among the workgroups: where one workgroup a row
// tile would leave CUs idle or wait for the longest sequence.
bool shared_form(int64_t nv, int64_t S) { return nv < 4 * kGroups && S > 16 * kTile; }

template <typename T, bool F8, int R, int P>
int launch(const kda_mla_absorbed_args& a, hipStream_t stream) {
    const int rts = row_tiles(a.T, a.H);
    const int64_t nv = a.B * rts;
    if (!shared_form(nv, a.S)) {
        absorbed_kernel<T, F8, R, P><<<static_cast<unsigned>(nv), 64 * kWaves, 0, stream>>>(a, rts);
    } else {
        absorbed_shared_kernel<T, F8, R, P><<<kGroups, 64 * kWaves, 0, stream>>>(a, rts);
        join_kernel<T><<<dim3(static_cast<unsigned>(nv), kRowTile, R / 64), 16 * kJoinGroups, 0, stream>>>(
            a, rts, static_cast<int>(kGroups));
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

template <typename T, bool F8, int R>
int launch_pos(const kda_mla_absorbed_args& a, hipStream_t stream) {
    switch (a.P) {
        case 64: return launch<T, F8, R, 64>(a, stream);
        case 32: return launch<T, F8, R, 32>(a, stream);
        default: return launch<T, F8, R, 0>(a, stream);
    }
}
template <typename T, bool F8>
int launch_rank(const kda_mla_absorbed_args& a, hipStream_t stream) {
    switch (a.R) {
        case 512: return launch_pos<T, F8, 512>(a, stream);
        case 256: return launch_pos<T, F8, 256>(a, stream);
        default: return launch_pos<T, F8, 128>(a, stream);
    }
}

}  // namespace

int64_t mla_absorbed_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t S, int64_t R) {
    const int64_t nv = B * row_tiles(T, H);
    if (nv == 0 || !shared_form(nv, S)) return 0;
    return slots(kGroups, nv) * kRowTile * (R * 4 + 8) + nv * 8;
}

int mla_absorbed_launch(const kda_mla_absorbed_args& a, hipStream_t stream) {
    if (a.cache_dtype == KDA_DTYPE_E4M3)
        return a.dtype == KDA_DTYPE_F16 ? launch_rank<_Float16, true>(a, stream) : launch_rank<bf16_t, true>(a, stream);
    return a.dtype == KDA_DTYPE_F16 ? launch_rank<_Float16, false>(a, stream) : launch_rank<bf16_t, false>(a, stream);
}

}  // namespace kda
