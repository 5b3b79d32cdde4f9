// Latent attention in its expanded form, backward.  With the forward's lse,
//
//   p_tj = 2^(s'_tj - lse_t),  dp_tj = do_t . v_j,  delta_t = do_t . o_t,
//   ds_tj = p_tj (dp_tj - delta_t),
//   dv_j = sum_t p_tj do_t,  dq_t = scale sum_j ds_tj [k_j | k_pe_j],
//   dk_j = scale sum_t ds_tj q_t  (its last P channels summed over the heads too).
//
// Two kernels that each form s and dp anew, one with a wave's 32 query rows
// standing and the keys passing (dq, and delta for the other), one with a
// wave's 32 keys standing and the queries passing (dk, dv): seven products
// instead of the five that adding dq's parts in memory would take, and no
// atomics, so the sums have one order.  Bound by the matrix cores, which are
// busy 40 % (dq) and 35 % (dk, dv) of the time: two waves a SIMD hide the steps
// between a wave's products from each other in part only.
//
// In both, the scores are formed with the standing index in the lanes, so p
// and ds, rounded to the activation type, are operands of the accumulating
// products as they lie in their registers; those products' other operand is
// the passing tile read transposed from LDS.  The position part's gradient is
// left per head in fp32 and summed over the heads by a third kernel.
//
// fp16: p is formed times 2^12 and ds times a power of two that follows its
// magnitude (per row in dq, per wave in dk), so neither long contexts nor
// small gradients fall below fp16's range; bf16 needs neither.
//
// Where lse is past 2^16 the scaled score is rounded first here too (kFar), and what
// lse's own rounding took is subtracted as well: keys that share a row's weight at
// such scores would have all of it each otherwise.
#include <hip/hip_runtime.h>

#include "kda_launch.h"
#include "kda_mla.h"
#include "kda_mla_tile.h"

namespace kda {
namespace {

using namespace mla;

constexpr int kKeys = 32;             // keys a tile of the dq kernel

template <typename T> constexpr bool kHalf = Elem<T>::code == KDA_DTYPE_F16;
template <typename T> constexpr float kPShift = kHalf<T> ? 12.f : 0.f;

// Where a sequence's queries and keys are.
struct Place {
    int64_t b, h;
    int len, start, exist;            // tokens; position of query 0; queries that exist
    __device__ __forceinline__ Place(const kda_mla_expanded_args& a, int64_t bh) {
        b = bh / a.H;
        h = bh - b * a.H;
        len = tokens(a.lengths, b, a.S);
        start = first_position(a.starts, b, a.S, a.T);
        exist = max(0, min(static_cast<int>(a.T), len - start));
    }
};

// A power of two for values up to m, so that their products with it stay
// within 2^14: the one in use, or where that is too large one that leaves 2^6
// of room.
__device__ __forceinline__ float follow(float f, float m) {
    return m * f > 0x1p14f ? __builtin_amdgcn_ldexpf(1.f, 8 - __builtin_amdgcn_frexp_expf(m)) : f;
}
constexpr float kFirst = 0x1p60f;     // before any value

__device__ __forceinline__ float dot8(uint4 x, uint4 y, float acc, _Float16) {
    const h8 a = __builtin_bit_cast(h8, x), b = __builtin_bit_cast(h8, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = fmaf(static_cast<float>(a[i]), static_cast<float>(b[i]), acc);
    return acc;
}
__device__ __forceinline__ float dot8(uint4 x, uint4 y, float acc, bf16_t) {
    const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        acc = fmaf(__uint_as_float(a[i] << 16), __uint_as_float(b[i] << 16), acc);
        acc = fmaf(__uint_as_float(a[i] & 0xffff0000u), __uint_as_float(b[i] & 0xffff0000u), acc);
    }
    return acc;
}

template <typename T>
__device__ __forceinline__ uint4 rest8(const f16v& x, int at) {
    return uint4{rest(x[at], x[at + 1], T{}), rest(x[at + 2], x[at + 3], T{}), rest(x[at + 4], x[at + 5], T{}),
                 rest(x[at + 6], x[at + 7], T{})};
}
// FEW: p and ds go into the products with what their rounding leaves.  In variants of
// their own: the others' registers are full (dk and dv 247 -> 277 us at 4 x 2048).
// dq of 32 rows a wave, and delta.  195 us at B=4 T=2048 H=16, 128 + 64 channels,
// bf16: 700 TFLOP/s.  RW waves of rows times KW that share the keys of each (of
// a step's KW kKeys keys, wave group g takes the g-th kKeys), joined at the end.
// Four groups' tiles of 128 + 64 channels fit LDS once, and the registers do not
// hold the next ones beside the sums: those are loaded after the products.  (The
// variants of 128 rows spill 8 to 10 registers at 128 + 64 channels.)
// Grid as the forward's.
template <typename T, int N, int P, int RW, int KW, bool FEW>
__global__ __launch_bounds__(64 * RW * KW, 2) void dq_kernel(kda_mla_expanded_bwd_args g, float* delta, int qtiles) {
    const kda_mla_expanded_args& a = g.fwd;
    constexpr int kStep = KW * kKeys, kRows = 32 * RW;
    using F = KvTile<T, N, P, 64 * RW * KW, kStep, 8>;
    constexpr int D = F::D, V = F::V;
    constexpr int kBufs = N == 128 && KW == 4 ? 1 : 2;
    constexpr int kJoin = KW / 2 * RW * (D / 32) * 16 * 64 * 4, kTiles = kBufs * F::kBuf * 2;
    constexpr int kBytes = kTiles > kJoin ? kTiles : kJoin;
    __shared__ __align__(16) char raw[kBytes];
    T* smem = reinterpret_cast<T*>(raw);
    const int64_t bhs = a.B * a.H, bh = blockIdx.x % bhs;
    const Place at(a, bh);
    const int t0 = (qtiles - 1 - static_cast<int>(blockIdx.x / bhs)) * kRows;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lq = lane & 31;
    const int half = lane >> 5, row = wave % RW, group = wave / RW;
    const int t = t0 + 32 * row + lq, nq = static_cast<int>(a.T);
    const bool live = t < at.exist;
    const int limit = live ? at.start + t : -1;
    const int w0 = t0 + 32 * row;
    const int wlast = w0 < at.exist ? at.start + min(w0 + 31, at.exist - 1) : -1;
    const int wall = w0 + 32 <= at.exist ? at.start + w0 : -1;
    const int keys = t0 < at.exist ? at.start + min(t0 + kRows, at.exist) : 0;
    const float c = a.scale * kLog2E;

    f16v dq[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[i][e] = 0.f;
    float f = kHalf<T> ? kFirst : 1.f;

    if (keys > 0) {
        // a row that does not exist, or at a position below 0, takes another's data: its own is not read
        const int tc = min(max(t, -at.start), at.exist - 1);
        const T* qr = static_cast<const T*>(a.q) + at.b * a.q_stride[0] + tc * a.q_stride[1] + at.h * a.q_stride[2] +
                      8 * half;
        const T* dor = static_cast<const T*>(g.d_o) + at.b * g.d_o_stride[0] + tc * g.d_o_stride[1] +
                       at.h * g.d_o_stride[2] + 8 * half;
        // delta from o as it was before rounding: its rounding is one value for the row and would
        // move every ds of it (fp16, T=203: dq off by 3.2e-4 with it, 3.0e-4 without)
        const int64_t from = ((at.b * a.T + tc) * a.H + at.h) * V + 8 * half;
        const T* orow = static_cast<const T*>(a.o) + from;
        const T* lrow = static_cast<const T*>(a.o_low) + from;
        uint4 q[D / 16], d_o[V / 16];
#pragma unroll
        for (int k = 0; k < D / 16; ++k) q[k] = *reinterpret_cast<const uint4*>(qr + 16 * k);
        float dl = 0.f;
#pragma unroll
        for (int k = 0; k < V / 16; ++k) {
            d_o[k] = *reinterpret_cast<const uint4*>(dor + 16 * k);
            dl = dot8(d_o[k], *reinterpret_cast<const uint4*>(orow + 16 * k), dl, T{});
            dl = dot8(d_o[k], *reinterpret_cast<const uint4*>(lrow + 16 * k), dl, T{});
        }
        dl = half_sum(dl);
        if (live && half == 0 && group == 0) delta[bh * a.T + t] = dl;
        float lse = live ? a.lse[bh * a.T + t] : INFINITY;
        const bool far = __any(far_from_zero(lse));
        if (!far) lse -= kPShift<T>;

        F tile(a, at.b, at.h);
        tile.fetch(a, 0, keys);
        tile.put(smem);
        __syncthreads();
        int cur = 0;
        for (int j0 = 0; j0 < keys; j0 += kStep) {
            if constexpr (kBufs == 2) tile.fetch(a, j0 + kStep, keys);
            const int jw = j0 + kKeys * group;                    // the wave's first key
            if (jw <= wlast) {
                const T* kt = smem + cur * F::kBuf + (kKeys * group + lq) * F::kK + 8 * half;
                const T* vt = smem + cur * F::kBuf + kStep * F::kK + (kKeys * group + lq) * F::kV + 8 * half;
                f16v s, dp;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) s = Act<T>::mma32(*reinterpret_cast<const uint4*>(kt + 16 * k), q[k], s);
#pragma unroll
                for (int k = 0; k < V / 16; ++k)
                    dp = Act<T>::mma32(*reinterpret_cast<const uint4*>(vt + 16 * k), d_o[k], dp);
                if (jw + kKeys - 1 > wall) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (jw + 8 * (e / 4) + 4 * half + e % 4 > limit) s[e] = -INFINITY;
                }
                float m = 0.f, by = c, less = lse;
                if (far) {
#pragma clang fp contract(off)
                    int r = static_cast<int>(__lane_id()) & 31;
                    asm volatile("" : "+v"(r));                   // read here, for no register to be kept for it
                    const float low = a.lse_low ? a.lse_low[bh * a.T + min(w0 + r, at.exist - 1)] : 0.f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = s[e] * c - lse - low;
                    by = 1.f;
                    less = -kPShift<T>;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    dp[e] = __builtin_amdgcn_exp2f(fmaf(s[e], by, -less)) * (dp[e] - dl);
                    if constexpr (kHalf<T>) m = fmaxf(m, fabsf(dp[e]));
                }
                if constexpr (kHalf<T>) {
                    m = half_max(m);
                    if (__any(m * f > 0x1p14f)) {
                        const float now = follow(f, m), ratio = now / f;
                        f = now;
#pragma unroll
                        for (int i = 0; i < D / 32; ++i)
#pragma unroll
                            for (int e = 0; e < 16; ++e) dq[i][e] *= ratio;
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) dp[e] *= f;
                }
                const T* tr = smem + cur * F::kBuf + (kKeys * group + 4 * half + ((lane & 15) >> 2)) * F::kK +
                              16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                if constexpr (FEW) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint4 ds = rest8<T>(dp, 8 * k);
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) {
                            const uint2 x = read_tr(tr + 16 * k * F::kK + 32 * i);
                            const uint2 y = read_tr(tr + (16 * k + 8) * F::kK + 32 * i);
                            dq[i] = Act<T>::mma32(uint4{x.x, x.y, y.x, y.y}, ds, dq[i]);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint4 ds{Act<T>::pair(dp[8 * k], dp[8 * k + 1]), Act<T>::pair(dp[8 * k + 2], dp[8 * k + 3]),
                                   Act<T>::pair(dp[8 * k + 4], dp[8 * k + 5]), Act<T>::pair(dp[8 * k + 6], dp[8 * k + 7])};
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const uint2 x = read_tr(tr + 16 * k * F::kK + 32 * i);
                        const uint2 y = read_tr(tr + (16 * k + 8) * F::kK + 32 * i);
                        dq[i] = Act<T>::mma32(uint4{x.x, x.y, y.x, y.y}, ds, dq[i]);
                    }
                }
            }
            if constexpr (kBufs == 2) {
                cur ^= 1;
            } else {
                __syncthreads();
                tile.fetch(a, j0 + kStep, keys);
            }
            tile.put(smem + cur * F::kBuf);
            __syncthreads();
        }
    }
    const float norm = a.scale * __builtin_amdgcn_exp2f(-kPShift<T>) / f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[i][e] *= norm;
    // the key groups' sums, half of them onto the other half at a time
#pragma unroll
    for (int n = KW / 2; n > 0; n /= 2) {
        f4* sums = reinterpret_cast<f4*>(raw) + (group % n * RW + row) * (D / 32) * 4 * 64 + lane;
        if (group >= n && group < 2 * n) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sums[(4 * i + e) * 64] = f4{dq[i][4 * e], dq[i][4 * e + 1], dq[i][4 * e + 2], dq[i][4 * e + 3]};
        }
        __syncthreads();
        if (group < n) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f4 y = sums[(4 * i + e) * 64];
#pragma unroll
                    for (int d = 0; d < 4; ++d) dq[i][4 * e + d] += y[d];
                }
        }
        __syncthreads();
    }
    if (group != 0 || t >= nq) return;
    T* out = static_cast<T*>(g.dq) + ((at.b * a.T + t) * a.H + at.h) * D + 4 * half;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint2*>(out + 32 * i + 8 * e) =
                uint2{Act<T>::pair(dq[i][4 * e], dq[i][4 * e + 1]), Act<T>::pair(dq[i][4 * e + 2], dq[i][4 * e + 3])};
}

// dk and dv.  A workgroup has 32 KG keys, whose rows of K and V stay in LDS, and
// takes 32 (8 / KG) queries a step: eight waves, each 32 of the keys and 32 of a
// step's queries, so that a SIMD has two waves and each holds a part of the
// sums of its keys, joined at the end.  (Four waves with K and V in registers
// need more than 256 of them, and moving values between the two halves of the
// register file took most of the time: 403 us at B=4 T=2048 H=16 with 128 + 64
// channels, 273 this way, 630 TFLOP/s.)
// Grid: (key tiles, the first have the most queries) x (batch, head), the latter inner.
template <typename T, int N, int P, int KG>
struct Dkv {
    static constexpr int D = N + P, V = N, NT = 512, kSides = 8 / KG, kStand = 32 * KG, kPass = 32 * kSides;
    // LDS rows, elements: sixteen rows' pieces and, nearly, four rows of a transposed
    // read in different banks (V + 8, which is right for the former alone: 274 us, V + 24 268)
    static constexpr int kK = D + 8, kV = V + 24;
    static constexpr int kStanding = kStand * (kK + kV), kPassing = kPass * (kK + kV);
    static constexpr int kJoin = 4 * 64 * (D / 32) * 16 * 4;      // bytes: one half's dk
    static constexpr int kTiles = (kStanding + kPassing) * 2;
    static constexpr int kBytes = (kTiles > kJoin ? kTiles : kJoin);
};

template <typename T, int N, int P, int KG, bool FEW>
__global__ __launch_bounds__(512, 2) void dkv_kernel(kda_mla_expanded_bwd_args g, const float* delta, float* dpe) {
    const kda_mla_expanded_args& a = g.fwd;
    using F = Dkv<T, N, P, KG>;
    constexpr int D = F::D, V = F::V, kK = F::kK, kV = F::kV, kStand = F::kStand, kPass = F::kPass;
    // the next step's queries in flight through the products where registers hold them
    // (128 queries of 128 + 64 channels took 46 registers to scratch memory: T=1000 48 us, 32 without)
    constexpr bool kEarly = KG == 4 || N == 64;
    __shared__ __align__(16) char raw[F::kBytes];
    // lse, delta and lse's rest of a step's queries; where one of 64 has an lse far from zero, zeros are in
    // its place and it is the last
    __shared__ __align__(16) float stats[4][kPass];
    __shared__ int fars[kPass / 64];
    T* ks = reinterpret_cast<T*>(raw);
    T* vs = ks + kStand * kK;
    T* qs = vs + kStand * kV;
    T* os = qs + kPass * kK;
    const int64_t bhs = a.B * a.H, bh = blockIdx.x % bhs;
    const Place at(a, bh);
    const int j0 = static_cast<int>(blockIdx.x / bhs) * kStand;
    const int lane = threadIdx.x & 63, lk = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = wave % KG, side = wave / KG;
    const int w0 = j0 + 32 * mine, j = w0 + lk;
    const float c = a.scale * kLog2E;

    f16v dk[D / 32], dv[V / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[i][e] = 0.f;
#pragma unroll
    for (int i = 0; i < V / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) dv[i][e] = 0.f;
    float f = kHalf<T> ? kFirst : 1.f;

    // the first queries that see a key of these; those before the first key are not read
    const int first = max(max(0, j0 - at.start) / kPass * kPass, -at.start);
    if (j0 < at.len && first < at.exist) {
        const T* qb = static_cast<const T*>(a.q) + at.b * a.q_stride[0] + at.h * a.q_stride[2];
        const T* ob = static_cast<const T*>(g.d_o) + at.b * g.d_o_stride[0] + at.h * g.d_o_stride[2];
        // kPass threads on each of lse, delta and lse's rest (the others repeat them)
        const int what = wave / (kPass / 64);
        const float* sb = (what & 1 ? delta : what == 2 && a.lse_low ? a.lse_low : a.lse) + bh * a.T;
        constexpr int kP = D % 64 == 0 ? 0 : 32;                     // so that each part is whole rounds of the threads
        Rows<T, kPass, D - kP, F::NT, kK> q;
        Rows<T, kPass, kP, F::NT, kK> qp;
        Rows<T, kPass, V, F::NT, kV> d_o;
        q.start(a.q_stride[1]);
        qp.start(a.q_stride[1]);
        d_o.start(g.d_o_stride[1]);
        float x;
        // rows past the last query that exists are zeros, and their lse makes p zero
        const auto fetch = [&](int t0) {
            q.fetch(qb, a.q_stride[1], t0, at.exist);
            qp.fetch(qb + D - kP, a.q_stride[1], t0, at.exist);
            d_o.fetch(ob, g.d_o_stride[1], t0, at.exist);
            x = sb[min(t0 + static_cast<int>(threadIdx.x & (kPass - 1)), at.exist - 1)];
            issued();
        };
        const auto put = [&](int t0) {
            q.put(qs);
            qp.put(qs + D - kP);
            d_o.put(os);
            if (what < 3) {
                const int i = threadIdx.x & (kPass - 1);
                const bool there = t0 + i < at.exist;
                float y = there ? x : 0.f;
                if (what == 0) {
                    const bool far = __any(there && far_from_zero(x));
                    if (far) stats[3][i] = there ? x : INFINITY;
                    if (lane == 0) fars[wave] = far;
                    y = there ? (far ? 0.f : x) - kPShift<T> : INFINITY;
                }
                stats[what][i] = what == 2 && !a.lse_low ? 0.f : y;
            }
        };
        fetch(first);
        {
            Rows<T, kStand, N, F::NT, kK> k;
            Rows<T, kStand, P, F::NT, kK> pe;
            Rows<T, kStand, V, F::NT, kV> v;
            k.start(a.k_stride[1]);
            pe.start(a.k_pe_stride[1]);
            v.start(a.v_stride[1]);
            k.fetch(static_cast<const T*>(a.k) + at.b * a.k_stride[0] + at.h * a.k_stride[2], a.k_stride[1], j0, at.len);
            pe.fetch(static_cast<const T*>(a.k_pe) + at.b * a.k_pe_stride[0], a.k_pe_stride[1], j0, at.len);
            v.fetch(static_cast<const T*>(a.v) + at.b * a.v_stride[0] + at.h * a.v_stride[2], a.v_stride[1], j0, at.len);
            k.put(ks);
            pe.put(ks + N);
            v.put(vs);
        }
        put(first);
        __syncthreads();
        for (int t0 = first; t0 < at.exist; t0 += kPass) {
            if constexpr (kEarly) fetch(t0 + kPass);
            const int tw = t0 + 32 * side;                            // the wave's queries
            if (tw < at.exist && at.start + tw + 31 >= w0 && w0 < at.len) {
                const T* qt = qs + (32 * side + lk) * kK + 8 * half;
                const T* ot = os + (32 * side + lk) * kV + 8 * half;
                const T* kt = ks + (32 * mine + lk) * kK + 8 * half;
                const T* vt = vs + (32 * mine + lk) * kV + 8 * half;
                f16v s, dp;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    s = Act<T>::mma32(*reinterpret_cast<const uint4*>(qt + 16 * i),
                                      *reinterpret_cast<const uint4*>(kt + 16 * i), s);
#pragma unroll
                for (int i = 0; i < V / 16; ++i)
                    dp = Act<T>::mma32(*reinterpret_cast<const uint4*>(ot + 16 * i),
                                       *reinterpret_cast<const uint4*>(vt + 16 * i), dp);
                if (at.start + tw < w0 + 31 || w0 + 32 > at.len) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (at.start + tw + 8 * (e / 4) + 4 * half + e % 4 < j || j >= at.len) s[e] = -INFINITY;
                }
                float m = 0.f;
                const float* st = &stats[0][32 * side + 4 * half];
                if (__builtin_amdgcn_readfirstlane(fars[32 * side / 64])) {
#pragma clang fp contract(off)
                    // in place, for the product with c below: the common path stays as it is
                    float opaque = c;
                    asm volatile("" : "+v"(opaque));      // (and forms nothing of this ahead, in registers)
                    const float back = __builtin_amdgcn_rcpf(opaque);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float* far = st + 2 * kPass + 8 * (e / 4) + e % 4;
                        s[e] = (s[e] * opaque - far[kPass] - far[0]) * back;
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const f4 l = *reinterpret_cast<const f4*>(st + 8 * u), d = *reinterpret_cast<const f4*>(st + kPass + 8 * u);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(s[4 * u + e], c, -l[e]));
                        s[4 * u + e] = p;
                        dp[4 * u + e] = p * (dp[4 * u + e] - d[e]);
                        if constexpr (kHalf<T>) m = fmaxf(m, fabsf(dp[4 * u + e]));
                    }
                }
                if constexpr (kHalf<T>) {
                    m = wave_max(m);
                    if (m * f > 0x1p14f) {
                        const float now = follow(f, m), ratio = now / f;
                        f = now;
#pragma unroll
                        for (int i = 0; i < D / 32; ++i)
#pragma unroll
                            for (int e = 0; e < 16; ++e) dk[i][e] *= ratio;
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) dp[e] *= f;
                }
                const int trow = 32 * side + 4 * half + ((lane & 15) >> 2), tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                const T* qtr = qs + trow * kK + tcol;
                const T* otr = os + trow * kV + tcol;
                if constexpr (FEW) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint4 pf = rest8<T>(s, 8 * u), df = rest8<T>(dp, 8 * u);
#pragma unroll
                        for (int i = 0; i < V / 32; ++i) {
                            const uint2 y = read_tr(otr + 16 * u * kV + 32 * i), z = read_tr(otr + (16 * u + 8) * kV + 32 * i);
                            dv[i] = Act<T>::mma32(uint4{y.x, y.y, z.x, z.y}, pf, dv[i]);
                        }
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) {
                            const uint2 y = read_tr(qtr + 16 * u * kK + 32 * i), z = read_tr(qtr + (16 * u + 8) * kK + 32 * i);
                            dk[i] = Act<T>::mma32(uint4{y.x, y.y, z.x, z.y}, df, dk[i]);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint4 pf{Act<T>::pair(s[8 * u], s[8 * u + 1]), Act<T>::pair(s[8 * u + 2], s[8 * u + 3]),
                                   Act<T>::pair(s[8 * u + 4], s[8 * u + 5]), Act<T>::pair(s[8 * u + 6], s[8 * u + 7])};
                    const uint4 df{Act<T>::pair(dp[8 * u], dp[8 * u + 1]), Act<T>::pair(dp[8 * u + 2], dp[8 * u + 3]),
                                   Act<T>::pair(dp[8 * u + 4], dp[8 * u + 5]), Act<T>::pair(dp[8 * u + 6], dp[8 * u + 7])};
#pragma unroll
                    for (int i = 0; i < V / 32; ++i) {
                        const uint2 y = read_tr(otr + 16 * u * kV + 32 * i), z = read_tr(otr + (16 * u + 8) * kV + 32 * i);
                        dv[i] = Act<T>::mma32(uint4{y.x, y.y, z.x, z.y}, pf, dv[i]);
                    }
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const uint2 y = read_tr(qtr + 16 * u * kK + 32 * i), z = read_tr(qtr + (16 * u + 8) * kK + 32 * i);
                        dk[i] = Act<T>::mma32(uint4{y.x, y.y, z.x, z.y}, df, dk[i]);
                    }
                }
            }
            __syncthreads();
            if constexpr (!kEarly) fetch(t0 + kPass);
            put(t0 + kPass);
            __syncthreads();
        }
    }
    // the sides' sums, half of them onto the other half at a time
    const float pn = __builtin_amdgcn_exp2f(-kPShift<T>), norm = a.scale * pn / f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[i][e] *= norm;
    const auto join = [&](auto& x, int tiles, int n) {
        f4* sums = reinterpret_cast<f4*>(raw) + (side % n * KG + mine) * tiles * 4 * 64 + lane;
        if (side >= n && side < 2 * n) {
#pragma unroll
            for (int i = 0; i < tiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sums[(4 * i + e) * 64] = f4{x[i][4 * e], x[i][4 * e + 1], x[i][4 * e + 2], x[i][4 * e + 3]};
        }
        __syncthreads();
        if (side < n) {
#pragma unroll
            for (int i = 0; i < tiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f4 y = sums[(4 * i + e) * 64];
#pragma unroll
                    for (int d = 0; d < 4; ++d) x[i][4 * e + d] += y[d];
                }
        }
        __syncthreads();
    };
#pragma unroll
    for (int n = F::kSides / 2; n > 0; n /= 2) {
        join(dk, D / 32, n);
        join(dv, V / 32, n);
    }
    if (side != 0 || j >= a.S) return;
    const int64_t row = (at.b * a.S + j) * a.H + at.h;
    T* kout = static_cast<T*>(g.dk) + row * N + 4 * half;
    T* vout = static_cast<T*>(g.dv) + row * V + 4 * half;
#pragma unroll
    for (int i = 0; i < N / 32; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            *reinterpret_cast<uint2*>(kout + 32 * i + 8 * e) = uint2{Act<T>::pair(dk[i][4 * e], dk[i][4 * e + 1]),
                                                                     Act<T>::pair(dk[i][4 * e + 2], dk[i][4 * e + 3])};
            *reinterpret_cast<uint2*>(vout + 32 * i + 8 * e) =
                uint2{Act<T>::pair(dv[i][4 * e] * pn, dv[i][4 * e + 1] * pn),
                      Act<T>::pair(dv[i][4 * e + 2] * pn, dv[i][4 * e + 3] * pn)};
        }
    if constexpr (P > 0) {
        float* out = dpe + (bh * a.S + j) * P + 4 * half;
#pragma unroll
        for (int i = 0; i < P / 32; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f16v& x = dk[N / 32 + i];
                *reinterpret_cast<f4*>(out + 32 * i + 8 * e) = f4{x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]};
            }
    }
}

// The heads' position gradients summed in order: four channels a thread.
template <typename T>
__global__ __launch_bounds__(256) void dpe_kernel(const float* dpe, T* out, int64_t B, int64_t H, int64_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;     // of B n, n = S P / 4
    if (i >= B * n) return;
    const int64_t b = i / n;
    const f4* from = reinterpret_cast<const f4*>(dpe) + (b * H) * n + (i - b * n);
    f4 sum = from[0];
    for (int64_t h = 1; h < H; ++h) {
        const f4 x = from[h * n];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += x[e];
    }
    reinterpret_cast<uint2*>(out)[i] = uint2{Act<T>::pair(sum[0], sum[1]), Act<T>::pair(sum[2], sum[3])};
}

int64_t delta_bytes(int64_t B, int64_t T, int64_t H) { return (B * T * H * 4 + 15) / 16 * 16; }

template <typename T, int N, int P, int RW, int KW, bool FEW = false>
void launch_dq(const kda_mla_expanded_bwd_args& g, float* delta, hipStream_t stream) {
    const int64_t qtiles = (g.fwd.T + 32 * RW - 1) / (32 * RW);
    dq_kernel<T, N, P, RW, KW, FEW><<<static_cast<unsigned>(qtiles * g.fwd.B * g.fwd.H), 64 * RW * KW, 0, stream>>>(
        g, delta, static_cast<int>(qtiles));
}

template <typename T, int N, int P>
int launch(const kda_mla_expanded_bwd_args& g, hipStream_t stream) {
    const kda_mla_expanded_args& a = g.fwd;
    float* delta = static_cast<float*>(g.workspace);
    float* dpe = reinterpret_cast<float*>(static_cast<char*>(g.workspace) + delta_bytes(a.B, a.T, a.H));
    const int64_t bhs = a.B * a.H, ktiles = (a.S + 127) / 128;
    // Tiles of 256 query rows where that leaves every CU two (a long one alone at the
    // end takes as long as all the others); of 64, whose waves share the keys four ways,
    // where those of 128 are no more than the CUs and these no more either or long;
    // else of 128, the keys shared two ways unless they are few (a wave group's start
    // costs more than it saves).  us, 128 rows alone / shared / 64
    // rows, B=1 H=16, 128 + 64 channels: T=203 19 / 20 / 20, T=500 34 / 32 / 24, T=1000
    // 60 / 48 / 33, T=2048 109 / 86 / 73, T=2200 - / 84 / 92, T=3000 159 / 112 / 132; 64 + 32:
    // T=500 H=8 21 / - / 14, T=3000 100 / 66 / 71.  256 rows / 128 shared, T=4096: 201 / 175.
    if (a.T > 0) {
        const int64_t wide = (a.T + 255) / 256, narrow = (a.T + 127) / 128, least = (a.T + 63) / 64;
        if (few(a)) launch_dq<T, N, P, 4, 1, true>(g, delta, stream);
        else if (wide * bhs >= 512) launch_dq<T, N, P, 8, 1>(g, delta, stream);
        else if (narrow * bhs <= 256 && (least * bhs <= 256 || a.S >= 1024) && (N == 64 || a.S > 256))
            launch_dq<T, N, P, 2, 4>(g, delta, stream);
        else if (a.S < (N == 128 ? 512 : 1024)) launch_dq<T, N, P, 4, 1>(g, delta, stream);
        else launch_dq<T, N, P, 4, 2>(g, delta, stream);
    }
    if (ktiles == 0) return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
    // Likewise 64 keys a workgroup instead of 128: B=1 H=16, 128 + 64 channels T=203 20 /
    // 15 us, T=1000 48 / 32, T=2048 89 / 69, T=2500 107 / 104, T=3000 125 / 133, B=4 T=300 (two
    // rounds of short ones) 24 / 27.
    if (few(a))
        dkv_kernel<T, N, P, 2, true><<<static_cast<unsigned>((a.S + 63) / 64 * bhs), 512, 0, stream>>>(g, delta, dpe);
    else if (ktiles * bhs > 320 || ((a.S + 63) / 64 * bhs > 256 && a.S < 1024))
        dkv_kernel<T, N, P, 4, false><<<static_cast<unsigned>(ktiles * bhs), 512, 0, stream>>>(g, delta, dpe);
    else
        dkv_kernel<T, N, P, 2, false><<<static_cast<unsigned>((a.S + 63) / 64 * bhs), 512, 0, stream>>>(g, delta, dpe);
    if constexpr (P > 0) {
        const int64_t n = a.S * P / 4;
        dpe_kernel<T><<<static_cast<unsigned>((a.B * n + 255) / 256), 256, 0, stream>>>(dpe, static_cast<T*>(g.dk_pe),
                                                                                       a.B, a.H, n);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

template <typename T>
int launch_dims(const kda_mla_expanded_bwd_args& g, hipStream_t stream) {
    switch (g.fwd.N + g.fwd.P) {
        case 192: return launch<T, 128, 64>(g, stream);
        case 160: return launch<T, 128, 32>(g, stream);
        case 128: return g.fwd.N == 128 ? launch<T, 128, 0>(g, stream) : launch<T, 64, 64>(g, stream);
        case 96: return launch<T, 64, 32>(g, stream);
        default: return launch<T, 64, 0>(g, stream);
    }
}

}  // namespace

int64_t mla_expanded_bwd_workspace_bytes(int64_t B, int64_t T, int64_t S, int64_t H, int64_t P) {
    return delta_bytes(B, T, H) + B * S * H * P * 4;
}

int mla_expanded_bwd_launch(const kda_mla_expanded_bwd_args& g, hipStream_t stream) {
    return g.fwd.dtype == KDA_DTYPE_F16 ? launch_dims<_Float16>(g, stream) : launch_dims<bf16_t>(g, stream);
}

}  // namespace kda
