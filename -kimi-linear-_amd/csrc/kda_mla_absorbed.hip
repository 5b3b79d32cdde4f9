// Latent attention in its absorbed form: a few query rows a sequence against
// the cache itself, whose rows are keys and (their first R channels) values.
//
//   s_mj = scale q_m . c_j,   o_m = sum_j 2^(s'_mj - M_m) c_j[0:R] / sum_j 2^(s'_mj - M_m),
//   s' = s log2(e),  M a running maximum (in fp16 less 15).
//
// Bound by reading the cache: 16 heads of one token make 2 (2R + P) 16 flops of
// each row's 2 (R + P) bytes, 30 a byte.  So sixteen query rows (a row tile: with up
// to 16 heads, a token's) read each row once, and more fetch it again for each
// sixteen of them, whole rows at a time (the score product's operand layout, a lane a row, would
// ask for 16 cache lines an instruction: a window's loads took 6.8 k cycles to
// issue that way, 2 k this way), and goes to LDS, from where the score product
// reads it by rows and the value product transposed.
//
// A workgroup's waves each take 16 keys of a window and leave their scores
// in LDS beside the rows; then every wave forms all of the window's weights
// for itself (a few exponentials a lane) and the value product for its own
// R / WAVES channels.  So the rows' sums are never spread over waves, and there
// is nothing to merge at the end of a sequence.
//
// The keys of all sequences are shared among the workgroups in units of 16 by
// what the lengths are (a decode batch's differ), and what a workgroup has of a
// sequence that others share goes to the workspace, to be joined by a second kernel.
//
// In 8 bits a value is widened to the activation type exactly; a key's scale
// multiplies its score, and enters the value product through the exponent,
// 2^(s' + log2 scale - M), so that P keeps its full precision in 16 bits whatever
// the scales' size (in fp16 down to 2^-29 of the largest: reference).  M is then the
// largest of the sums, and the terms of the softmax's denominator are divided by the
// scale again.
//
// At 16 heads, R=512 P=64 (a copy reaches 4.8 TB/s): B=64 of 8192 tokens 115 us
// (5.2 TB/s), of 64 to 4096 tokens 40.5 us from HBM, in 8 bits 128 to 8192 43.5 us,
// with 5 us of them the join; one sequence of 32768 17.8 us, in 8 bits 15.5; of 200,
// in one workgroup, 10 us: a window is 1.5 us and the way to the first one 3.  32 heads
// of that batch 67 us, 64 121, 128 169.
#include <hip/hip_runtime.h>

#include "kda_launch.h"
#include "kda_mla.h"

namespace kda {
namespace {

using namespace mla;

constexpr int kUnit = 16;         // keys of a wave's part of a window
constexpr int kRows = 16;         // query rows of a workgroup
constexpr int WAVES = 4, kThreads = 64 * WAVES;

// Workspace: for every slot (a workgroup's part of a row tile's sequence) the
// rows' sums, [16][R] fp32, and their (maximum, denominator); for every row
// tile the first and last workgroup that has a part of it.
struct Workspace {
    float* o;
    float2* ml;
    int2* span;
};
__host__ __device__ inline int64_t slots(int64_t groups, int64_t tiles) { return groups + tiles; }
__host__ __device__ inline Workspace carve(void* p, int64_t n_slots, int64_t R) {
    Workspace w;
    w.o = static_cast<float*>(p);
    w.ml = reinterpret_cast<float2*>(w.o + n_slots * kRows * R);
    w.span = reinterpret_cast<int2*>(w.ml + n_slots * kRows);
    return w;
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));      // (arrays of uint4 may stay in scratch memory)

// Query rows m0.. as (token, head): row m0 + r, past the last repeating it.
struct Queries {
    int H, t0, h0, last;
    float inv;
    __device__ __forceinline__ Queries(const kda_mla_absorbed_args& a, int m0) {
        H = static_cast<int>(a.H);
        t0 = m0 / H;
        h0 = m0 - t0 * H;
        last = static_cast<int>(a.T) * H - 1 - m0;
        inv = __builtin_amdgcn_rcpf(static_cast<float>(H));
    }
    // h0 + r < H + 16: with 16 heads or more it passes H once at most, with
    // fewer it is below 32, which the reciprocal divides exactly
    __device__ __forceinline__ int token(int r) const {
        const int x = h0 + min(r, last);
        return t0 + (H >= kRows ? (x >= H ? 1 : 0) : static_cast<int>((static_cast<float>(x) + 0.5f) * inv));
    }
    __device__ __forceinline__ int head(int r, int t) const { return h0 + min(r, last) - (t - t0) * H; }
};

// Reads issued before this stay before it.
__device__ __forceinline__ void stay() { asm volatile("" ::: "memory"); }
// A barrier for what the waves leave each other in LDS, that does not wait for loads under way as __syncthreads does.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 64 lanes' 16 (or 4) bytes each, from base + offset bytes, on end to LDS; waited
// for by the reader (landed).  In assembly for the compiler not to wait: it takes
// a transposed LDS read for one that may be of any load's place.  (m0 is
// reserved: the compiler keeps nothing in it.)
__device__ __forceinline__ uint32_t lds_address(void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)(p)));
}
__device__ __forceinline__ void to_lds(const void* base, int offset, char* lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds_address(lds)), "v"(offset), "s"(base)
                 : "memory");
}
__device__ __forceinline__ void word_to_lds(const void* base, int offset, char* lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(lds_address(lds)), "v"(offset), "s"(base)
                 : "memory");
}
// This wave's loads into LDS are there.
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Rows go straight to LDS as they are in the cache, asynchronously: two buffers,
// the next window's rows under way while this one is worked on, none in
// registers.  LDS rows have no padding (a load fills 1 KB on end); instead the
// 16-byte piece c of row r lies at c turned by bits of r, so that sixteen rows'
// pieces (the score product's reads) and the rows of a transposed read (the value
// product's) are in different banks.  8-bit values are widened after they are
// read from LDS, by each product for itself.
template <typename T, bool F8, int R, int P>
struct Kernel {
    static constexpr int D = R + P, kWindow = kUnit * WAVES, kSteps = D / 32, kScore = kWindow + 4;
    static constexpr int kTiles = R / 16 / WAVES;               // 16-channel tiles of a wave
    static constexpr int ES = F8 ? 1 : 2, RB = R * ES, PB = P * ES;              // bytes
    static constexpr int kLatRows = 1024 / RB, kLat = kUnit / kLatRows;          // rows a load, loads a unit
    static constexpr int kPosRows = P == 0 || 1024 / PB > kUnit ? kUnit : 1024 / PB, kPos = P == 0 ? 0 : kUnit / kPosRows;
    static constexpr int kPosUnit = kPos * 1024;                // bytes of a unit's position parts (whole loads)
    static constexpr int kPosAt = kWindow * RB, kScaleAt = kPosAt + WAVES * kPosUnit;
    static constexpr int kBuffer = kScaleAt + (F8 ? WAVES * 256 : 0);
    static_assert(kBuffer >= kRows * (D + 8) * 2, "the queries pass through a buffer");

    struct Shared {
        char buf[2][kBuffer];            // [kWindow][R], [WAVES][kPosUnit], scales
        float s[kRows][kScore];
        float inv[F8 ? kWindow : 4];
    };

    // Where piece c of row r lies: of the latent, with r = r0 + x, r0 a multiple of the rows of a load and x
    // within one, and of the position part.
    static __device__ __forceinline__ int turn(int r) {
        return RB >= 256 ? ((r << 1) & 14) | ((r >> 3) & 1) : (r >> 1) & 7;
    }
    static __device__ __forceinline__ int turn(int r0, int x) { return turn(r0) ^ (RB >= 256 ? x << 1 : x >> 1); }
    static __device__ __forceinline__ int pos_piece(int r, int c) {
        return c ^ (PB == 128 ? (r >> 1) & 7 : (PB == 64 ? (r >> 2) & 3 : (r >> 3) & 1));
    }

    // A unit's rows, keys j.. of which those past hi - 1 repeat it, into their place in a buffer.
    static __device__ __forceinline__ void load(const kda_mla_absorbed_args& a, int64_t b, int j, int hi, int wave, int lane,
                                                char* buf) {
        const int base = min(j, hi - 1), last = hi - 1 - base, stride = static_cast<int>(a.cache_stride[1]) * ES;
        const char* rows = static_cast<const char*>(a.cache) + (b * a.cache_stride[0] + base * a.cache_stride[1]) * ES;
        constexpr int per = RB / 16;                             // lanes of a row
        const int x = lane / per, c = lane % per;
#pragma unroll
        for (int i = 0; i < kLat; ++i)
            to_lds(rows, min(kLatRows * i + x, last) * stride + 16 * (c ^ turn(kLatRows * i, x)),
                   buf + (kUnit * wave + kLatRows * i) * RB);
        if constexpr (P > 0) {
            constexpr int pp = PB / 16;
#pragma unroll
            for (int i = 0; i < kPos; ++i) {
                const int r = kPosRows * i + lane / pp % kPosRows;       // (lanes past the unit's rows fill the rest)
                to_lds(rows, min(r, last) * stride + RB + 16 * pos_piece(r, lane % pp),
                       buf + kPosAt + wave * kPosUnit + 1024 * i);
            }
        }
        if constexpr (F8) {
            const int r = (lane >> 1) & 15;
            word_to_lds(a.cache_scale + b * a.scale_stride[0] + base * a.scale_stride[1],
                        (min(r, last) * static_cast<int>(a.scale_stride[1]) + (lane & 1)) * 4, buf + kScaleAt + 256 * wave);
        }
    }

    struct State {
        uint4 q[kSteps];
        f4 o[kTiles];
        float top, sum;
    };
    // Channels of step k that lane group lg has: in 8 bits a 16-byte piece is two steps'.
    static __device__ __forceinline__ int channel(int k, int lg) {
        return F8 && k < R / 32 ? 64 * (k / 2) + 16 * lg + 8 * (k % 2) : 32 * k + 8 * lg;
    }

    // The scores of the wave's unit, keys 4 lg + i of row ln: times scale log2(e), plus log2 of the key's scale.
    static __device__ __forceinline__ f4 scores(const char* buf, const State& st, float c, float* inv, int wave, int ln,
                                                int lg) {
        const char* row = buf + (kUnit * wave + ln) * RB;
        const char* pos = buf + kPosAt + wave * kPosUnit + ln * PB;
        const int f = turn(ln);
        constexpr int kReads = RB / 64;
        u4 piece[kReads];                // all asked for before the first product: nothing else hides their latency
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        u4 tail[F8 || P == 0 ? 1 : P / 32];
        u2 tail8[F8 && P ? P / 32 : 1];
#pragma unroll
        for (int k = 0; k < kReads; ++k) {
            constexpr int kLow = RB >= 256 ? 4 : 2;              // reads whose pieces are turned among themselves
            piece[k] = *reinterpret_cast<const u4*>(row + 64 * kLow * (k / kLow) + 16 * ((4 * (k % kLow) + lg) ^ f));
        }
#pragma unroll
        for (int k = 0; k < P / 32; ++k) {
            if constexpr (F8) tail8[k] = *reinterpret_cast<const u2*>(pos + 16 * pos_piece(ln, 2 * k + (lg >> 1)) + 8 * (lg & 1));
            else tail[k] = *reinterpret_cast<const u4*>(pos + 16 * pos_piece(ln, 4 * k + lg));
        }
        f4 s;
        if constexpr (F8) {
            const f4* sc = reinterpret_cast<const f4*>(buf + kScaleAt + 256 * wave + 32 * lg);
            const f4 s01 = sc[0], s23 = sc[1];
            stay();
            f4 lat{}, odd{}, far{};
#pragma unroll
            for (int k = 0; k < kReads; ++k) {
                lat = Act<T>::mma16(widen8<T>(piece[k][0], piece[k][1]), st.q[2 * k], lat);
                odd = Act<T>::mma16(widen8<T>(piece[k][2], piece[k][3]), st.q[2 * k + 1], odd);
            }
#pragma unroll
            for (int k = 0; k < P / 32; ++k)
                far = Act<T>::mma16(widen8<T>(tail8[k][0], tail8[k][1]), st.q[R / 32 + k], far);
            const float sl[4] = {s01[0], s01[2], s23[0], s23[2]}, sp[4] = {s01[1], s01[3], s23[1], s23[3]};
            f4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = fmaf((lat[i] + odd[i]) * sl[i] + far[i] * sp[i], c, __builtin_amdgcn_logf(sl[i]));
                r[i] = __builtin_amdgcn_rcpf(sl[i]);
            }
            if (ln == 0) *reinterpret_cast<f4*>(inv + kUnit * wave + 4 * lg) = r;
        } else {
            stay();
            f4 acc{}, odd{};
#pragma unroll
            for (int k = 0; k < kReads; ++k) {
                const uint4 x = __builtin_bit_cast(uint4, piece[k]);
                if (k % 2 == 0) acc = Act<T>::mma16(x, st.q[k], acc);
                else odd = Act<T>::mma16(x, st.q[k], odd);
            }
#pragma unroll
            for (int k = 0; k < P / 32; ++k) acc = Act<T>::mma16(__builtin_bit_cast(uint4, tail[k]), st.q[R / 32 + k], acc);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = (acc[i] + odd[i]) * c;
        }
        return s;
    }

    // A window at keys j0..; its rows are in `buf`, the next window's are asked for into `next`.
    static __device__ __forceinline__ void window(const kda_mla_absorbed_args& a, int64_t b, int j0, int hi, int limit,
                                                  float c, int wave, int lane, const char* buf, char* next, Shared& sh,
                                                  State& st) {
        const int ln = lane & 15, lg = lane >> 4;
        if (j0 + kWindow < hi) load(a, b, j0 + kWindow + kUnit * wave, hi, wave, lane, next);
        f4 s = scores(buf, st, c, sh.inv, wave, ln, lg);
        const int key = j0 + kUnit * wave + 4 * lg;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (key + i > limit) s[i] = -INFINITY;
        *reinterpret_cast<f4*>(&sh.s[ln][kUnit * wave + 4 * lg]) = s;
        lds_barrier();

        uint4 p[kWindow / 32];
        float x[kWindow / 32][8], mx = kNoMax;
#pragma unroll
        for (int k = 0; k < kWindow / 32; ++k) {
            const f4* from = reinterpret_cast<const f4*>(&sh.s[ln][32 * k + 8 * lg]);
            const f4 lo4 = from[0], hi4 = from[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[k][e] = lo4[e];
                x[k][4 + e] = hi4[e];
                mx = fmaxf(mx, fmaxf(lo4[e], hi4[e]));
            }
        }
        mx = fmaxf(st.top, reference<T>(lanegroup4_max(mx)));
        const float alpha = __builtin_amdgcn_exp2f(st.top - mx);
        st.top = mx;
        float part = 0.f;
#pragma unroll
        for (int k = 0; k < kWindow / 32; ++k) {
            f4 inv[2];
            if constexpr (F8) {
                inv[0] = *reinterpret_cast<const f4*>(&sh.inv[32 * k + 8 * lg]);
                inv[1] = *reinterpret_cast<const f4*>(&sh.inv[32 * k + 8 * lg + 4]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[k][e] = __builtin_amdgcn_exp2f(x[k][e] - mx);
                part = F8 ? fmaf(x[k][e], inv[e / 4][e % 4], part) : part + x[k][e];
            }
            p[k] = uint4{Act<T>::pair(x[k][0], x[k][1]), Act<T>::pair(x[k][2], x[k][3]), Act<T>::pair(x[k][4], x[k][5]),
                         Act<T>::pair(x[k][6], x[k][7])};
        }
        st.sum = fmaf(st.sum, alpha, part);
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[i][e] *= alpha;
        values(buf, p, wave, ln, lg, st);
        landed();                        // the next window's
        lds_barrier();
    }

    // O^T += V^T P^T: keys 32 k + 8 lg.. of channel ln of each of the wave's tiles.
    static __device__ __forceinline__ void values(const char* buf, const uint4 (&p)[kWindow / 32], int wave, int ln, int lg,
                                                  State& st) {
        constexpr int kAtOnce = kTiles < 4 ? kTiles : 4;
        constexpr int kMask = RB >= 256 ? 15 : 7;
#pragma unroll
        for (int i0 = 0; i0 < kTiles; i0 += kAtOnce) {
            uint2 y[kAtOnce][kWindow / 32][F8 ? 1 : 2];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if constexpr (F8) {
                    // eight rows of sixteen channels: a lane points at eight channels of row ln / 2
                    const int r = 8 * lg + (ln >> 1), at = kTiles * wave + i0 + i;
                    const char* v = buf + r * RB + 16 * ((at & ~kMask) | ((at & kMask) ^ turn(r & 15))) + 8 * (ln & 1);
#pragma unroll
                    for (int k = 0; k < kWindow / 32; ++k) y[i][k][0] = read_tr8(v + 32 * k * RB);
                } else {
                    // four rows of sixteen channels, twice: a lane points at four channels of row ln / 4
                    const int at = 2 * (kTiles * wave + i0 + i) + ((ln >> 1) & 1);
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const int r = 8 * lg + 4 * n + (ln >> 2);
                        const char* v = buf + r * RB + 16 * ((at & ~kMask) | ((at & kMask) ^ turn(r & 15))) + 8 * (ln & 1);
#pragma unroll
                        for (int k = 0; k < kWindow / 32; ++k) y[i][k][n] = read_tr(v + 32 * k * RB);
                    }
                }
            }
            stay();
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                for (int k = 0; k < kWindow / 32; ++k) {
                    uint4 v;
                    if constexpr (F8) v = widen8<T>(y[i][k][0].x, y[i][k][0].y);
                    else v = uint4{y[i][k][0].x, y[i][k][0].y, y[i][k][1].x, y[i][k][1].y};
                    st.o[i0 + i] = Act<T>::mma16(v, p[k], st.o[i0 + i]);
                }
        }
    }

    // One row tile's part, keys [lo, hi), of sequence b; the whole of it if
    // `whole`, else into the workspace's slot.
    static __device__ __forceinline__ void segment(const kda_mla_absorbed_args& a, Shared& sh, int64_t b, int rt, int len,
                                                   int lo, int hi, bool whole, const Workspace& ws, int64_t slot) {
        const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int rows = static_cast<int>(a.T * a.H), m0 = rt * kRows;
        const float c = a.scale * kLog2E;
        load(a, b, lo + kUnit * wave, hi, wave, lane, sh.buf[0]);
        // the queries through the other buffer: each piece is read from memory once
        const Queries rq(a, m0);
        constexpr int kQStride = D + 8, kPieces = kRows * (D / 8), kPer = (kPieces + kThreads - 1) / kThreads;
        u4 qr[kPer];
        const T* qb = static_cast<const T*>(a.q) + b * a.q_stride[0];
        T* qs = reinterpret_cast<T*>(sh.buf[1]);
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const int i = min(static_cast<int>(threadIdx.x) + n * kThreads, kPieces - 1), r = i / (D / 8);
            const int t = rq.token(r);
            qr[n] = *reinterpret_cast<const u4*>(qb + t * a.q_stride[1] + rq.head(r, t) * a.q_stride[2] + i % (D / 8) * 8);
        }
        const int limit = min(hi - 1, len - static_cast<int>(a.T) + rq.token(ln));    // last key that the lane's row sees
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const int i = min(static_cast<int>(threadIdx.x) + n * kThreads, kPieces - 1);
            *reinterpret_cast<u4*>(qs + i / (D / 8) * kQStride + i % (D / 8) * 8) = qr[n];
        }
        __syncthreads();
        State st;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) st.q[k] = *reinterpret_cast<const uint4*>(qs + ln * kQStride + channel(k, lg));
#pragma unroll
        for (int i = 0; i < kTiles; ++i) st.o[i] = f4{0.f, 0.f, 0.f, 0.f};
        st.top = kNoMax;
        st.sum = 0.f;
        landed();
        lds_barrier();
        for (int j0 = lo; j0 < hi; j0 += 2 * kWindow) {
            window(a, b, j0, hi, limit, c, wave, lane, sh.buf[0], sh.buf[1], sh, st);
            if (j0 + kWindow < hi) window(a, b, j0 + kWindow, hi, limit, c, wave, lane, sh.buf[1], sh.buf[0], sh, st);
        }
        const float den = lanegroup4_sum(st.sum), norm = den == 0.f ? 0.f : 1.f / den;
        const int ch = 16 * kTiles * wave + 4 * lg;
        if (whole) {
            if (m0 + ln >= rows) return;
            T* out = static_cast<T*>(a.o) + (b * rows + m0 + ln) * R + ch;
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
                *reinterpret_cast<uint2*>(out + 16 * i) = uint2{Act<T>::pair(st.o[i][0] * norm, st.o[i][1] * norm),
                                                                Act<T>::pair(st.o[i][2] * norm, st.o[i][3] * norm)};
        } else {
            float* out = ws.o + (slot * kRows + ln) * R + ch;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) *reinterpret_cast<f4*>(out + 16 * i) = st.o[i];
            if (wave == 0 && lg == 0) ws.ml[slot * kRows + ln] = float2{st.top, den};
        }
    }
};

__device__ __forceinline__ int units(int len) { return (len + kUnit - 1) / kUnit; }
__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}

// Grid: a workgroup for each row tile of each sequence (`alone`), or more than
// kCut workgroups, each with its share of all units, at least kLeast.
//
// Up to kCut row tiles are cut each for itself into even parts, one a workgroup;
// of more, the shares run on from one row tile into the next, which evens them out
// but gives most workgroups two parts to start (1.3 us each) and more parts to join.
// us at 16 heads, R=512 P=64, run on / cut: 64 sequences of 64 to 4096 tokens 36.6 /
// 32.6, of 1 to 1000 23.7 / 16.8, 16 of 1900 with 4 tokens each 31 / 25, 37 of 8192
// 74 / 73; in 8 bits 64 of 64 to 4096 29 / 24, but 52 of 8192 52 / 57.  One rule for both
// widths: batches whose lengths differ gain in both.
constexpr int kLeast = 8, kCut = 64;
template <typename T, bool F8, int R, int P>
__global__ __launch_bounds__(kThreads, F8 ? 2 : 1) void absorbed_kernel(kda_mla_absorbed_args a, int rts, bool alone) {
    using K = Kernel<T, F8, R, P>;
    __shared__ __align__(16) typename K::Shared sh;
    const int lane = threadIdx.x & 63, nv = static_cast<int>(a.B) * rts, group = static_cast<int>(blockIdx.x);
    if (alone) {
        const int b = group / rts, rt = group - b * rts, len = tokens(a.lengths, b, a.S);
        if (len > 0) {
            K::segment(a, sh, b, rt, len, 0, len, true, Workspace{}, 0);
        } else {
            const int rows = static_cast<int>(a.T * a.H), m0 = rt * kRows, n = min(rows - m0, kRows) * (R / 8);
            uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + (static_cast<int64_t>(b) * rows + m0) * R);
            for (int i = threadIdx.x; i < n; i += kThreads) out[i] = uint4{0, 0, 0, 0};
        }
        return;
    }
    const Workspace ws = carve(a.workspace, slots(gridDim.x, nv), R);
    // 64 row tiles at a time, one a lane: their tokens, and where their units end in the list
    int len = 0, end = 0;
    const auto look = [&](int v0) {
        len = v0 + lane < nv ? tokens(a.lengths, (v0 + lane) / rts, a.S) : 0;
        end = wave_scan(units(len), lane);
        return __builtin_amdgcn_readlane(end, 63);
    };
    int64_t total = 0;
    for (int v0 = (nv - 1) / 64 * 64; v0 >= 0; v0 -= 64) total += look(v0);       // ends with the first 64
    if (total == 0) return;
    if (nv <= kCut && total < INT32_MAX / 2) {       // cut by row tile; every workgroup returns in here
        // The share: whole windows, so that the parts, each row tile's even, are no
        // more than the workgroups.  Rounding up adds less than one part a row tile,
        // so leaving nv workgroups out of the division always suffices; half as many
        // mostly do.
        const int n = units(len), all = static_cast<int>(total), groups = static_cast<int>(gridDim.x);
        int k = 0;
        for (int spare = nv / 2;; spare = nv) {
            const int share = max((all / (groups - spare) + WAVES) / WAVES * WAVES, kLeast);
            k = (n + share - 1) / share;
            end = wave_scan(k, lane);
            if (spare == nv || __builtin_amdgcn_readlane(end, 63) <= groups) break;
        }
        const uint64_t mine = __ballot(end - k <= group && group < end);
        if (mine == 0) return;
        const int v = __builtin_ctzll(mine), b = v / rts, size = __builtin_amdgcn_readlane(len, v);
        const int parts = __builtin_amdgcn_readlane(k, v), at = group - (__builtin_amdgcn_readlane(end, v) - parts);
        const int per = (units(size) + parts - 1) / parts, lo = at * per;
        K::segment(a, sh, b, v - b * rts, size, kUnit * lo, min(kUnit * (lo + per), size), parts == 1, ws,
                   static_cast<int64_t>(group) + v);
        if (threadIdx.x == 0) {
            if (at == 0) ws.span[v].x = group;
            if (at == parts - 1) ws.span[v].y = group;
        }
        return;
    }
    // A part is not worth its place in the workspace below kLeast units; short
    // sequences have a workgroup each.
    int64_t share;
    if (total < INT32_MAX / 2) {     // (a 64-bit division takes ten times as long)
        const int all = static_cast<int>(total), groups = static_cast<int>(gridDim.x);
        share = max((all + groups - 1) / groups, min(kLeast, (all + nv - 1) / nv));
    } else {
        share = (total + gridDim.x - 1) / gridDim.x;
    }
    const int64_t from = group * share, to = min(from + share, total);
    int64_t before = 0;              // units of the row tiles before these 64
    for (int v0 = 0; v0 < nv && before < to; v0 += 64) {
        if (v0 > 0) look(v0);
        const int n = units(len);
        const int64_t first = before + end - n;      // this lane's first unit in the list
        uint64_t todo = __ballot(n > 0 && first < to && first + n > from);
        while (todo) {
            const int i = __builtin_ctzll(todo);
            todo &= todo - 1;
            const int v = v0 + i, b = v / rts, size = __builtin_amdgcn_readlane(len, i), n = units(size);
            const int64_t at = before + __builtin_amdgcn_readlane(end, i) - n;
            const int lo = static_cast<int>(max(from - at, static_cast<int64_t>(0)));
            const int hi = static_cast<int>(min(to - at, static_cast<int64_t>(n)));
            K::segment(a, sh, b, v - b * rts, size, kUnit * lo, min(kUnit * hi, size), lo == 0 && hi == n, ws,
                       static_cast<int64_t>(group) + v);
            if (threadIdx.x == 0) {
                if (lo == 0) ws.span[v].x = group;
                if (hi == n) ws.span[v].y = group;
            }
        }
        before += __builtin_amdgcn_readlane(end, 63);
    }
}

// The parts of one row's sequence joined: grid (row tiles, their rows, R / 4 /
// LANES), LANES lanes on 4 channels each and 256 / LANES groups of them on every
// so-manieth part, whose sums meet in LDS, in an order that the lengths alone decide.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void join_kernel(kda_mla_absorbed_args a, int rts, int groups) {
    const int64_t v = blockIdx.x, b = v / rts, nv = a.B * rts;
    const int rows = static_cast<int>(a.T * a.H), m = static_cast<int>(v - b * rts) * kRows + blockIdx.y;
    if (m >= rows) return;
    constexpr int kJoinGroups = 256 / LANES;
    const int at = threadIdx.x % LANES, c = 4 * LANES * blockIdx.z + 4 * at, group = threadIdx.x / LANES;
    const Workspace ws = carve(a.workspace, slots(groups, nv), a.R);
    int2 span = ws.span[v];                      // (asked for with the length; unwritten where that is zero)
    if (tokens(a.lengths, b, a.S) == 0) span = int2{0, -1};
    if (span.x == span.y) return;                // one workgroup had it all, and wrote the result
    const float2* ml = ws.ml + v * kRows + blockIdx.y;
    const float* o = ws.o + (v * kRows + blockIdx.y) * a.R + c;
    float top = kNoMax, den = 0.f;
    f4 r{};
    // four parts' loads in flight together; one past the last counts as empty
    constexpr int kAhead = 4;
    for (int g = span.x + group; g <= span.y; g += kAhead * kJoinGroups) {
        float2 x[kAhead];
        f4 y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int at_g = min(g + i * kJoinGroups, span.y);
            x[i] = ml[at_g * kRows];
            y[i] = *reinterpret_cast<const f4*>(o + static_cast<int64_t>(at_g) * kRows * a.R);
        }
        float now = top;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (g + i * kJoinGroups > span.y) x[i] = float2{kNoMax, 0.f};
            now = fmaxf(now, x[i].x);
        }
        const float f0 = __builtin_amdgcn_exp2f(top - now);
        top = now;
        den *= f0;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] *= f0;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const float f = x[i].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x[i].x - now);
            den = fmaf(f, x[i].y, den);
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = fmaf(f, y[i][e], r[e]);
        }
    }
    __shared__ f4 sums[kJoinGroups][LANES];
    __shared__ float2 stats[kJoinGroups];
    sums[group][at] = r;
    if (at == 0) stats[group] = float2{top, den};
    __syncthreads();
    if (group != 0) return;
    const int n = min(kJoinGroups, span.y - span.x + 1);
    for (int g = 0; g < n; ++g) top = fmaxf(top, stats[g].x);
    den = 0.f;
    r = f4{};
    for (int g = 0; g < n; ++g) {
        const float w = __builtin_amdgcn_exp2f(stats[g].x - top);
        den = fmaf(w, stats[g].y, den);
        const f4 y = sums[g][at];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = fmaf(w, y[e], r[e]);
    }
    const float norm = den == 0.f ? 0.f : 1.f / den;
    *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + (b * rows + m) * a.R + c) =
        uint2{Act<T>::pair(r[0] * norm, r[1] * norm), Act<T>::pair(r[2] * norm, r[3] * norm)};
}

int row_tiles(int64_t T, int64_t H) { return static_cast<int>((T * H + kRows - 1) / kRows); }

// Workgroups of the shared form: one a CU.  Two leave twice the parts to join
// and are no faster in between; us at 16 heads, 256 / 512 workgroups: B=64 of 64
// to 4096 tokens 36.8 / 44.4, in 8 bits 29.7 / 29.6; B=16 of 8192 34.1 / 40.2, in 8
// bits 23.9 / 25.8.
constexpr int64_t kGroups = 256;
static_assert(kGroups > kCut);
// Whether the units are shared among the workgroups: where one workgroup a row
// tile would leave CUs idle or wait for the longest sequence.  us, shared /
// one a row tile, lengths spread evenly: 300 sequences up to 4096 tokens 158 /
// 183, up to 1024 46 / 44; 600 up to 1024 104 / 97, in 8 bits 71 / 57.
bool shared_form(int64_t nv, int64_t S) { return nv < 512 && S > 512; }

template <typename T, bool F8, int R, int P>
int launch(const kda_mla_absorbed_args& a, hipStream_t stream) {
    const int rts = row_tiles(a.T, a.H);
    const int64_t nv = a.B * rts;
    if (!shared_form(nv, a.S)) {
        absorbed_kernel<T, F8, R, P><<<static_cast<unsigned>(nv), kThreads, 0, stream>>>(a, rts, true);
    } else {
        constexpr int groups = static_cast<int>(kGroups);
        absorbed_kernel<T, F8, R, P><<<groups, kThreads, 0, stream>>>(a, rts, false);
        // many rows have few parts each, and few rows may have many
        const dim3 grid(static_cast<unsigned>(nv), kRows);
        if (nv >= 32)
            join_kernel<T, R / 4><<<grid, 256, 0, stream>>>(a, rts, groups);
        else
            join_kernel<T, 16><<<dim3(grid.x, grid.y, R / 64), 256, 0, stream>>>(a, rts, groups);
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
    return slots(kGroups, nv) * kRows * (R * 4 + 8) + nv * 8;
}

int mla_absorbed_launch(const kda_mla_absorbed_args& a, hipStream_t stream) {
    if (a.cache_dtype == KDA_DTYPE_E4M3)
        return a.dtype == KDA_DTYPE_F16 ? launch_rank<_Float16, true>(a, stream) : launch_rank<bf16_t, true>(a, stream);
    return a.dtype == KDA_DTYPE_F16 ? launch_rank<_Float16, false>(a, stream) : launch_rank<bf16_t, false>(a, stream);
}

}  // namespace kda
