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
// largest of those sums.  The denominator knows no scales, which may lie 2^187 apart: a lane
// sums 2^s' of the keys whose scores it forms, and a segment ends with its output, 2^M / denominator
// times what was summed.  Where a row's largest score D is far from zero, fp32 holds no such sums
// and a score no scale's exponent beside it: then the segment is gone over again with scores less D.
//
// In 4 bits (e2m1) each 128 channels have a power of two.  The score product's pieces
// are 32 channels of a key, so a scale is one operand of the conversion that widens them (in fp16,
// which holds fewer powers, it multiplies the group's products instead).  In the value product a
// wave's channels are of one group, so as in 8 bits the scale enters through the exponent, each
// wave for its own: a wave has its own maximum M.  A transposed read gives a lane sixteen
// keys of a channel, the window's quarter of its lane group.  The arithmetic, and not the bytes, is most of a window: 386 vector
// operations before the scales went into the conversions, sums were rescaled only where there is a new
// maximum, load offsets became constants and masks were only applied where there is one, about 290 after.
//
// At 16 heads, R=512 P=64 (a copy reaches 4.8 TB/s): B=64 of 8192 tokens 115 us
// (5.2 TB/s), of 64 to 4096 tokens 40.6 us from HBM, in 8 bits 128 to 8192 43.8 us,
// with 5 us of them the join; one sequence of 32768 17.8 us, in 8 bits 15.5; of 200,
// in one workgroup, 10 us: a window is 1.5 us and the way to the first one 3.  32 heads
// of that batch 67 us, 64 121, 128 169.  In 4 bits B=64 of 8192 tokens 48 us, of 128 to 8192
// 33, one of 65536 20, of 200 8.7.
#include <hip/hip_runtime.h>

#include "kda_launch.h"
#include "kda_mla.h"

namespace kda {
namespace {

using namespace mla;

constexpr int kUnit = 16;         // keys of a wave's part of a window
constexpr int kRows = 16;         // query rows of a workgroup
constexpr int kGroup = 128;       // latent channels of a 4-bit cache's scale
constexpr int WAVES = 4, kThreads = 64 * WAVES;

// Workspace: for every slot (a workgroup's part of a row tile's sequence) the
// rows' sums, [16][R] fp32, and their (maximum, denominator), in 8 and 4 bits the rows' outputs in
// place of the sums, times kOutRoom and kDenRoom; for every row tile the first and last workgroup that has a part of it.
struct Workspace {
    float* o;
    float2* ml;
    int2* span;
};
// A row's output is below 2^130 and its denominator, against its largest score, at most 2^30: with this off both, no sum of
// their products overflows.
constexpr float kOutRoom = 0x1p-4f, kDenRoom = 0x1p-30f;
// Rows whose largest score is further from zero count from that: 2^96 2^30 is still a number, and what ends below
// 2^-126 is 2^-30 of the largest.
constexpr float kAway = 96.f;
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

// Rows go straight to LDS as they are in the cache, asynchronously: two buffers,
// the next window's rows under way while this one is worked on, none in
// registers.  LDS rows have no padding (a load fills 1 KB on end); instead the
// 16-byte piece c of row r lies at c turned by bits of r, so that sixteen rows'
// pieces (the score product's reads) and the rows of a transposed read (the value
// product's) are in different banks.  8-bit values are widened after they are
// read from LDS, by each product for itself.
template <typename T, int BITS, int R, int P>
struct Kernel {
    static constexpr bool F8 = BITS == 8, F4 = BITS == 4;
    static constexpr bool kApart = BITS < 16;                   // the denominator apart from the scales
    static constexpr int D = R + P, kWindow = kUnit * WAVES, kSteps = D / 32, kScore = kWindow + 4;
    static constexpr int kTiles = R / 16 / WAVES;               // 16-channel tiles of a wave
    static constexpr int ES = BITS == 16 ? 2 : 1, RB = R * BITS / 8, PB = P * BITS / 8;   // bytes (of a stride's unit, a row)
    static constexpr int kScales = F4 ? R / kGroup : 1;         // scales of a row's latent part
    // bf16 holds every value times its scale: the conversion of a 4-bit row's values takes it in.
    static constexpr bool kWide = Elem<T>::code == KDA_DTYPE_BF16;
    static constexpr int kLatRows = 1024 / RB, kLat = kUnit / kLatRows;          // rows a load, loads a unit
    static constexpr int kPosRows = P == 0 || 1024 / PB > kUnit ? kUnit : 1024 / PB, kPos = P == 0 ? 0 : kUnit / kPosRows;
    static constexpr int kPosUnit = kPos * 1024;                // bytes of a unit's position parts (whole loads)
    static constexpr int kPosAt = kWindow * RB, kScaleAt = kPosAt + WAVES * kPosUnit;
    static constexpr int kBuffer = kScaleAt + (BITS < 16 ? WAVES * 256 : 0);
    static_assert(kBuffer >= kRows * (D + 8) * 2, "the queries pass through a buffer");

    struct Shared {
        char buf[2][kBuffer];            // [kWindow][R], [WAVES][kPosUnit], scales
        float s[kRows][kScore];
        float e[kApart ? kScales : 1][kApart ? kWindow : 4];     // log2 of the scales
        float2 den[kApart ? WAVES : 1][kRows];                   // each wave's keys: largest score, and their sum
    };

    // Where piece c of row r lies: of the latent, with r = r0 + x, r0 a multiple of the rows of a load and x
    // within one, and of the position part.
    static __device__ __forceinline__ int turn(int r) {
        return RB >= 256 ? ((r << 1) & 14) | ((r >> 3) & 1) : (RB == 128 ? (r >> 1) & 7 : (r >> 2) & 3);
    }
    static __device__ __forceinline__ int turn(int r0, int x) {
        return turn(r0) ^ (RB >= 256 ? x << 1 : (RB == 128 ? x >> 1 : x >> 2));
    }
    static __device__ __forceinline__ int pos_piece(int r, int c) {
        return PB < 32 ? c : c ^ (PB == 128 ? (r >> 1) & 7 : (PB == 64 ? (r >> 2) & 3 : (r >> 3) & 1));
    }

    // Offsets of what a lane loads of a 4-bit unit's rows: the same for every unit whose rows all exist.
    struct Offsets {
        int lat[F4 ? kLat : 1], pos, scale;
    };
    static __device__ __forceinline__ Offsets offsets(const kda_mla_absorbed_args& a, int lane) {
        Offsets o{};
        if constexpr (F4) {
            const int stride = static_cast<int>(a.cache_stride[1]), x = lane / (RB / 16), c = lane % (RB / 16);
#pragma unroll
            for (int i = 0; i < kLat; ++i) o.lat[i] = (kLatRows * i + x) * stride + 16 * (c ^ turn(kLatRows * i, x));
            if constexpr (P > 0) {
                const int r = lane / (PB / 16) % kUnit;
                o.pos = r * stride + RB + 16 * pos_piece(r, lane % (PB / 16));
            }
            o.scale = ((lane >> 1) & 15) * static_cast<int>(a.scale_stride[1]) + 4 * (lane & 1);
        }
        return o;
    }
    static __device__ __forceinline__ void load_whole(const kda_mla_absorbed_args& a, int64_t b, int j, int wave, const Offsets& o,
                                                      char* buf) {
        const char* rows = static_cast<const char*>(a.cache) + (b * a.cache_stride[0] + j * a.cache_stride[1]);
        const char* scales = static_cast<const char*>(a.cache_scale) + (b * a.scale_stride[0] + j * a.scale_stride[1]);
#pragma unroll
        for (int i = 0; i < kLat; ++i) to_lds(rows, o.lat[i], buf + (kUnit * wave + kLatRows * i) * RB);
        if constexpr (P > 0) to_lds(rows, o.pos, buf + kPosAt + wave * kPosUnit);
        word_to_lds(scales, o.scale, buf + kScaleAt + 256 * wave);
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
            word_to_lds(static_cast<const float*>(a.cache_scale) + b * a.scale_stride[0] + base * a.scale_stride[1],
                        (min(r, last) * static_cast<int>(a.scale_stride[1]) + (lane & 1)) * 4, buf + kScaleAt + 256 * wave);
        }
        if constexpr (F4) {
            const int r = (lane >> 1) & 15;
            word_to_lds(static_cast<const uint8_t*>(a.cache_scale) + b * a.scale_stride[0] + base * a.scale_stride[1],
                        min(r, last) * static_cast<int>(a.scale_stride[1]) + 4 * (lane & 1), buf + kScaleAt + 256 * wave);
        }
    }

    struct State {
        uint4 q[kSteps];
        f4 o[kTiles];
        float top, sum;
        float most, from;        // apart: the largest score less what they count from, 0 or D
    };
    // Channels of step k that lane group lg has: in 8 bits a 16-byte piece is two steps', in 4 bits four steps'.
    static __device__ __forceinline__ int channel(int k, int lg) {
        if constexpr (F4) return k < R / 32 ? 128 * (k / 4) + 32 * lg + 8 * (k % 4) : 32 * k + 8 * lg;
        return F8 && k < R / 32 ? 64 * (k / 2) + 16 * lg + 8 * (k % 2) : 32 * k + 8 * lg;
    }

    // A scale of a 4-bit cache, byte i of a row's word: NaN's code gives infinity.
    static __device__ __forceinline__ float power(uint32_t w, int i) {
        return __uint_as_float((w >> (8 * i) & 255u) << 23);
    }

    // The scores of the wave's unit, keys 4 lg + i of row ln: times scale log2(e).
    static __device__ __forceinline__ f4 scores(const char* buf, const State& st, float c, Shared& sh, int wave, int ln,
                                                int lg) {
        const char* row = buf + (kUnit * wave + ln) * RB;
        const char* pos = buf + kPosAt + wave * kPosUnit + ln * PB;
        const int f = turn(ln);
        constexpr int kReads = RB / 64;
        u4 piece[kReads];                // all asked for before the first product: nothing else hides their latency
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        u4 tail[BITS < 16 || P == 0 ? 1 : P / 32];
        u2 tail8[F8 && P ? P / 32 : 1];
        uint32_t tail4[F4 && P ? P / 32 : 1];
#pragma unroll
        for (int k = 0; k < kReads; ++k) {
            constexpr int kLow = RB >= 256 ? 4 : RB / 64;        // reads whose pieces are turned among themselves
            piece[k] = *reinterpret_cast<const u4*>(row + 64 * kLow * (k / kLow) + 16 * ((4 * (k % kLow) + lg) ^ f));
        }
#pragma unroll
        for (int k = 0; k < P / 32; ++k) {
            if constexpr (F4) tail4[k] = *reinterpret_cast<const uint32_t*>(pos + 16 * pos_piece(ln, k) + 4 * lg);
            else if constexpr (F8) tail8[k] = *reinterpret_cast<const u2*>(pos + 16 * pos_piece(ln, 2 * k + (lg >> 1)) + 8 * (lg & 1));
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
            f4 e;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = ((lat[i] + odd[i]) * sl[i] + far[i] * sp[i]) * c;
                e[i] = __builtin_amdgcn_logf(sl[i]);
            }
            if (ln == 0) *reinterpret_cast<f4*>(&sh.e[0][kUnit * wave + 4 * lg]) = e;
        } else if constexpr (F4) {
            // a piece is one key's 32 channels, so four products on end are of one group
            const uint2 own = *reinterpret_cast<const uint2*>(buf + kScaleAt + 256 * wave + 8 * ln);    // key ln's scales
            u4 w01{}, w23{};
            if constexpr (!kWide) {
                w01 = *reinterpret_cast<const u4*>(buf + kScaleAt + 256 * wave + 32 * lg);              // keys 4 lg + i's
                w23 = *reinterpret_cast<const u4*>(buf + kScaleAt + 256 * wave + 32 * lg + 16);
            }
            const int byte = static_cast<int>(own.x >> (8 * (lg < kScales ? lg : 0)) & 255u);
            stay();
            f4 lat[kReads], far{};
#pragma unroll
            for (int k = 0; k < kReads; ++k) lat[k] = f4{};
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int k = 0; k < kReads; ++k)
                    lat[k] = Act<T>::mma16(widen4<T>(piece[k][n], kWide ? power(own.x, k) : 1.f), st.q[4 * k + n], lat[k]);
#pragma unroll
            for (int k = 0; k < P / 32; ++k)
                far = Act<T>::mma16(widen4<T>(tail4[k], kWide ? power(kScales == 4 ? own.y : own.x, kScales % 4) : 1.f),
                                    st.q[R / 32 + k], far);
            if constexpr (kWide) {               // (a scale's NaN has made its key's products NaN)
#pragma unroll
                for (int k = 0; k < kReads; ++k) far += lat[k];
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = far[i] * c;
            } else {
                const uint32_t w[4][2] = {{w01[0], w01[1]}, {w01[2], w01[3]}, {w23[0], w23[1]}, {w23[2], w23[3]}};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = P > 0 ? far[i] * power(w[i][kScales / 4], kScales % 4) : 0.f;
#pragma unroll
                    for (int k = 0; k < kReads; ++k) x = fmaf(lat[k][i], power(w[i][0], k), x);
                    x *= c;
                    s[i] = fmaf(x, 0.f, x);      // an infinity is a scale's NaN
                }
            }
            if (lg < kScales) sh.e[lg][kUnit * wave + ln] = byte == 255 ? __builtin_nanf("") : static_cast<float>(byte - 127);
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

    // First of the eight keys of a window that lane group lg has in step k of the value product.
    static __device__ __forceinline__ int at(int k, int lg) { return F4 ? 16 * lg + 8 * k : 32 * k + 8 * lg; }

    static __device__ __forceinline__ void rescale(State& st, float alpha) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[i][e] *= alpha;
    }

    // What the lane's own scores add to the denominator.
    static __device__ __forceinline__ void count(State& st, const f4& s) {
        st.most = fmaxf(st.most, fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
#pragma unroll
        for (int i = 0; i < 4; ++i) st.sum += __builtin_amdgcn_exp2f(s[i]);
    }

    // A window's scores plus log2 of the scales of the wave's channels, and the largest of a lane's.
    static __device__ __forceinline__ float scaled(const Shared& sh, int wave, int ln, int lg,
                                                   float (&x)[kWindow / 32][8]) {
        float mx = kNoMax;
#pragma unroll
        for (int k = 0; k < kWindow / 32; ++k) {
            const f4* from = reinterpret_cast<const f4*>(&sh.s[ln][at(k, lg)]);
            const f4* more = reinterpret_cast<const f4*>(&sh.e[kScales * wave / WAVES][at(k, lg)]);
            const f4 s[2] = {from[0], from[1]}, e[2] = {more[0], more[1]};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[k][i] = s[i / 4][i % 4] + e[i / 4][i % 4];
                mx = fmaxf(mx, x[k][i]);
            }
        }
        return mx;
    }

    // A window at keys j0..; its rows are in `buf`, the next window's are asked for into `next`.
    static __device__ __forceinline__ void window(const kda_mla_absorbed_args& a, int64_t b, int j0, int hi, int limit,
                                                  float c, int wave, int lane, const Offsets& offs, const char* buf, char* next,
                                                  Shared& sh, State& st) {
        const int ln = lane & 15, lg = lane >> 4;
        if (j0 + kWindow < hi) {
            const int j = j0 + kWindow + kUnit * wave;
            if (F4 && j + kUnit <= hi) load_whole(a, b, j, wave, offs, next);
            else load(a, b, j, hi, wave, lane, next);
        }
        f4 s = scores(buf, st, c, sh, wave, ln, lg);
        const int key = j0 + kUnit * wave + 4 * lg;
        if (!F4 || __any(key + 3 > limit)) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (key + i > limit) s[i] = -INFINITY;
        }
        if constexpr (kApart) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] -= st.from;
        }
        *reinterpret_cast<f4*>(&sh.s[ln][kUnit * wave + 4 * lg]) = s;
        lds_barrier();

        uint4 p[kWindow / 32];
        float x[kWindow / 32][8], mx = kNoMax;
        if constexpr (kApart) {
            count(st, s);
        } else {
#pragma unroll
            for (int k = 0; k < kWindow / 32; ++k) {
                const f4* from = reinterpret_cast<const f4*>(&sh.s[ln][at(k, lg)]);
                const f4 lo4 = from[0], hi4 = from[1];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[k][e] = lo4[e];
                    x[k][4 + e] = hi4[e];
                    mx = fmaxf(mx, fmaxf(lo4[e], hi4[e]));
                }
            }
        }
        float alpha = 1.f;
        if constexpr (kApart) {
            // Later windows mostly hold no new maximum, and leave the sums as they are.  (In bf16 the maximum might lag
            // by 2^8 as well, but a largest weight of 1 has no rounding, and where it is most of the softmax that
            // shows: 64 sequences of up to 8192 tokens 1.8e-3 off, with the lag 2.1e-3, in the same time.)  In 8 bits, where
            // a window has less to do beside, the question costs what it saves: 600 of up to 1024 44.5 us with it, 43.3.
            mx = reference<T>(lanegroup4_max(scaled(sh, wave, ln, lg, x)));
            if (F8 || __any(mx > st.top)) {
                mx = fmaxf(st.top, mx);
                rescale(st, __builtin_amdgcn_exp2f(st.top - mx));
                st.top = mx;
            }
            mx = st.top;
        } else {
            mx = fmaxf(st.top, reference<T>(lanegroup4_max(mx)));
            alpha = __builtin_amdgcn_exp2f(st.top - mx);
            st.top = mx;
        }
        float part = 0.f;
#pragma unroll
        for (int k = 0; k < kWindow / 32; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[k][e] = __builtin_amdgcn_exp2f(x[k][e] - mx);
                if constexpr (!kApart) part += x[k][e];
            }
            p[k] = uint4{Act<T>::pair(x[k][0], x[k][1]), Act<T>::pair(x[k][2], x[k][3]), Act<T>::pair(x[k][4], x[k][5]),
                         Act<T>::pair(x[k][6], x[k][7])};
        }
        if constexpr (!kApart) {
            st.sum = fmaf(st.sum, alpha, part);
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[i][e] *= alpha;
        }
        values(buf, p, wave, ln, lg, st);
        landed<0>();                        // the next window's
        lds_barrier();
    }

    // O^T += V^T P^T: keys 32 k + 8 lg.. of channel ln of each of the wave's tiles.
    static __device__ __forceinline__ void values(const char* buf, const uint4 (&p)[kWindow / 32], int wave, int ln, int lg,
                                                  State& st) {
        constexpr int kAtOnce = kTiles < 4 ? kTiles : 4;
        constexpr int kMask = RB >= 256 ? 15 : RB / 16 - 1;
        static_assert(!F4 || kWindow == 64, "a 4-bit transposed read gives a lane group a quarter of the window");
#pragma unroll
        for (int i0 = 0; i0 < kTiles; i0 += kAtOnce) {
            uint2 y[kAtOnce][F4 ? 1 : kWindow / 32][F8 || F4 ? 1 : 2];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if constexpr (F4) {
                    // sixteen rows of sixteen channels, all of the lane group's keys: a lane points at row ln's
                    const int tile = kTiles * wave + i0 + i, c = tile >> 1;
                    y[i][0][0] = read_tr4(buf + (16 * lg + ln) * RB + 16 * ((c & ~kMask) | ((c & kMask) ^ turn(ln))) +
                                          8 * (tile & 1));
                } else if constexpr (F8) {
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
                    if constexpr (F4) v = widen4<T>(k == 0 ? y[i][0][0].x : y[i][0][0].y);
                    else if constexpr (F8) v = widen8<T>(y[i][k][0].x, y[i][k][0].y);
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
        const Offsets offs = offsets(a, lane);
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
        st.from = 0.f;
        float den, norm;
        for (bool again = false;; again = true) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i) st.o[i] = f4{0.f, 0.f, 0.f, 0.f};
            st.top = st.most = kNoMax;
            st.sum = 0.f;
            landed<0>();
            lds_barrier();
            for (int j0 = lo; j0 < hi; j0 += 2 * kWindow) {
                window(a, b, j0, hi, limit, c, wave, lane, offs, sh.buf[0], sh.buf[1], sh, st);
                if (j0 + kWindow < hi)
                    window(a, b, j0 + kWindow, hi, limit, c, wave, lane, offs, sh.buf[1], sh.buf[0], sh, st);
            }
            if constexpr (kApart) {
                const float most = lanegroup4_max(st.most), sum = lanegroup4_sum(st.sum);
                if (lg == 0) sh.den[wave][ln] = float2{most, sum};
                lds_barrier();
                float all = kNoMax;
                den = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float2 part = sh.den[w][ln];
                    all = fmaxf(all, part.x);
                    den += part.y;
                }
                if (!again && __any(fabsf(all) > kAway && all > kNoMax)) {       // the same in every wave
                    st.from = fabsf(all) > kAway ? all : 0.f;
                    // (unknown to be the first load's: its addresses would be kept for this, in 14 registers more than there are)
                    int first = lo, own = lane;
                    asm volatile("" : "+v"(first), "+v"(own));
                    load(a, b, __builtin_amdgcn_readfirstlane(first) + kUnit * wave, hi, wave, own, sh.buf[0]);
                    continue;
                }
                const bool none = all == kNoMax;
                den = none ? 0.f : den * __builtin_amdgcn_exp2f(-all);           // against the largest score
                norm = none ? 0.f : (whole ? 1.f : kOutRoom) * __builtin_amdgcn_exp2f(st.top - all) / den;
                st.top = none ? kNoMax : st.from + all;
                den *= kDenRoom;
            } else {
                den = lanegroup4_sum(st.sum);
                norm = den == 0.f ? 0.f : 1.f / den;
            }
            break;
        }
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
            for (int i = 0; i < kTiles; ++i) {
                if constexpr (kApart) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.o[i][e] *= norm;
                }
                *reinterpret_cast<f4*>(out + 16 * i) = st.o[i];
            }
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
template <typename T, int BITS, int R, int P>
__global__ __launch_bounds__(kThreads, BITS < 16 ? 2 : 1) void absorbed_kernel(kda_mla_absorbed_args a, int rts, bool alone) {
    using K = Kernel<T, BITS, R, P>;
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
// APART: the parts are outputs, to be weighted with their denominators.
template <typename T, int LANES, bool APART>
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
            float f = x[i].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x[i].x - now);
            den = fmaf(f, x[i].y, den);
            if constexpr (APART) f *= x[i].y;
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
    const float norm = den == 0.f ? 0.f : (APART ? 1.f / kOutRoom : 1.f) / den;
    *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + (b * rows + m) * a.R + c) =
        uint2{Act<T>::pair(r[0] * norm, r[1] * norm), Act<T>::pair(r[2] * norm, r[3] * norm)};
}

int row_tiles(int64_t T, int64_t H) { return static_cast<int>((T * H + kRows - 1) / kRows); }

// Workgroups of the shared form: one a CU.  Two leave twice the parts to join
// and are no faster in between; us at 16 heads, 256 / 512 workgroups: B=64 of 64
// to 4096 tokens 36.8 / 44.4, in 8 bits 29.7 / 29.6; B=16 of 8192 34.1 / 40.2, in 8
// bits 23.9 / 25.8.  In 4 bits a window is mostly arithmetic, which two workgroups hide for each
// other where there are four windows for each: 64 of 128 to 8192 36.2 / 35.0, 200 of 10 to 2000
// 59.5 / 47.6, 16 of 8192 at 64 heads 34.7 / 32.3, but 64 of 16 to 1024 15.7 / 17.4, one of 65536 20.3 / 23.7.
constexpr int64_t kGroups = 256;
static_assert(kGroups > kCut);
int64_t most_groups(int64_t nv, int64_t S, bool four) {
    return four && nv * ((S + 63) / 64) >= 8 * kGroups ? 2 * kGroups : kGroups;
}
// Whether the units are shared among the workgroups: where one workgroup a row
// tile would leave CUs idle or wait for the longest sequence.  us, shared /
// one a row tile, lengths spread evenly: 300 sequences up to 4096 tokens 158 /
// 183, up to 1024 46 / 44; 600 up to 1024 104 / 97, in 8 bits 71 / 57.
bool shared_form(int64_t nv, int64_t S) { return nv < 512 && S > 512; }

template <typename T, int BITS, int R, int P>
int launch(const kda_mla_absorbed_args& a, hipStream_t stream) {
    const int rts = row_tiles(a.T, a.H);
    const int64_t nv = a.B * rts;
    if (!shared_form(nv, a.S)) {
        absorbed_kernel<T, BITS, R, P><<<static_cast<unsigned>(nv), kThreads, 0, stream>>>(a, rts, true);
    } else {
        const int groups = static_cast<int>(most_groups(nv, a.S, BITS == 4));
        absorbed_kernel<T, BITS, R, P><<<groups, kThreads, 0, stream>>>(a, rts, false);
        // many rows have few parts each, and few rows may have many
        const dim3 grid(static_cast<unsigned>(nv), kRows);
        constexpr bool apart = Kernel<T, BITS, R, P>::kApart;
        if (nv >= 32)
            join_kernel<T, R / 4, apart><<<grid, 256, 0, stream>>>(a, rts, groups);
        else
            join_kernel<T, 16, apart><<<dim3(grid.x, grid.y, R / 64), 256, 0, stream>>>(a, rts, groups);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

template <typename T, int BITS, int R>
int launch_pos(const kda_mla_absorbed_args& a, hipStream_t stream) {
    switch (a.P) {
        case 64: return launch<T, BITS, R, 64>(a, stream);
        case 32: return launch<T, BITS, R, 32>(a, stream);
        default: return launch<T, BITS, R, 0>(a, stream);
    }
}
template <typename T, int BITS>
int launch_rank(const kda_mla_absorbed_args& a, hipStream_t stream) {
    switch (a.R) {
        case 512: return launch_pos<T, BITS, 512>(a, stream);
        case 256: return launch_pos<T, BITS, 256>(a, stream);
        default: return launch_pos<T, BITS, 128>(a, stream);
    }
}

}  // namespace

int64_t mla_absorbed_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t S, int64_t R, int32_t cache_dtype) {
    const int64_t nv = B * row_tiles(T, H);
    if (nv == 0 || !shared_form(nv, S)) return 0;
    return slots(most_groups(nv, S, cache_dtype == KDA_DTYPE_E2M1), nv) * kRows * (R * 4 + 8) + nv * 8;
}

int mla_absorbed_launch(const kda_mla_absorbed_args& a, hipStream_t stream) {
    const bool half = a.dtype == KDA_DTYPE_F16;
    switch (a.cache_dtype) {
        case KDA_DTYPE_E2M1: return half ? launch_rank<_Float16, 4>(a, stream) : launch_rank<bf16_t, 4>(a, stream);
        case KDA_DTYPE_E4M3: return half ? launch_rank<_Float16, 8>(a, stream) : launch_rank<bf16_t, 8>(a, stream);
        default: return half ? launch_rank<_Float16, 16>(a, stream) : launch_rank<bf16_t, 16>(a, stream);
    }
}

}  // namespace kda
