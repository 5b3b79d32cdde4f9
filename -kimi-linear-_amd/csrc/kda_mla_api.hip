// C ABI of the latent attention: argument validation and dispatch.  Declared
// in include/kda_hip.h; as in kda_api.hip no exception crosses it and no call
// allocates, frees or synchronises.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "kda_hip.h"
#include "kda_launch.h"

namespace {

constexpr int64_t kMaxTokens = int64_t{1} << 30;      // positions are 32-bit in the kernels
constexpr int64_t kMaxGrid = INT32_MAX;

bool act(int32_t d) { return d == KDA_DTYPE_F16 || d == KDA_DTYPE_BF16; }
bool at16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// 16-byte rows of `bytes`-wide elements: base and every stride.
bool rows_ok(const void* p, const int64_t* stride, int n, int64_t bytes) {
    if (!at16(p)) return false;
    for (int i = 0; i < n; ++i)
        if (stride[i] < 0 || stride[i] * bytes % 16 != 0) return false;
    return true;
}

// Token strides whose tiles of up to 128 rows a 32-bit offset reaches.
bool near(int64_t stride) { return stride < (int64_t{1} << 23); }

// Rows of scale pairs, read and written 8 bytes at a time.  (The kernels' offsets
// from a row are unsigned.)
bool scale_rows_ok(const void* p, const int64_t (&stride)[2]) {
    return reinterpret_cast<uintptr_t>(p) % 8 == 0 && stride[0] >= 0 && stride[1] >= 0 && stride[0] % 2 == 0 &&
           stride[1] % 2 == 0;
}

bool scale_ok(float s) { return std::isfinite(s) && s > 0.f; }
bool pos_ok(int64_t P) { return P == 0 || P == 32 || P == 64; }

bool sizes_ok(int64_t B, int64_t T, int64_t S, int64_t H) {
    return B >= 0 && T >= 0 && S >= 0 && H >= 0 && T <= kMaxTokens && S <= kMaxTokens && B <= kMaxGrid && H <= kMaxGrid;
}

// 16 bits a channel as the activations, or 8 or 4.
bool cache_type(int32_t d, int32_t act_dtype) { return d == act_dtype || d == KDA_DTYPE_E4M3 || d == KDA_DTYPE_E2M1; }
bool scaled(int32_t d) { return d == KDA_DTYPE_E4M3 || d == KDA_DTYPE_E2M1; }
// A cache row's width in the units of its strides: elements, or of a 4-bit cache bytes.
int64_t width(int32_t d, int64_t D) { return d == KDA_DTYPE_E2M1 ? D / 2 : D; }
// Its scales' rows: 4 bits, eight bytes with byte strides.
bool scales_ok(int32_t d, const void* p, const int64_t (&stride)[2]) {
    if (d != KDA_DTYPE_E2M1) return scale_rows_ok(p, stride);
    return reinterpret_cast<uintptr_t>(p) % 8 == 0 && stride[0] >= 0 && stride[1] >= 0 && stride[0] % 8 == 0 && stride[1] % 8 == 0;
}

// [n0, n1] rows of `width` elements of which no two share any, by strides that nest.
bool distinct(const int64_t (&stride)[2], int64_t n0, int64_t n1, int64_t width) {
    const int64_t s0 = n0 > 1 ? stride[0] : 0, s1 = n1 > 1 ? stride[1] : 0;
    const bool rows = (n0 <= 1 || s0 >= width) && (n1 <= 1 || s1 >= width);
    return rows && (n0 <= 1 || n1 <= 1 || s0 - width >= (n1 - 1) * s1 || s1 - width >= (n0 - 1) * s0);
}

// [p, p + bytes) of two arrays.
bool apart(const void* a, int64_t na, const void* b, int64_t nb) {
    const auto a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    return a0 + static_cast<uintptr_t>(na) <= b0 || b0 + static_cast<uintptr_t>(nb) <= a0;
}

int expanded_check(const kda_mla_expanded_args& a) {
    if (!sizes_ok(a.B, a.T, a.S, a.H) || a.T + a.S > INT32_MAX) return KDA_ERR_BAD_SHAPE;
    if (!act(a.dtype)) return KDA_ERR_BAD_DTYPE;
    if ((a.N != 64 && a.N != 128) || a.V != a.N || !pos_ok(a.P) || !scale_ok(a.scale)) return KDA_ERR_UNSUPPORTED;
    if (a.B * a.H > kMaxGrid) return KDA_ERR_BAD_SHAPE;
    if (a.B * a.H * ((a.T > a.S ? a.T : a.S) / 64 + 1) > kMaxGrid) return KDA_ERR_BAD_SHAPE;
    if (a.B == 0 || a.H == 0) return KDA_OK;
    if (a.T > 0 && (!a.q || !a.o)) return KDA_ERR_NULL_POINTER;
    if (a.S > 0 && (!a.k || !a.v || (a.P > 0 && !a.k_pe))) return KDA_ERR_NULL_POINTER;
    if (!rows_ok(a.q, a.q_stride, 3, 2) || !rows_ok(a.k, a.k_stride, 3, 2) || !rows_ok(a.v, a.v_stride, 3, 2) ||
        (a.P > 0 && !rows_ok(a.k_pe, a.k_pe_stride, 2, 2)) || !at16(a.o) ||
        !at16(a.o_low) || !near(a.q_stride[1]) || !near(a.k_stride[1]) || !near(a.v_stride[1]) || (a.P > 0 && !near(a.k_pe_stride[1])))
        return KDA_ERR_UNSUPPORTED;
    return KDA_OK;
}

}  // namespace

extern "C" {

size_t kda_mla_expanded_workspace_size(int64_t B, int64_t T, int64_t S, int64_t H, int64_t V) {
    if (!sizes_ok(B, T, S, H) || (V != 64 && V != 128)) return 0;
    return static_cast<size_t>(kda::mla_expanded_workspace_bytes(B, T, S, H, V));
}

int kda_mla_expanded_fwd(const kda_mla_expanded_args* a, void* stream) {
    if (a == nullptr) return KDA_ERR_NULL_POINTER;
    if (const int st = expanded_check(*a); st != KDA_OK) return st;
    if (a->B == 0 || a->H == 0 || a->T == 0) return KDA_OK;
    if (!a->workspace && kda::mla_expanded_workspace_bytes(a->B, a->T, a->S, a->H, a->V) > 0) return KDA_ERR_NULL_POINTER;
    if (!at16(a->workspace)) return KDA_ERR_UNSUPPORTED;
    return kda::mla_expanded_launch(*a, static_cast<hipStream_t>(stream));
}

size_t kda_mla_expanded_bwd_workspace_size(int64_t B, int64_t T, int64_t S, int64_t H, int64_t P) {
    if (!sizes_ok(B, T, S, H) || !pos_ok(P)) return 0;
    return static_cast<size_t>(kda::mla_expanded_bwd_workspace_bytes(B, T, S, H, P));
}

int kda_mla_expanded_bwd(const kda_mla_expanded_bwd_args* g, void* stream) {
    if (g == nullptr) return KDA_ERR_NULL_POINTER;
    const kda_mla_expanded_args& a = g->fwd;
    if (const int st = expanded_check(a); st != KDA_OK) return st;
    if (a.B == 0 || a.H == 0) return KDA_OK;
    if (a.T > 0 && (!a.lse || !a.o_low || !g->d_o || !g->dq)) return KDA_ERR_NULL_POINTER;
    if (a.S > 0 && (!g->dk || !g->dv || (a.P > 0 && !g->dk_pe))) return KDA_ERR_NULL_POINTER;
    if (!g->workspace && kda::mla_expanded_bwd_workspace_bytes(a.B, a.T, a.S, a.H, a.P) > 0) return KDA_ERR_NULL_POINTER;
    if (!rows_ok(g->d_o, g->d_o_stride, 3, 2) || !near(g->d_o_stride[1]) || !at16(g->dq) || !at16(g->dk) || !at16(g->dk_pe) || !at16(g->dv) ||
        !at16(g->workspace))
        return KDA_ERR_UNSUPPORTED;
    return kda::mla_expanded_bwd_launch(*g, static_cast<hipStream_t>(stream));
}

size_t kda_mla_absorbed_workspace_size(int64_t B, int64_t T, int64_t H, int64_t S, int64_t R) {
    if (!sizes_ok(B, T, S, H) || (R != 128 && R != 256 && R != 512)) return 0;
    return static_cast<size_t>(kda::mla_absorbed_workspace_bytes(B, T, H, S, R, KDA_DTYPE_E2M1));
}

size_t kda_mla_absorbed_cache_workspace_size(int64_t B, int64_t T, int64_t H, int64_t S, int64_t R, int32_t cache_dtype) {
    if (!sizes_ok(B, T, S, H) || (R != 128 && R != 256 && R != 512) || !(act(cache_dtype) || scaled(cache_dtype))) return 0;
    return static_cast<size_t>(kda::mla_absorbed_workspace_bytes(B, T, H, S, R, cache_dtype));
}

int kda_mla_absorbed_fwd(const kda_mla_absorbed_args* a, void* stream) {
    if (a == nullptr) return KDA_ERR_NULL_POINTER;
    if (!sizes_ok(a->B, a->T, a->S, a->H)) return KDA_ERR_BAD_SHAPE;
    if (!act(a->dtype) || !cache_type(a->cache_dtype, a->dtype)) return KDA_ERR_BAD_DTYPE;
    if ((a->R != 128 && a->R != 256 && a->R != 512) || !pos_ok(a->P) || !scale_ok(a->scale)) return KDA_ERR_UNSUPPORTED;
    if (a->H > 0 && a->T > kMaxGrid / 16 / a->H) return KDA_ERR_BAD_SHAPE;
    if (a->B * ((a->T * a->H + 15) / 16) > kMaxGrid) return KDA_ERR_BAD_SHAPE;
    if (a->B == 0 || a->H == 0 || a->T == 0) return KDA_OK;
    const bool few = scaled(a->cache_dtype);
    if (!a->q || !a->o || !a->lengths) return KDA_ERR_NULL_POINTER;
    if (a->S > 0 && (!a->cache || (few && !a->cache_scale))) return KDA_ERR_NULL_POINTER;
    if (!a->workspace && kda::mla_absorbed_workspace_bytes(a->B, a->T, a->H, a->S, a->R, a->cache_dtype) > 0) return KDA_ERR_NULL_POINTER;
    if (!rows_ok(a->q, a->q_stride, 3, 2) || !rows_ok(a->cache, a->cache_stride, 2, few ? 1 : 2) || !at16(a->o) ||
        !at16(a->workspace) || !near(a->cache_stride[1]))
        return KDA_ERR_UNSUPPORTED;
    if (few && (!scales_ok(a->cache_dtype, a->cache_scale, a->scale_stride) || !near(a->scale_stride[1])))
        return KDA_ERR_UNSUPPORTED;
    return kda::mla_absorbed_launch(*a, static_cast<hipStream_t>(stream));
}

int kda_mla_cache_append(const kda_mla_append_args* a, void* stream) {
    if (a == nullptr) return KDA_ERR_NULL_POINTER;
    if (!sizes_ok(a->B, a->T, a->S, 1) || (a->T > 0 && a->B > kMaxGrid / a->T)) return KDA_ERR_BAD_SHAPE;
    if (!act(a->x_dtype) || !cache_type(a->cache_dtype, a->x_dtype)) return KDA_ERR_BAD_DTYPE;
    if (a->norm_f32 != 0 && a->norm_f32 != 1) return KDA_ERR_BAD_DTYPE;
    if ((a->R != 128 && a->R != 256 && a->R != 512) || !pos_ok(a->P)) return KDA_ERR_UNSUPPORTED;
    if (a->B == 0 || a->T == 0 || a->S == 0) return KDA_OK;
    const bool few = scaled(a->cache_dtype);
    if (!a->x || !a->cache || !a->lengths || (few && !a->cache_scale)) return KDA_ERR_NULL_POINTER;
    if (!rows_ok(a->x, a->x_stride, 2, 2) || !rows_ok(a->cache, a->cache_stride, 2, few ? 1 : 2) || !at16(a->norm_weight))
        return KDA_ERR_UNSUPPORTED;
    // distinct rows of the cache, so that no two waves write one
    if (!distinct(a->cache_stride, a->B, a->S, width(a->cache_dtype, a->R + a->P))) return KDA_ERR_UNSUPPORTED;
    if (few && (!scales_ok(a->cache_dtype, a->cache_scale, a->scale_stride) ||
                !distinct(a->scale_stride, a->B, a->S, a->cache_dtype == KDA_DTYPE_E2M1 ? 8 : 2)))
        return KDA_ERR_UNSUPPORTED;
    return kda::mla_append_launch(*a, static_cast<hipStream_t>(stream));
}

int kda_mla_cache_read(const kda_mla_read_args* a, void* stream) {
    if (a == nullptr) return KDA_ERR_NULL_POINTER;
    if (!sizes_ok(a->B, 0, a->S, 1) || a->B * (a->S / 7 + 1) > kMaxGrid) return KDA_ERR_BAD_SHAPE;
    if (!act(a->out_dtype) || (a->cache_dtype != 0 && !scaled(a->cache_dtype))) return KDA_ERR_BAD_DTYPE;
    if ((a->R != 128 && a->R != 256 && a->R != 512) || !pos_ok(a->P)) return KDA_ERR_UNSUPPORTED;
    if (a->B == 0 || a->S == 0) return KDA_OK;
    if (!a->cache || !a->cache_scale || !a->out) return KDA_ERR_NULL_POINTER;
    if (!rows_ok(a->cache, a->cache_stride, 2, 1) || !at16(a->out) || !scales_ok(a->cache_dtype, a->cache_scale, a->scale_stride))
        return KDA_ERR_UNSUPPORTED;
    const int64_t D = a->R + a->P;
    if (!apart(a->out, a->B * a->S * D * 2, a->cache,
               (a->B - 1) * a->cache_stride[0] + (a->S - 1) * a->cache_stride[1] + width(a->cache_dtype, D)))
        return KDA_ERR_ALIAS;
    return kda::mla_read_launch(*a, static_cast<hipStream_t>(stream));
}

}  // extern "C"
