// capi.hip -- the extern "C" boundary (include/lcml_fp8.h): argument
// validation, kernel selection and error reporting.  No entry point
// synchronises the host or allocates device memory.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <atomic>

#include "../../include/lcml_fp8.h"
#include "kv_cache.hpp"
#include "lcml_internal.hpp"

namespace {

thread_local char g_err[512] = "";
// names of the kernels launched on this thread since the last
// lcml_fp8_kernel_trace() call, comma separated (truncated when full)
thread_local char g_trace[1024] = "";
thread_local char g_trace_out[1024] = "";
thread_local size_t g_trace_len = 0;

void note(const char *label) {
    const size_t n = strlen(label), sep = g_trace_len ? 2 : 0;
    if (g_trace_len + sep + n + 1 > sizeof(g_trace)) return;
    if (sep) memcpy(g_trace + g_trace_len, ", ", 2);
    memcpy(g_trace + g_trace_len + sep, label, n + 1);
    g_trace_len += sep + n;
}

int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

// a launch's status; on success the launch is noted in the kernel trace
// under `label` (the entry point's name when none is given)
int hip_status(hipError_t err, const char *what, const char *label = nullptr) {
    if (err == hipSuccess) {
        note(label ? label : what);
        return LCML_OK;
    }
    return fail(LCML_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
}

bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool float_or_bf16(int dtype) { return dtype == LCML_DTYPE_FLOAT || dtype == LCML_DTYPE_BFLOAT16; }
bool elem_aligned(const void *p, int dtype) { return aligned(p, dtype == LCML_DTYPE_BFLOAT16 ? 2 : 4); }

int check_view(int64_t outer, int64_t axis_len, int64_t inner, const char *fn) {
    if (outer < 0 || axis_len < 1 || inner < 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: invalid view [outer=%lld, axis_len=%lld, inner=%lld]", fn,
                    (long long)outer, (long long)axis_len, (long long)inner);
    return LCML_OK;
}

// Shared validation of the GEMM epilogue arguments.
int make_epilogue(lcml::Epilogue &e, const char *fn, int64_t M, int64_t N, const float *a_scale,
                  const float *b_scale, int per_channel, float alpha, const float *c, int c_ndim,
                  int64_t c0, int64_t c1, float beta, int act, void *y, int y_dtype, int64_t ldy,
                  bool scales_optional = false) {
    if (!b_scale && !scales_optional) return fail(LCML_ERR_INVALID_ARG, "%s: b_scale is NULL", fn);
    if (!y && M > 0 && N > 0) return fail(LCML_ERR_INVALID_ARG, "%s: y is NULL", fn);
    if (y_dtype != LCML_DTYPE_FLOAT && y_dtype != LCML_DTYPE_BFLOAT16)
        return fail(LCML_ERR_UNSUPPORTED, "%s: output dtype %d (FLOAT=1 or BFLOAT16=16 supported)", fn, y_dtype);
    if (ldy < N) return fail(LCML_ERR_INVALID_ARG, "%s: ldy=%lld < N=%lld", fn, (long long)ldy, (long long)N);
    if (act < LCML_ACT_NONE || act > LCML_ACT_GELU_TANH)
        return fail(LCML_ERR_UNSUPPORTED, "%s: activation %d", fn, act);
    const bool has_c = c != nullptr && beta != 0.0f;
    if (has_c) {
        if (c_ndim < 0 || c_ndim > 2) return fail(LCML_ERR_INVALID_ARG, "%s: C ndim %d", fn, c_ndim);
        if (c_ndim == 1 && !(c0 == 1 || c0 == N || c0 == M))
            return fail(LCML_ERR_INVALID_ARG, "%s: 1-D C of length %lld broadcasts to neither N nor M", fn,
                        (long long)c0);
        if (c_ndim == 2 && (!(c0 == 1 || c0 == M) || !(c1 == 1 || c1 == N)))
            return fail(LCML_ERR_INVALID_ARG, "%s: C shape [%lld, %lld] does not broadcast to [%lld, %lld]",
                        fn, (long long)c0, (long long)c1, (long long)M, (long long)N);
    }
    e.a_scale = a_scale;
    e.b_scale = b_scale;
    e.b_per_channel = per_channel ? 1 : 0;
    e.alpha = alpha;
    e.c = has_c ? c : nullptr;
    e.c_ndim = c_ndim;
    e.c0 = c0;
    e.c1 = c1;
    e.beta = beta;
    e.act = act;
    e.y = y;
    e.y_bf16 = y_dtype == LCML_DTYPE_BFLOAT16;
    e.ldy = ldy;
    e.M = M;
    e.N = N;
    e.amax_part = nullptr;
    return LCML_OK;
}

}  // namespace

extern "C" {

const char *lcml_fp8_last_error(void) { return g_err; }

const char *lcml_fp8_kernel_trace(void) {
    memcpy(g_trace_out, g_trace, g_trace_len + 1);
    g_trace[0] = 0;
    g_trace_len = 0;
    return g_trace_out;
}

int lcml_fp8_abi_version(void) { return LCML_FP8_ABI_VERSION; }

int lcml_fp8_quantize(const float *x, uint8_t *y, int64_t outer, int64_t axis_len, int64_t inner,
                      const float *y_scale, void *stream) {
    if (int rc = check_view(outer, axis_len, inner, "lcml_fp8_quantize")) return rc;
    if (outer * axis_len * inner == 0) return LCML_OK;
    if (!x || !y || !y_scale) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_quantize: NULL pointer");
    const char *label = nullptr;
    const hipError_t err = lcml::launch_quantize(x, y, outer, axis_len, inner, y_scale, (hipStream_t)stream, &label);
    return hip_status(err, "lcml_fp8_quantize", label);
}

int lcml_fp8_dequantize(const uint8_t *x, float *y, int64_t outer, int64_t axis_len, int64_t inner,
                        const float *x_scale, void *stream) {
    if (int rc = check_view(outer, axis_len, inner, "lcml_fp8_dequantize")) return rc;
    if (outer * axis_len * inner == 0) return LCML_OK;
    if (!x || !y || !x_scale) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_dequantize: NULL pointer");
    const char *label = nullptr;
    const hipError_t err = lcml::launch_dequantize(x, y, outer, axis_len, inner, x_scale, (hipStream_t)stream, &label);
    return hip_status(err, "lcml_fp8_dequantize", label);
}

int lcml_fp8_quantize_dynamic(const float *x, uint8_t *y, int64_t n, float *scale_out, void *workspace,
                              void *stream) {
    if (n < 0) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_quantize_dynamic: n < 0");
    if (!scale_out) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_quantize_dynamic: scale_out is NULL");
    if (n > 0 && (!x || !y)) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_quantize_dynamic: NULL pointer");
    if (n > LCML_FP8_DYNAMIC_SMALL_MAX && !workspace)
        return fail(LCML_ERR_INVALID_ARG,
                    "lcml_fp8_quantize_dynamic: n=%lld needs a workspace of %d bytes", (long long)n,
                    LCML_FP8_DYNAMIC_WORKSPACE_BYTES);
    const char *label = nullptr;
    const hipError_t err = lcml::launch_quantize_dynamic(x, y, n, scale_out, static_cast<uint32_t *>(workspace),
                                                         (hipStream_t)stream, &label);
    return hip_status(err, "lcml_fp8_quantize_dynamic", label);
}

int lcml_fp8_amax(const float *x, int64_t n, float *amax_out, void *stream) {
    if (n < 0 || !amax_out || (n > 0 && !x)) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_amax: bad argument");
    // The amax word is amax_out itself (fp32 bits of a non-negative float).
    hipStream_t s = (hipStream_t)stream;
    uint32_t *word = reinterpret_cast<uint32_t *>(amax_out);
    hipError_t err = lcml::launch_fill_u32(word, 0u, 1, s);
    if (err == hipSuccess && n > 0) err = lcml::launch_amax(x, n, word, s);
    return hip_status(err, "lcml_fp8_amax");
}

int64_t lcml_fp8_packed_weight_bytes(int64_t K, int64_t N) {
    if (K <= 0 || N <= 0) return 0;
    return lcml::pad_to(K, lcml::kPackK) * lcml::pad_to(N, lcml::kPanelCols);
}

int lcml_fp8_pack_weight(const uint8_t *w, int64_t K, int64_t N, int w_is_nk, uint8_t *packed,
                         void *stream) {
    if (K <= 0 || N <= 0 || !w || !packed)
        return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_pack_weight: bad argument (K=%lld N=%lld)", (long long)K,
                    (long long)N);
    if (!aligned(packed, 16)) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_pack_weight: packed not 16-byte aligned");
    return hip_status(lcml::launch_pack_weight(w, K, N, w_is_nk, packed, (hipStream_t)stream),
                      "lcml_fp8_pack_weight");
}

int lcml_fp8_unpack_weight(const uint8_t *packed, int64_t K, int64_t N, int w_is_nk, uint8_t *w,
                           void *stream) {
    if (K <= 0 || N <= 0 || !w || !packed)
        return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_unpack_weight: bad argument");
    if (!aligned(packed, 16)) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_unpack_weight: packed not 16-byte aligned");
    return hip_status(lcml::launch_unpack_weight(packed, K, N, w_is_nk, w, (hipStream_t)stream),
                      "lcml_fp8_unpack_weight");
}

namespace {
// AUTO's kernel for an M x N x K GEMM.  All times grow about linearly in K;
// in units of one skinny workgroup with 4 row blocks (19 us at K = 4096,
// 38 us at K = 11008), measured on 4096x11008, 11008x4096 and 4096x4096:
//   * 256x256 tiles: one round of up to 256 tiles takes 4.5 units;
//   * 128x128 tiles: 2.2 units per 256 tiles (two workgroups share a CU);
//   * the skinny kernel: lcml::skinny_row_blocks.
// M <= 16 always takes the skinny kernel; a 256x256 grid of at least 256
// tiles keeps the 256x256 kernel.  Examples: 4096x11008 at M = 512: 128x128
// tiles 64 us against 83 (skinny) and 93 (256x256); 4096x4096 at M = 1024:
// 46 us against 66 and 91; 11008x4096 at M = 512: skinny 73 us against 91.
// the native-FP8 kernel of the same tiling (LCML_KERNEL_AUTO_FP8)
int fp8_twin(int kernel) {
    switch (kernel) {
    case LCML_KERNEL_MFMA: return LCML_KERNEL_MFMA_FP8;
    case LCML_KERNEL_MFMA_128: return LCML_KERNEL_MFMA_128_FP8;
    case LCML_KERNEL_SKINNY: return LCML_KERNEL_SKINNY_FP8;
    default: return kernel;
    }
}

// the kernel trace's name of a resolved GEMM kernel choice
const char *kernel_label(int kernel) {
    switch (kernel) {
    case LCML_KERNEL_MFMA: return "gemm_mfma_256";
    case LCML_KERNEL_MFMA_FP8: return "gemm_mfma_256_fp8";
    case LCML_KERNEL_MFMA_128: return "gemm_mfma_128";
    case LCML_KERNEL_MFMA_128_FP8: return "gemm_mfma_128_fp8";
    case LCML_KERNEL_SKINNY: return "gemm_skinny";
    case LCML_KERNEL_SKINNY_FP8: return "gemm_skinny_fp8";
    case LCML_KERNEL_VALU: return "gemv_valu";
    default: return "gemm";
    }
}

// AUTO's kernel and its modelled time in those units
struct AutoChoice {
    int kernel;
    double units;
};
AutoChoice auto_gemm_choice(int64_t M, int64_t N, int64_t K) {
    if (M <= 16) return {LCML_KERNEL_SKINNY, 0.0};
    const int64_t tiles = (M + 255) / 256 * ((N + 255) / 256);
    if (tiles >= 256) return {LCML_KERNEL_MFMA, 4.5 * (double)tiles / 256.0};
    double skinny = 0;
    lcml::skinny_row_blocks(M, N, K, &skinny);
    const double t128 = (double)((M + 127) / 128 * ((N + 127) / 128));
    const double small = 2.2 * (t128 > 256 ? t128 / 256 : 1.0);
    if (skinny <= small && skinny < 4.5) return {LCML_KERNEL_SKINNY, skinny};
    return small < 4.5 ? AutoChoice{LCML_KERNEL_MFMA_128, small} : AutoChoice{LCML_KERNEL_MFMA, 4.5};
}

int auto_gemm_kernel(int64_t M, int64_t N, int64_t K) { return auto_gemm_choice(M, N, K).kernel; }

// Whether AUTO's dynamically quantised linear of M > 16 rows takes the codes
// in 16-row blocks and the kernel that reads them: where the row-major choice
// is the small-M kernel, whose sums that kernel's equal bit for bit (the tiles
// sum K in one chain, and a linear in one call equals its two calls), and its
// modelled time is a seventh below (19 us a unit at K = 4096, 3 us besides).
// N = 12288, K = 4096, with the quantiser: M = 100 31.7 us row-major against
// 28.1.  Up to 65536 elements of x the row-major codes take one launch where
// these take two (unless x's partial maxima are given): 0.6 us on the
// modelled times (N = 8192, K = 512, M = 32 8.9 us row-major against 9.9).
// Up to 32 rows of 128 panels or more take 32 x 64 tiles and need a long K, in us
// with the quantisers, row-major / these: N = 8192, M = 17 K = 2048 11.3 / 12.0,
// 3072 13.0 / 13.2, 4096 16.4 / 14.9; N = 9216 11.3 / 12.0, 13.7 / 14.1, 16.6 / 14.9.
bool dynamic_by_rows(int64_t M, int64_t N, int64_t K, bool x_parts) {
    const AutoChoice c = auto_gemm_choice(M, N, K);
    const double launch = M * K <= LCML_FP8_DYNAMIC_SMALL_MAX && !x_parts ? 0.6 : 0.0;
    return M > 16 && c.kernel == LCML_KERNEL_SKINNY && !(M <= 32 && N > 127 * 64 && K < 3584) &&
           lcml::gemm_rows_us(M, N, K) + launch < 0.86 * (c.units * 19.0 * (double)K / 4096.0 + 3.0);
}
}  // namespace

namespace {
// Amax partials of y (optional, y_amax_part non-null): the caller checked
// y is fp32, dense (ldy == N) and the buffer holds lcml_fp8_amax_parts_max
// words; *y_amax_npart receives the count written.
struct YAmax {
    uint32_t *part = nullptr;
    int *npart = nullptr;
};

// lcml_fp8_gemm with an optional amax-partials output
int gemm_core(const char *fn, int64_t M, int64_t N, int64_t K, const uint8_t *a, int64_t lda, const float *a_scale,
              const uint8_t *b_packed, const float *b_scale, int b_scale_per_channel, float alpha, const float *c,
              int c_ndim, int64_t c_dim0, int64_t c_dim1, float beta, int act, void *y, int y_dtype, int64_t ldy,
              int kernel, void *stream, YAmax ya) {
    if (M < 0 || N <= 0 || K <= 0) return fail(LCML_ERR_INVALID_ARG, "%s: M=%lld N=%lld K=%lld", fn,
                                               (long long)M, (long long)N, (long long)K);
    lcml::Epilogue e;
    if (int rc = make_epilogue(e, fn, M, N, a_scale, b_scale, b_scale_per_channel, alpha, c, c_ndim, c_dim0,
                               c_dim1, beta, act, y, y_dtype, ldy))
        return rc;
    if (M == 0) {
        if (ya.npart) *ya.npart = 0;
        return LCML_OK;
    }
    if (!a || !b_packed) return fail(LCML_ERR_INVALID_ARG, "%s: NULL operand", fn);
    if (K % 16 != 0) return fail(LCML_ERR_UNSUPPORTED, "%s: K=%lld is not a multiple of 16", fn, (long long)K);
    if (lda < K || lda % 16 != 0 || !aligned(a, 16))
        return fail(LCML_ERR_INVALID_ARG, "%s: a must be 16-byte aligned with lda >= K, lda %% 16 == 0", fn);
    if (!aligned(b_packed, 16)) return fail(LCML_ERR_INVALID_ARG, "%s: b_packed not 16-byte aligned", fn);
    hipStream_t s = (hipStream_t)stream;
    if (kernel == LCML_KERNEL_AUTO) kernel = auto_gemm_kernel(M, N, K);
    if (kernel == LCML_KERNEL_AUTO_FP8) kernel = fp8_twin(auto_gemm_kernel(M, N, K));
    hipError_t err;
    const char *label = kernel_label(kernel);
    switch (kernel) {
    case LCML_KERNEL_MFMA:
    case LCML_KERNEL_MFMA_FP8:
    case LCML_KERNEL_MFMA_128:
    case LCML_KERNEL_MFMA_128_FP8:
        // buffer offsets are 32-bit with 0x80000000 as the out-of-range marker
        if ((M - 1) * lda + K >= (int64_t)0x80000000 || lcml_fp8_packed_weight_bytes(K, N) >= (int64_t)0x80000000)
            return fail(LCML_ERR_UNSUPPORTED, "%s: operand larger than 2 GiB for the MFMA kernel", fn);
        if ((M + 127) / 128 * ((N + 127) / 128) >= (int64_t)0x80000000)
            return fail(LCML_ERR_UNSUPPORTED, "%s: M=%lld N=%lld exceeds the tile grid", fn, (long long)M, (long long)N);
        if (ya.part) {  // the tile kernels write one partial per workgroup
            e.amax_part = ya.part;
            *ya.npart = (int)lcml::gemm_mfma_workgroups(
                M, N, kernel == LCML_KERNEL_MFMA_128 || kernel == LCML_KERNEL_MFMA_128_FP8);
        }
        err = lcml::launch_gemm_mfma(M, N, K, a, lda, b_packed, e,
                                     kernel == LCML_KERNEL_MFMA || kernel == LCML_KERNEL_MFMA_128, s,
                                     kernel == LCML_KERNEL_MFMA_128 || kernel == LCML_KERNEL_MFMA_128_FP8);
        if (ya.part) label = kernel == LCML_KERNEL_MFMA_128 || kernel == LCML_KERNEL_MFMA_128_FP8
                                 ? (kernel == LCML_KERNEL_MFMA_128 ? "gemm_mfma_128_amax" : "gemm_mfma_128_fp8_amax")
                                 : (kernel == LCML_KERNEL_MFMA ? "gemm_mfma_256_amax" : "gemm_mfma_256_fp8_amax");
        ya.part = nullptr;  // written
        break;
    case LCML_KERNEL_SKINNY:
    case LCML_KERNEL_SKINNY_FP8:
        // buffer extents are 32-bit: the activations and one weight panel
        if ((M - 1) * lda + K >= (int64_t)0x80000000 || lcml::pad_to(K, lcml::kPackK) * 64 >= (int64_t)0x80000000)
            return fail(LCML_ERR_UNSUPPORTED, "%s: operand larger than 2 GiB for the skinny kernel", fn);
        if ((M + 63) / 64 * ((N + 63) / 64) >= (int64_t)0x80000000)
            return fail(LCML_ERR_UNSUPPORTED, "%s: M=%lld N=%lld exceeds the skinny kernel's grid", fn, (long long)M,
                        (long long)N);
        err = lcml::launch_gemm_skinny(M, N, K, a, lda, b_packed, e, kernel == LCML_KERNEL_SKINNY, s);
        if (M <= 16 && lcml::skinny_col_blocks(N, K, false) < 4)
            label = kernel == LCML_KERNEL_SKINNY ? "gemm_skinny_part" : "gemm_skinny_part_fp8";
        break;
    case LCML_KERNEL_VALU: err = lcml::launch_gemv_valu_fp8(M, N, K, a, lda, b_packed, e, s); break;
    default: return fail(LCML_ERR_INVALID_ARG, "%s: unknown kernel %d", fn, kernel);
    }
    if (int rc = hip_status(err, fn, label)) return rc;
    if (ya.part)  // kernels without the epilogue partials: an amax pass over y
        return hip_status(lcml::launch_amax_partials(static_cast<const float *>(y), M * N, ya.part, ya.npart, s),
                          fn, "amax_partials");
    return LCML_OK;
}
}  // namespace

int lcml_fp8_gemm(int64_t M, int64_t N, int64_t K, const uint8_t *a, int64_t lda, const float *a_scale,
                  const uint8_t *b_packed, const float *b_scale, int b_scale_per_channel, float alpha,
                  const float *c, int c_ndim, int64_t c_dim0, int64_t c_dim1, float beta, int act, void *y,
                  int y_dtype, int64_t ldy, int kernel, void *stream) {
    return gemm_core("lcml_fp8_gemm", M, N, K, a, lda, a_scale, b_packed, b_scale, b_scale_per_channel, alpha, c,
                     c_ndim, c_dim0, c_dim1, beta, act, y, y_dtype, ldy, kernel, stream, YAmax{});
}

int64_t lcml_fp8_amax_parts_max(int64_t M, int64_t N) {
    if (M <= 0 || N <= 0) return 0;
    const int64_t tiles = lcml::gemm_mfma_workgroups(M, N, true);  // 128x128 tiles: the most workgroups
    const int64_t pass = lcml::amax_partials_count(M * N);
    return tiles > pass ? tiles : pass;
}

namespace {
// The fused kernel applies when the quantised activations fit its LDS copy.
// Every workgroup of it reads and encodes all M*K activations; on the
// 4096x11008 linear that redundant pass beats the separate quantise launch
// up to M = 4 (13.9 us against 15.6 us; at M = 8 it loses, 18.6 against
// 16 us), so AUTO fuses while M*K <= 16384.
constexpr int64_t kAutoFuseMaxElems = 16384;
bool dynamic_fusable(int64_t M, int64_t K, const float *x, int64_t ldx, int kernel) {
    const bool fits = M <= 16 && lcml::skinny_dynamic_lds_bytes(M, K) <= lcml::kSkinnyDynLdsMax &&
                      (!x || aligned(x, 16)) && ldx % 4 == 0 && ((M - 1) * ldx + K) * 4 < (int64_t)0x80000000;
    if (kernel == LCML_KERNEL_AUTO || kernel == LCML_KERNEL_AUTO_FP8) return fits && M * K <= kAutoFuseMaxElems;
    return fits && (kernel == LCML_KERNEL_SKINNY || kernel == LCML_KERNEL_SKINNY_FP8);
}
int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }
static_assert(LCML_FP8_DYNAMIC_WORKSPACE_BYTES >= lcml::kMaxAmaxPartials * 4, "workspace holds the partial maxima");
// quantised activations, the partial maxima, the scale (when not returned)
int64_t two_step_workspace_bytes(int64_t M, int64_t K) { return pad256(M * K) + LCML_FP8_DYNAMIC_WORKSPACE_BYTES + 256; }
}  // namespace

int64_t lcml_fp8_gemm_dynamic_workspace_bytes(int64_t M, int64_t K, int kernel) {
    if (M <= 0 || K <= 0) return 0;
    if (dynamic_fusable(M, K, nullptr, K, kernel)) return 0;
    return two_step_workspace_bytes(M, K);
}

}  // extern "C"

namespace {
// lcml_fp8_gemm_dynamic with the workspace resolved by the caller: the
// caller's buffer, or the no-allocation entry point's device array.
// x partial maxima given (x_amax_part, x_amax_npart > 0): the two-step path
// encodes from them instead of an amax pass over x (the fused small-M
// kernel computes the same maximum itself)
struct XAmax {
    const uint32_t *part = nullptr;
    int npart = 0;
};

int gemm_dynamic_impl(const char *fn, int64_t M, int64_t N, int64_t K, const float *x, int64_t ldx,
                      const uint8_t *b_packed, const float *b_scale, int b_scale_per_channel, float alpha,
                      const float *c, int c_ndim, int64_t c_dim0, int64_t c_dim1, float beta, int act, void *y,
                      int y_dtype, int64_t ldy, float *x_scale_out, void *workspace, int64_t workspace_bytes,
                      int kernel, void *stream, XAmax xa = XAmax{}, YAmax ya = YAmax{}) {
    if (M < 0 || N <= 0 || K <= 0) return fail(LCML_ERR_INVALID_ARG, "%s: M=%lld N=%lld K=%lld", fn,
                                               (long long)M, (long long)N, (long long)K);
    lcml::Epilogue e;
    if (int rc = make_epilogue(e, fn, M, N, nullptr, b_scale, b_scale_per_channel, alpha, c, c_ndim, c_dim0,
                               c_dim1, beta, act, y, y_dtype, ldy))
        return rc;
    if (M == 0) {
        if (ya.npart) *ya.npart = 0;
        return LCML_OK;
    }
    if (!x || !b_packed) return fail(LCML_ERR_INVALID_ARG, "%s: NULL operand", fn);
    if (K % 16 != 0) return fail(LCML_ERR_UNSUPPORTED, "%s: K=%lld is not a multiple of 16", fn, (long long)K);
    if (ldx < K) return fail(LCML_ERR_INVALID_ARG, "%s: ldx=%lld < K=%lld", fn, (long long)ldx, (long long)K);
    if (!aligned(b_packed, 16)) return fail(LCML_ERR_INVALID_ARG, "%s: b_packed not 16-byte aligned", fn);
    hipStream_t s = (hipStream_t)stream;
    if (dynamic_fusable(M, K, x, ldx, kernel)) {
        if (int rc = hip_status(lcml::launch_gemm_skinny_dynamic(M, N, K, x, ldx, b_packed, e, x_scale_out,
                                                                 kernel != LCML_KERNEL_SKINNY_FP8 &&
                                                                     kernel != LCML_KERNEL_AUTO_FP8,
                                                                 s),
                                fn,
                                kernel == LCML_KERNEL_SKINNY_FP8 || kernel == LCML_KERNEL_AUTO_FP8
                                    ? "gemm_skinny_dynamic_fp8"
                                    : "gemm_skinny_dynamic"))
            return rc;
        if (ya.part)
            return hip_status(lcml::launch_amax_partials(static_cast<const float *>(y), M * N, ya.part, ya.npart, s),
                              fn, "amax_partials");
        return LCML_OK;
    }
    // two-step path: quantise into the workspace, then the selected GEMM.
    // The size is that of this path whatever the size query said: the query
    // cannot see x, and a misaligned x takes this path where an aligned one
    // would have fused.
    if (ldx != K) return fail(LCML_ERR_UNSUPPORTED, "%s: x must be contiguous (ldx == K) for M=%lld", fn, (long long)M);
    const int64_t need = two_step_workspace_bytes(M, K);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
        return fail(LCML_ERR_INVALID_ARG, "%s: needs a 256-byte aligned workspace of %lld bytes", fn,
                    (long long)need);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    uint8_t *q = ws;
    uint32_t *part = reinterpret_cast<uint32_t *>(ws + pad256(M * K));
    float *scale = x_scale_out ? x_scale_out : reinterpret_cast<float *>(ws + pad256(M * K) + LCML_FP8_DYNAMIC_WORKSPACE_BYTES);
    if (kernel == LCML_KERNEL_AUTO && aligned(x, 16) && dynamic_by_rows(M, N, K, xa.part != nullptr)) {
        // medium M: the codes in the layout of the GEMM that reads them
        int npart = xa.npart;
        if (!xa.part)
            if (int rc = hip_status(lcml::launch_amax_partials(x, M * K, part, &npart, s), fn, "amax_partials")) return rc;
        if (int rc = hip_status(lcml::launch_quantize_rows(x, q, M, K, xa.part ? xa.part : part, npart, scale, s), fn,
                                "quantize_rows"))
            return rc;
        e.a_scale = scale;
        if (int rc = hip_status(lcml::launch_gemm_rows(M, N, K, q, b_packed, e, s), fn, "gemm_rows")) return rc;
        if (ya.part)
            return hip_status(lcml::launch_amax_partials(static_cast<const float *>(y), M * N, ya.part, ya.npart, s),
                              fn, "amax_partials");
        return LCML_OK;
    }
    hipError_t err = xa.part ? lcml::launch_quantize_dynamic_parts(x, q, M * K, xa.part, xa.npart, scale, s)
                             : lcml::launch_quantize_dynamic(x, q, M * K, scale, part, s);
    if (int rc = hip_status(err, fn, xa.part ? "quantize_dynamic_parts" : "quantize_dynamic")) return rc;
    return gemm_core(fn, M, N, K, q, K, scale, b_packed, b_scale, b_scale_per_channel, alpha, c, c_ndim, c_dim0,
                     c_dim1, beta, act, y, y_dtype, ldy, kernel, stream, ya);
}

// The no-allocation variant's workspace: one array per device, in device
// memory from the moment the library's code object is loaded on that device
// until the process ends.  `scratch` names a host-side shadow of it; its
// device address comes from hipGetSymbolAddress, resolved once per device
// (with that device current) and kept in scratch_addr.  Calls that overlap
// on one device share it and race.
constexpr int64_t kNoAllocScratchBytes = LCML_FP8_NOALLOC_SCRATCH_BYTES;
static_assert(kNoAllocScratchBytes >= LCML_FP8_NOALLOC_MAX_ELEMS + LCML_FP8_DYNAMIC_WORKSPACE_BYTES + 256,
              "scratch holds the two-step workspace of the largest accepted M*K");
static __device__ __align__(256) uint8_t scratch[kNoAllocScratchBytes];
constexpr int kMaxDevices = 64;
std::atomic<void *> scratch_addr[kMaxDevices];

int noalloc_scratch(const char *fn, void **out) {
    int dev = 0;
    if (hipError_t err = hipGetDevice(&dev); err != hipSuccess) return hip_status(err, fn);
    if (dev < 0 || dev >= kMaxDevices) return fail(LCML_ERR_UNSUPPORTED, "%s: device %d (at most %d)", fn, dev, kMaxDevices);
    void *p = scratch_addr[dev].load(std::memory_order_acquire);
    if (!p) {
        // the same address on every call: threads racing here store equal values
        if (hipError_t err = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)); err != hipSuccess)
            return hip_status(err, fn);
        if (!p) return fail(LCML_ERR_HIP, "%s: no device address for the scratch array", fn);
        scratch_addr[dev].store(p, std::memory_order_release);
    }
    *out = p;
    return LCML_OK;
}
}  // namespace

extern "C" {

int lcml_fp8_gemm_dynamic(int64_t M, int64_t N, int64_t K, const float *x, int64_t ldx, const uint8_t *b_packed,
                          const float *b_scale, int b_scale_per_channel, float alpha, const float *c, int c_ndim,
                          int64_t c_dim0, int64_t c_dim1, float beta, int act, void *y, int y_dtype, int64_t ldy,
                          float *x_scale_out, void *workspace, int64_t workspace_bytes, int kernel, void *stream) {
    return gemm_dynamic_impl("lcml_fp8_gemm_dynamic", M, N, K, x, ldx, b_packed, b_scale, b_scale_per_channel, alpha,
                             c, c_ndim, c_dim0, c_dim1, beta, act, y, y_dtype, ldy, x_scale_out, workspace,
                             workspace_bytes, kernel, stream);
}

int lcml_fp8_gemm_dynamic_ex(int64_t M, int64_t N, int64_t K, const float *x, int64_t ldx, const uint8_t *b_packed,
                             const float *b_scale, int b_scale_per_channel, float alpha, const float *c, int c_ndim,
                             int64_t c_dim0, int64_t c_dim1, float beta, int act, void *y, int y_dtype, int64_t ldy,
                             float *x_scale_out, const uint32_t *x_amax_part, int x_amax_npart, uint32_t *y_amax_part,
                             int64_t y_amax_capacity, int *y_amax_npart, void *workspace, int64_t workspace_bytes,
                             int kernel, void *stream) {
    const char *fn = "lcml_fp8_gemm_dynamic_ex";
    XAmax xa;
    if (x_amax_part) {
        if (x_amax_npart < 1) return fail(LCML_ERR_INVALID_ARG, "%s: x_amax_npart=%d", fn, x_amax_npart);
        xa.part = x_amax_part;
        xa.npart = x_amax_npart;
    }
    YAmax ya;
    if (y_amax_part) {
        if (y_dtype != LCML_DTYPE_FLOAT || ldy != N)
            return fail(LCML_ERR_UNSUPPORTED, "%s: amax partials of y need a dense fp32 y (ldy == N)", fn);
        if (!y_amax_npart) return fail(LCML_ERR_INVALID_ARG, "%s: y_amax_npart is NULL", fn);
        if (y_amax_capacity < lcml_fp8_amax_parts_max(M, N))
            return fail(LCML_ERR_INVALID_ARG, "%s: y_amax_capacity=%lld < lcml_fp8_amax_parts_max=%lld", fn,
                        (long long)y_amax_capacity, (long long)lcml_fp8_amax_parts_max(M, N));
        ya.part = y_amax_part;
        ya.npart = y_amax_npart;
    }
    return gemm_dynamic_impl(fn, M, N, K, x, ldx, b_packed, b_scale, b_scale_per_channel, alpha, c, c_ndim, c_dim0,
                             c_dim1, beta, act, y, y_dtype, ldy, x_scale_out, workspace, workspace_bytes, kernel,
                             stream, xa, ya);
}

int lcml_fp8_gemm_dynamic_noalloc(int64_t M, int64_t N, int64_t K, const float *x, int64_t ldx,
                                  const uint8_t *b_packed, const float *b_scale, int b_scale_per_channel, float alpha,
                                  const float *c, int c_ndim, int64_t c_dim0, int64_t c_dim1, float beta, int act,
                                  void *y, int y_dtype, int64_t ldy, float *x_scale_out, int kernel, void *stream) {
    const char *fn = "lcml_fp8_gemm_dynamic_noalloc";
    if (M > 0 && K > 0 && M * K > LCML_FP8_NOALLOC_MAX_ELEMS)
        return fail(LCML_ERR_UNSUPPORTED, "%s: M*K=%lld exceeds the no-allocation limit of %lld elements", fn,
                    (long long)(M * K), (long long)LCML_FP8_NOALLOC_MAX_ELEMS);
    if (M < 0 || N <= 0 || K <= 0) return fail(LCML_ERR_INVALID_ARG, "%s: M=%lld N=%lld K=%lld", fn,
                                               (long long)M, (long long)N, (long long)K);
    if (M == 0) return gemm_dynamic_impl(fn, M, N, K, x, ldx, b_packed, b_scale, b_scale_per_channel, alpha, c,
                                         c_ndim, c_dim0, c_dim1, beta, act, y, y_dtype, ldy, x_scale_out, nullptr, 0,
                                         kernel, stream);
    void *ws = nullptr;
    if (int rc = noalloc_scratch(fn, &ws)) return rc;
    return gemm_dynamic_impl(fn, M, N, K, x, ldx, b_packed, b_scale, b_scale_per_channel, alpha, c, c_ndim, c_dim0,
                             c_dim1, beta, act, y, y_dtype, ldy, x_scale_out, ws, kNoAllocScratchBytes, kernel,
                             stream);
}

int lcml_fp8_quantize_nhwc(const float *x, uint8_t *y, int64_t n, int64_t c, int64_t h, int64_t w,
                           const float *y_scale, float *scale_out, void *workspace, void *stream) {
    const char *fn = "lcml_fp8_quantize_nhwc";
    if (n < 0 || c <= 0 || h <= 0 || w <= 0) return fail(LCML_ERR_INVALID_ARG, "%s: bad shape", fn);
    if (c % 4 != 0) return fail(LCML_ERR_UNSUPPORTED, "%s: c=%lld is not a multiple of 4", fn, (long long)c);
    if (n * c * h * w >= (int64_t)1 << 31 || n * h >= ((int64_t)1 << 31))
        return fail(LCML_ERR_UNSUPPORTED, "%s: tensor too large", fn);
    if (n == 0) return LCML_OK;
    if (!x || !y) return fail(LCML_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    if (!aligned(y, 4)) return fail(LCML_ERR_INVALID_ARG, "%s: y must be 4-byte aligned", fn);
    hipStream_t s = (hipStream_t)stream;
    if (y_scale)
        return hip_status(lcml::launch_quantize_nhwc(x, y, n, (int)c, (int)h, (int)w, y_scale, nullptr, 0, nullptr, s),
                          fn);
    if (!scale_out || !workspace)
        return fail(LCML_ERR_INVALID_ARG, "%s: the dynamic scale needs scale_out and a workspace", fn);
    uint32_t *part = static_cast<uint32_t *>(workspace);
    int npart = 0;
    hipError_t err = lcml::launch_amax_partials(x, n * c * h * w, part, &npart, s);
    if (err == hipSuccess)
        err = lcml::launch_quantize_nhwc(x, y, n, (int)c, (int)h, (int)w, nullptr, part, npart, scale_out, s);
    return hip_status(err, fn);
}

int64_t lcml_fp8_packed_conv_weight_bytes(int64_t cout, int64_t cin_g, int64_t kh, int64_t kw, int64_t group) {
    if (cout <= 0 || cin_g <= 0 || kh <= 0 || kw <= 0 || group <= 0 || cout % group != 0) return 0;
    return group * lcml_fp8_packed_weight_bytes(kh * kw * cin_g, cout / group);
}

int lcml_fp8_pack_conv_weight(const uint8_t *w, int64_t cout, int64_t cin_g, int64_t kh, int64_t kw, int64_t group,
                              uint8_t *packed, void *stream) {
    const char *fn = "lcml_fp8_pack_conv_weight";
    if (cout <= 0 || cin_g <= 0 || kh <= 0 || kw <= 0 || group <= 0 || cout % group != 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: bad shape or group", fn);
    if (!w || !packed) return fail(LCML_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    if (!aligned(packed, 16)) return fail(LCML_ERR_INVALID_ARG, "%s: packed not 16-byte aligned", fn);
    if (lcml_fp8_packed_conv_weight_bytes(cout, cin_g, kh, kw, group) >= (int64_t)1 << 31)
        return fail(LCML_ERR_UNSUPPORTED, "%s: packed weight larger than 2 GiB", fn);
    return hip_status(lcml::launch_pack_conv_weight(w, (int)cout, (int)cin_g, (int)kh, (int)kw, (int)group, packed,
                                                    (hipStream_t)stream),
                      fn);
}

int lcml_fp8_conv2d(const uint8_t *x_nhwc, const float *x_scale, int64_t n, int64_t c, int64_t h, int64_t w,
                    const uint8_t *w_packed, const float *w_scale, int w_scale_per_channel, int64_t cout, int64_t kh,
                    int64_t kw, int64_t stride_h, int64_t stride_w, int64_t pad_h, int64_t pad_w, int64_t dil_h,
                    int64_t dil_w, int64_t group, int64_t oh, int64_t ow, const float *bias, int act, void *y,
                    int y_dtype, int kernel, void *stream) {
    const char *fn = "lcml_fp8_conv2d";
    if (n < 0 || c <= 0 || h <= 0 || w <= 0 || cout <= 0 || kh <= 0 || kw <= 0 || oh <= 0 || ow <= 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: bad shape", fn);
    if (stride_h <= 0 || stride_w <= 0 || dil_h <= 0 || dil_w <= 0 || pad_h < 0 || pad_w < 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: strides and dilations must be >= 1, pads >= 0", fn);
    if (group <= 0 || c % group != 0 || cout % group != 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: group=%lld must divide c=%lld and cout=%lld", fn, (long long)group,
                    (long long)c, (long long)cout);
    if ((c / group) % 16 != 0)
        return fail(LCML_ERR_UNSUPPORTED, "%s: channels per group (%lld) not a multiple of 16", fn,
                    (long long)(c / group));
    const int64_t M = n * oh * ow;
    if (n * h * w * c >= (int64_t)1 << 31 || M >= (int64_t)1 << 31 ||
        lcml_fp8_packed_conv_weight_bytes(cout, c / group, kh, kw, group) >= (int64_t)1 << 31)
        return fail(LCML_ERR_UNSUPPORTED, "%s: operand larger than 2 GiB", fn);
    if (kernel == LCML_KERNEL_AUTO || kernel == LCML_KERNEL_AUTO_FP8) {
        // as auto_gemm_kernel without the skinny kernel; groups add grid rows
        const int64_t N = cout / group;
        const double big = (double)((M + 255) / 256 * ((N + 255) / 256) * group);
        const double t128 = (double)((M + 127) / 128 * ((N + 127) / 128) * group);
        const double small = 2.2 * (t128 > 256 ? t128 / 256 : 1.0);
        const int tiles = big < 256 && small < 4.5 ? LCML_KERNEL_MFMA_128 : LCML_KERNEL_MFMA;
        kernel = kernel == LCML_KERNEL_AUTO_FP8 ? fp8_twin(tiles) : tiles;
    }
    if (kernel != LCML_KERNEL_MFMA && kernel != LCML_KERNEL_MFMA_FP8 && kernel != LCML_KERNEL_MFMA_128 &&
        kernel != LCML_KERNEL_MFMA_128_FP8)
        return fail(LCML_ERR_UNSUPPORTED, "%s: kernel %d (AUTO, AUTO_FP8 or one of the MFMA tile kernels)", fn,
                    kernel);
    lcml::Epilogue e;
    if (int rc = make_epilogue(e, fn, M, cout, x_scale, w_scale, w_scale_per_channel, 1.0f, bias, 1, cout, 0, 1.0f,
                               act, y, y_dtype, cout))
        return rc;
    // per group: N = cout/group columns; the scale and bias pointers are
    // advanced to the group's channels in the kernel
    e.N = cout / group;
    e.c0 = cout / group;
    if (n == 0) return LCML_OK;
    if (!x_nhwc || !w_packed) return fail(LCML_ERR_INVALID_ARG, "%s: NULL operand", fn);
    if (!aligned(x_nhwc, 16) || !aligned(w_packed, 16))
        return fail(LCML_ERR_INVALID_ARG, "%s: x_nhwc and w_packed must be 16-byte aligned", fn);
    return hip_status(lcml::launch_conv_mfma(x_nhwc, n, (int)c, (int)h, (int)w, w_packed, (int)cout, (int)kh, (int)kw,
                                             (int)stride_h, (int)stride_w, (int)pad_h, (int)pad_w, (int)dil_h,
                                             (int)dil_w, (int)group, (int)oh, (int)ow, e,
                                             kernel == LCML_KERNEL_MFMA || kernel == LCML_KERNEL_MFMA_128,
                                             (hipStream_t)stream,
                                             kernel == LCML_KERNEL_MFMA_128 || kernel == LCML_KERNEL_MFMA_128_FP8),
                      fn,
                      kernel == LCML_KERNEL_MFMA       ? "conv_mfma_256"
                      : kernel == LCML_KERNEL_MFMA_FP8 ? "conv_mfma_256_fp8"
                      : kernel == LCML_KERNEL_MFMA_128 ? "conv_mfma_128"
                                                       : "conv_mfma_128_fp8");
}

int lcml_fp8_gemm_w8a32(int64_t M, int64_t N, int64_t K, const float *a, int64_t lda, const uint8_t *b_packed,
                        const float *b_scale, int b_scale_per_channel, float alpha, const float *c, int c_ndim,
                        int64_t c_dim0, int64_t c_dim1, float beta, int act, void *y, int y_dtype, int64_t ldy,
                        void *stream) {
    const char *fn = "lcml_fp8_gemm_w8a32";
    if (M < 0 || N <= 0 || K <= 0) return fail(LCML_ERR_INVALID_ARG, "%s: M=%lld N=%lld K=%lld", fn,
                                               (long long)M, (long long)N, (long long)K);
    lcml::Epilogue e;
    if (int rc = make_epilogue(e, fn, M, N, nullptr, b_scale, b_scale_per_channel, alpha, c, c_ndim, c_dim0,
                               c_dim1, beta, act, y, y_dtype, ldy))
        return rc;
    if (M == 0) return LCML_OK;
    if (!a || !b_packed) return fail(LCML_ERR_INVALID_ARG, "%s: NULL operand", fn);
    if (lda < K || !aligned(a, 4)) return fail(LCML_ERR_INVALID_ARG, "%s: lda < K or a misaligned", fn);
    if (!aligned(b_packed, 16)) return fail(LCML_ERR_INVALID_ARG, "%s: b_packed not 16-byte aligned", fn);
    if (lcml::w8a32_mfma_wins(M, N, K, a, lda))
        return hip_status(lcml::launch_gemm_w8a32(M, N, K, a, lda, b_packed, e, (hipStream_t)stream), fn,
                          "gemm_w8a32_mfma");
    return hip_status(lcml::launch_gemv_valu_f32(M, N, K, a, lda, b_packed, e, (hipStream_t)stream), fn,
                      "gemv_valu_w8a32");
}

int lcml_fp8_conv2d_f32(const float *x, const float *w, const float *bias, float *y, int64_t n, int64_t c, int64_t h,
                        int64_t wd, int64_t cout, int64_t kh, int64_t kw, int64_t stride_h, int64_t stride_w,
                        int64_t pad_h, int64_t pad_w, int64_t dil_h, int64_t dil_w, int64_t group, int64_t oh,
                        int64_t ow, int act, void *stream) {
    const char *fn = "lcml_fp8_conv2d_f32";
    if (n < 0 || c <= 0 || h <= 0 || wd <= 0 || cout <= 0 || kh <= 0 || kw <= 0 || oh <= 0 || ow <= 0 ||
        group <= 0 || c % group != 0 || cout % group != 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: bad shape or group", fn);
    if (stride_h <= 0 || stride_w <= 0 || dil_h <= 0 || dil_w <= 0 || pad_h < 0 || pad_w < 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: strides and dilations must be >= 1, pads >= 0", fn);
    if (act < LCML_ACT_NONE || act > LCML_ACT_GELU_TANH) return fail(LCML_ERR_UNSUPPORTED, "%s: activation %d", fn, act);
    if (n == 0) return LCML_OK;
    if (!x || !w || !y) return fail(LCML_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    if (n * cout * oh * ow >= (int64_t)1 << 40) return fail(LCML_ERR_UNSUPPORTED, "%s: output too large", fn);
    const char *label = nullptr;
    const hipError_t err = lcml::launch_conv2d_f32(
        x, w, bias, y, n, (int)c, (int)h, (int)wd, (int)cout, (int)kh, (int)kw, (int)stride_h, (int)stride_w,
        (int)pad_h, (int)pad_w, (int)dil_h, (int)dil_w, (int)group, (int)oh, (int)ow, act, (hipStream_t)stream, &label);
    return hip_status(err, fn, label);
}

int lcml_fp8_sgemm(int64_t M, int64_t N, int64_t K, const float *a, int64_t lda, int trans_a, const float *b,
                   int64_t ldb, int trans_b, float alpha, const float *c, int c_ndim, int64_t c_dim0,
                   int64_t c_dim1, float beta, int act, void *y, int y_dtype, int64_t ldy, void *stream) {
    const char *fn = "lcml_fp8_sgemm";
    if (M < 0 || N <= 0 || K <= 0) return fail(LCML_ERR_INVALID_ARG, "%s: M=%lld N=%lld K=%lld", fn,
                                               (long long)M, (long long)N, (long long)K);
    lcml::Epilogue e;
    if (int rc = make_epilogue(e, fn, M, N, nullptr, nullptr, 0, alpha, c, c_ndim, c_dim0, c_dim1, beta, act, y,
                               y_dtype, ldy, true))
        return rc;
    if (M == 0) return LCML_OK;
    if (!a || !b) return fail(LCML_ERR_INVALID_ARG, "%s: NULL operand", fn);
    if (lda < (trans_a ? M : K) || ldb < (trans_b ? K : N))
        return fail(LCML_ERR_INVALID_ARG, "%s: leading dimension too small", fn);
    const char *label = nullptr;
    const hipError_t err = lcml::launch_sgemm(M, N, K, a, lda, trans_a, b, ldb, trans_b, e, (hipStream_t)stream, &label);
    return hip_status(err, fn, label);
}

int lcml_fp8_activation(const float *x, float *y, int64_t n, int act, void *stream) {
    if (n < 0 || act < LCML_ACT_NONE || act > LCML_ACT_GELU_TANH)
        return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_activation: n=%lld act=%d", (long long)n, act);
    if (n == 0) return LCML_OK;
    if (!x || !y) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_activation: NULL pointer");
    return hip_status(lcml::launch_activation(x, y, n, act, (hipStream_t)stream), "lcml_fp8_activation");
}

int lcml_fp8_stream_read(const void *p, int64_t bytes, int workgroups, uint32_t *sink, void *stream) {
    const char *fn = "lcml_fp8_stream_read";
    if (bytes < 0 || bytes % 16 != 0 || workgroups < 1 || workgroups > (1 << 20))
        return fail(LCML_ERR_INVALID_ARG, "%s: bytes=%lld (multiple of 16) workgroups=%d", fn, (long long)bytes,
                    workgroups);
    if (bytes == 0) return LCML_OK;
    if (!p || !sink || !aligned(p, 16)) return fail(LCML_ERR_INVALID_ARG, "%s: p must be 16-byte aligned, sink set", fn);
    if ((bytes / 16 + workgroups - 1) / workgroups >= ((int64_t)1 << 27))
        return fail(LCML_ERR_UNSUPPORTED, "%s: a workgroup's share of %lld bytes over %d workgroups exceeds 2 GiB", fn,
                    (long long)bytes, workgroups);
    return hip_status(lcml::launch_stream_read(p, bytes, workgroups, sink, (hipStream_t)stream), fn);
}

namespace {
bool fp8_dtype_ok(int dt) {
    return dt == LCML_DTYPE_FLOAT || dt == LCML_DTYPE_FLOAT8E4M3FN || dt == LCML_DTYPE_FLOAT8E5M2;
}
}  // namespace

int lcml_fp8_cast(const void *x, int x_dtype, void *y, int y_dtype, int64_t n, void *stream) {
    const char *fn = "lcml_fp8_cast";
    if (n < 0) return fail(LCML_ERR_INVALID_ARG, "%s: n < 0", fn);
    if (!fp8_dtype_ok(x_dtype) || !fp8_dtype_ok(y_dtype))
        return fail(LCML_ERR_UNSUPPORTED, "%s: dtypes %d -> %d (FLOAT, FLOAT8E4M3FN, FLOAT8E5M2 only)", fn, x_dtype,
                    y_dtype);
    if (n == 0) return LCML_OK;
    if (!x || !y) return fail(LCML_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    if (x_dtype == LCML_DTYPE_FLOAT ? !aligned(x, 4) : false) return fail(LCML_ERR_INVALID_ARG, "%s: x misaligned", fn);
    if (y_dtype == LCML_DTYPE_FLOAT ? !aligned(y, 4) : false) return fail(LCML_ERR_INVALID_ARG, "%s: y misaligned", fn);
    return hip_status(lcml::launch_cast(x, x_dtype, y, y_dtype, n, (hipStream_t)stream), fn);
}

int lcml_fp8_quantize_e5m2(const float *x, uint8_t *y, int64_t outer, int64_t axis_len, int64_t inner,
                           const float *y_scale, int saturate, void *stream) {
    if (int rc = check_view(outer, axis_len, inner, "lcml_fp8_quantize_e5m2")) return rc;
    if (outer * axis_len * inner == 0) return LCML_OK;
    if (!x || !y || !y_scale) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_quantize_e5m2: NULL pointer");
    if (saturate != 0 && saturate != 1) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_quantize_e5m2: saturate %d", saturate);
    return hip_status(lcml::launch_quantize_e5m2(x, y, outer, axis_len, inner, y_scale, saturate == 1,
                                                 (hipStream_t)stream),
                      "lcml_fp8_quantize_e5m2");
}

int lcml_fp8_dequantize_e5m2(const uint8_t *x, float *y, int64_t outer, int64_t axis_len, int64_t inner,
                             const float *x_scale, void *stream) {
    if (int rc = check_view(outer, axis_len, inner, "lcml_fp8_dequantize_e5m2")) return rc;
    if (outer * axis_len * inner == 0) return LCML_OK;
    if (!x || !y || !x_scale) return fail(LCML_ERR_INVALID_ARG, "lcml_fp8_dequantize_e5m2: NULL pointer");
    return hip_status(lcml::launch_dequantize_e5m2(x, y, outer, axis_len, inner, x_scale, (hipStream_t)stream),
                      "lcml_fp8_dequantize_e5m2");
}

int lcml_fp8_binary(int op, int dtype, const void *a, const int64_t *a_shape, int a_ndim, const void *b,
                    const int64_t *b_shape, int b_ndim, void *y, const int64_t *y_shape, int y_ndim, void *stream) {
    const char *fn = "lcml_fp8_binary";
    if (op < LCML_BINARY_ADD || op > LCML_BINARY_DIV) return fail(LCML_ERR_INVALID_ARG, "%s: op %d", fn, op);
    if (!fp8_dtype_ok(dtype)) return fail(LCML_ERR_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    if (a_ndim < 0 || b_ndim < 0 || y_ndim < 0 || y_ndim > lcml::kMaxBcastDims || a_ndim > y_ndim || b_ndim > y_ndim)
        return fail(LCML_ERR_INVALID_ARG, "%s: ranks a=%d b=%d y=%d (at most %d, y the largest)", fn, a_ndim, b_ndim,
                    y_ndim, lcml::kMaxBcastDims);
    if ((a_ndim && !a_shape) || (b_ndim && !b_shape) || (y_ndim && !y_shape))
        return fail(LCML_ERR_INVALID_ARG, "%s: NULL shape", fn);
    // numpy broadcasting, right-aligned; element strides of a and b per output dim
    lcml::BcastGeom g{};
    g.ndim = y_ndim;
    int64_t n = 1, acc_a = 1, acc_b = 1;
    bool same = a_ndim == y_ndim && b_ndim == y_ndim;
    for (int d = y_ndim - 1; d >= 0; --d) {
        const int da = d - (y_ndim - a_ndim), db = d - (y_ndim - b_ndim);
        const int64_t ea = da >= 0 ? a_shape[da] : 1, eb = db >= 0 ? b_shape[db] : 1, ey = y_shape[d];
        if (ea < 0 || eb < 0 || ey < 0) return fail(LCML_ERR_INVALID_ARG, "%s: negative dimension", fn);
        const int64_t want = ea == 1 ? eb : (eb == 1 || eb == ea ? ea : -1);
        if (want < 0 || want != ey)
            return fail(LCML_ERR_INVALID_ARG, "%s: dim %d: a %lld, b %lld do not broadcast to y %lld", fn, d,
                        (long long)ea, (long long)eb, (long long)ey);
        same = same && ea == ey && eb == ey;
        g.dims[d] = ey;
        g.sa[d] = ea == 1 ? 0 : acc_a;
        g.sb[d] = eb == 1 ? 0 : acc_b;
        acc_a *= ea;
        acc_b *= eb;
        if (ey && n > ((int64_t)1 << 40) / ey) return fail(LCML_ERR_UNSUPPORTED, "%s: tensor too large", fn);
        n *= ey;
    }
    if (n == 0) return LCML_OK;
    if (!a || !b || !y) return fail(LCML_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    if (dtype == LCML_DTYPE_FLOAT && (!aligned(a, 4) || !aligned(b, 4) || !aligned(y, 4)))
        return fail(LCML_ERR_INVALID_ARG, "%s: fp32 tensors must be 4-byte aligned", fn);
    return hip_status(lcml::launch_fp8_binary(op, dtype, a, b, y, n, same, g, (hipStream_t)stream), fn);
}

int64_t lcml_fp8_rms_norm_workspace_bytes(int64_t M, int64_t H, int mode) {
    return M > 1 && H > 0 && mode == LCML_SCALE_TENSOR ? lcml::rms_norm_workspace(M) : 0;
}

int lcml_fp8_rms_norm(int64_t M, int64_t H, const void *x, int x_dtype, int64_t ldx, const void *residual,
                      void *residual_out, int r_dtype, int64_t ldr, int64_t ldro, const float *gamma, float eps,
                      uint8_t *y, int64_t ldy, int mode, float *scale, void *workspace, int64_t workspace_bytes,
                      void *stream) {
    const char *fn = "lcml_fp8_rms_norm";
    if (M < 0 || H <= 0) return fail(LCML_ERR_INVALID_ARG, "%s: M=%lld H=%lld", fn, (long long)M, (long long)H);
    if (!float_or_bf16(x_dtype)) return fail(LCML_ERR_UNSUPPORTED, "%s: x dtype %d", fn, x_dtype);
    if (mode < LCML_SCALE_STATIC || mode > LCML_SCALE_ROW) return fail(LCML_ERR_INVALID_ARG, "%s: mode %d", fn, mode);
    if (!(eps >= 0.0f)) return fail(LCML_ERR_INVALID_ARG, "%s: eps %g", fn, (double)eps);
    if (residual) {
        if (!float_or_bf16(r_dtype)) return fail(LCML_ERR_UNSUPPORTED, "%s: residual dtype %d", fn, r_dtype);
        if (ldr < H || (residual_out && ldro < H))
            return fail(LCML_ERR_INVALID_ARG, "%s: residual pitch below H=%lld", fn, (long long)H);
    } else if (residual_out) {
        return fail(LCML_ERR_INVALID_ARG, "%s: residual_out without residual", fn);
    }
    if (ldx < H || ldy < H) return fail(LCML_ERR_INVALID_ARG, "%s: pitch below H=%lld", fn, (long long)H);
    if (M >= (int64_t)1 << 31 || H >= (int64_t)1 << 31)
        return fail(LCML_ERR_UNSUPPORTED, "%s: M=%lld H=%lld", fn, (long long)M, (long long)H);
    if (M == 0) return LCML_OK;
    if (!x || !gamma || !y || !scale) return fail(LCML_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    if (!elem_aligned(x, x_dtype) || (residual && (!elem_aligned(residual, r_dtype) || !elem_aligned(residual_out, r_dtype))) ||
        !aligned(gamma, 4) || !aligned(scale, 4))
        return fail(LCML_ERR_INVALID_ARG, "%s: pointer not aligned to its elements", fn);
    if (const int64_t need = lcml_fp8_rms_norm_workspace_bytes(M, H, mode);
        need && (!workspace || workspace_bytes < need || !aligned(workspace, 4)))
        return fail(LCML_ERR_INVALID_ARG, "%s: needs a workspace of %lld bytes", fn, (long long)need);
    return hip_status(lcml::launch_rms_norm(M, H, x, x_dtype == LCML_DTYPE_BFLOAT16, ldx, residual, residual_out,
                                            r_dtype == LCML_DTYPE_BFLOAT16, ldr, ldro, gamma, eps, y, ldy, mode, scale,
                                            workspace, (hipStream_t)stream),
                      fn);
}

namespace {
// The cache arguments of the three KV entry points.
int make_tokens(lcml::KvTokens &t, const char *fn, int64_t tokens, const void *k_cache, const void *v_cache,
                const float *k_scale, const float *v_scale, int64_t pages, int64_t kv_heads, int64_t head_dim,
                int64_t page_tokens, const int32_t *block_table, int64_t table_stride, int64_t table_cols,
                const int32_t *kv_len, const int32_t *cu_q, int64_t seqs, int64_t max_q) {
    if (tokens < 0 || seqs < 0 || max_q < 0 || pages < 0 || table_cols < 0 || kv_heads <= 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: tokens=%lld seqs=%lld max_q=%lld pages=%lld table_cols=%lld kv_heads=%lld",
                    fn, (long long)tokens, (long long)seqs, (long long)max_q, (long long)pages, (long long)table_cols,
                    (long long)kv_heads);
    if (head_dim < 16 || head_dim > 256 || head_dim % 16)
        return fail(LCML_ERR_UNSUPPORTED, "%s: head_dim=%lld (16 to 256, in steps of 16)", fn, (long long)head_dim);
    if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)))
        return fail(LCML_ERR_UNSUPPORTED, "%s: page_tokens=%lld (16, 32, 64, 128 or 256)", fn, (long long)page_tokens);
    const int64_t most = ((int64_t)1 << 31) - 1;
    if (tokens > most || seqs > most || pages > most || table_cols > most || kv_heads > 65535 || max_q > most)
        return fail(LCML_ERR_UNSUPPORTED, "%s: a size of 2^31 or more", fn);
    if (table_stride < table_cols)
        return fail(LCML_ERR_INVALID_ARG, "%s: table_stride=%lld < table_cols=%lld", fn, (long long)table_stride,
                    (long long)table_cols);
    if (tokens == 0 || seqs == 0 || max_q == 0) return LCML_OK;
    if ((table_cols && !block_table) || !kv_len || !cu_q) return fail(LCML_ERR_INVALID_ARG, "%s: NULL index array", fn);
    if (!aligned(block_table, 4) || !aligned(kv_len, 4) || !aligned(cu_q, 4))
        return fail(LCML_ERR_INVALID_ARG, "%s: index arrays not 4-byte aligned", fn);
    if (pages && (!k_cache || !v_cache || !k_scale || !v_scale)) return fail(LCML_ERR_INVALID_ARG, "%s: NULL cache", fn);
    if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
        return fail(LCML_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned, scales 4-byte aligned", fn);
    t = lcml::KvTokens{block_table,         kv_len,           cu_q,           table_stride,      (int32_t)table_cols,
                       (int32_t)seqs,       (int32_t)tokens,  (int32_t)pages, (int32_t)kv_heads, (int32_t)head_dim,
                       __builtin_ctzll((unsigned long long)page_tokens)};
    return LCML_OK;
}

// 2^32 work items a launch, with `threads` for a page and head of K or of V
int check_kv_grid(const char *fn, const lcml::KvTokens &t, int64_t max_q, int64_t threads) {
    const int64_t per_seq = lcml::kv_pages_per_seq(max_q, t.tshift) * 2 * t.heads;
    if (per_seq > (((int64_t)1 << 32) - 256) / threads / t.seqs)
        return fail(LCML_ERR_UNSUPPORTED, "%s: seqs=%lld max_q=%lld exceeds one launch", fn, (long long)t.seqs,
                    (long long)max_q);
    return LCML_OK;
}
}  // namespace

int lcml_fp8_kv_cache_write(const void *k, const void *v, int dtype, int64_t tokens, int64_t k_token_stride,
                            int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, uint8_t *k_cache,
                            uint8_t *v_cache, float *k_scale, float *v_scale, int64_t pages, int64_t kv_heads,
                            int64_t head_dim, int64_t page_tokens, const int32_t *block_table, int64_t table_stride,
                            int64_t table_cols, const int32_t *kv_len, const int32_t *cu_q, int64_t seqs,
                            int64_t max_q, void *stream) {
    const char *fn = "lcml_fp8_kv_cache_write";
    if (!float_or_bf16(dtype)) return fail(LCML_ERR_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    lcml::KvTokens t;
    if (int rc = make_tokens(t, fn, tokens, k_cache, v_cache, k_scale, v_scale, pages, kv_heads, head_dim, page_tokens,
                             block_table, table_stride, table_cols, kv_len, cu_q, seqs, max_q))
        return rc;
    if (tokens == 0 || seqs == 0 || max_q == 0 || pages == 0) return LCML_OK;
    if (!k || !v || !elem_aligned(k, dtype) || !elem_aligned(v, dtype))
        return fail(LCML_ERR_INVALID_ARG, "%s: k or v NULL or not aligned to its elements", fn);
    if (int rc = check_kv_grid(fn, t, max_q, lcml::kv_write_threads(max_q, t.dim, t.tshift))) return rc;
    return hip_status(lcml::launch_kv_write(t, max_q, k, v, dtype == LCML_DTYPE_BFLOAT16, k_token_stride, k_head_stride,
                                            v_token_stride, v_head_stride, k_cache, v_cache, k_scale, v_scale,
                                            (hipStream_t)stream),
                      fn);
}

int lcml_fp8_kv_cache_read(const uint8_t *k_cache, const uint8_t *v_cache, const float *k_scale, const float *v_scale,
                           int64_t pages, int64_t kv_heads, int64_t head_dim, int64_t page_tokens,
                           const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *kv_len,
                           const int32_t *cu_q, int64_t seqs, int64_t max_q, void *k, void *v, int dtype,
                           int64_t tokens, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                           int64_t v_head_stride, void *stream) {
    const char *fn = "lcml_fp8_kv_cache_read";
    if (!float_or_bf16(dtype)) return fail(LCML_ERR_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    lcml::KvTokens t;
    if (int rc = make_tokens(t, fn, tokens, k_cache, v_cache, k_scale, v_scale, pages, kv_heads, head_dim, page_tokens,
                             block_table, table_stride, table_cols, kv_len, cu_q, seqs, max_q))
        return rc;
    if (tokens == 0 || seqs == 0 || max_q == 0 || pages == 0) return LCML_OK;
    if (!k || !v || !elem_aligned(k, dtype) || !elem_aligned(v, dtype))
        return fail(LCML_ERR_INVALID_ARG, "%s: k or v NULL or not aligned to its elements", fn);
    const int64_t units = (int64_t)(t.dim >> 3) << (t.tshift - 2);  // of 4 tokens x 8 elements, a thread each
    if (int rc = check_kv_grid(fn, t, max_q, units)) return rc;
    return hip_status(lcml::launch_kv_read(t, max_q, k, v, dtype == LCML_DTYPE_BFLOAT16, k_token_stride, k_head_stride,
                                           v_token_stride, v_head_stride, k_cache, v_cache, k_scale, v_scale,
                                           (hipStream_t)stream),
                      fn);
}

int64_t lcml_fp8_kv_cache_plan_workspace_bytes(int64_t seqs, int64_t tokens) {
    return seqs < 0 || tokens < 0 ? 0 : lcml::kv_plan_workspace(seqs, tokens);
}

int lcml_fp8_kv_cache_plan(const int32_t *new_tokens, const int32_t *kv_len_in, const int32_t *ended,
                           const int32_t *first_own, int64_t seqs, int32_t *free_pages, const int32_t *free_count,
                           int64_t pages, int64_t page_tokens, int32_t *block_table, int64_t table_stride,
                           int64_t table_cols, int32_t *kv_len, int32_t *cu_q, int32_t *left, int32_t *positions,
                           int64_t *slots, int64_t tokens, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *fn = "lcml_fp8_kv_cache_plan";
    if (seqs < 0 || pages < 0 || table_cols < 0 || tokens < 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: seqs=%lld pages=%lld table_cols=%lld tokens=%lld", fn, (long long)seqs,
                    (long long)pages, (long long)table_cols, (long long)tokens);
    if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)))
        return fail(LCML_ERR_UNSUPPORTED, "%s: page_tokens=%lld (16, 32, 64, 128 or 256)", fn, (long long)page_tokens);
    const int64_t most = ((int64_t)1 << 31) - 1;
    if (pages > most || table_cols > most || tokens > most)
        return fail(LCML_ERR_UNSUPPORTED, "%s: a size of 2^31 or more", fn);
    if (seqs > (int64_t)1 << 30)  // indexes of sequences are added in 32 bits
        return fail(LCML_ERR_UNSUPPORTED, "%s: seqs=%lld (2^30 at most)", fn, (long long)seqs);
    if (table_stride < table_cols)
        return fail(LCML_ERR_INVALID_ARG, "%s: table_stride=%lld < table_cols=%lld", fn, (long long)table_stride,
                    (long long)table_cols);
    if ((seqs && (!new_tokens || !kv_len_in || !kv_len || (table_cols && !block_table))) || (pages && !free_pages) ||
        !free_count || !cu_q || !left)
        return fail(LCML_ERR_INVALID_ARG, "%s: NULL index array", fn);
    for (const void *p : {(const void *)new_tokens, (const void *)kv_len_in, (const void *)ended, (const void *)first_own,
                          (const void *)free_pages, (const void *)free_count, (const void *)block_table,
                          (const void *)kv_len, (const void *)cu_q, (const void *)left, (const void *)positions})
        if (!aligned(p, 4)) return fail(LCML_ERR_INVALID_ARG, "%s: index arrays not 4-byte aligned", fn);
    if (!aligned(slots, 8)) return fail(LCML_ERR_INVALID_ARG, "%s: slots not 8-byte aligned", fn);
    if (const int64_t need = lcml::kv_plan_workspace(seqs, tokens);
        need && (!workspace || workspace_bytes < need || !aligned(workspace, 8)))
        return fail(LCML_ERR_INVALID_ARG, "%s: needs an 8-byte aligned workspace of %lld bytes", fn, (long long)need);
    const lcml::KvPlan p{new_tokens, ended, first_own, kv_len_in, free_count, free_pages, block_table, table_stride,
                         (int32_t)table_cols, (int32_t)seqs, (int32_t)pages,
                         __builtin_ctzll((unsigned long long)page_tokens), kv_len, cu_q, left, positions, slots, tokens,
                         static_cast<int64_t *>(workspace)};
    const char *label = nullptr;
    const hipError_t err = lcml::launch_kv_plan(p, (hipStream_t)stream, &label);
    return hip_status(err, fn, label);
}

int lcml_fp8_qk_norm_rope(const void *q, const void *k, int dtype, int64_t tokens, int64_t q_heads, int64_t k_heads,
                          int64_t head_dim, int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                          int64_t k_head_stride, const float *q_gamma, const float *k_gamma, float eps,
                          const int32_t *positions, const float *table, int64_t table_rows, int64_t rot_dim,
                          int interleaved, void *q_out, void *k_out, int out_dtype, int64_t qo_token_stride,
                          int64_t qo_head_stride, int64_t ko_token_stride, int64_t ko_head_stride, void *stream) {
    const char *fn = "lcml_fp8_qk_norm_rope";
    if (!float_or_bf16(dtype) || !float_or_bf16(out_dtype))
        return fail(LCML_ERR_UNSUPPORTED, "%s: dtypes %d, out %d", fn, dtype, out_dtype);
    if (tokens < 0 || q_heads < 0 || k_heads < 0 || table_rows < 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: tokens=%lld q_heads=%lld k_heads=%lld table_rows=%lld", fn,
                    (long long)tokens, (long long)q_heads, (long long)k_heads, (long long)table_rows);
    if (head_dim < 16 || head_dim > 256 || head_dim % 16)
        return fail(LCML_ERR_UNSUPPORTED, "%s: head_dim=%lld (16 to 256, in steps of 16)", fn, (long long)head_dim);
    if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2)
        return fail(LCML_ERR_INVALID_ARG, "%s: rot_dim=%lld (even, up to head_dim=%lld)", fn, (long long)rot_dim,
                    (long long)head_dim);
    if (!(eps >= 0.0f)) return fail(LCML_ERR_INVALID_ARG, "%s: eps %g", fn, (double)eps);
    if (q_heads > 65535 || k_heads > 65535 || tokens >= (int64_t)1 << 31 || table_rows >= (int64_t)1 << 31)
        return fail(LCML_ERR_UNSUPPORTED, "%s: tokens=%lld q_heads=%lld k_heads=%lld table_rows=%lld", fn,
                    (long long)tokens, (long long)q_heads, (long long)k_heads, (long long)table_rows);
    if (tokens == 0 || q_heads + k_heads == 0) return LCML_OK;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) ||
        (q_heads && (!elem_aligned(q, dtype) || !elem_aligned(q_out, out_dtype))) ||
        (k_heads && (!elem_aligned(k, dtype) || !elem_aligned(k_out, out_dtype))))
        return fail(LCML_ERR_INVALID_ARG, "%s: q, k or an output NULL or not aligned to its elements", fn);
    if (rot_dim && (!positions || (table_rows && !table)))
        return fail(LCML_ERR_INVALID_ARG, "%s: a rotation takes positions and a table", fn);
    if (!aligned(q_gamma, 4) || !aligned(k_gamma, 4) || !aligned(positions, 4) || !aligned(table, 4))
        return fail(LCML_ERR_INVALID_ARG, "%s: gammas, positions or table not 4-byte aligned", fn);
    // 64 threads each, 2^32 work items a launch
    if (tokens * lcml::qk_norm_rope_parts(tokens, (int32_t)q_heads, (int32_t)k_heads, (int32_t)head_dim) >= ((int64_t)1 << 26) - 4)
        return fail(LCML_ERR_UNSUPPORTED, "%s: tokens=%lld exceeds one launch", fn, (long long)tokens);
    const lcml::RopeArgs a{q, k, q_out, k_out, q_gamma, k_gamma, table, positions, q_token_stride,
                           q_head_stride, k_token_stride, k_head_stride, qo_token_stride, qo_head_stride,
                           ko_token_stride, ko_head_stride, tokens, (int32_t)q_heads, (int32_t)k_heads,
                           (int32_t)head_dim, (int32_t)rot_dim,
                           rot_dim ? (int32_t)table_rows : 0x7fffffff, interleaved != 0, eps,
                           1.0f / (float)head_dim, 0};
    return hip_status(lcml::launch_qk_norm_rope(a, dtype == LCML_DTYPE_BFLOAT16, out_dtype == LCML_DTYPE_BFLOAT16,
                                                (hipStream_t)stream),
                      fn);
}

int64_t lcml_fp8_attention_workspace_bytes(int64_t tokens, int64_t seqs, int64_t q_heads, int64_t kv_heads,
                                           int64_t head_dim, int64_t max_q, int64_t max_kv) {
    if (tokens <= 0 || seqs <= 0 || kv_heads <= 0 || q_heads < kv_heads || head_dim <= 0 || max_q <= 0 || max_kv <= 0)
        return 0;
    return lcml::attention_workspace(tokens, seqs, q_heads, kv_heads, head_dim, max_q, max_kv);
}

namespace {
// what the attention entry points are given alike
struct AttentionCall {
    const void *q;
    int q_dtype;
    int64_t tokens, q_heads, q_token_stride, q_head_stride;
    void *o;
    int o_dtype;
    int64_t o_token_stride, o_head_stride;
    const uint8_t *k_cache, *v_cache;
    const float *k_scale, *v_scale;
    int64_t pages, kv_heads, head_dim, page_tokens;
    const int32_t *block_table;
    int64_t table_stride, table_cols;
    const int32_t *kv_len, *cu_q;
    int64_t seqs, max_q, max_kv;
    float scale;
    int causal;
    int64_t window;
};
// 256 threads each, 2^32 work items a launch, and a workgroup for each row
// where parts are joined; sizes whose products would pass 64 bits are past
// that by far
constexpr int64_t kMostGroups = (int64_t)1 << 24;

int too_large(const char *fn, const AttentionCall &c) {
    return fail(LCML_ERR_UNSUPPORTED, "%s: seqs=%lld max_q=%lld q_heads=%lld exceeds one launch", fn, (long long)c.seqs,
                (long long)c.max_q, (long long)c.q_heads);
}
// Checks c and fills a; *rows false: a call without rows.
int make_attention(lcml::AttentionArgs &a, const char *fn, const AttentionCall &c, bool *rows) {
    if (!float_or_bf16(c.q_dtype) || !float_or_bf16(c.o_dtype))
        return fail(LCML_ERR_UNSUPPORTED, "%s: dtypes q %d, o %d", fn, c.q_dtype, c.o_dtype);
    if (!(c.scale > 0.0f) || c.scale > 3.0e38f) return fail(LCML_ERR_INVALID_ARG, "%s: scale %g", fn, (double)c.scale);
    if (c.window < 0 || c.max_kv < 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: window=%lld max_kv=%lld", fn, (long long)c.window, (long long)c.max_kv);
    if (int rc = make_tokens(a.t, fn, c.tokens, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.pages, c.kv_heads,
                             c.head_dim, c.page_tokens, c.block_table, c.table_stride, c.table_cols, c.kv_len, c.cu_q,
                             c.seqs, c.max_q))
        return rc;
    if (c.q_heads <= 0 || c.q_heads % c.kv_heads)
        return fail(LCML_ERR_INVALID_ARG, "%s: q_heads=%lld is not a multiple of kv_heads=%lld", fn,
                    (long long)c.q_heads, (long long)c.kv_heads);
    if (c.q_heads > 65535 || c.max_kv >= (int64_t)1 << 31)
        return fail(LCML_ERR_UNSUPPORTED, "%s: q_heads=%lld max_kv=%lld", fn, (long long)c.q_heads, (long long)c.max_kv);
    *rows = c.tokens > 0 && c.seqs > 0 && c.max_q > 0;
    if (!*rows) return LCML_OK;
    if (!c.q || !c.o || !elem_aligned(c.q, c.q_dtype) || !elem_aligned(c.o, c.o_dtype))
        return fail(LCML_ERR_INVALID_ARG, "%s: q or o NULL or not aligned to its elements", fn);
    if (c.max_q * c.q_heads / c.kv_heads > kMostGroups * 16 || c.seqs * c.kv_heads > kMostGroups) return too_large(fn, c);
    a.q = c.q, a.o = c.o, a.k = c.k_cache, a.v = c.v_cache, a.ks = c.k_scale, a.vs = c.v_scale;
    a.q_token = c.q_token_stride, a.q_head = c.q_head_stride, a.o_token = c.o_token_stride, a.o_head = c.o_head_stride;
    a.max_q = c.max_q, a.max_kv = c.max_kv;
    a.window = c.window < (int64_t)1 << 31 ? c.window : 0;  // a longer one hides nothing
    a.q_heads = (int32_t)c.q_heads, a.causal = c.causal != 0;
    a.q_bf16 = c.q_dtype == LCML_DTYPE_BFLOAT16, a.o_bf16 = c.o_dtype == LCML_DTYPE_BFLOAT16;
    a.scale = c.scale;
    return LCML_OK;
}

// lcml_fp8_attention, and with sinks > 0 lcml_fp8_attention_sinks
int attend(const char *fn, const AttentionCall &c, int64_t sinks, void *workspace, int64_t workspace_bytes, void *stream) {
    lcml::AttentionArgs a{};
    bool rows = false;
    if (int rc = make_attention(a, fn, c, &rows)) return rc;
    if (!rows) return LCML_OK;
    if (lcml::attention_groups(c.seqs, c.q_heads, c.kv_heads, c.head_dim, c.max_q, c.max_kv) >= kMostGroups)
        return too_large(fn, c);
    const int64_t need = lcml::attention_workspace(c.tokens, c.seqs, c.q_heads, c.kv_heads, c.head_dim, c.max_q, c.max_kv);
    if (need && c.seqs * c.max_q >= kMostGroups / c.q_heads) return too_large(fn, c);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return fail(LCML_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)need);
    a.sinks = sinks < (int64_t)1 << 31 ? (uint32_t)sinks : 0x7fffffffu;
    const char *label = nullptr;
    const hipError_t err = a.window > 0 && sinks > 0 ? lcml::launch_attention_sinks(a, workspace, (hipStream_t)stream, &label)
                                                     : lcml::launch_attention(a, workspace, (hipStream_t)stream, &label);
    return hip_status(err, fn, label);
}
}  // namespace

int lcml_fp8_attention(const void *q, int q_dtype, int64_t tokens, int64_t q_heads, int64_t q_token_stride,
                       int64_t q_head_stride, void *o, int o_dtype, int64_t o_token_stride, int64_t o_head_stride,
                       const uint8_t *k_cache, const uint8_t *v_cache, const float *k_scale, const float *v_scale,
                       int64_t pages, int64_t kv_heads, int64_t head_dim, int64_t page_tokens,
                       const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *kv_len,
                       const int32_t *cu_q, int64_t seqs, int64_t max_q, int64_t max_kv, float scale, int causal,
                       int64_t window, void *workspace, int64_t workspace_bytes, void *stream) {
    return attend("lcml_fp8_attention",
                  AttentionCall{q, q_dtype, tokens, q_heads, q_token_stride, q_head_stride, o, o_dtype, o_token_stride,
                                o_head_stride, k_cache, v_cache, k_scale, v_scale, pages, kv_heads, head_dim, page_tokens,
                                block_table, table_stride, table_cols, kv_len, cu_q, seqs, max_q, max_kv, scale, causal,
                                window},
                  0, workspace, workspace_bytes, stream);
}

int lcml_fp8_attention_sinks(const void *q, int q_dtype, int64_t tokens, int64_t q_heads, int64_t q_token_stride,
                             int64_t q_head_stride, void *o, int o_dtype, int64_t o_token_stride, int64_t o_head_stride,
                             const uint8_t *k_cache, const uint8_t *v_cache, const float *k_scale, const float *v_scale,
                             int64_t pages, int64_t kv_heads, int64_t head_dim, int64_t page_tokens,
                             const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *kv_len,
                             const int32_t *cu_q, int64_t seqs, int64_t max_q, int64_t max_kv, float scale, int causal,
                             int64_t window, int64_t sinks, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *fn = "lcml_fp8_attention_sinks";
    if (sinks < 0) return fail(LCML_ERR_INVALID_ARG, "%s: sinks=%lld", fn, (long long)sinks);
    return attend(fn,
                  AttentionCall{q, q_dtype, tokens, q_heads, q_token_stride, q_head_stride, o, o_dtype, o_token_stride,
                                o_head_stride, k_cache, v_cache, k_scale, v_scale, pages, kv_heads, head_dim, page_tokens,
                                block_table, table_stride, table_cols, kv_len, cu_q, seqs, max_q, max_kv, scale, causal,
                                window},
                  sinks, workspace, workspace_bytes, stream);
}

int64_t lcml_fp8_attention_shared_workspace_bytes(int64_t tokens, int64_t seqs, int64_t groups, int64_t q_heads,
                                                  int64_t kv_heads, int64_t head_dim, int64_t max_q, int64_t max_own,
                                                  int64_t max_prefix) {
    if (tokens <= 0 || seqs <= 0 || groups < 0 || kv_heads <= 0 || q_heads < kv_heads || head_dim <= 0 || max_q <= 0 ||
        max_own < 0 || max_prefix < 0)
        return 0;
    int64_t workgroups = 0;
    return lcml::attention_shared_workspace(tokens, seqs, groups, q_heads, kv_heads, head_dim, max_q, max_own, max_prefix,
                                            &workgroups);
}

int lcml_fp8_attention_shared(const void *q, int q_dtype, int64_t tokens, int64_t q_heads, int64_t q_token_stride,
                              int64_t q_head_stride, void *o, int o_dtype, int64_t o_token_stride, int64_t o_head_stride,
                              const uint8_t *k_cache, const uint8_t *v_cache, const float *k_scale, const float *v_scale,
                              int64_t pages, int64_t kv_heads, int64_t head_dim, int64_t page_tokens,
                              const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *kv_len,
                              const int32_t *cu_q, int64_t seqs, const int32_t *group_seq, const int32_t *prefix_table,
                              int64_t prefix_stride, int64_t prefix_cols, const int32_t *prefix_len, int64_t groups,
                              int64_t max_q, int64_t max_own, int64_t max_prefix, float scale, int causal,
                              void *workspace, int64_t workspace_bytes, void *stream) {
    const char *fn = "lcml_fp8_attention_shared";
    const AttentionCall c{q, q_dtype, tokens, q_heads, q_token_stride, q_head_stride, o, o_dtype, o_token_stride,
                          o_head_stride, k_cache, v_cache, k_scale, v_scale, pages, kv_heads, head_dim, page_tokens,
                          block_table, table_stride, table_cols, kv_len, cu_q, seqs, max_q, max_own, scale, causal, 0};
    lcml::AttentionArgs a{};
    bool rows = false;
    if (int rc = make_attention(a, fn, c, &rows)) return rc;
    if (groups < 0 || prefix_cols < 0 || max_prefix < 0)
        return fail(LCML_ERR_INVALID_ARG, "%s: groups=%lld prefix_cols=%lld max_prefix=%lld", fn, (long long)groups,
                    (long long)prefix_cols, (long long)max_prefix);
    if (prefix_stride < prefix_cols)
        return fail(LCML_ERR_INVALID_ARG, "%s: prefix_stride=%lld < prefix_cols=%lld", fn, (long long)prefix_stride,
                    (long long)prefix_cols);
    if (groups > kMostGroups || prefix_cols >= (int64_t)1 << 31 || max_prefix >= (int64_t)1 << 31)
        return fail(LCML_ERR_UNSUPPORTED, "%s: groups=%lld prefix_cols=%lld max_prefix=%lld", fn, (long long)groups,
                    (long long)prefix_cols, (long long)max_prefix);
    if (!rows) return LCML_OK;
    if (groups && (!group_seq || !prefix_len || (prefix_cols && !prefix_table)))
        return fail(LCML_ERR_INVALID_ARG, "%s: NULL index array", fn);
    if (!aligned(group_seq, 4) || !aligned(prefix_len, 4) || !aligned(prefix_table, 4))
        return fail(LCML_ERR_INVALID_ARG, "%s: index arrays not 4-byte aligned", fn);
    if (tokens * (q_heads / kv_heads) > kMostGroups * 16) return too_large(fn, c);
    int64_t workgroups = 0;
    const int64_t need = lcml::attention_shared_workspace(tokens, seqs, groups, q_heads, kv_heads, head_dim, max_q, max_own,
                                                          max_prefix, &workgroups);
    if (workgroups >= kMostGroups) return too_large(fn, c);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
        return fail(LCML_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)need);
    a.group_seq = group_seq, a.prefix_len = prefix_len, a.groups = (int32_t)groups;
    const char *label = nullptr;
    const hipError_t err = lcml::launch_attention_shared(a, prefix_table, prefix_stride, prefix_cols, max_prefix, workspace,
                                                         (hipStream_t)stream, &label);
    return hip_status(err, fn, label);
}

}  // extern "C"
