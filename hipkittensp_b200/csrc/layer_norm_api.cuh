// Host side of the layer norm: argument checks, choice of the kernel variant, launches (entry points in mxfp6_api.cu).
#pragma once
#include "layer_norm_kernel.cuh"

namespace mxfp6 {

typedef void (*LnKernel)(const LnParams);
struct LnChoice {
    LnKernel kern;
    int warps;       // warps that share a row; one: eight rows per CTA; none: a CTA of 1024 threads passes over the row again
    int smem;        // dynamic shared memory
};

// Whole 8-element chunks: a thread holds up to four, sixteen warps a row: 16384 elements.
template <typename T, int FMT>
static LnChoice ln_forward_vec(int H) {
    const int smem = 8 * H;          // w and b as fp32
    if (H <= 256) return {layer_norm_kernel<T, 1, 1, FMT>, 1, smem};
    if (H <= 1024) return {layer_norm_kernel<T, 4, 1, FMT>, 1, smem};
    if (H <= 2048) return {layer_norm_kernel<T, 4, 2, FMT>, 2, smem};
    if (H <= 4096) return {layer_norm_kernel<T, 4, 4, FMT>, 4, smem};
    if (H <= 8192) return {layer_norm_kernel<T, 4, 8, FMT>, 8, smem};
    if (H <= 16384) return {layer_norm_kernel<T, 4, 16, FMT>, 16, smem};
    return {layer_norm_long_kernel<T, 8, FMT>, 0, 0};
}
template <typename T>
static LnChoice ln_forward_odd(int H) {
    if (H <= 256) return {layer_norm_odd_kernel<T, 8, 1>, 1, 0};
    if (H <= 512) return {layer_norm_odd_kernel<T, 8, 2>, 2, 0};
    if (H <= 1024) return {layer_norm_odd_kernel<T, 8, 4>, 4, 0};
    if (H <= 2048) return {layer_norm_odd_kernel<T, 8, 8>, 8, 0};
    if (H <= 4096) return {layer_norm_odd_kernel<T, 8, 16>, 16, 0};
    if (H <= 8192) return {layer_norm_odd_kernel<T, 16, 16>, 16, 0};
    if (H <= 16384) return {layer_norm_odd_kernel<T, 32, 16>, 16, 0};
    return {layer_norm_long_kernel<T, 1, -1>, 0, 0};
}
// fmt: format of an MX result, negative for one in x's type
template <typename T>
static LnChoice ln_forward_kernel(bool vec, int fmt, int H) {
    if (!vec) return ln_forward_odd<T>(H);
    switch (fmt) {
        case MXFP6_E2M3: return ln_forward_vec<T, MXFP6_E2M3>(H);
        case MXFP6_E3M2: return ln_forward_vec<T, MXFP6_E3M2>(H);
        case MXFP8_E4M3: return ln_forward_vec<T, MXFP8_E4M3>(H);
        case MXFP8_E5M2: return ln_forward_vec<T, MXFP8_E5M2>(H);
        case MXFP4_E2M1: return ln_forward_vec<T, MXFP4_E2M1>(H);
        default: return ln_forward_vec<T, -1>(H);
    }
}

// Backward holds x, dy and both column sums: 16 elements a thread, 8192 a row; bf16 rows of whole chunks up to 16384 keep x and dy
// in shared memory.
constexpr int kLnBackwardMax = 8192, kLnBackwardWide = 16384;
static int ln_backward_warps(int H) { return H <= 512 ? 1 : H <= 1024 ? 2 : H <= 2048 ? 4 : H <= 4096 ? 8 : 16; }
template <typename T>
static LnChoice ln_backward_kernel(bool vec, int H) {
    const int warps = ln_backward_warps(H);
    if (vec) {
        // w as fp32; one warp per row: room for the eight warps' column sums
        if (H <= 256) return {layer_norm_backward_kernel<T, 1, 1>, 1, 8 * 256 * 4};
        switch (warps) {
            case 1: return {layer_norm_backward_kernel<T, 2, 1>, 1, 8 * 512 * 4};
            case 2: return {layer_norm_backward_kernel<T, 2, 2>, 2, 4 * H};
            case 4: return {layer_norm_backward_kernel<T, 2, 4>, 4, 4 * H};
            case 8: return {layer_norm_backward_kernel<T, 2, 8>, 8, 4 * H};
            default: return {layer_norm_backward_kernel<T, 2, 16>, 16, 4 * H};
        }
    }
    if (H <= 256) return {layer_norm_backward_odd_kernel<T, 8, 1>, 1, 0};
    switch (warps) {
        case 1: return {layer_norm_backward_odd_kernel<T, 16, 1>, 1, 0};
        case 2: return {layer_norm_backward_odd_kernel<T, 16, 2>, 2, 0};
        case 4: return {layer_norm_backward_odd_kernel<T, 16, 4>, 4, 0};
        case 8: return {layer_norm_backward_odd_kernel<T, 16, 8>, 8, 0};
        default: return {layer_norm_backward_odd_kernel<T, 16, 16>, 16, 0};
    }
}

// Number of partial sums per column of the parameter gradients: the grid of the kernel that writes them.
static int ln_parts(int64_t rows, int64_t H, int sm_count) {
    if (H <= kLnBackwardMax) {
        const int warps = ln_backward_warps((int)H);
        const int64_t want = warps == 1 ? (rows + 7) / 8 : rows;
        const int64_t cap = (int64_t)sm_count * (warps == 1 ? 2 : 16 / warps);      // 512 threads of 128 registers per SM
        return (int)(want < cap ? want : cap);
    }
    int64_t y = 8 * (int64_t)sm_count / ((H + 255) / 256);
    if (y > (rows + 15) / 16) y = (rows + 15) / 16;
    return (int)(y < 1 ? 1 : y);
}
static int ln_parts_wide(int64_t rows, int sm_count) { return (int)(rows < sm_count ? rows : sm_count); }
// ... the most that any kernel which may serve such rows writes (their type and alignment are not known here)
static int ln_parts_most(int64_t rows, int64_t H, int sm_count) {
    if (rows <= 0) return 0;
    const int n = ln_parts(rows, H, sm_count), w = H > kLnBackwardMax && H <= kLnBackwardWide ? ln_parts_wide(rows, sm_count) : 0;
    return n > w ? n : w;
}

static int ln_check(const char* what, int64_t rows, int64_t H, int x_dtype, int w_dtype) {
    if (rows < 0 || H < 1) return fail(MXFP6_ERR_BAD_ARG, "%s: rows=%lld H=%lld (rows >= 0 and H >= 1)", what, (long long)rows, (long long)H);
    if (rows > 0x7fffffffLL || H > 0x3fffffffLL) return fail(MXFP6_ERR_BAD_ARG, "%s: dimension too large", what);
    if (x_dtype != 0 && x_dtype != 1) return fail(MXFP6_ERR_BAD_ARG, "%s: dtype must be 0 (fp32) or 1 (bf16)", what);
    if (w_dtype != 0 && w_dtype != 1) return fail(MXFP6_ERR_BAD_ARG, "%s: w_dtype must be 0 (fp32) or 1 (bf16)", what);
    return MXFP6_OK;
}
static bool ln_natural(const void* p, int dtype) { return !((uintptr_t)p & (dtype == 0 ? 3 : 1)); }
// whole 8-element loads of the row matrices (32 or 16 bytes) and of the parameter vectors (16 bytes at a time)
static bool ln_rows_vec(const void* p, int dtype) { return !((uintptr_t)p & (dtype == 0 ? 31 : 15)); }

static int ln_forward(const char* what, const void* x, int x_dtype, const void* w, const void* b, int w_dtype, void* y, int fmt,
                      void* packed, void* scales, float* mean, float* rstd, int64_t rows, int64_t H, float eps, void* stream) {
    const bool mx = fmt >= 0;
    int rc = ln_check(what, rows, H, x_dtype, w_dtype);
    if (rc) return rc;
    if (!(eps >= 0.f) || eps > 3e38f) return fail(MXFP6_ERR_BAD_ARG, "%s: eps must be finite and not negative", what);
    if (mx && !fmt_valid(fmt)) return fail(MXFP6_ERR_BAD_ARG, "%s: bad format %d", what, fmt);
    if (mx && H % 32) return fail(MXFP6_ERR_BAD_ARG, "%s: H=%lld must be a multiple of 32", what, (long long)H);
    if (rows == 0) return MXFP6_OK;
    if (!x || (mx ? !packed || !scales : !y)) return fail(MXFP6_ERR_BAD_ARG, "%s: null pointer", what);
    if (!ln_natural(x, x_dtype) || !ln_natural(y, x_dtype) || !ln_natural(w, w_dtype) || !ln_natural(b, w_dtype) ||
        !ln_natural(mean, 0) || !ln_natural(rstd, 0))
        return fail(MXFP6_ERR_BAD_ARG, "%s: misaligned pointer", what);
    const bool vec = H % 8 == 0 && ln_rows_vec(x, x_dtype) && ln_rows_vec(y, x_dtype) && !((uintptr_t)w & 15) && !((uintptr_t)b & 15);
    if (mx && (!vec || ((uintptr_t)packed & 15)))
        return fail(MXFP6_ERR_BAD_ARG, "%s: x must be 32-byte (fp32) or 16-byte (bf16) aligned, weight, bias and codes 16-byte", what);
    DeviceState* d = nullptr;
    if ((rc = get_device_state(&d))) return rc;
    const LnChoice k = x_dtype == 0 ? ln_forward_kernel<float>(vec, fmt, (int)H) : ln_forward_kernel<__nv_bfloat16>(vec, fmt, (int)H);
    const int threads = k.warps == 0 ? 1024 : k.warps == 1 ? 256 : 32 * k.warps;
    int per_sm = 0;
    if ((rc = resident_ctas(*d, (const void*)k.kern, threads, k.smem, &per_sm))) return rc;
    const int64_t want = k.warps == 1 ? (rows + 7) / 8 : rows, cap = (int64_t)d->sm_count * per_sm;
    LnParams P{};
    P.x = x; P.y = y; P.w = w; P.b = b; P.w_bf16 = w_dtype;
    P.mean = mean; P.rstd = rstd;
    P.q_out = (uint8_t*)packed; P.q_scales = (uint8_t*)scales;
    P.rows = rows; P.H = (int)H; P.inv_h = 1.f / (float)H; P.eps = eps;
    return launch_pdl(k.kern, (unsigned)(want < cap ? want : cap), (unsigned)threads, (size_t)k.smem, (cudaStream_t)stream, P);
}

static int ln_backward(const void* dy, const void* x, int x_dtype, const float* mean, const float* rstd, const void* w, int w_dtype,
                       void* dx, float* dw, float* db, int64_t rows, int64_t H, void* ws, size_t ws_bytes, void* stream) {
    const char* what = "layer_norm_backward";
    int rc = ln_check(what, rows, H, x_dtype, w_dtype);
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (((uintptr_t)dw & 3) || ((uintptr_t)db & 3)) return fail(MXFP6_ERR_BAD_ARG, "%s: misaligned pointer", what);
    if (rows == 0) {        // sums over no rows
        if (dw) CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)H * 4, st));
        if (db) CUDA_TRY(cudaMemsetAsync(db, 0, (size_t)H * 4, st));
        return MXFP6_OK;
    }
    if (!dy || !x || !mean || !rstd || !dx) return fail(MXFP6_ERR_BAD_ARG, "%s: null pointer", what);
    if (!ln_natural(x, x_dtype) || !ln_natural(dy, x_dtype) || !ln_natural(dx, x_dtype) || !ln_natural(w, w_dtype) ||
        !ln_natural(mean, 0) || !ln_natural(rstd, 0))
        return fail(MXFP6_ERR_BAD_ARG, "%s: misaligned pointer", what);
    DeviceState* d = nullptr;
    if ((rc = get_device_state(&d))) return rc;
    const bool sums = dw || db;
    // one size for every type and alignment of such rows
    const size_t need = sums ? (size_t)ln_parts_most(rows, H, d->sm_count) * 2 * (size_t)H * 4 : 0;
    if (sums && (!ws || ws_bytes < need)) return fail(MXFP6_ERR_BAD_ARG, "%s: workspace too small: need %zu bytes, got %zu", what, need, ws ? ws_bytes : 0);
    if (sums && ((uintptr_t)ws & 15)) return fail(MXFP6_ERR_BAD_ARG, "%s: workspace must be 16-byte aligned", what);
    const bool vec = H % 8 == 0 && ln_rows_vec(x, x_dtype) && ln_rows_vec(dy, x_dtype) && ln_rows_vec(dx, x_dtype) && !((uintptr_t)w & 15);
    LnParams P{};
    P.x = x; P.dy = dy; P.y = dx; P.w = w; P.w_bf16 = w_dtype;
    P.mean = const_cast<float*>(mean); P.rstd = const_cast<float*>(rstd);
    P.part = sums ? (float*)ws : nullptr;
    P.rows = rows; P.H = (int)H; P.inv_h = 1.f / (float)H;
    int parts = ln_parts(rows, H, d->sm_count);
    if (H <= kLnBackwardMax) {
        const LnChoice k = x_dtype == 0 ? ln_backward_kernel<float>(vec, (int)H) : ln_backward_kernel<__nv_bfloat16>(vec, (int)H);
        if ((rc = launch_pdl(k.kern, (unsigned)parts, (unsigned)(k.warps == 1 ? 256 : 32 * k.warps), (size_t)k.smem, st, P))) return rc;
    } else if (vec && x_dtype == 1 && H <= kLnBackwardWide) {
        const int smem = 4 * (int)H + 2 * 2 * 4 * 512 * 16;
        parts = ln_parts_wide(rows, d->sm_count);
        if ((rc = ensure_smem_attr(*d, (const void*)layer_norm_backward_wide_kernel, 4 * kLnBackwardWide + 2 * 2 * 4 * 512 * 16))) return rc;
        if ((rc = launch_pdl(layer_norm_backward_wide_kernel, (unsigned)parts, 512, (size_t)smem, st, P))) return rc;
    } else {
        if (sums) {
            LnKernel k = x_dtype == 0 ? layer_norm_columns_kernel<float> : layer_norm_columns_kernel<__nv_bfloat16>;
            k<<<dim3((unsigned)((H + 255) / 256), (unsigned)parts), 256, 0, st>>>(P);
            CUDA_TRY(cudaGetLastError());
        }
        const LnKernel k = x_dtype == 0 ? (vec ? layer_norm_backward_long_kernel<float, 8> : layer_norm_backward_long_kernel<float, 1>)
                                        : (vec ? layer_norm_backward_long_kernel<__nv_bfloat16, 8> : layer_norm_backward_long_kernel<__nv_bfloat16, 1>);
        const int64_t cap = 2 * (int64_t)d->sm_count;
        if ((rc = launch_pdl(k, (unsigned)(rows < cap ? rows : cap), 1024, 0, st, P))) return rc;
    }
    if (!sums) return MXFP6_OK;
    return launch_pdl(layer_norm_fold_kernel, (unsigned)((2 * H + 31) / 32), 1024, 0, st, (const float*)ws, parts, (int)H, dw, db);
}

}  // namespace mxfp6
