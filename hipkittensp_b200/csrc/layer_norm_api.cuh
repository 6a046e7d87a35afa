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

// How the rows of the matrices lie: whole aligned chunks of 8 elements; any width and start, but the same place in the 16- or
// 32-byte units of memory in each matrix; or anything else.
enum LnRows : int { kLnWhole, kLnOdd, kLnApart };
static LnRows ln_rows(int64_t H, int dtype, const void* w, const void* b, const void* p, const void* q, const void* r) {
    const uintptr_t unit = dtype == 0 ? 31 : 15, at = (uintptr_t)p & unit;
    if (((uintptr_t)q & unit) != at || ((uintptr_t)r & unit) != at) return kLnApart;
    return at == 0 && H % 8 == 0 && !((uintptr_t)w & 15) && !((uintptr_t)b & 15) ? kLnWhole : kLnOdd;
}

// A thread holds up to four chunks, sixteen warps a row: 16384 elements, and 7 fewer where the row may start anywhere in its chunk.
template <typename T, int FMT, bool ODD>
static LnChoice ln_forward_choice(int H) {
    const int smem = 8 * H + (ODD ? 128 : 0);          // w and b as fp32
    const int span = H + (ODD ? 7 : 0);
    if (span <= 256) return {layer_norm_kernel<T, 1, 1, FMT, ODD>, 1, smem};
    if (span <= 512) return {layer_norm_kernel<T, 2, 1, FMT, ODD>, 1, smem};
    // three chunks per thread where they are enough: with four, up to half of the threads would work on nothing
    // (8192 x 5000 bf16 41 -> 39 us, 30000 x 700 27 -> 22 us)
    if constexpr (FMT < 0) {
        if (span <= 768) return {layer_norm_kernel<T, 3, 1, FMT, ODD>, 1, smem};
        if (span > 1024 && span <= 1536) return {layer_norm_kernel<T, 3, 2, FMT, ODD>, 2, smem};
        if (span > 2048 && span <= 3 * 1024) return {layer_norm_kernel<T, 3, 4, FMT, ODD>, 4, smem};
        if (span > 4096 && span <= 6144) return {layer_norm_kernel<T, 3, 8, FMT, ODD>, 8, smem};
        if (span > 8192 && span <= 12288) return {layer_norm_kernel<T, 3, 16, FMT, ODD>, 16, smem};
    }
    if (span <= 1024) return {layer_norm_kernel<T, 4, 1, FMT, ODD>, 1, smem};
    if (span <= 2048) return {layer_norm_kernel<T, 4, 2, FMT, ODD>, 2, smem};
    if (span <= 4096) return {layer_norm_kernel<T, 4, 4, FMT, ODD>, 4, smem};
    if (span <= 8192) return {layer_norm_kernel<T, 4, 8, FMT, ODD>, 8, smem};
    if (span <= 16384) return {layer_norm_kernel<T, 4, 16, FMT, ODD>, 16, smem};
    return {layer_norm_long_kernel<T, ODD ? 1 : 8, FMT>, 0, 0};
}
// fmt: format of an MX result, negative for one in x's type
template <typename T>
static LnChoice ln_forward_kernel(LnRows rows, int fmt, int H) {
    if (rows == kLnApart) return {layer_norm_long_kernel<T, 1, -1>, 0, 0};
    if (rows == kLnOdd) return ln_forward_choice<T, -1, true>(H);
    switch (fmt) {
        case MXFP6_E2M3: return ln_forward_choice<T, MXFP6_E2M3, false>(H);
        case MXFP6_E3M2: return ln_forward_choice<T, MXFP6_E3M2, false>(H);
        case MXFP8_E4M3: return ln_forward_choice<T, MXFP8_E4M3, false>(H);
        case MXFP8_E5M2: return ln_forward_choice<T, MXFP8_E5M2, false>(H);
        case MXFP4_E2M1: return ln_forward_choice<T, MXFP4_E2M1, false>(H);
        default: return ln_forward_choice<T, -1, false>(H);
    }
}

// Backward holds x, dy and both column sums: 16 elements a thread, 8192 a row; bf16 rows up to 16384 keep x and dy in shared
// memory; the rest (kern = null) goes over its rows again.
constexpr int kLnBackwardMax = 8192, kLnBackwardWide = 16384;
static int ln_backward_warps(int span) { return span <= 512 ? 1 : span <= 1024 ? 2 : span <= 2048 ? 4 : span <= 4096 ? 8 : 16; }
template <typename T, bool ODD>
static LnChoice ln_backward_choice(int H) {
    const int span = H + (ODD ? 7 : 0);
    if (span > kLnBackwardMax) return {nullptr, 0, 0};
    const int smem = 4 * H + (ODD ? 64 : 0);           // w as fp32; one warp per row: room for the eight warps' column sums
    if (span <= 256) return {layer_norm_backward_kernel<T, 1, 1, ODD>, 1, 8 * 256 * 4};
    switch (ln_backward_warps(span)) {
        case 1: return {layer_norm_backward_kernel<T, 2, 1, ODD>, 1, 8 * 512 * 4};
        case 2: return {layer_norm_backward_kernel<T, 2, 2, ODD>, 2, smem};
        case 4: return {layer_norm_backward_kernel<T, 2, 4, ODD>, 4, smem};
        case 8: return {layer_norm_backward_kernel<T, 2, 8, ODD>, 8, smem};
        default: return {layer_norm_backward_kernel<T, 2, 16, ODD>, 16, smem};
    }
}
template <typename T>
static LnChoice ln_backward_kernel(LnRows rows, int H) {
    if (rows == kLnApart) return {nullptr, 0, 0};
    const int span = H + (rows == kLnOdd ? 7 : 0);
    if constexpr (sizeof(T) == 2)
        if (span > kLnBackwardMax && span <= kLnBackwardWide)
            return {rows == kLnOdd ? layer_norm_backward_wide_kernel<true> : layer_norm_backward_wide_kernel<false>, 16, 4 * H + 64 + 2 * 2 * 4 * 512 * 16};
    return rows == kLnOdd ? ln_backward_choice<T, true>(H) : ln_backward_choice<T, false>(H);
}

// CTAs for `rows` rows at a time (eight rows per CTA when a warp owns one), at most cap, and the step from one of a CTA's rows to
// its next.  Rows that start anywhere are dealt so that a CTA's rows lie a multiple of eight apart.
static int ln_grid(int64_t rows, int warps, bool odd, int64_t cap, int64_t* step) {
    int64_t grid;
    if (odd) {
        const int64_t want = warps == 1 ? 8 * ((rows + 63) / 64) : rows;
        cap = cap / 8 * 8;
        grid = want <= cap ? want : cap;
        *step = want <= cap ? (warps == 1 ? 8 * grid : rows) : (warps == 1 ? 8 * grid : grid);
    } else {
        const int64_t want = warps == 1 ? (rows + 7) / 8 : rows;
        grid = want < cap ? want : cap;
        *step = warps == 1 ? 8 * grid : grid;
    }
    return (int)grid;
}

// Number of partial sums per column of the parameter gradients: the grid of the kernel that writes them.
// At most what is resident (512 threads of 128 registers per SM), and no more than keeps the partials' 8 bytes per column and part
// at a third of the 6 or 12 bytes per element that the rows move, as long as every SM has a CTA (1500 x 1001 fp32: 562 instead of
// 1184 parts).
static int64_t ln_backward_cap(int warps, int sm_count, int64_t rows, int elem_bytes) {
    const int64_t resident = (int64_t)sm_count * (warps == 1 ? 2 : 16 / warps);
    const int64_t few = rows * elem_bytes * 3 / 32, least = few > sm_count ? few : sm_count;
    return least < resident ? least : resident;
}
static int ln_parts_columns(int64_t rows, int64_t H, int sm_count) {
    int64_t y = 8 * (int64_t)sm_count / ((H + 255) / 256);
    if (y > (rows + 15) / 16) y = (rows + 15) / 16;
    return (int)(y < 1 ? 1 : y);
}
// ... the most that any kernel which may serve such rows writes (their type and place are not known here)
static int64_t ln_parts_most(int64_t rows, int64_t H, int sm_count) {
    if (rows <= 0) return 0;
    int64_t most = ln_parts_columns(rows, H, sm_count), step;
    auto take = [&](int64_t n) { if (n > most) most = n; };
    for (int odd = 0; odd < 2; ++odd) {
        const int64_t span = H + 7 * odd;
        if (span > kLnBackwardMax) continue;
        const int warps = ln_backward_warps((int)span);
        take(ln_grid(rows, warps, odd != 0, ln_backward_cap(warps, sm_count, rows, 4), &step));
    }
    if (H + 7 > kLnBackwardMax && H <= kLnBackwardWide) take(rows < sm_count ? rows : sm_count);
    return most;
}

// Elements of a partial vector: whole chunks, wherever in its first one the row starts.
static int ln_part_ld(int64_t H) { return (int)((H + 14) / 8 * 8); }
static size_t ln_workspace(int64_t rows, int64_t H, int sm_count) { return (size_t)ln_parts_most(rows, H, sm_count) * 2 * (size_t)ln_part_ld(H) * 4; }

static int ln_check(const char* what, int64_t rows, int64_t H, int x_dtype, int w_dtype) {
    if (rows < 0 || H < 1) return fail(MXFP6_ERR_BAD_ARG, "%s: rows=%lld H=%lld (rows >= 0 and H >= 1)", what, (long long)rows, (long long)H);
    if (rows > 0x7fffffffLL || H > 0x3fffffffLL) return fail(MXFP6_ERR_BAD_ARG, "%s: dimension too large", what);
    if (x_dtype != 0 && x_dtype != 1) return fail(MXFP6_ERR_BAD_ARG, "%s: dtype must be 0 (fp32) or 1 (bf16)", what);
    if (w_dtype != 0 && w_dtype != 1) return fail(MXFP6_ERR_BAD_ARG, "%s: w_dtype must be 0 (fp32) or 1 (bf16)", what);
    return MXFP6_OK;
}
static bool ln_natural(const void* p, int dtype) { return !((uintptr_t)p & (dtype == 0 ? 3 : 1)); }

// Do the ranges share bytes?  A CTA writes its rows while others still read theirs, so a result may lie on an operand of its own
// shape, row upon row, or apart from it.
static bool ln_overlap(const void* p, uint64_t p_bytes, const void* q, uint64_t q_bytes) {
    const uint64_t a = (uintptr_t)p, b = (uintptr_t)q;
    return a < b ? b - a < p_bytes : a - b < q_bytes;
}

struct LnRange { const char* name; const void* p; uint64_t bytes; };
// A result that lies on an operand, or on another result, whose bytes other CTAs read or write at any time (null ranges lie nowhere).
static int ln_apart(const char* what, std::initializer_list<LnRange> results, std::initializer_list<LnRange> operands, bool among = false) {
    for (const LnRange* r = results.begin(); r != results.end(); ++r) {
        if (!r->p) continue;
        for (const LnRange& o : operands)
            if (o.p && ln_overlap(r->p, r->bytes, o.p, o.bytes)) return fail(MXFP6_ERR_BAD_ARG, "%s: %s overlaps %s", what, r->name, o.name);
        for (const LnRange* q = r + 1; among && q != results.end(); ++q)
            if (q->p && ln_overlap(r->p, r->bytes, q->p, q->bytes)) return fail(MXFP6_ERR_BAD_ARG, "%s: %s overlaps %s", what, r->name, q->name);
    }
    return MXFP6_OK;
}

// elements from the 16- or 32-byte boundary in front of p to p
static int ln_offset(const void* p, int dtype) { return (int)((uintptr_t)p & (dtype == 0 ? 31 : 15)) / (dtype == 0 ? 4 : 2); }

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
    const LnRows place = ln_rows(H, x_dtype, w, b, x, mx ? x : y, x);
    if (mx && (place != kLnWhole || ((uintptr_t)packed & 15)))
        return fail(MXFP6_ERR_BAD_ARG, "%s: x must be 32-byte (fp32) or 16-byte (bf16) aligned, weight, bias and codes 16-byte", what);
    const uint64_t bytes = (uint64_t)rows * (uint64_t)H * (x_dtype == 0 ? 4 : 2);
    if (mx ? ln_overlap(x, bytes, packed, (uint64_t)rows * (uint64_t)(H / 32) * fmt_block_bytes(fmt)) ||
                 ln_overlap(x, bytes, scales, (uint64_t)rows * (uint64_t)(H / 32))
           : x != y && ln_overlap(x, bytes, y, bytes))
        return fail(MXFP6_ERR_BAD_ARG, "%s: the result overlaps x", what);
    {
        const uint64_t params = (uint64_t)H * (w_dtype == 0 ? 4 : 2), stats = (uint64_t)rows * 4;
        const LnRange y_range{"the result", mx ? packed : y, mx ? (uint64_t)rows * (uint64_t)(H / 32) * fmt_block_bytes(fmt) : bytes},
            scale_range{"the scales", mx ? scales : nullptr, (uint64_t)rows * (uint64_t)(H / 32)}, mean_range{"mean", mean, stats}, rstd_range{"rstd", rstd, stats};
        if ((rc = ln_apart(what, {y_range, scale_range, mean_range, rstd_range}, {{"weight", w, params}, {"bias", b, params}}, true))) return rc;
        if ((rc = ln_apart(what, {mean_range, rstd_range}, {{"x", x, bytes}}))) return rc;
    }
    DeviceState* d = nullptr;
    if ((rc = get_device_state(&d))) return rc;
    const LnChoice k = x_dtype == 0 ? ln_forward_kernel<float>(place, fmt, (int)H) : ln_forward_kernel<__nv_bfloat16>(place, fmt, (int)H);
    const int threads = k.warps == 0 ? 1024 : k.warps == 1 ? 256 : 32 * k.warps;
    int per_sm = 0;
    if ((rc = resident_ctas(*d, (const void*)k.kern, threads, k.smem, &per_sm))) return rc;
    LnParams P{};
    P.x = x; P.y = y; P.w = w; P.b = b; P.w_bf16 = w_dtype;
    P.mean = mean; P.rstd = rstd;
    P.q_out = (uint8_t*)packed; P.q_scales = (uint8_t*)scales;
    P.rows = rows; P.H = (int)H; P.inv_h = (float)(1.0 / (double)H); P.inv_h_low = (float)(1.0 / (double)H - (double)P.inv_h); P.eps = eps;
    P.offset = ln_offset(x, x_dtype);
    const int grid = ln_grid(rows, k.warps, place == kLnOdd && k.warps > 0, (int64_t)d->sm_count * per_sm, &P.step);
    return launch_pdl(k.kern, (unsigned)grid, (unsigned)threads, (size_t)k.smem, (cudaStream_t)stream, P);
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
    const uint64_t bytes = (uint64_t)rows * (uint64_t)H * (x_dtype == 0 ? 4 : 2);
    if ((dx != x && ln_overlap(dx, bytes, x, bytes)) || (dx != dy && ln_overlap(dx, bytes, dy, bytes)))
        return fail(MXFP6_ERR_BAD_ARG, "%s: dx overlaps x or dy without being it", what);
    const uint64_t params = (uint64_t)H * (w_dtype == 0 ? 4 : 2), sum_bytes = (uint64_t)H * 4, stats = (uint64_t)rows * 4;
    const LnRange dx_range{"dx", dx, bytes}, dw_range{"dweight", dw, sum_bytes}, db_range{"dbias", db, sum_bytes}, x_range{"x", x, bytes}, dy_range{"dy", dy, bytes},
        w_range{"weight", w, params}, mean_range{"mean", mean, stats}, rstd_range{"rstd", rstd, stats};
    if ((rc = ln_apart(what, {dx_range}, {w_range, mean_range, rstd_range}))) return rc;
    DeviceState* d = nullptr;
    if ((rc = get_device_state(&d))) return rc;
    const bool sums = dw || db;
    // one size for every type and alignment of such rows
    const size_t need = sums ? ln_workspace(rows, H, d->sm_count) : 0;
    if (sums && (!ws || ws_bytes < need)) return fail(MXFP6_ERR_BAD_ARG, "%s: workspace too small: need %zu bytes, got %zu", what, need, ws ? ws_bytes : 0);
    if (sums && ((uintptr_t)ws & 15)) return fail(MXFP6_ERR_BAD_ARG, "%s: workspace must be 16-byte aligned", what);
    // (the sums are written when all else has been read, but into no other result, and the workspace while rows are read and written)
    if (sums && ((rc = ln_apart(what, {{"the workspace", ws, need}}, {dx_range, dw_range, db_range, x_range, dy_range, w_range, mean_range, rstd_range})) ||
                 (rc = ln_apart(what, {dx_range, dw_range, db_range}, {}, true))))
        return rc;
    const LnRows place = ln_rows(H, x_dtype, w, nullptr, x, dy, dx);
    LnParams P{};
    P.x = x; P.dy = dy; P.y = dx; P.w = w; P.w_bf16 = w_dtype;
    P.mean = const_cast<float*>(mean); P.rstd = const_cast<float*>(rstd);
    P.part = sums ? (float*)ws : nullptr;
    P.rows = rows; P.H = (int)H; P.inv_h = (float)(1.0 / (double)H); P.inv_h_low = (float)(1.0 / (double)H - (double)P.inv_h);
    P.offset = ln_offset(x, x_dtype);
    P.part_ld = place == kLnWhole ? (int)H : ln_part_ld(H);
    const LnChoice k = x_dtype == 0 ? ln_backward_kernel<float>(place, (int)H) : ln_backward_kernel<__nv_bfloat16>(place, (int)H);
    int parts;
    if (k.kern) {
        parts = ln_grid(rows, k.warps, place == kLnOdd, ln_backward_cap(k.warps, d->sm_count, rows, x_dtype == 0 ? 4 : 2), &P.step);
        if (k.smem > 32 * 1024 && (rc = ensure_smem_attr(*d, (const void*)k.kern, 4 * kLnBackwardWide + 64 + 2 * 2 * 4 * 512 * 16))) return rc;
        if ((rc = launch_pdl(k.kern, (unsigned)parts, (unsigned)(k.warps == 1 ? 256 : 32 * k.warps), (size_t)k.smem, st, P))) return rc;
    } else {
        parts = ln_parts_columns(rows, H, d->sm_count);
        if (sums) {
            const LnKernel columns = x_dtype == 0 ? layer_norm_columns_kernel<float> : layer_norm_columns_kernel<__nv_bfloat16>;
            columns<<<dim3((unsigned)((H + 255) / 256), (unsigned)parts), 256, 0, st>>>(P);
            CUDA_TRY(cudaGetLastError());
        }
        const bool vec = place == kLnWhole;
        const LnKernel over = x_dtype == 0 ? (vec ? layer_norm_backward_long_kernel<float, 8> : layer_norm_backward_long_kernel<float, 1>)
                                        : (vec ? layer_norm_backward_long_kernel<__nv_bfloat16, 8> : layer_norm_backward_long_kernel<__nv_bfloat16, 1>);
        const int64_t cap = 2 * (int64_t)d->sm_count;
        if ((rc = launch_pdl(over, (unsigned)(rows < cap ? rows : cap), 1024, 0, st, P))) return rc;
    }
    if (!sums) return MXFP6_OK;
    return launch_pdl(layer_norm_fold_kernel, (unsigned)((2 * H + 31) / 32), 1024, 0, st, (const float*)ws, parts, (int)H, P.part_ld,
                      k.kern && place == kLnOdd ? 1 : 0, P.offset, dw, db);
}

}  // namespace mxfp6
