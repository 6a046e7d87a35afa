// Layer norm over the rows of a [rows, H] matrix (fp32 or bf16), its gradient, and the form that hands its result on as an MX
// operand.  All sums and statistics are fp32, and 64 bits for the rows whose squares leave the range of fp32.
//
//   forward    mean = sum(x) / H,  var = sum((x - mean)^2) / H,  rstd = 1 / sqrt(var + eps),  y = (x - mean) * rstd * w + b
//   backward   xhat = (x - mean) * rstd,  g = dy * w,
//              dx = (g - sum(g) / H - xhat * sum(g * xhat) / H) * rstd,   dw = sum over rows(dy * xhat),   db = sum over rows(dy)
//
// Both are bound by HBM: forward reads x and writes y once, backward reads x and dy and writes dx once.  A row is held in
// registers between its passes (the variance is the sum of squared distances from the mean, not E[x^2] - mean^2, which loses
// every digit of rows whose mean is far above their spread; the second pass also sums the distances themselves, whose mean is
// what the first pass's rounding left out of the mean).  One warp or one CTA owns a row; CTAs are persistent.
//
// The parameter gradients: every CTA sums its rows in registers (each thread owns the same columns of every row) and writes one
// partial per column; a second kernel adds the partials in a fixed order, so results do not depend on timing.
#pragma once
#include <cuda_bf16.h>

#include "ptx.cuh"
#include "quant.cuh"

namespace mxfp6 {

struct LnParams {
    const void* x;           // [rows, H]
    const void* dy;          // backward: [rows, H]
    void* y;                 // forward: result, [rows, H] in x's type; backward: dx
    const void* w;           // [H] or null (ones)
    const void* b;           // [H] or null (zeros)
    int w_bf16;              // type of w and b: 0 = fp32, 1 = bf16
    float* mean;             // [rows]; forward: may be null, like rstd
    float* rstd;             // [rows]
    float* part;             // backward: [grid][2][part_ld] partial sums of dw and db, or null when they are not wanted
    uint8_t* q_out;          // forward to an MX operand: codes [rows, H * bits / 8] ...
    uint8_t* q_scales;       // ... and scales [rows, H / 32]
    int64_t rows;
    int64_t step;            // rows from one of a thread's rows to its next
    int H;
    int offset;              // elements from a chunk boundary (16 or 32 bytes) back to the first row's start
    float inv_h, inv_h_low;  // 1 / H as the sum of two fp32 values
    float eps;
    int part_ld;             // H, or the row's place among its chunks: element col + a of a vector, like the row itself
};
// x / H with one rounding of x's size (1 / H rounded to fp32 alone would add as much again to every mean and variance); x finite
__device__ __forceinline__ float over_h(const LnParams& P, float x) { return fmaf(x, P.inv_h_low, x * P.inv_h); }
// ... and an infinite x stays infinite: its product with the low part, which may be 0 or negative, is left out
__device__ __forceinline__ float over_h_inf(const LnParams& P, float x) {
    const float t = x * P.inv_h;
    return isinf(t) ? t : fmaf(x, P.inv_h_low, t);
}

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// V consecutive elements as they lie in memory (V = 8: one 16- or 32-byte load; V = 1: any alignment), not kept in L1.
template <typename T, int V> struct Raw { uint32_t u[V == 8 ? (sizeof(T) == 4 ? 8 : 4) : 1]; };

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> ld_raw(const T* p) {
    Raw<T, V> r;
    if constexpr (V == 8 && sizeof(T) == 4) {
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3]), "=r"(r.u[4]), "=r"(r.u[5]), "=r"(r.u[6]), "=r"(r.u[7]) : "l"(p) : "memory");
    } else if constexpr (V == 8) {
        asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3]) : "l"(p) : "memory");
    } else if constexpr (sizeof(T) == 4) {
        r.u[0] = *reinterpret_cast<const volatile uint32_t*>(p);
    } else {
        r.u[0] = *reinterpret_cast<const volatile uint16_t*>(p);
    }
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __uint_as_float(r.u[i]);
    } else if constexpr (V == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(r.u[i]); v[2 * i + 1] = bf16_hi(r.u[i]); }
    } else {
        v[0] = bf16_lo(r.u[0]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void st_row(T* p, const float (&v)[V]) {
    if constexpr (V == 8 && sizeof(T) == 4) {
        st_global_v8(p, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]),
                     __float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else if constexpr (V == 8) {
        uint4 q;
        q.x = pack_bf16x2(v[0], v[1]); q.y = pack_bf16x2(v[2], v[3]); q.z = pack_bf16x2(v[4], v[5]); q.w = pack_bf16x2(v[6], v[7]);
        *reinterpret_cast<uint4*>(p) = q;
    } else if constexpr (sizeof(T) == 4) {
        *p = v[0];
    } else {
        *p = __float2bfloat16_rn(v[0]);
    }
}
// V elements of a parameter vector (fill where there is none).  Plain loads, which the wait for the preceding kernel orders and which
// the CTAs of an SM share in L1 (not the read-only path, which promises nothing about a kernel that was still writing; loads that
// go past L1 cost 16 x 8192 a microsecond and rows that start anywhere 20 to 40 %)
template <int V>
__device__ __forceinline__ void ld_param(const void* w, int is_bf16, int col, float fill, float (&v)[V]) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = fill;
    } else if (is_bf16) {
        const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(w) + col;
        if constexpr (V == 8) {
            const uint4 q = *reinterpret_cast<const uint4*>(p);
            const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(u[i]); v[2 * i + 1] = bf16_hi(u[i]); }
        } else {
            v[0] = bf16_lo(*reinterpret_cast<const unsigned short*>(p));
        }
    } else {
        const float* p = reinterpret_cast<const float*>(w) + col;
        if constexpr (V == 8) {
            const float4 a = *reinterpret_cast<const float4*>(p), c = *reinterpret_cast<const float4*>(p + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = c.x; v[5] = c.y; v[6] = c.z; v[7] = c.w;
        } else {
            v[0] = *p;
        }
    }
}

// Sums of N values over the WARPS warps that share a row (one warp: shuffles alone).  `red` has N * WARPS floats per call of a
// row pass; the barrier in front of the reads is the only one a pass needs because consecutive passes use different buffers.
template <int N, int WARPS>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    if constexpr (WARPS > 1) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) red[n * WARPS + warp] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float s = lane < WARPS ? red[n * WARPS + lane] : 0.f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
                if (o < WARPS) s += __shfl_xor_sync(0xffffffffu, s, o);
            v[n] = WARPS < 32 ? __shfl_sync(0xffffffffu, s, 0) : s;
        }
    }
}

// C chunks of eight fp32 values, each a quarter of a 32-element block held by four consecutive lanes -> codes and scales; chunk c holds
// the elements from col + c * stride on.  Step by step for all chunks, so that their shuffles are in flight together.
template <int FMT, int C>
__device__ __forceinline__ void mx_store(float2 (&v)[C][4], uint8_t* codes_row, uint8_t* scales_row, int col, int stride, int cols) {
    float amax[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
        amax[c] = amax3(amax3(v[c][0].x, v[c][0].y, v[c][1].x), amax3(v[c][1].y, v[c][2].x, v[c][2].y), fmaxf(fabsf(v[c][3].x), fabsf(v[c][3].y)));
#pragma unroll
    for (int c = 0; c < C; ++c) amax[c] = fmaxf(amax[c], __shfl_xor_sync(0xffffffffu, amax[c], 1));
#pragma unroll
    for (int c = 0; c < C; ++c) amax[c] = fmaxf(amax[c], __shfl_xor_sync(0xffffffffu, amax[c], 2));
    const int j = (col >> 3) & 3;                   // place of these eight in their block (the stride is a multiple of 32)
    uint32_t w0[C], w1[C];
    int sb[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        sb[c] = quant_scale_byte(amax[c], FMT);
        const float f = quant_inv_scale(sb[c]);
        float s[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __fmul2_rn(v[c][i], make_float2(f, f));
            s[2 * i] = t.x; s[2 * i + 1] = t.y;
        }
        if constexpr (FMT == kE2M1) {
            w0[c] = cvt_oct_e2m1(s);
            w1[c] = 0;
        } else {
            const uint32_t lo = cvt_quad<FMT>(s[0], s[1], s[2], s[3]), hi = cvt_quad<FMT>(s[4], s[5], s[6], s[7]);
            // 6-bit codes: 24 bits each, 48 a lane
            w0[c] = fmt_fp8(FMT) ? lo : lo | (hi << 24);
            w1[c] = fmt_fp8(FMT) ? hi : hi >> 8;
        }
    }
    if constexpr (FMT == kE2M1 || fmt_fp8(FMT)) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = col + c * stride;
            if (at >= cols) continue;
            if constexpr (FMT == kE2M1) *reinterpret_cast<uint32_t*>(codes_row + at / 2) = w0[c];
            else *reinterpret_cast<uint2*>(codes_row + at) = make_uint2(w0[c], w1[c]);
        }
    } else {
        // four lanes hold 24 bytes, which three of them write, 8 each: lane j the bits from 64 j on, which start at bit 16 j of its
        // own 48 and run on into its neighbour's
        uint32_t n0[C], n1[C];
#pragma unroll
        for (int c = 0; c < C; ++c) { n0[c] = __shfl_down_sync(0xffffffffu, w0[c], 1); n1[c] = __shfl_down_sync(0xffffffffu, w1[c], 1); }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = col + c * stride;
            const uint32_t a = j == 2 ? w1[c] : w0[c], b = j == 2 ? n0[c] : w1[c], d = j == 2 ? n1[c] : n0[c];
            const uint32_t o0 = __byte_perm(a, b, j == 0 ? 0x3210 : j == 1 ? 0x5432 : 0x5410);
            const uint32_t o1 = __byte_perm(b, d, j == 0 ? 0x5410 : j == 1 ? 0x7654 : 0x5432);
            if (at < cols && j < 3) *reinterpret_cast<uint2*>(codes_row + (at / 32) * 24 + 8 * j) = make_uint2(o0, o1);
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
        if (col + c * stride < cols && j == 0) scales_row[(col + c * stride) / 32] = (uint8_t)sb[c];
}

// A row that fp32 statistics cannot carry, by the TPR = 32 * WARPS threads that share it, in 64 bits and straight from memory: the sum
// or the sum of squares overflows (values past about 1e17), the squares vanish below the range and eps does not cover them, or
// the row holds an infinity or a NaN (whose mean and rstd come out as the formulas give them).  Not inlined: no
// register of the usual path is held for it.  Three passes with one element per load: 16384 x 8192 bf16, every row of that kind, 0.85 ms
// against 0.095.
template <int WARPS>
__device__ __forceinline__ double row_sum64(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (WARPS > 1) {
        __syncthreads();                                        // (what the buffer held has been read)
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0;
        for (int w = 0; w < WARPS; ++w) v += red[w];
    }
    return v;
}
template <typename T, int WARPS, int FMT>
__device__ __noinline__ void norm_row_64(const LnParams P, int64_t row, int tid, double* red) {
    constexpr int TPR = 32 * WARPS;
    const T* x = reinterpret_cast<const T*>(P.x) + row * P.H;
    auto at = [&](int col) {
        float v[1];
        unpack<T, 1>(ld_raw<T, 1>(x + col), v);
        return (double)v[0];
    };
    double s = 0.0, q = 0.0;
    for (int col = tid; col < P.H; col += TPR) s += at(col);
    const double mean = row_sum64<WARPS>(s, red) / P.H;
    for (int col = tid; col < P.H; col += TPR) {
        const double d = at(col) - mean;
        q += d * d;
    }
    const double rstd = 1.0 / sqrt(row_sum64<WARPS>(q, red) / P.H + (double)P.eps);
    if (tid == 0) {
        if (P.mean) P.mean[row] = (float)mean;
        if (P.rstd) P.rstd[row] = (float)rstd;
    }
    auto result = [&](int col) {
        float w[1], b[1];
        ld_param<1>(P.w, P.w_bf16, col, 1.f, w);
        ld_param<1>(P.b, P.w_bf16, col, 0.f, b);
        return (float)((at(col) - mean) * rstd * (double)w[0] + (double)b[0]);
    };
    if constexpr (FMT < 0) {
        for (int col = tid; col < P.H; col += TPR) {
            const float v[1] = {result(col)};
            st_row<T, 1>(reinterpret_cast<T*>(P.y) + row * P.H + col, v);
        }
    } else {
        // every thread makes the same number of rounds: the lanes of a block exchange their largest magnitudes
        for (int c0 = 0; c0 < P.H; c0 += 8 * TPR) {
            const int col = c0 + 8 * tid;
            float v[8];
#pragma unroll 1
            for (int i = 0; i < 8; ++i) v[i] = col < P.H ? result(col + i) : 0.f;
            float2 o[1][4] = {{make_float2(v[0], v[1]), make_float2(v[2], v[3]), make_float2(v[4], v[5]), make_float2(v[6], v[7])}};
            mx_store<FMT, 1>(o, P.q_out + row * (P.H / 32) * fmt_block_bytes(FMT), P.q_scales + row * (P.H / 32), col, 0, P.H);
        }
    }
}
// Does the sum of squares of a row say that it is such a row?  (A sum that is not finite makes it so too.)  Below 2^-100 it has lost digits to
// the end of the range, which matter where eps is small beside the variance.  (The bound is made here: as a member of LnParams it moved
// the registers of the MX forms about, E2M3 113 -> 119 us.)
__device__ __forceinline__ bool beyond_fp32(const LnParams& P, float q) { return !(q >= (P.eps < 0x1p-70f ? 0x1p-100f : 0.f) && q <= 3.402823466e38f); }

// ---- rows as chunks of 8 elements
// Rows of whole, aligned chunks (ODD = false) are n = H / 8 chunks.  Other rows are cut at the same 16- or 32-byte boundaries of
// memory: the row starts `a` elements behind a boundary, its first and last chunk may hold neighbours' elements (which are
// masked when read and never written), and column `col` is element col + a of the chunks.  `a` is
// the same for rows that lie a multiple of 8 rows apart, so a CTA takes only such rows, its threads own the same columns in each
// of them, and the parameters are staged once, shifted by a.
template <bool ODD>
struct Chunks {
    int a, n, H;
    __device__ __forceinline__ int lo(int chunk) const { return ODD ? min(max(a - 8 * chunk, 0), 8) : 0; }                // first element of the row in this chunk
    __device__ __forceinline__ int hi(int chunk) const { return ODD ? min(max(a + H - 8 * chunk, 0), 8) : (chunk < n ? 8 : 0); }      // one past its last
    __device__ __forceinline__ bool whole(int chunk) const { return ODD ? 8 * chunk >= a && 8 * chunk + 8 <= a + H : chunk < n; }
};
template <bool ODD>
__device__ __forceinline__ Chunks<ODD> chunks_of(const LnParams& P, int64_t row) {
    Chunks<ODD> k;
    k.H = P.H;
    k.a = ODD ? (int)((P.offset + row * P.H) & 7) : 0;
    k.n = ODD ? (k.a + P.H + 7) >> 3 : P.H >> 3;
    return k;
}
// first row of a group of WARPS warps (warp w of eight when one warp owns a row)
template <bool ODD, int WARPS>
__device__ __forceinline__ int64_t first_row(int w) {
    if constexpr (ODD) return (blockIdx.x & 7) + 8 * ((int64_t)w + (WARPS == 1 ? 8 : 1) * (int64_t)(blockIdx.x >> 3));
    return WARPS == 1 ? (int64_t)blockIdx.x * 8 + w : blockIdx.x;
}
// Chunk `chunk` of the row whose first chunk starts at element `at` of the matrix m (which may be before its first element).  A chunk
// at an end of the row is loaded whole, with what it holds of the neighbouring rows, and masked when it is used (loading it
// element by element would wait for the elements to put them together, a row ahead of their use: 8192 x 4097 bf16 in 95 us);
// only a row whose chunks reach past the matrix (inner = false) is loaded element by element.
template <typename T, bool ODD>
__device__ __forceinline__ void ld_chunk(const T* m, int64_t at, bool inner, int chunk, const Chunks<ODD>& k, Raw<T, 8>& r) {
    if constexpr (!ODD) {
        if (chunk < k.n) r = ld_raw<T, 8>(m + at + 8 * chunk);
    } else if (chunk < k.n) {
        const int64_t e = at + 8 * chunk;
        if (inner) {
            r = ld_raw<T, 8>(m + e);
        } else {
            const int lo = k.lo(chunk), hi = k.hi(chunk);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t u = 0;
                if (i >= lo && i < hi) u = ld_raw<T, 1>(m + e + i).u[0];
                if constexpr (sizeof(T) == 4) r.u[i] = u;
                else r.u[i >> 1] = (i & 1) ? r.u[i >> 1] | (u << 16) : u;
            }
        }
    }
}
// zeros for the elements of a chunk that belong to other rows
template <typename T>
__device__ __forceinline__ void mask_chunk(const Chunks<true>& k, int chunk, Raw<T, 8>& r) {
    const int lo = k.lo(chunk), hi = k.hi(chunk);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < lo || i >= hi) r.u[i] = 0;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r.u[i] &= (2 * i >= lo && 2 * i < hi ? 0xffffu : 0u) | (2 * i + 1 >= lo && 2 * i + 1 < hi ? 0xffff0000u : 0u);
    }
}
// `value` for the elements of a chunk that belong to other rows
__device__ __forceinline__ void fill_outside(const Chunks<true>& k, int chunk, float value, float2 (&v)[4]) {
    const int lo = k.lo(chunk), hi = k.hi(chunk);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (2 * i < lo || 2 * i >= hi) v[i].x = value;
        if (2 * i + 1 < lo || 2 * i + 1 >= hi) v[i].y = value;
    }
}
// Parameter vectors in shared memory, as fp32 whatever their type and filled where they are absent: float4 planes of n chunks
// (the low halves, then the high halves), so that neighbouring threads read neighbouring 16 bytes.
template <bool ODD>
__device__ __forceinline__ void stage_param(const void* w, int is_bf16, float fill, const Chunks<ODD>& k, float4* plane) {
    for (int c = threadIdx.x; c < k.n; c += blockDim.x) {
        float v[8];
        if constexpr (ODD) {
            // eight loads in flight whatever the chunk holds of the row (one after another, this staging alone took 5 us of a call)
            const int lo = k.lo(c), hi = k.hi(c);
            int col[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) col[i] = min(max(8 * c - k.a + i, 0), k.H - 1);
            if (!w) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = fill;
            } else if (is_bf16) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = bf16_lo(reinterpret_cast<const unsigned short*>(w)[col[i]]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = reinterpret_cast<const float*>(w)[col[i]];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < lo || i >= hi) v[i] = 0.f;
        } else {
            ld_param<8>(w, is_bf16, 8 * c, fill, v);
        }
        plane[c] = make_float4(v[0], v[1], v[2], v[3]);
        plane[k.n + c] = make_float4(v[4], v[5], v[6], v[7]);
    }
}
__device__ __forceinline__ void ld_staged(const float4* plane, int n, int chunk, float2 (&v)[4]) {
    const float4 lo = plane[chunk], hi = plane[n + chunk];
    v[0] = make_float2(lo.x, lo.y); v[1] = make_float2(lo.z, lo.w); v[2] = make_float2(hi.x, hi.y); v[3] = make_float2(hi.z, hi.w);
}
template <typename T>
__device__ __forceinline__ void unpack2(const Raw<T, 8>& r, float2 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = make_float2(__uint_as_float(r.u[2 * i]), __uint_as_float(r.u[2 * i + 1]));
        else v[i] = make_float2(bf16_lo(r.u[i]), bf16_hi(r.u[i]));
    }
}
template <typename T>
__device__ __forceinline__ void st_row2(T* p, const float2 (&v)[4]) {
    const float t[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
    st_row<T, 8>(p, t);
}

template <typename T, bool ODD>
__device__ __forceinline__ void st_chunk(T* rowp, int chunk, const Chunks<ODD>& k, const float2 (&v)[4]) {
    if (k.whole(chunk)) {
        st_row2<T>(rowp + 8 * chunk, v);
    } else if constexpr (ODD) {
        const float t[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
        const int lo = k.lo(chunk), hi = k.hi(chunk);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float o[1] = {t[i]};
            if (i >= lo && i < hi) st_row<T, 1>(rowp + 8 * chunk + i, o);
        }
    }
}

// ---------------------------------------------------------------------------------- forward
// WARPS warps own a row, C chunks of 8 elements per thread.  WARPS = 1: eight warps per CTA with a row each.  FMT < 0: the result is
// written in x's type; otherwise it leaves as codes and scales.  The next row is on its way in registers while this one is worked
// on, the arithmetic runs on pairs (fma.f32x2), and the parameters are staged once per CTA: bf16 rows are bound by issue, not by
// HBM, when each element costs 25 instructions (16384 x 8192 in 124 us).  Threads whose columns lie past H take part in everything
// but the stores, on zeros: a branch per chunk would keep the chunks' instructions from being interleaved.
template <typename T, int C, int WARPS, int FMT, bool ODD>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : 32 * WARPS, WARPS == 1 ? 2 : 16 / WARPS)
layer_norm_kernel(const LnParams P) {
    constexpr int TPR = 32 * WARPS;
    static_assert(!ODD || FMT < 0, "an MX result has whole blocks");
    // the chunks' codes made together (16384 x 8192 bf16: E2M1 100 us, 104 one by one; E4M3 100, 105) or, where that takes too many
    // registers, one by one (E2M3 111 us, 124 together)
    constexpr bool together = FMT == kE2M1 || fmt_fp8(FMT);
    __shared__ float red[2][WARPS], red2[2][2 * WARPS];         // [row parity]
    __shared__ double red64[WARPS];
    extern __shared__ float4 prm[];                             // w, then b
    pdl_launch_dependents();
    pdl_wait();
    const int tid = WARPS == 1 ? (threadIdx.x & 31) : threadIdx.x;
    int64_t row = first_row<ODD, WARPS>(WARPS == 1 ? threadIdx.x >> 5 : 0);
    const Chunks<ODD> K = chunks_of<ODD>(P, row);
    const T* x = reinterpret_cast<const T*>(P.x);
    const int64_t elements = P.rows * P.H;
    Raw<T, 8> raw[C];
    auto load = [&](int64_t r) {
        if (r < P.rows) {
            const int64_t at = r * P.H - K.a;
            const bool inner = at >= 0 && at + 8 * K.n <= elements;
#pragma unroll
            for (int c = 0; c < C; ++c) ld_chunk<T, ODD>(x, at, inner, tid + c * TPR, K, raw[c]);
        }
    };
    auto begin = [&](int64_t r) {
#pragma unroll
        for (int c = 0; c < C; ++c) raw[c] = Raw<T, 8>{};       // elements outside the row stay zero
        load(r);
    };
    begin(row);
    stage_param(P.w, P.w_bf16, 1.f, K, prm);
    stage_param(P.b, P.w_bf16, 0.f, K, prm + 2 * K.n);
    // does this warp hold elements outside the row?  (one decision per row; the same for all of this thread's rows)
    bool inside = true;
#pragma unroll
    for (int c = 0; c < C; ++c) inside = inside && K.whole(tid + c * TPR);
    const bool edge = !__all_sync(0xffffffffu, inside);
    __syncthreads();
    for (int par = 0;; par ^= 1) {
        for (; row < P.rows; row += P.step, par ^= 1) {
            float2 v[C][4];
            if constexpr (ODD) {
                if (edge)
#pragma unroll
                    for (int c = 0; c < C; ++c) mask_chunk<T>(K, tid + c * TPR, raw[c]);
            }
#pragma unroll
            for (int c = 0; c < C; ++c) unpack2<T>(raw[c], v[c]);
            load(row + P.step);
            float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) s2 = __fadd2_rn(s2, v[c][i]);
            float s[1] = {s2.x + s2.y};
            row_sum<1, WARPS>(s, red[par]);
            const float mean0 = over_h(P, s[0]);
            float2 q2 = make_float2(0.f, 0.f), d2 = make_float2(0.f, 0.f);
            if (ODD && edge) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int lo = K.lo(tid + c * TPR), hi = K.hi(tid + c * TPR);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 m = make_float2(2 * i >= lo && 2 * i < hi ? -mean0 : 0.f, 2 * i + 1 >= lo && 2 * i + 1 < hi ? -mean0 : 0.f);
                        v[c][i] = __fadd2_rn(v[c][i], m);
                        q2 = __ffma2_rn(v[c][i], v[c][i], q2);
                        d2 = __fadd2_rn(d2, v[c][i]);
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const float m = ODD || tid + c * TPR < K.n ? -mean0 : 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[c][i] = __fadd2_rn(v[c][i], make_float2(m, m));
                        q2 = __ffma2_rn(v[c][i], v[c][i], q2);
                        d2 = __fadd2_rn(d2, v[c][i]);
                    }
                }
            }
            float q[2] = {q2.x + q2.y, d2.x + d2.y};
            row_sum<2, WARPS>(q, red2[par]);
            if (beyond_fp32(P, q[0])) break;                        // (equal for all threads of the row)
            const float corr = over_h(P, q[1]);
            const float rstd = 1.f / sqrtf(fmaxf(fmaf(-corr, corr, over_h(P, q[0])), 0.f) + P.eps);
            if (tid == 0) {
                if (P.mean) P.mean[row] = mean0 + corr;
                if (P.rstd) P.rstd[row] = rstd;
            }
            const float shift = -corr * rstd;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int chunk = tid + c * TPR;
                const bool live = chunk < K.n;
                float2 w[4], b[4];
                ld_staged(prm, K.n, live ? chunk : 0, w);
                ld_staged(prm + 2 * K.n, K.n, live ? chunk : 0, b);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[c][i] = __ffma2_rn(__ffma2_rn(v[c][i], make_float2(rstd, rstd), make_float2(shift, shift)), w[i], b[i]);
                if constexpr (FMT < 0) {
                    st_chunk<T, ODD>(reinterpret_cast<T*>(P.y) + row * P.H - K.a, chunk, K, v[c]);
                } else if constexpr (!together) {
                    float2 o[1][4] = {{v[c][0], v[c][1], v[c][2], v[c][3]}};
                    mx_store<FMT, 1>(o, P.q_out + row * (P.H / 32) * fmt_block_bytes(FMT), P.q_scales + row * (P.H / 32), 8 * chunk, 0, P.H);
                }
            }
            if constexpr (FMT >= 0 && together)
                mx_store<FMT, C>(v, P.q_out + row * (P.H / 32) * fmt_block_bytes(FMT), P.q_scales + row * (P.H / 32), 8 * tid, 8 * TPR, P.H);
        }
        if (row >= P.rows) break;
        // (the call stands outside the loop over the rows: inside it E2M1 takes 105 us instead of 101, E4M3 106 instead of 101)
        norm_row_64<T, WARPS, FMT>(P, row, tid, red64);
        row += P.step;
        begin(row);
    }
}

// Rows longer than the registers of a CTA hold, and rows of x and y that lie differently in their 16- or 32-byte units (V = 1): a CTA
// of 1024 threads passes over its row three times (the second and third pass find it in L2).
template <typename T, int V, int FMT>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(const LnParams P) {
    __shared__ float red[32], red2[64];
    __shared__ double red64[32];
    pdl_launch_dependents();
    pdl_wait();
    const T* x = reinterpret_cast<const T*>(P.x);
    for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x) {
        const T* xr = x + row * P.H;
        float s[1] = {0.f};
        for (int col = threadIdx.x * V; col < P.H; col += 1024 * V) {
            float v[V];
            unpack<T, V>(ld_raw<T, V>(xr + col), v);
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += v[i];
        }
        row_sum<1, 32>(s, red);
        const float mean0 = over_h(P, s[0]);
        float q[2] = {0.f, 0.f};
        for (int col = threadIdx.x * V; col < P.H; col += 1024 * V) {
            float v[V];
            unpack<T, V>(ld_raw<T, V>(xr + col), v);
#pragma unroll
            for (int i = 0; i < V; ++i) { const float d = v[i] - mean0; q[0] = fmaf(d, d, q[0]); q[1] += d; }
        }
        row_sum<2, 32>(q, red2);
        if (beyond_fp32(P, q[0])) {
            norm_row_64<T, 32, FMT>(P, row, threadIdx.x, red64);
            continue;
        }
        const float corr = over_h(P, q[1]);
        const float rstd = 1.f / sqrtf(fmaxf(fmaf(-corr, corr, over_h(P, q[0])), 0.f) + P.eps);
        if (threadIdx.x == 0 && P.mean) P.mean[row] = mean0 + corr;
        if (threadIdx.x == 0 && P.rstd) P.rstd[row] = rstd;
        const float shift = -corr * rstd;
        // every thread makes the same number of rounds: the lanes of a block exchange their largest magnitudes
        for (int c0 = 0; c0 < P.H; c0 += 1024 * V) {
            const int col = c0 + threadIdx.x * V;
            const bool live = col < P.H;
            float v[V], w[V], b[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = 0.f;
            if (live) {
                unpack<T, V>(ld_raw<T, V>(xr + col), v);
                ld_param<V>(P.w, P.w_bf16, col, 1.f, w);
                ld_param<V>(P.b, P.w_bf16, col, 0.f, b);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = fmaf(fmaf(v[i] - mean0, rstd, shift), w[i], b[i]);
            }
            if constexpr (FMT >= 0) {
                float2 o[1][4] = {{make_float2(v[0], v[1]), make_float2(v[2], v[3]), make_float2(v[4], v[5]), make_float2(v[6], v[7])}};
                mx_store<FMT, 1>(o, P.q_out + row * (P.H / 32) * fmt_block_bytes(FMT), P.q_scales + row * (P.H / 32), col, 0, P.H);
            } else if (live) {
                st_row<T, V>(reinterpret_cast<T*>(P.y) + row * P.H + col, v);
            }
        }
    }
}

// a thread's column sums to their chunks of a partial vector
template <int C, int TPR, bool ODD>
__device__ __forceinline__ void st_sums(float* out, int tid, const Chunks<ODD>& k, const float2 (&v)[C][4]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int chunk = tid + c * TPR;
        if (chunk >= k.n) continue;
        float4* o = reinterpret_cast<float4*>(out + 8 * chunk);
        o[0] = make_float4(v[c][0].x, v[c][0].y, v[c][1].x, v[c][1].y);
        o[1] = make_float4(v[c][2].x, v[c][2].y, v[c][3].x, v[c][3].y);
    }
}

// ---------------------------------------------------------------------------------- backward
// WARPS warps own a row, C chunks of 8 columns per thread; the same columns of every row, whose parameter gradients the thread
// sums in registers.  As in the forward kernel the next row is on its way while this one is worked on (without that, HBM idles
// through every row's reduction: 16384 x 8192 bf16 in 273 us) and the arithmetic runs on pairs.
template <typename T, int C, int WARPS, bool ODD>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : 32 * WARPS, WARPS == 1 ? 2 : 16 / WARPS)
layer_norm_backward_kernel(const LnParams P) {
    constexpr int TPR = 32 * WARPS;
    __shared__ float red[2][2 * WARPS];
    extern __shared__ float4 prm[];                             // w; at the end the warps' column sums (one warp per row)
    pdl_launch_dependents();
    pdl_wait();
    const int tid = WARPS == 1 ? (threadIdx.x & 31) : threadIdx.x;
    int64_t row = first_row<ODD, WARPS>(WARPS == 1 ? threadIdx.x >> 5 : 0);
    const Chunks<ODD> K = chunks_of<ODD>(P, row);
    const T* x = reinterpret_cast<const T*>(P.x);
    const T* dy = reinterpret_cast<const T*>(P.dy);
    const int64_t elements = P.rows * P.H;
    Raw<T, 8> rx[C], rg[C];
    float mean_n = 0.f, rstd_n = 0.f;
    auto load = [&](int64_t r) {
        if (r < P.rows) {
            const int64_t at = r * P.H - K.a;
            const bool inner = at >= 0 && at + 8 * K.n <= elements;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                ld_chunk<T, ODD>(x, at, inner, tid + c * TPR, K, rx[c]);
                ld_chunk<T, ODD>(dy, at, inner, tid + c * TPR, K, rg[c]);
            }
            mean_n = __ldcg(P.mean + r);
            rstd_n = __ldcg(P.rstd + r);
        }
    };
    float2 dw[C][4], db[C][4];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        rx[c] = Raw<T, 8>{}; rg[c] = Raw<T, 8>{};
#pragma unroll
        for (int i = 0; i < 4; ++i) dw[c][i] = db[c][i] = make_float2(0.f, 0.f);
    }
    load(row);
    stage_param(P.w, P.w_bf16, 1.f, K, prm);
    bool inside = true;
#pragma unroll
    for (int c = 0; c < C; ++c) inside = inside && K.whole(tid + c * TPR);
    const bool edge = !__all_sync(0xffffffffu, inside);         // (one decision per row, as in the forward kernel)
    __syncthreads();
    for (int par = 0; row < P.rows; row += P.step, par ^= 1) {
        const float mean = mean_n, rstd = rstd_n;
        float2 xh[C][4], g[C][4];
        if constexpr (ODD) {
            if (edge)
#pragma unroll
                for (int c = 0; c < C; ++c) { mask_chunk<T>(K, tid + c * TPR, rx[c]); mask_chunk<T>(K, tid + c * TPR, rg[c]); }
        }
#pragma unroll
        for (int c = 0; c < C; ++c) { unpack2<T>(rx[c], xh[c]); unpack2<T>(rg[c], g[c]); }
        if constexpr (ODD) {
            // (dy is zero outside the row, and so are its products, unless the zero that stands there for x lies infinitely many rstd from the mean)
            if (edge && isinf(mean * rstd))
#pragma unroll
                for (int c = 0; c < C; ++c) fill_outside(K, tid + c * TPR, mean, xh[c]);
        }
        load(row + P.step);
        float2 a2 = make_float2(0.f, 0.f), b2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            // (outside the row dy is zero, and so is all that is summed)
            // (the branch costs nothing here and keeps the registers of fp32 rows down: 16384 x 8192 in 256 us, 279 without it)
            const int chunk = tid + c * TPR;
            if (chunk >= K.n) continue;
            float2 w[4];
            ld_staged(prm, K.n, chunk, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // (the distance from the mean is taken before the scaling: x * rstd - mean * rstd loses digits of rows far from zero)
                xh[c][i] = __fmul2_rn(__fadd2_rn(xh[c][i], make_float2(-mean, -mean)), make_float2(rstd, rstd));
                dw[c][i] = __ffma2_rn(g[c][i], xh[c][i], dw[c][i]);
                db[c][i] = __fadd2_rn(db[c][i], g[c][i]);
                g[c][i] = __fmul2_rn(g[c][i], w[i]);
                a2 = __fadd2_rn(a2, g[c][i]);
                b2 = __ffma2_rn(g[c][i], xh[c][i], b2);
            }
        }
        float s[2] = {a2.x + a2.y, b2.x + b2.y};
        row_sum<2, WARPS>(s, red[par]);
        const float m1 = -over_h_inf(P, s[0]), m2 = -over_h_inf(P, s[1]);
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                g[c][i] = __fmul2_rn(__fadd2_rn(g[c][i], __ffma2_rn(xh[c][i], make_float2(m2, m2), make_float2(m1, m1))), make_float2(rstd, rstd));
            st_chunk<T, ODD>(reinterpret_cast<T*>(P.y) + row * P.H - K.a, tid + c * TPR, K, g[c]);
        }
    }
    if (!P.part) return;
    float* out = P.part + (int64_t)blockIdx.x * 2 * P.part_ld;
    if constexpr (WARPS == 1) {
        // eight warps hold sums of the same columns
        float* fold = reinterpret_cast<float*>(prm);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    reinterpret_cast<float2*>(fold)[(threadIdx.x >> 5) * (TPR * 4 * C) + (tid + c * TPR) * 4 + i] = k ? db[c][i] : dw[c][i];
            __syncthreads();
            for (int col = threadIdx.x; col < P.H; col += 256) {
                float a = 0.f;
#pragma unroll
                for (int r = 0; r < 8; ++r) a += fold[r * (TPR * 8 * C) + K.a + col];
                out[(int64_t)k * P.part_ld + K.a + col] = a;
            }
        }
    } else {
        st_sums<C, TPR, ODD>(out, tid, K, dw);
        st_sums<C, TPR, ODD>(out + P.part_ld, tid, K, db);
    }
}

// bf16 rows of 8192 to 16384 elements: four chunks per thread, whose column sums alone take 64 of its 128 registers.  x and dy of
// the next two rows are copied by cp.async into slots of shared memory that only this thread reads (no barrier), and both passes
// over a row read them there (4096 x 16384 in 81 us; passing over global memory again and summing the columns in a kernel of
// their own took 311 us).
template <bool ODD>
__global__ void __launch_bounds__(512, 1) layer_norm_backward_wide_kernel(const LnParams P) {
    typedef __nv_bfloat16 T;
    constexpr int C = 4, D = 2, TPR = 512, SLOT = TPR * 16;
    __shared__ float red[2][2 * 16];
    extern __shared__ float4 prm[];                             // w, then the slots: [x, dy][row][chunk][thread]
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x;
    int64_t row = blockIdx.x;
    const Chunks<ODD> K = chunks_of<ODD>(P, row);
    const T* x = reinterpret_cast<const T*>(P.x);
    const T* dy = reinterpret_cast<const T*>(P.dy);
    const int64_t elements = P.rows * P.H;
    const uint32_t sx = smem_u32(prm + 2 * K.n) + tid * 16, sg = sx + D * C * SLOT;
    auto put = [&](uint32_t slot, const Raw<T, 8>& r) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot), "r"(r.u[0]), "r"(r.u[1]), "r"(r.u[2]), "r"(r.u[3]) : "memory");
    };
    auto get = [&](uint32_t slot) {
        Raw<T, 8> r;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3]) : "r"(slot) : "memory");
        return r;
    };
    // columns past H are never copied and stay zero
#pragma unroll
    for (int i = 0; i < 2 * D * C; ++i) put(sx + i * SLOT, Raw<T, 8>{});
    auto load = [&](int d, int64_t r) {
        if (r < P.rows) {
            const int64_t at = r * P.H - K.a;
            const bool inner = at >= 0 && at + 8 * K.n <= elements;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int chunk = tid + c * TPR;
                const uint32_t px = sx + (d * C + c) * SLOT, pg = sg + (d * C + c) * SLOT;
                if (chunk >= K.n) continue;
                if (!ODD || inner) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(px), "l"(x + at + 8 * chunk) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(pg), "l"(dy + at + 8 * chunk) : "memory");
                } else {
                    Raw<T, 8> t{};
                    ld_chunk<T, ODD>(x, at, false, chunk, K, t);
                    put(px, t);
                    ld_chunk<T, ODD>(dy, at, false, chunk, K, t);
                    put(pg, t);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto take = [&](uint32_t slot, int chunk, float2 (&v)[4]) {
        Raw<T, 8> r = get(slot);
        if constexpr (ODD) {
            if (!K.whole(chunk)) mask_chunk<T>(K, chunk, r);
        }
        unpack2<T>(r, v);
    };
    float2 dw[C][4], db[C][4];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) dw[c][i] = db[c][i] = make_float2(0.f, 0.f);
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, row + d * P.step);
    float mean_n = 0.f, rstd_n = 0.f;
    if (row < P.rows) { mean_n = __ldcg(P.mean + row); rstd_n = __ldcg(P.rstd + row); }
    stage_param(P.w, P.w_bf16, 1.f, K, prm);
    __syncthreads();
    for (int par = 0; row < P.rows; row += P.step, par ^= 1) {
        static_assert(D == 2, "the slot alternates with the parity of the reduction");
        const float mean = mean_n, rstd = rstd_n;
        const int64_t next = row + P.step;
        if (next < P.rows) { mean_n = __ldcg(P.mean + next); rstd_n = __ldcg(P.rstd + next); }
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
        float2 a2 = make_float2(0.f, 0.f), b2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int chunk = tid + c * TPR;
            if (chunk >= K.n) continue;
            float2 xh[4], g[4], w[4];
            take(sx + (par * C + c) * SLOT, chunk, xh);
            take(sg + (par * C + c) * SLOT, chunk, g);
            if constexpr (ODD) {
                if (!K.whole(chunk)) fill_outside(K, chunk, mean, xh);      // (0 - mean may be infinitely many rstd)
            }
            ld_staged(prm, K.n, chunk, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xh[i] = __fmul2_rn(__fadd2_rn(xh[i], make_float2(-mean, -mean)), make_float2(rstd, rstd));
                dw[c][i] = __ffma2_rn(g[i], xh[i], dw[c][i]);
                db[c][i] = __fadd2_rn(db[c][i], g[i]);
                g[i] = __fmul2_rn(g[i], w[i]);
                a2 = __fadd2_rn(a2, g[i]);
                b2 = __ffma2_rn(g[i], xh[i], b2);
            }
        }
        float s[2] = {a2.x + a2.y, b2.x + b2.y};
        row_sum<2, 16>(s, red[par]);
        const float m1 = -over_h_inf(P, s[0]), m2 = -over_h_inf(P, s[1]);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int chunk = tid + c * TPR;
            if (chunk >= K.n) continue;
            float2 xh[4], g[4], w[4];
            take(sx + (par * C + c) * SLOT, chunk, xh);
            take(sg + (par * C + c) * SLOT, chunk, g);
            ld_staged(prm, K.n, chunk, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xh[i] = __fmul2_rn(__fadd2_rn(xh[i], make_float2(-mean, -mean)), make_float2(rstd, rstd));
                g[i] = __fmul2_rn(g[i], w[i]);
                g[i] = __fmul2_rn(__fadd2_rn(g[i], __ffma2_rn(xh[i], make_float2(m2, m2), make_float2(m1, m1))), make_float2(rstd, rstd));
            }
            st_chunk<T, ODD>(reinterpret_cast<T*>(P.y) + row * P.H - K.a, chunk, K, g);
        }
        load(par, row + D * P.step);                            // the slots of this row have been read
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!P.part) return;
    float* out = P.part + (int64_t)blockIdx.x * 2 * P.part_ld;
    st_sums<C, TPR, ODD>(out, tid, K, dw);
    st_sums<C, TPR, ODD>(out + P.part_ld, tid, K, db);
}

// Rows longer than a CTA's registers hold: dx with a second pass over the row, and the parameter gradients by a kernel whose
// threads own a column each and walk down a share of the rows.
template <typename T, int V>
__global__ void __launch_bounds__(1024) layer_norm_backward_long_kernel(const LnParams P) {
    __shared__ float red[2][64];
    pdl_launch_dependents();
    pdl_wait();
    int par = 0;
    for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x, par ^= 1) {
        const T* x = reinterpret_cast<const T*>(P.x) + row * P.H;
        const T* dy = reinterpret_cast<const T*>(P.dy) + row * P.H;
        const float mean = __ldcg(P.mean + row), rstd = __ldcg(P.rstd + row);
        float s[2] = {0.f, 0.f};
        for (int col = threadIdx.x * V; col < P.H; col += 1024 * V) {
            float v[V], g[V], w[V];
            unpack<T, V>(ld_raw<T, V>(x + col), v);
            unpack<T, V>(ld_raw<T, V>(dy + col), g);
            ld_param<V>(P.w, P.w_bf16, col, 1.f, w);
#pragma unroll
            for (int i = 0; i < V; ++i) { const float gw = g[i] * w[i]; s[0] += gw; s[1] = fmaf(gw, (v[i] - mean) * rstd, s[1]); }
        }
        row_sum<2, 32>(s, red[par]);
        const float m1 = over_h_inf(P, s[0]), m2 = over_h_inf(P, s[1]);
        for (int col = threadIdx.x * V; col < P.H; col += 1024 * V) {
            float v[V], g[V], w[V];
            unpack<T, V>(ld_raw<T, V>(x + col), v);
            unpack<T, V>(ld_raw<T, V>(dy + col), g);
            ld_param<V>(P.w, P.w_bf16, col, 1.f, w);
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] = (g[i] * w[i] - fmaf((v[i] - mean) * rstd, m2, m1)) * rstd;
            st_row<T, V>(reinterpret_cast<T*>(P.y) + row * P.H + col, g);
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const LnParams P) {
    pdl_launch_dependents();
    pdl_wait();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= P.H) return;
    const int64_t per = (P.rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = blockIdx.y * per, r1 = r0 + per < P.rows ? r0 + per : P.rows;
    const T* x = reinterpret_cast<const T*>(P.x);
    const T* dy = reinterpret_cast<const T*>(P.dy);
    float dw = 0.f, db = 0.f;
#pragma unroll 4
    for (int64_t r = r0; r < r1; ++r) {
        float v[1], g[1];
        unpack<T, 1>(ld_raw<T, 1>(x + r * P.H + col), v);
        unpack<T, 1>(ld_raw<T, 1>(dy + r * P.H + col), g);
        dw = fmaf(g[0], (v[0] - __ldcg(P.mean + r)) * __ldcg(P.rstd + r), dw);
        db += g[0];
    }
    float* out = P.part + (int64_t)blockIdx.y * 2 * P.part_ld;
    out[col] = dw;
    out[P.part_ld + col] = db;
}

// [parts][2][ld] partial sums -> dw [H], db [H] (either may be null): 32 columns per CTA, 32 threads per column, each adding
// every 32nd partial; the 32 sums meet in shared memory in a fixed order.  odd: the vectors of part p start a elements late, as the
// rows of that CTA do.
__global__ void __launch_bounds__(1024) layer_norm_fold_kernel(const float* part, int parts, int H, int ld, int odd, int offset, float* dw, float* db) {
    __shared__ float s[32][33];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t two_h = 2 * (int64_t)H;
    const int64_t col = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int lane = threadIdx.x >> 5;
    float a = 0.f;
    if (col < two_h) {
        const float* p0 = part + (col < H ? col : col - H + ld);
#pragma unroll 8
        for (int p = lane; p < parts; p += 32) a += __ldcg(p0 + (int64_t)p * 2 * ld + (odd ? (offset + (p & 7) * (H & 7)) & 7 : 0));
    }
    s[lane][threadIdx.x & 31] = a;
    __syncthreads();
    // warp `lane` sums the 32 shares of column `lane`
    float t = s[threadIdx.x & 31][lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    if ((threadIdx.x & 31) == 0 && c < two_h) {
        if (c < H) { if (dw) dw[c] = t; }
        else if (db) db[c - H] = t;
    }
}

}  // namespace mxfp6
