// MX operand bytes + E8M0 scales -> fp32 or bf16 values: value = element * 2^(scale - 127).
//
// Byte work bound by HBM (reads 0.53, 0.78 or 1.03 bytes per element, writes 4 or 2).  One thread takes 8 consecutive
// elements (4, 6 or 8 code bytes, a quarter of a block), so that its fp32 result is one whole 32-byte sector and a warp's
// results are consecutive; four independent loads per thread are in flight.  The hardware conversions to half precision
// are exact for every element format; the product with a power of two is exact too unless it leaves the fp32 range.
// Rounding to bf16 (to nearest even) changes no value inside the normal range: the elements have at most four
// significant bits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"
#include "quant.cuh"

namespace mxfp6 {

// two codes (in the low two bytes; for E2M1 in the low byte) -> two fp32 values
template <int FMT>
__device__ __forceinline__ float2 decode_pair(uint32_t c) {
    uint32_t h;
    const uint16_t c16 = (uint16_t)c;
    if constexpr (FMT == kE2M3) asm("cvt.rn.f16x2.e2m3x2 %0, %1;" : "=r"(h) : "h"(c16));
    else if constexpr (FMT == kE3M2) asm("cvt.rn.f16x2.e3m2x2 %0, %1;" : "=r"(h) : "h"(c16));
    else if constexpr (FMT == kE4M3) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c16));
    else if constexpr (FMT == kE5M2) asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(c16));
    else asm("{\n\t.reg .b8 t, u;\n\tmov.b16 {t, u}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "h"(c16));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// code bytes of 8 elements, lowest first; VEC: the operand is aligned for one load (fp4, fp8) or 2-byte loads (fp6)
template <int FMT, bool VEC>
__device__ __forceinline__ uint64_t load_codes8(const uint8_t* p) {
    constexpr int B = fmt_block_bytes(FMT) / 4;
    if constexpr (VEC && B == 4) return __ldcg(reinterpret_cast<const uint32_t*>(p));
    if constexpr (VEC && B == 8) return __ldcg(reinterpret_cast<const unsigned long long*>(p));
    uint64_t w = 0;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < B / 2; ++i) w |= (uint64_t)__ldcg(reinterpret_cast<const uint16_t*>(p) + i) << (16 * i);
    } else {
#pragma unroll
        for (int i = 0; i < B; ++i) w |= (uint64_t)__ldcg(p + i) << (8 * i);
    }
    return w;
}

template <int FMT>
__device__ __forceinline__ void decode8(uint64_t w, uint32_t scale_byte, float (&v)[8]) {
    // 2^(byte - 127); byte 0 is the fp32 subnormal 2^-127, byte 255 a NaN
    const float s = scale_byte == 255 ? __uint_as_float(0x7fc00000u) : scale_byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(scale_byte << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t c;
        if constexpr (FMT == kE2M1) c = (uint32_t)(w >> (8 * i)) & 0xffu;
        else if constexpr (FMT == kE4M3 || FMT == kE5M2) c = (uint32_t)(w >> (16 * i)) & 0xffffu;
        else { const uint32_t t = (uint32_t)(w >> (12 * i)) & 0xfffu; c = (t & 63u) | ((t >> 6) << 8); }
        const float2 x = decode_pair<FMT>(c);
        v[2 * i] = x.x * s; v[2 * i + 1] = x.y * s;
    }
}

template <int FMT, typename OutT, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* packed, const uint8_t* scales,
                                                         int64_t n_oct, OutT* out) {
    constexpr int U = 4;
    // Programmatic dependent launch: the codes may be the preceding kernel's output, so nothing is read before the wait,
    // and the loads go to L2 (a read-only path may hold lines from before that kernel wrote them).
    pdl_launch_dependents();
    pdl_wait();
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t o0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; o0 < n_oct; o0 += U * step) {
        uint64_t w[U];
        uint32_t sb[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t o = o0 + u * step;
            w[u] = 0; sb[u] = 0;
            if (o < n_oct) { w[u] = load_codes8<FMT, VEC>(packed + o * (fmt_block_bytes(FMT) / 4)); sb[u] = __ldcg(scales + (o >> 2)); }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t o = o0 + u * step;
            if (o >= n_oct) break;
            float v[8];
            decode8<FMT>(w[u], sb[u], v);
            if constexpr (sizeof(OutT) == 4) {
                float* d = reinterpret_cast<float*>(out) + o * 8;
                if constexpr (VEC) {
                    st_global_v8(d, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]),
                                 __float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
                } else {
                    *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>(d + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            } else {
                uint4 q;
                q.x = pack_bf16x2(v[0], v[1]); q.y = pack_bf16x2(v[2], v[3]);
                q.z = pack_bf16x2(v[4], v[5]); q.w = pack_bf16x2(v[6], v[7]);
                *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + o * 8) = q;
            }
        }
    }
}

}  // namespace mxfp6
