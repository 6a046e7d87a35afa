// MX operand bytes + E8M0 scales -> fp32 or bf16 values: value = element * 2^(scale - 127).
//
// Byte work bound by HBM (reads 0.53, 0.78 or 1.03 bytes per element, writes 4 or 2).  The hardware conversions to half
// precision are exact for every element format; the product with a power of two is exact too unless it leaves the fp32 range.
// Rounding to bf16 (to nearest even) changes no value inside the normal range: the elements have at most four significant bits.
//
// dequantize_tma_kernel, the mirror image of the quantiser: every warp works on its own, on tiles of 64 blocks.  Bulk copies
// bring the codes and scales of the next tiles into the warp's ring while each lane decodes two blocks and writes the 32 values of
// each as a swizzled row of a staging buffer, which one TMA store takes to memory (the output viewed as [blocks, 32]).  The plain
// kernel behind it (8 elements per thread, four loads in flight) serves operands whose codes or scales do not start on 16 bytes.
// 16384 x 8192, streaming against plain: E2M1 to fp32 108 / 119 us (5.6 TB/s), E2M3 to bf16 68 / 81 us (5.5 TB/s).  Of the 108 us
// the stores alone take 86 (6.2 TB/s, measured without the loads) and the codes 11 at the copy rate.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"
#include "quant.cuh"
#include "quantize_kernel.cuh"

namespace mxfp6 {

// 2^(byte - 127); byte 0 is the fp32 subnormal 2^-127, byte 255 a NaN
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return byte == 255 ? __uint_as_float(0x7fc00000u) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ float2 half2_bits_to_float2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// four codes of a byte each (fp6 in the low six bits) -> four fp32 values times s
template <int FMT>
__device__ __forceinline__ void decode_bytes4(uint32_t c, float s, float2 (&v)[2]) {
    uint32_t h0, h1;
#define MX_CVT2(T) asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.rn.f16x2." T " %0, l;\n\tcvt.rn.f16x2." T " %1, u;\n\t}" : "=r"(h0), "=r"(h1) : "r"(c))
    if constexpr (FMT == kE2M3) MX_CVT2("e2m3x2");
    else if constexpr (FMT == kE3M2) MX_CVT2("e3m2x2");
    else if constexpr (FMT == kE4M3) MX_CVT2("e4m3x2");
    else MX_CVT2("e5m2x2");
#undef MX_CVT2
    v[0] = __fmul2_rn(half2_bits_to_float2(h0), make_float2(s, s));
    v[1] = __fmul2_rn(half2_bits_to_float2(h1), make_float2(s, s));
}
// 24 bits of four 6-bit codes -> one code per byte
__device__ __forceinline__ uint32_t spread_fp6(uint32_t q) {
    const uint32_t t = (q & 0xfffu) | ((q & 0xfff000u) << 4);
    return (t & 0x003f003fu) | ((t & 0x0fc00fc0u) << 2);
}
// eight codes of a block in the low bits of w -> eight values times s
template <int FMT>
__device__ __forceinline__ void decode8(uint64_t w, float s, float2 (&v)[4]) {
    if constexpr (FMT == kE2M1) {
        uint32_t h[4];
        asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
            : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"((uint32_t)w));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fmul2_rn(half2_bits_to_float2(h[i]), make_float2(s, s));
    } else {
        const uint32_t lo = (uint32_t)w, hi = (uint32_t)(w >> 32);
        float2 t[2], u[2];
        if constexpr (fmt_fp8(FMT)) {
            decode_bytes4<FMT>(lo, s, t);
            decode_bytes4<FMT>(hi, s, u);
        } else {
            decode_bytes4<FMT>(spread_fp6(lo & 0xffffffu), s, t);
            decode_bytes4<FMT>(spread_fp6(__funnelshift_r(lo, hi, 24) & 0xffffffu), s, u);
        }
        v[0] = t[0]; v[1] = t[1]; v[2] = u[0]; v[3] = u[1];
    }
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
            float2 v[4];
            decode8<FMT>(w[u], e8m0_value(sb[u]), v);
            if constexpr (sizeof(OutT) == 4) {
                float* d = reinterpret_cast<float*>(out) + o * 8;
                *reinterpret_cast<float4*>(d) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
                *reinterpret_cast<float4*>(d + 4) = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
            } else {
                uint4 q;
                q.x = pack_bf16x2(v[0].x, v[0].y); q.y = pack_bf16x2(v[1].x, v[1].y);
                q.z = pack_bf16x2(v[2].x, v[2].y); q.w = pack_bf16x2(v[3].x, v[3].y);
                *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + o * 8) = q;
            }
        }
    }
}

// ---------------------------------------------------------------------------------- streaming kernel
constexpr int kStatusTimeoutDequant = 0x23;     // a warp waited for the codes of a tile

template <int FMT, typename OutT>
struct DequantCfg {
    static constexpr int WARPS = 4;
    static constexpr int LB = 2;                                     // blocks per lane and tile
    static constexpr int STAGES = 3;
    static constexpr int TILE = 32 * LB;                             // blocks of a warp's tile
    static constexpr int CODES = TILE * fmt_block_bytes(FMT);        // 1, 1.5 or 2 KB
    static constexpr int ROW = 32 * (int)sizeof(OutT);               // bytes of one block's values
    static constexpr int OUT = TILE * ROW;                           // 8 KB or 4 KB
    static constexpr int OUT_BUFS = 2;
    static constexpr int SMEM_BYTES = WARPS * (OUT_BUFS * OUT + STAGES * (CODES + TILE + 8)) + 16;
    static constexpr int SMEM_ALLOC = SMEM_BYTES + 1024;
    static constexpr int CTAS_PER_SM = 232448 / (SMEM_ALLOC + 1024) < 6 ? 232448 / (SMEM_ALLOC + 1024) : 6;
};

template <int FMT, typename OutT>
__global__ void __launch_bounds__(128, (DequantCfg<FMT, OutT>::CTAS_PER_SM))
dequantize_tma_kernel(const __grid_constant__ CUtensorMap tm_out, const uint8_t* packed, const uint8_t* scales, long long n_blocks,
                      int* status, unsigned long long wait_cycles) {
    using Cfg = DequantCfg<FMT, OutT>;
    constexpr int B = fmt_block_bytes(FMT);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t out_off = warp * Cfg::OUT_BUFS * Cfg::OUT;
    const uint32_t code_off = Cfg::WARPS * Cfg::OUT_BUFS * Cfg::OUT + warp * Cfg::STAGES * Cfg::CODES;
    const uint32_t scale_off = Cfg::WARPS * (Cfg::OUT_BUFS * Cfg::OUT + Cfg::STAGES * Cfg::CODES) + warp * Cfg::STAGES * Cfg::TILE;
    const uint32_t bar_off = Cfg::WARPS * (Cfg::OUT_BUFS * Cfg::OUT + Cfg::STAGES * (Cfg::CODES + Cfg::TILE)) + warp * Cfg::STAGES * 8;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + Cfg::SMEM_BYTES - 16);
    auto bar = [&](uint32_t s) { return smem_base + bar_off + 8u * s; };
    if (lane == 0) {
        for (int s = 0; s < Cfg::STAGES; ++s) mbar_init(bar(s), 1);
        fence_barrier_init();
    }
    if (threadIdx.x == 0) { *abort_flag = 0; tma_prefetch_desc(&tm_out); }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();

    constexpr int TILE = Cfg::TILE;
    const int tiles = (int)((n_blocks + TILE - 1) / TILE), whole = (int)(n_blocks / TILE);
    const int step = (int)gridDim.x * Cfg::WARPS;
    const int first = (int)blockIdx.x * Cfg::WARPS + warp;
    auto request = [&](uint32_t s, int t) {                     // one lane; the last, partial tile is read with plain loads
        if (t >= whole) return;
        mbar_arrive_expect_tx(bar(s), Cfg::CODES + TILE);
        bulk_load_1d(smem_base + code_off + s * Cfg::CODES, packed + (long long)t * Cfg::CODES, Cfg::CODES, bar(s));
        bulk_load_1d(smem_base + scale_off + s * TILE, scales + (long long)t * TILE, TILE, bar(s));
    };
    if (lane == 0)
        for (int s = 0; s < Cfg::STAGES; ++s) request(s, first + s * step);
    uint32_t s = 0, phase = 0, ob = 0;
    for (int t = first; t < tiles; t += step) {
        uint64_t w[Cfg::LB][4];                                 // this lane's blocks: 8 elements each
        float sc[Cfg::LB];
        if (t < whole) {
            if (!__all_sync(0xffffffffu, quant_wait(bar(s), phase, abort_flag, status, wait_cycles, kStatusTimeoutDequant))) break;
#pragma unroll
            for (int b = 0; b < Cfg::LB; ++b) {
                const uint8_t* c = smem_gen + code_off + s * Cfg::CODES + (b * 32 + lane) * B;
                if constexpr (B == 16) {
                    const uint4 q = *reinterpret_cast<const uint4*>(c);
                    w[b][0] = q.x; w[b][1] = q.y; w[b][2] = q.z; w[b][3] = q.w;
                } else if constexpr (B == 24) {
                    const uint2 q0 = *reinterpret_cast<const uint2*>(c), q1 = *reinterpret_cast<const uint2*>(c + 8), q2 = *reinterpret_cast<const uint2*>(c + 16);
                    w[b][0] = q0.x | ((uint64_t)q0.y << 32);
                    w[b][1] = __funnelshift_r(q0.y, q1.x, 16) | ((uint64_t)(q1.x >> 16) << 32);
                    w[b][2] = q1.y | ((uint64_t)q2.x << 32);
                    w[b][3] = __funnelshift_r(q2.x, q2.y, 16) | ((uint64_t)(q2.y >> 16) << 32);
                } else {
                    const uint4 q0 = *reinterpret_cast<const uint4*>(c), q1 = *reinterpret_cast<const uint4*>(c + 16);
                    w[b][0] = q0.x | ((uint64_t)q0.y << 32); w[b][1] = q0.z | ((uint64_t)q0.w << 32);
                    w[b][2] = q1.x | ((uint64_t)q1.y << 32); w[b][3] = q1.z | ((uint64_t)q1.w << 32);
                }
                sc[b] = e8m0_value(smem_gen[scale_off + s * TILE + b * 32 + lane]);
            }
            __syncwarp();                                       // the stage is in registers
            if (lane == 0) request(s, t + Cfg::STAGES * step);
        } else {
#pragma unroll
            for (int b = 0; b < Cfg::LB; ++b) {
                const long long blk = (long long)t * TILE + b * 32 + lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[b][i] = blk < n_blocks ? load_codes8<FMT, false>(packed + blk * B + i * (B / 4)) : 0;
                sc[b] = blk < n_blocks ? e8m0_value(__ldcg(scales + blk)) : 0.f;
            }
        }
        if (++s == Cfg::STAGES) { s = 0; phase ^= 1; }
        // the store that last read this staging buffer is done with it
        if (lane == 0) bulk_wait_group_read<Cfg::OUT_BUFS - 1>();
        __syncwarp();
#pragma unroll
        for (int b = 0; b < Cfg::LB; ++b) {
            const uint32_t row = smem_base + out_off + ob * Cfg::OUT + (b * 32 + lane) * Cfg::ROW;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 v[4];
                decode8<FMT>(w[b][i], sc[b], v);
                if constexpr (sizeof(OutT) == 4) {
                    // 128-byte rows, 128-byte swizzle: 16-byte chunk c of row r sits at chunk c ^ (r % 8)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + (((2 * i + h) ^ (lane & 7)) << 4)), "r"(__float_as_uint(v[2 * h].x)),
                                     "r"(__float_as_uint(v[2 * h].y)), "r"(__float_as_uint(v[2 * h + 1].x)), "r"(__float_as_uint(v[2 * h + 1].y)) : "memory");
                } else {
                    // 64-byte rows, 64-byte swizzle: chunk c of row r sits at chunk c ^ ((r / 2) % 4)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((i ^ ((lane >> 1) & 3)) << 4)), "r"(pack_bf16x2(v[0].x, v[0].y)),
                                 "r"(pack_bf16x2(v[1].x, v[1].y)), "r"(pack_bf16x2(v[2].x, v[2].y)), "r"(pack_bf16x2(v[3].x, v[3].y)) : "memory");
                }
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            // (rows past the last block are clipped; values on their way to DRAM leave L2 first: bf16 64.8 -> 60.9 us for 16384 x
            // 8192 from E2M1, while fp32 loses 1 % by it)
            if constexpr (sizeof(OutT) == 2) tma_store_2d_hint(&tm_out, smem_base + out_off + ob * Cfg::OUT, 0, t * TILE, l2_policy_evict_first());
            else tma_store_2d(&tm_out, smem_base + out_off + ob * Cfg::OUT, 0, t * TILE);
            bulk_commit_group();
        }
        ob ^= 1;
    }
    if (lane == 0) bulk_wait_group<0>();
    if (*abort_flag) {
        // give loads that are still in flight time to land before shared memory goes away
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) { __nanosleep(1000); }
    }
}

}  // namespace mxfp6
