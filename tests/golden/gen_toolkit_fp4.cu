// Generates tests/golden/toolkit_fp4_kat.json: known answers for FP4 E2M1 from the CUDA toolkit's HOST conversion
// routines (cuda_fp4.h), saturating and round-to-nearest-even.  Runs on the CPU only.
//   nvcc -o /tmp/gen_toolkit_fp4 tests/golden/gen_toolkit_fp4.cu && /tmp/gen_toolkit_fp4 > tests/golden/toolkit_fp4_kat.json
#include <cuda_fp16.h>
#include <cuda_fp4.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

static uint32_t bits(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
static float value(int c) { return __half2float(__half(__nv_cvt_fp4_to_halfraw((__nv_fp4_storage_t)c, __NV_E2M1))); }

int main() {
    std::vector<float> xs;
    // every value, every midpoint between neighbours, the fp32 neighbours of each midpoint, and the saturation gap
    for (int c = 1; c < 8; ++c) {
        const float v = value(c), mid = 0.5f * (value(c - 1) + v);
        const float cand[] = {v, nextafterf(v, 0.f), nextafterf(v, 1e30f), mid, nextafterf(mid, 0.f), nextafterf(mid, 1e30f)};
        for (float x : cand) { xs.push_back(x); xs.push_back(-x); }
    }
    const float extra[] = {0.f, 1e-30f, 1e-9f, 0.1f, 0.2f, 6.5f, 7.f, 7.5f, 7.999f, 8.f, 100.f, 1e30f};
    for (float e : extra) { xs.push_back(e); xs.push_back(-e); }
    uint32_t s = 12345u;                               // values spread over the range
    for (int i = 0; i < 400; ++i) { s = s * 1664525u + 1013904223u; xs.push_back(((float)(s >> 8) / 16777216.f - 0.5f) * 16.f); }
    printf("{\n\"encode\": [\n");
    for (size_t i = 0; i < xs.size(); ++i) {
        const unsigned c = __nv_cvt_float_to_fp4(xs[i], __NV_E2M1, cudaRoundNearest);
        printf("[%u,%u]%s\n", bits(xs[i]), c & 15u, i + 1 < xs.size() ? "," : "");
    }
    printf("],\n\"decode\": [");
    for (int c = 0; c < 16; ++c) printf("%u%s", bits(value(c)), c < 15 ? "," : "");
    // a pair conversion puts its first element into the low nibble
    const unsigned pair = __nv_cvt_float2_to_fp4x2(make_float2(1.5f, -4.f), __NV_E2M1, cudaRoundNearest);
    printf("],\n\"pair\": [%u, %u, %u]\n}\n", bits(1.5f), bits(-4.f), pair & 255u);
    return 0;
}
