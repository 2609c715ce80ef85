// Helpers of the two attentions over the cache in 4 bits.
#pragma once

#include <cuda_bf16.h>

#include "cache4.h"

namespace bk {

inline uint32_t multiprocessors() {
    int dev = 0, count = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
    return uint32_t(count);
}

// A weight is 2^(score - level) as one f16 or, for f32, two: what is below 2^-24 is lost, what is above 65504 does not fit. A level is set
// kBelow under its row's maximum and stays until a score is 2^kMost above it, so that the largest weight of a row lies between 2^kBelow
// and 2^kMost and the smallest that keep their bits lie as far below it as an f16 allows: 11 bits (one f16) down to 2^-21 of the
// largest, 22 (two) down to 2^-15, to within 2^-32 and 2^-37 of the largest from there. With the level at the maximum those were 2^-25, and a
// tail of 32 000 equal weights behind one heavy position 1e-4 off. The f32 level moves a little more often for it (past 2^3 times the
// maximum it was set by instead of 2^8).
//
// One f16, 11 bits, for f16 and bf16 queries: as many as the result has, or more; another part would double the products with the values. Against
// 64 bits the results are 2.9e-4 off with f16 queries, 2.1e-4 with weights of 32 bits, and with bf16 ones 1.7e-3 either way: what is left is the
// rounding of the result. Two, 22 bits, for f32: three would add half to the products again, and the errors are those of sums in 32 bits
// without it (3e-7 to 8e-7; everything in 32 bits: 5e-7 to 1.2e-6).
template <bool TWO> struct Level {
    static constexpr float kBelow = TWO ? 12.0f : 7.0f, kMost = 15.0f;
};

#ifdef __CUDACC__
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 halves(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// From 8192 on -8 times a scale is past the largest f16, while scales are held up to 65280. The kernel of few rows folds a tile of positions
// that holds such a scale of values: their scales are an eighth (65280 / 8 = 8160) and the weights 8 times what they are, for which the
// level is 3 less, and the running sum 8 times as much, while the tile lasts; what Level says of the largest weight holds as it is. Eighths
// are exact for scales from 2^-14 on; a value of a smaller one that shares its tile with one of 8192 is rounded to 2^-21. (Scales of
// keys are multiplied in 32 bits there.) The kernel of many rows computes such rows in another way.
constexpr float kFold = 0.125f, kUnfold = 8.0f, kFoldBits = 3.0f;
__device__ __forceinline__ bool past_f16(__half scale) { return __hge(__habs(scale), __half(8192.0f)); }
__device__ __forceinline__ __half2 larger(__half2 a, __half2 b) { return __hmax2(__habs2(a), __habs2(b)); }

// The eight numbers of a word, n - 8 times the scale, as four pairs: (low of bytes 0, 2), (high of 0, 2), (low of 1, 3), (high of 1, 3).
// A number set into the mantissa of 1024 (or, 16 times it, of 1024) is exact, so is n - 8, and so is the product with a scale of 8
// bits that is not past_f16: three instructions a pair and no rounding.
__device__ __forceinline__ void widen(uint32_t w, __half2 scale, uint32_t (&v)[4]) {
    const uint32_t magic = 0x64006400u, u = w >> 8;
    const __half2 bias = halves(0x64086408u), sixteenth = halves(0x2c002c00u), less = halves(0xd480d480u);  // 1032, 1 / 16, -72
    v[0] = bits(__hmul2(__hsub2(halves((w & 0x000f000fu) | magic), bias), scale));
    v[1] = bits(__hmul2(__hfma2(halves((w & 0x00f000f0u) | magic), sixteenth, less), scale));
    v[2] = bits(__hmul2(__hsub2(halves((u & 0x000f000fu) | magic), bias), scale));
    v[3] = bits(__hmul2(__hfma2(halves((u & 0x00f000f0u) | magic), sixteenth, less), scale));
}
#endif

}  // namespace bk
