// Attention over the paged cache in 4 bits.
#include <cuda_bf16.h>

#include <cmath>

#include "cache4.h"
#include "pdl.cuh"

namespace bk {
namespace {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A CTA of four warps to a (row, query head). Each warp walks every fourth position with a running maximum and sum.
template <class T, int E>
__global__ void __launch_bounds__(128) cache4_rows_kernel(const Cache4 c, const Cache4Batch b, const Cache4Attend a) {
    __shared__ float part[4][32 * E], top[4], total[4];
    wait_for_previous();
    release_next();
    const uint32_t row = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t sequence;
    long long position;
    if (!row_place(b, row, sequence, position)) return;
    const uint32_t kv = head / (a.heads / c.kv_heads);
    const long long last = min(position, (long long)b.columns * c.page_size - 1);
    const long long first = a.window != 0 ? max(0ll, position - (long long)a.window + 1) : 0;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        q[j] = to_float(static_cast<const T*>(a.q)[size_t(row) * a.q_stride + head * 32 * E + lane * E + j]) * a.scale;
        o[j] = 0.0f;
    }
    constexpr int kLanes = 32 / E;
    const uint32_t block = lane / kLanes, in_block = lane % kLanes, shift = in_block < kLanes / 2 ? 0 : 4, byte = block * 16 + (in_block % (kLanes / 2)) * E;
    for (long long p = first + warp; p <= last; p += 4) {
        const int32_t page = page_of(c, b, sequence, uint32_t(p >> c.page_shift));
        float k[E], v[E], s = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) k[j] = v[j] = 0.0f;
        if (page >= 0) {
            const size_t at = ((size_t(page) * c.kv_heads + kv) * c.page_size + (uint32_t(p) & (c.page_size - 1))) * E;
            const float dk = __half2float(c.k_scales[at + block]), dv = __half2float(c.v_scales[at + block]);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                k[j] = (float((c.k_quants[at * 16 + byte + j] >> shift) & 15) - 8.0f) * dk;
                v[j] = (float((c.v_quants[at * 16 + byte + j] >> shift) & 15) - 8.0f) * dv;
            }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) s = fmaf(q[j], k[j], s);
        s = warp_sum(s);
        const float next = fmaxf(m, s), keep = __expf(m - next), w = expf(s - next);
        m = next;
        l = fmaf(l, keep, w);
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] = fmaf(o[j], keep, w * v[j]);
    }
    if (lane == 0) {
        top[warp] = m;
        total[warp] = l;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) part[warp][lane * E + j] = o[j];
    __syncthreads();
    const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    float sum = 0.0f, keep[4];
    for (int w = 0; w < 4; ++w) {
        keep[w] = top[w] == -INFINITY ? 0.0f : expf(top[w] - most);
        sum = fmaf(total[w], keep[w], sum);
    }
    for (uint32_t i = threadIdx.x; i < 32 * E; i += 128) {
        float x = 0.0f;
        for (int w = 0; w < 4; ++w) x = fmaf(part[w][i], keep[w], x);
        put(static_cast<T*>(a.out) + size_t(row) * a.out_stride + head * 32 * E + i, sum > 0.0f ? x / sum : 0.0f);
    }
}

template <class T>
void attend(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, bool dependent, cudaStream_t s) {
    const auto kernel = c.dim == 64 ? cache4_rows_kernel<T, 2> : c.dim == 128 ? cache4_rows_kernel<T, 4> : cache4_rows_kernel<T, 8>;
    const dim3 grid(b.tokens, a.heads);
    if (dependent) {
        launch_dependent(kernel, grid, dim3(128), 0, s, c, b, a);
    } else {
        kernel<<<grid, 128, 0, s>>>(c, b, a);
        BK_CUDA(cudaGetLastError());
    }
}

}  // namespace

void launch_cache4_attention(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, int type, bool dependent, cudaStream_t s) {
    if (type == T_F32) attend<float>(c, b, a, dependent, s);
    else if (type == T_F16) attend<__half>(c, b, a, dependent, s);
    else attend<__nv_bfloat16>(c, b, a, dependent, s);
}

}  // namespace bk
