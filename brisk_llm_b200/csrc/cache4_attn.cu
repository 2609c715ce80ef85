// Attention over the paged cache in 4 bits, for few rows: single tokens, verify steps, and whatever cache4_prompt.cu leaves.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "cache4.h"
#include "pdl.cuh"

namespace bk {
namespace {

namespace cg = cooperative_groups;

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
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // an 8 x 8 matrix of f16, lane (g, t) holding row g, columns 2 t and 2 t + 1
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(v));
    return y;
}
__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 halves(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// 16 bytes to shared memory; zeros where !there (src is then any valid address).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The eight numbers of a word, n - 8 times the scale, as four pairs: (low of bytes 0, 2), (high of 0, 2), (low of 1, 3), (high of 1, 3).
// A number set into the mantissa of 1024 (or, 16 times it, of 1024) is exact, so is n - 8, and so is the product with a scale of 8
// bits: three instructions a pair and no rounding.
__device__ __forceinline__ void widen(uint32_t w, __half2 scale, uint32_t (&v)[4]) {
    const uint32_t magic = 0x64006400u, u = w >> 8;
    const __half2 bias = halves(0x64086408u), sixteenth = halves(0x2c002c00u), less = halves(0xd480d480u);  // 1032, 1 / 16, -72
    v[0] = bits(__hmul2(__hsub2(halves((w & 0x000f000fu) | magic), bias), scale));
    v[1] = bits(__hmul2(__hfma2(halves((w & 0x00f000f0u) | magic), sixteenth, less), scale));
    v[2] = bits(__hmul2(__hsub2(halves((u & 0x000f000fu) | magic), bias), scale));
    v[3] = bits(__hmul2(__hfma2(halves((u & 0x00f000f0u) | magic), sixteenth, less), scale));
}

template <int D> struct Split {
    static constexpr int kTile = 32;                      // positions a warp takes at a time
    static constexpr int kWarps = D == 256 ? 4 : 8;
    static constexpr int kStages = D == 64 ? 4 : 3;
    static constexpr int kRow = D / 2, kScales = D / 16;  // bytes of a position
    static constexpr int kK = 0, kV = kTile * kRow, kKs = 2 * kTile * kRow, kVs = kKs + kTile * kScales, kStage = kVs + kTile * kScales;
    static constexpr int kPitch = D + 4;                  // floats between two rows of a warp's result
    static constexpr int kSteps = D / 16;
    static constexpr size_t ring() { return size_t(kWarps) * kStages * kStage; }
    static constexpr size_t parts(int nt) { return size_t(kWarps) * 8 * nt * kPitch * 4; }
    static constexpr size_t body(int nt) { return ring() > parts(nt) ? ring() : parts(nt); }
    static constexpr size_t queries(int nt, bool two) { return size_t(nt) * kSteps * 32 * 8 * (two ? 2 : 1); }
    static constexpr size_t smem(int nt, bool two) { return body(nt) + queries(nt, two) + size_t(8 * nt) * (2 * kWarps + 4 + 16) * 4; }
};

// Where 16 bytes of a position's row lie in a stage, and which position a row of a matrix instruction is: chosen so that the loads of
// keys (8 rows, a quarter of each to a lane) and of values (4 rows, an eighth to a lane) meet no shared-memory bank twice.
template <int D> __device__ __forceinline__ uint32_t chunk_of(uint32_t position, uint32_t chunk) {
    if (D == 64) return chunk;
    return D == 128 ? chunk ^ (((position >> 1) & 1) << 1) : chunk ^ ((position & 3) << 1);
}
template <int D> __device__ __forceinline__ uint32_t position_of(uint32_t g) {  // g < 8
    return (g & 1) ? 4 + ((g >> 1) ^ (D == 128 ? 1 : 2)) : g >> 1;
}

// softmax(q k) v for 8 NT rows - tokens times the query heads of one key/value head - of one sequence. A cluster of CTAs shares the
// positions, each warp takes tiles of 32 of them with a running maximum and sum of its own; the warps' results are joined in
// shared memory, the CTAs' over the cluster's. Positions are the rows (M) and queries the columns (N = 8) of both products,
//     S^T = K Q^T (16 positions x 8 queries),     O^T = V^T P^T (16 dims x 8 queries),
// so that eight query heads fill an instruction and the 4-bit words become its A operand in registers, straight from the
// stage that cp.async filled: any order of the head's values does for K Q^T as long as Q has the same. P^T is S^T transposed in the warp.
// f32 queries and weights are two f16 parts each (22 bits); others one.
template <class T, int D, int NT>
__global__ void __launch_bounds__(Split<D>::kWarps * 32, NT == 1 || (NT == 2 && D == 64) ? 2 : 1) cache4_split_kernel(const Cache4 c, const Cache4Batch b, const Cache4Attend a) {
    using G = Split<D>;
    constexpr bool kTwo = sizeof(T) == 4;
    constexpr int kRows = 8 * NT, kThreads = G::kWarps * 32;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* q_frag = smem + G::body(NT);
    float* row_scale = reinterpret_cast<float*>(q_frag + G::queries(NT, kTwo));  // [kRows]
    float* warp_top = row_scale + kRows;                                         // [kWarps][kRows], then the sums
    float* warp_sum_ = warp_top + G::kWarps * kRows;
    float* cta_top = warp_sum_ + G::kWarps * kRows;  // [kRows], read by the cluster
    float* cta_sum = cta_top + kRows;
    float* weight = cta_sum + kRows;  // [16][kRows]

    wait_for_previous();
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t S = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t unit = blockIdx.x / S, kv = unit % c.kv_heads, tile = unit / c.kv_heads, sequence = blockIdx.y;
    const uint32_t group = a.heads / c.kv_heads;
    uint32_t first_row, count;
    sequence_rows(b, sequence, first_row, count);
    const uint32_t total = count * group, row0 = tile * kRows;
    if (row0 >= total) return;  // the whole cluster
    const uint32_t rows = min(total - row0, uint32_t(kRows));
    const long long context = b.context[sequence], held = (long long)b.columns * c.page_size;
    const long long first_pos = context + row0 / group, last_pos = context + (row0 + rows - 1) / group;
    const int hi = int(min(last_pos, held - 1));  // -1 and less: nothing
    const int lo = a.window != 0 ? int(min(max(first_pos - (long long)a.window + 1, 0ll), held)) : 0;

    // ---- queries: a power of two brings a row's largest value to 2^10, so that bf16 and both parts of f32 fit f16 ----
    for (uint32_t r = warp; r < kRows; r += G::kWarps) {
        float x[D / 32], most = 0.0f;
        const T* src = static_cast<const T*>(a.q) + size_t(first_row + (row0 + r) / group) * a.q_stride + size_t(kv * group + (row0 + r) % group) * D;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            x[j] = r < rows ? to_float(src[lane + 32 * j]) : 0.0f;
            most = fmaxf(most, fabsf(x[j]));
        }
        most = warp_max(most);
        const int up = most > 0.0f && most < INFINITY ? 10 - ilogbf(most) : 0;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const float v = ldexpf(a.scale < 0.0f ? -x[j] : x[j], up);
            const __half high = __float2half_rn(v);
            // value `lane` of block j: which lane's fragment of which step takes it (see widen and the loads of keys below)
            const uint32_t byte = lane & 15, word = byte >> 2;
            const uint32_t owner = D == 64 ? j * 2 + (word >> 1) : j & 3;
            const uint32_t step = (D == 64 ? 2 * (word & 1) : D == 128 ? 2 * word : (j >> 2) * 8 + 2 * word) + (byte & 1);
            const uint32_t at = ((((r >> 3) * G::kSteps + step) * 32 + (r & 7) * 4 + owner) * 2 + (lane >> 4)) * 2 + ((byte & 3) >> 1);
            __half* dst = reinterpret_cast<__half*>(q_frag);
            dst[at] = high;
            if (kTwo) dst[at + NT * G::kSteps * 128] = __float2half_rn(v - __half2float(high));
        }
        if (lane == 0) row_scale[r] = ldexpf(fabsf(a.scale) * 1.4426950408889634f, -up);
    }
    __syncthreads();

    float o[G::kSteps][NT][4], m[NT][2], l[NT][2], scale[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < G::kSteps; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            m[n][e] = -INFINITY;
            l[n][e] = 0.0f;
            scale[n][e] = row_scale[n * 8 + 2 * t + e];
        }
    }

    // ---- the warp's tiles: begin + 32 (rank + S (warp + W i)) and on ----
    const int begin = lo & ~31;
    const int tiles = hi >= lo ? (hi - begin) / 32 + 1 : 0, stride = int(S) * G::kWarps, mine = int(warp * S + rank);
    unsigned char* ring = smem + size_t(warp) * G::kStages * G::kStage;
    const uint32_t ring_at = uint32_t(__cvta_generic_to_shared(ring));
    // lanes 0 and 1 know the pages of the tile's two halves, asked for a tile ahead of the copies
    auto page_for = [&](int j) {
        const int p = begin + 32 * j + 16 * int(lane & 1);
        return j < tiles && p <= hi && p + 16 > lo ? page_of(c, b, sequence, uint32_t(p) >> c.page_shift) : -1;
    };
    auto request = [&](int j, int page, uint32_t slot) {  // copies of tile j into the slot; the same number of groups whether there is one
        const uint32_t base = ring_at + slot * G::kStage;
        const int page0 = __shfl_sync(0xffffffffu, page, 0), page1 = __shfl_sync(0xffffffffu, page, 1);
        if (j < tiles) {
            const uint32_t p0 = uint32_t(begin + 32 * j) & (c.page_size - 1), p1 = uint32_t(begin + 32 * j + 16) & (c.page_size - 1);
            const size_t at0 = (size_t(max(page0, 0)) * c.kv_heads + kv) * c.page_size + p0, at1 = (size_t(max(page1, 0)) * c.kv_heads + kv) * c.page_size + p1;
            constexpr int kChunks = G::kRow / 16;  // of a position's row
#pragma unroll
            for (int i = 0; i < 16 * kChunks / 32; ++i) {
                const uint32_t x = i * 32 + lane, p = x / kChunks, ch = x % kChunks;
                const size_t from = size_t(p) * G::kRow + ch * 16;
                const uint32_t to = p * G::kRow + chunk_of<D>(p, ch) * 16;
                copy16(base + G::kK + to, c.k_quants + at0 * G::kRow + from, page0 >= 0);
                copy16(base + G::kK + 16 * G::kRow + to, c.k_quants + at1 * G::kRow + from, page1 >= 0);
                copy16(base + G::kV + to, c.v_quants + at0 * G::kRow + from, page0 >= 0);
                copy16(base + G::kV + 16 * G::kRow + to, c.v_quants + at1 * G::kRow + from, page1 >= 0);
            }
            constexpr int kScaleChunks = G::kScales;  // of 16 positions: 16 * kScales / 16
#pragma unroll
            for (int x0 = 0; x0 < 4 * kScaleChunks; x0 += 32) {
                const uint32_t x = x0 + lane;
                if (x < 4 * kScaleChunks) {
                    const uint32_t which = x / (2 * kScaleChunks), half = (x / kScaleChunks) & 1, ch = x % kScaleChunks;
                    const char* from = reinterpret_cast<const char*>(which ? c.v_scales : c.k_scales) + (half ? at1 : at0) * G::kScales + ch * 16;
                    copy16(base + (which ? G::kVs : G::kKs) + (half * kScaleChunks + ch) * 16, from, (half ? page1 : page0) >= 0);
                }
            }
        }
        copies_commit();
    };

    int page_next = page_for(mine);
#pragma unroll
    for (int s = 0; s < G::kStages - 1; ++s) {
        const int page = page_next;
        page_next = page_for(mine + (s + 1) * stride);
        request(mine + s * stride, page, s);
    }
    const uint2* frag = reinterpret_cast<const uint2*>(q_frag) + lane;
    uint32_t slot = 0;
    for (int j = mine; j < tiles; j += stride) {
        {
            const int page = page_next, ahead = j + (G::kStages - 1) * stride;
            page_next = page_for(ahead + stride);
            request(ahead, page, slot == 0 ? G::kStages - 1 : slot - 1);
        }
        copies_wait<G::kStages - 1>();
        __syncwarp();
        const unsigned char* st = ring + slot * G::kStage;
        const int base = begin + 32 * j;

        float s[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int n = 0; n < NT; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.0f;
            const uint32_t pa = 16 * h + position_of<D>(g), pb = pa + 8;
#pragma unroll
            for (int part = 0; part < (D == 256 ? 2 : 1); ++part) {
                constexpr int kWords = D == 64 ? 2 : 4;
                uint32_t wa[kWords], wb[kWords];
                const uint32_t block = D == 64 ? t >> 1 : part * 4 + t;
                if (D == 64) {
                    const uint2 x = *reinterpret_cast<const uint2*>(st + G::kK + pa * G::kRow + t * 8), y = *reinterpret_cast<const uint2*>(st + G::kK + pb * G::kRow + t * 8);
                    wa[0] = x.x; wa[1] = x.y; wb[0] = y.x; wb[1] = y.y;
                } else {
                    const uint4 x = *reinterpret_cast<const uint4*>(st + G::kK + pa * G::kRow + chunk_of<D>(pa, block) * 16);
                    const uint4 y = *reinterpret_cast<const uint4*>(st + G::kK + pb * G::kRow + chunk_of<D>(pb, block) * 16);
                    wa[0] = x.x; wa[1] = x.y; wa[kWords - 2] = x.z; wa[kWords - 1] = x.w;
                    wb[0] = y.x; wb[1] = y.y; wb[kWords - 2] = y.z; wb[kWords - 1] = y.w;
                }
                const __half2 da = __half2half2(*reinterpret_cast<const __half*>(st + G::kKs + pa * G::kScales + block * 2));
                const __half2 db = __half2half2(*reinterpret_cast<const __half*>(st + G::kKs + pb * G::kScales + block * 2));
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    uint32_t va[4], vb[4];
                    widen(wa[w], da, va);
                    widen(wb[w], db, vb);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int step = part * 8 + 2 * w + u;
                            const uint2 q = frag[(n * G::kSteps + step) * 32];
                            mma16816(s[h][n], va[2 * u], vb[2 * u], va[2 * u + 1], vb[2 * u + 1], q.x, q.y);
                            if (kTwo) {
                                const uint2 r = frag[((NT + n) * G::kSteps + step) * 32];
                                mma16816(s[h][n], va[2 * u], vb[2 * u], va[2 * u + 1], vb[2 * u + 1], r.x, r.y);
                            }
                        }
                    }
                }
            }
        }

        // scores in powers of two, hidden ones to -inf
        const bool whole = base + 31 <= first_pos && base + 31 <= hi && (a.window == 0 || (long long)base > last_pos - (long long)a.window);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[h][n][e] *= scale[n][e & 1];
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const long long at = context + (row0 + n * 8 + 2 * t + e) / group;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int p = base + 16 * h + 8 * u + int(position_of<D>(g));
                            const bool seen = p <= at && p <= hi && (a.window == 0 || p > at - (long long)a.window);
                            if (!seen) s[h][n][2 * u + e] = -INFINITY;
                        }
                    }
                }
            }
        }
        // The maximum moves only where a score is 2^8 above it: weights up to 256 fit f16 as well as those up to 1 do.
        bool above = false;
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[n][e] = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
                above = above || top[n][e] > m[n][e] + 8.0f;
            }
        }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float keep[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = top[n][e];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    x = fmaxf(x, m[n][e]);
                    keep[e] = m[n][e] == -INFINITY ? 0.0f : exp2_fast(m[n][e] - x);
                    m[n][e] = x;
                    l[n][e] *= keep[e];
                }
#pragma unroll
                for (int i = 0; i < G::kSteps; ++i) {
                    o[i][n][0] *= keep[0];
                    o[i][n][1] *= keep[1];
                    o[i][n][2] *= keep[0];
                    o[i][n][3] *= keep[1];
                }
            }
        }
        uint32_t p_high[2][NT][2], p_low[2][NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float base0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], base1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float x = exp2_fast(s[h][n][2 * u] - base0), y = exp2_fast(s[h][n][2 * u + 1] - base1);
                    l[n][0] += x;
                    l[n][1] += y;
                    const __half2 high = __floats2half2_rn(x, y);
                    p_high[h][n][u] = transposed(bits(high));
                    if (kTwo) p_low[h][n][u] = transposed(bits(__floats2half2_rn(x - __low2float(high), y - __high2float(high))));
                }
            }
        }

#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // the positions of this lane's two pairs (see position_of); what the tile's rows do not see has scale 0, whatever lies there
            const uint32_t pos[4] = {16 * h + t, 16 * h + 4 + (t ^ (D == 128 ? 1 : 2)), 16 * h + 8 + t, 16 * h + 12 + (t ^ (D == 128 ? 1 : 2))};
            constexpr int kWords = D / 64;
            uint32_t w[4][kWords];
            __half d[4];
            const uint32_t block = D == 64 ? g >> 2 : D == 128 ? g >> 1 : g;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned char* row = st + G::kV + pos[i] * G::kRow;
                if (D == 64) {
                    w[i][0] = *reinterpret_cast<const uint32_t*>(row + g * 4);
                } else if (D == 128) {
                    const uint2 x = *reinterpret_cast<const uint2*>(row + chunk_of<D>(pos[i], g >> 1) * 16 + (g & 1) * 8);
                    w[i][0] = x.x; w[i][kWords - 1] = x.y;
                } else {
                    const uint4 x = *reinterpret_cast<const uint4*>(row + chunk_of<D>(pos[i], g) * 16);
                    w[i][0] = x.x; w[i][1 % kWords] = x.y; w[i][2 % kWords] = x.z; w[i][kWords - 1] = x.w;
                }
                const int p = base + int(pos[i]);
                d[i] = p >= lo && p <= hi ? *reinterpret_cast<const __half*>(st + G::kVs + pos[i] * G::kScales + block * 2) : __half(0.0f);
            }
            const __half2 d0 = __halves2half2(d[0], d[1]), d1 = __halves2half2(d[2], d[3]);
#pragma unroll
            for (int x = 0; x < kWords; ++x) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    uint32_t v0[4], v1[4];
                    widen(__byte_perm(w[0][x], w[1][x], z ? 0x7632 : 0x5410), d0, v0);
                    widen(__byte_perm(w[2][x], w[3][x], z ? 0x7632 : 0x5410), d1, v1);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int i = x * 4 + z * 2 + u;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma16816(o[i][n], v0[2 * u], v0[2 * u + 1], v1[2 * u], v1[2 * u + 1], p_high[h][n][0], p_high[h][n][1]);
                            if (kTwo) mma16816(o[i][n], v0[2 * u], v0[2 * u + 1], v1[2 * u], v1[2 * u + 1], p_low[h][n][0], p_low[h][n][1]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        slot = slot + 1 == G::kStages ? 0 : slot + 1;
    }
    copies_wait<0>();
    release_next();
    __syncthreads();  // the rings become the warps' results

    // ---- join ----
    float* part = reinterpret_cast<float*>(smem) + size_t(warp) * kRows * G::kPitch;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = l[n][e];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            const uint32_t r = n * 8 + 2 * t + e;
            if (g == 0) {
                warp_top[warp * kRows + r] = m[n][e];
                warp_sum_[warp * kRows + r] = x;
            }
#pragma unroll
            for (int i = 0; i < G::kSteps; ++i) {  // value f = (2 i + upper) 8 + g of the row is dim (B / 16) 32 + B % 16 + 16 upper, B = g D / 16 + i
                part[r * G::kPitch + (2 * i) * 8 + g] = o[i][n][e];
                part[r * G::kPitch + (2 * i + 1) * 8 + g] = o[i][n][2 + e];
            }
        }
    }
    __syncthreads();
    for (uint32_t x = tid; x < uint32_t(G::kWarps * kRows); x += kThreads) {  // warp_top becomes each warp's factor
        const uint32_t r = x % kRows;
        float most = -INFINITY;
        for (int w = 0; w < G::kWarps; ++w) most = fmaxf(most, warp_top[w * kRows + r]);
        const float mine_top = warp_top[x];
        weight[x] = mine_top == -INFINITY ? 0.0f : exp2_fast(mine_top - most);
        if (x < kRows) cta_top[r] = most;
    }
    __syncthreads();
    if (tid < kRows) {
        float sum = 0.0f;
        for (int w = 0; w < G::kWarps; ++w) sum = fmaf(warp_sum_[w * kRows + tid], weight[w * kRows + tid], sum);
        cta_sum[tid] = sum;
    }
    float* joined = reinterpret_cast<float*>(smem);
    for (uint32_t x = tid; x < uint32_t(kRows * D); x += kThreads) {
        const uint32_t at = (x / D) * G::kPitch + x % D;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < G::kWarps; ++w) sum = fmaf(joined[size_t(w) * kRows * G::kPitch + at], weight[w * kRows + x / D], sum);
        joined[at] = sum;  // of its own value only: no other thread reads it here
    }
    if (S > 1) cluster.sync();
    else __syncthreads();
    // the CTAs' factors over the sum of all
    if (tid < kRows) {
        float most = -INFINITY, sum = 0.0f;
        for (uint32_t k = 0; k < S; ++k) most = fmaxf(most, *cluster.map_shared_rank(cta_top + tid, k));
        for (uint32_t k = 0; k < S; ++k) {
            const float top = *cluster.map_shared_rank(cta_top + tid, k), w = top == -INFINITY ? 0.0f : exp2_fast(top - most);
            sum = fmaf(*cluster.map_shared_rank(cta_sum + tid, k), w, sum);
            weight[k * kRows + tid] = w;
        }
        row_scale[tid] = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
    }
    __syncthreads();
    for (uint32_t x = rank * kThreads + tid; x < rows * D; x += S * kThreads) {
        const uint32_t r = x / D, f = x % D, at = r * G::kPitch + f;
        float sum = 0.0f;
        for (uint32_t k = 0; k < S; ++k) sum = fmaf(*cluster.map_shared_rank(joined + at, k), weight[k * kRows + r], sum);
        const uint32_t B = (f & 7) * (D / 16) + (f >> 4), dim = (B >> 4) * 32 + (B & 15) + ((f >> 3) & 1) * 16;
        put(static_cast<T*>(a.out) + size_t(first_row + (row0 + r) / group) * a.out_stride + size_t(kv * group + (row0 + r) % group) * D + dim, sum * row_scale[r]);
    }
    if (S > 1) cluster.sync();  // nobody leaves while its shared memory is read
}

uint32_t multiprocessors() {
    int dev = 0, count = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
    return uint32_t(count);
}

template <class T, int D, int NT>
void attend_split(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, bool dependent, cudaStream_t s) {
    using G = Split<D>;
    const auto kernel = cache4_split_kernel<T, D, NT>;
    constexpr size_t smem = G::smem(NT, sizeof(T) == 4);
    static_assert(smem <= 227 * 1024);
    static DeviceOnce once;
    if (once.first()) {
        BK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
        BK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    }
    const uint64_t rows = uint64_t(b.max_tokens) * (a.heads / c.kv_heads), tiles = (rows + 8 * NT - 1) / (8 * NT);
    const uint64_t units = tiles * c.kv_heads * b.sequences;
    const uint64_t length = a.window != 0 ? std::min<uint64_t>(b.max_length, uint64_t(a.window) + 8 * NT + 31) : b.max_length;
    uint32_t split = 1;
    while (split < 16 && units * split < 2 * multiprocessors() && length > uint64_t(split) * G::kWarps * 64) split *= 2;
    if (units / b.sequences * split > 0x7fffffffull) throw CudaError("cuda: the 4-bit cache's attention takes fewer rows than these");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(uint32_t(units / b.sequences * split), b.sequences);
    cfg.blockDim = dim3(G::kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    BK_CUDA(cudaLaunchKernelEx(&cfg, kernel, c, b, a));
}

template <class T, int D>
void attend_sized(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, bool dependent, cudaStream_t s) {
    const uint64_t rows = uint64_t(b.max_tokens) * (a.heads / c.kv_heads);
    if (rows <= 8) attend_split<T, D, 1>(c, b, a, dependent, s);
    else if (rows <= 16 || D == 256) attend_split<T, D, 2>(c, b, a, dependent, s);
    else if constexpr (D < 256) attend_split<T, D, 4>(c, b, a, dependent, s);
}

template <class T>
void attend(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, bool dependent, cudaStream_t s) {
    if (c.dim == 64) attend_sized<T, 64>(c, b, a, dependent, s);
    else if (c.dim == 128) attend_sized<T, 128>(c, b, a, dependent, s);
    else attend_sized<T, 256>(c, b, a, dependent, s);
}

}  // namespace

void launch_cache4_attention(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, int type, bool dependent, cudaStream_t s) {
    if (type == T_F32) attend<float>(c, b, a, dependent, s);
    else if (type == T_F16) attend<__half>(c, b, a, dependent, s);
    else attend<__nv_bfloat16>(c, b, a, dependent, s);
}

}  // namespace bk
