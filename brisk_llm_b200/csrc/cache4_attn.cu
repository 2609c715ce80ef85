// Attention over the paged cache in 4 bits, for few rows: single tokens, verify steps, and whatever cache4_prompt.cu leaves.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "cache4_math.cuh"
#include "pdl.cuh"

namespace bk {
namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // an 8 x 8 matrix of f16, lane (g, t) holding row g, columns 2 t and 2 t + 1
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(v));
    return y;
}

// 16 bytes to shared memory; zeros where !there (src is then any valid address).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The eight numbers of a word (see widen) without a scale.
__device__ __forceinline__ void centred(uint32_t w, uint32_t (&v)[4]) {
    const uint32_t magic = 0x64006400u, u = w >> 8;
    const __half2 bias = halves(0x64086408u), sixteenth = halves(0x2c002c00u), less = halves(0xd480d480u);  // 1032, 1 / 16, -72
    v[0] = bits(__hsub2(halves((w & 0x000f000fu) | magic), bias));
    v[1] = bits(__hfma2(halves((w & 0x00f000f0u) | magic), sixteenth, less));
    v[2] = bits(__hsub2(halves((u & 0x000f000fu) | magic), bias));
    v[3] = bits(__hfma2(halves((u & 0x00f000f0u) | magic), sixteenth, less));
}
// The numbers n, not n - 8, as they are: four bits at the bottom of an f16 are n 2^-24, at bit 4 they are 16 n 2^-24, both exact.
__device__ __forceinline__ void as_they_are(uint32_t w, uint32_t (&v)[4]) {
    const uint32_t u = w >> 8;
    v[0] = w & 0x000f000fu;
    v[1] = w & 0x00f000f0u;
    v[2] = u & 0x000f000fu;
    v[3] = u & 0x00f000f0u;
}

// .aligned: by whole warps
__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// W warps a CTA, 8 NT rows, f32 (two f16 parts) or not.
template <int D, int NT, int W, bool TWO> struct Split {
    static constexpr int kTile = 32;  // positions a warp takes at a time
    static constexpr int kRows = 8 * NT, kThreads = 32 * W;
    static constexpr int kStages = D == 64 ? 4 : 3;
    static constexpr int kRow = D / 2, kScales = D / 16;  // bytes of a position
    static constexpr int kK = 0, kV = kTile * kRow, kKs = 2 * kTile * kRow, kVs = kKs + kTile * kScales, kStage = kVs + kTile * kScales;
    static constexpr int kOrdered = kThreads < 128 ? kThreads : 128;  // sequences that are put in order
    static constexpr uint32_t kManyCtas = 296;
    static constexpr int kPitch = D + 4;  // floats between two rows of a warp's result
    static constexpr int kSteps = D / 16;
    static constexpr bool kHeld = NT == 1 && !TWO && D <= 128;  // the queries stay in registers
    static constexpr size_t kRing = size_t(W) * kStages * kStage, kParts = size_t(W) * kRows * kPitch * 4;
    // behind the loop, in the ring's place: the warps' results, this CTA's share of all CTAs', each warp's maximum, sum and factor and the
    // CTAs' maxima and sums of each row
    static constexpr size_t kJoining = kParts + size_t(kRows) * D * 4 + size_t(kRows) * (3 * W + 32) * 4;
    static constexpr size_t kBody = kRing > kJoining ? kRing : kJoining;
    static constexpr size_t kQueries = size_t(NT) * kSteps * 32 * 8 * (TWO ? 2 : 1);
    // queries that go to registers pass through the last stage of the first warp, which the loop fills first
    static constexpr size_t kQueriesAt = kHeld ? size_t(kStages - 1) * kStage : kBody;
    static_assert(!kHeld || kQueries <= size_t(kStage));
    static constexpr size_t kRowsAt = kBody + (kHeld ? 0 : kQueries), kBytes = kRowsAt + size_t(kRows) * (3 + D / 32) * 4;
    // CTAs of an SM that registers and shared memory are meant for
    static constexpr int kResident = D < 256 && (NT == 1 || (NT == 2 && D == 64)) ? 16 / W : W == 4 ? 2 : 1;
};

// Where 16 bytes of a position's row lie in a stage, and which position a row of a matrix instruction is: chosen so that the loads of
// keys (8 rows, 4 bytes of one block to a lane) and of values (4 rows, an eighth to a lane) meet no shared-memory bank twice.
template <int D> __device__ __forceinline__ uint32_t chunk_of(uint32_t position, uint32_t chunk) {
    if (D == 64) return chunk ^ ((position >> 2) & 1);
    if (D == 128) return chunk ^ (((position >> 1) & 1) << 1) ^ ((position >> 2) & 1);
    return chunk ^ ((position & 3) << 1) ^ ((position >> 2) & 1);
}
template <int D> __device__ __forceinline__ uint32_t position_of(uint32_t g) {  // g < 8
    return (g & 1) ? 4 + ((g >> 1) ^ (D == 128 ? 1 : 2)) : g >> 1;
}

// softmax(q k) v for 8 NT rows - tokens times the query heads of one key/value head - of one sequence. A cluster of CTAs shares the
// positions, each warp takes tiles of 32 of them with a running level (of the maximum) and sum of its own; the warps' results are joined in
// shared memory, the CTAs' over the cluster's. Positions are the rows (M) and queries the columns (N = 8) of both products,
//     S^T = K Q^T (16 positions x 8 queries),     O^T = V^T P^T (16 dims x 8 queries),
// so that eight query heads fill an instruction and the 4-bit words become its A operand in registers, straight from the
// stage that cp.async filled: any order of the head's values does for K Q^T as long as Q has the same. P^T is S^T transposed in the warp.
// f32 queries and weights are two f16 parts each (22 bits); others one.
template <class T, int D, int NT, int W>
__global__ void __launch_bounds__(32 * W, Split<D, NT, W, sizeof(T) == 4>::kResident) cache4_split_kernel(const Cache4 c, const Cache4Batch b, const Cache4Attend a) {
    constexpr bool kTwo = sizeof(T) == 4;
    using G = Split<D, NT, W, kTwo>;
    constexpr int kRows = G::kRows, kThreads = G::kThreads;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* q_frag = smem + G::kQueriesAt;
    float* row_scale = reinterpret_cast<float*>(smem + G::kRowsAt);  // [kRows]
    int* row_last = reinterpret_cast<int*>(row_scale + kRows);       // [kRows] the last position a row sees
    int* row_first = row_last + kRows;                               // [kRows] and the first
    float* offset = reinterpret_cast<float*>(row_first + kRows);     // [D / 32][kRows]
    float* received = reinterpret_cast<float*>(smem + G::kParts);    // [S][kRows D / S]: this CTA's share of every CTA's result
    float* warp_top = received + kRows * D;                          // [W][kRows]
    float* warp_total = warp_top + W * kRows;
    float* factor = warp_total + W * kRows;
    float* tops = factor + W * kRows;  // [16][kRows], of the cluster's CTAs
    float* totals = tops + 16 * kRows;

    wait_for_previous();
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t S = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t unit = blockIdx.x / S, kv = unit % c.kv_heads, tile = unit / c.kv_heads;
    uint32_t sequence = blockIdx.y;
    if (gridDim.y > 1 && gridDim.y <= uint32_t(G::kOrdered) && gridDim.x * gridDim.y > G::kManyCtas) {
        // Ragged sequences and more CTAs than fit at a time: the longest go first, so that none begins when the others are done. Every CTA finds
        // the sequence of its place for itself (one token of 64 sequences of up to 8000 positions 107 -> 83 us).
        int* length = reinterpret_cast<int*>(smem);  // the rings are empty yet
        uint32_t* chosen = reinterpret_cast<uint32_t*>(length + G::kOrdered);
        if (tid < gridDim.y) length[tid] = b.context[tid];
        __syncthreads();
        if (tid < gridDim.y) {
            const int mine = length[tid];
            uint32_t before = 0;
#pragma unroll 8
            for (uint32_t i = 0; i < gridDim.y; ++i) before += length[i] > mine || (length[i] == mine && i < tid);
            if (before == blockIdx.y) *chosen = tid;
        }
        __syncthreads();
        sequence = *chosen;
        __syncthreads();
    }
    const uint32_t group = a.heads / c.kv_heads;
    const long long context = b.context[sequence];
    uint32_t first_row, count;
    sequence_rows(b, sequence, first_row, count);
    const uint32_t total = count * group, row0 = tile * kRows;
    if (row0 >= total) return;  // the whole cluster
    const uint32_t rows = min(total - row0, uint32_t(kRows));
    // the positions that a token of the sequence sees; last < first: none
    const long long held = (long long)b.columns * c.page_size;
    auto last_of = [&](uint32_t token) { return int(max(min(context + token, held - 1), -1ll)); };
    auto first_of = [&](uint32_t token) { return a.window != 0 ? int(min(max(context + token - (long long)a.window + 1, 0ll), held)) : 0; };
    const uint32_t token0 = row0 / group, token1 = (row0 + rows - 1) / group;
    const int lo = first_of(token0), hi = last_of(token1);
    const int whole_from = first_of(token1), whole_to = last_of(token0);  // what every row sees

    // ---- the warp's tiles: begin + 32 (rank + S (warp + W i)) and on ----
    const int begin = lo & ~31;
    const int tiles = hi >= lo ? (hi - begin) / 32 + 1 : 0, stride = int(S) * W, mine = int(warp * S + rank);
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
    // ---- queries: a power of two brings a row's largest value to 2^10, so that bf16 and both parts of f32 fit f16. For f16 and bf16 the
    // keys' numbers are used as they are: values that meet the high four bits of a byte are a sixteenth, and the -8 of a block's numbers is
    // -8 times the sum of its queries, where the sum begins. That takes a third of the instructions and, as the sums cancel, two bits of
    // 32-bit sums that f32 queries would miss: theirs are n - 8. ----
    for (uint32_t r = warp; r < kRows; r += W) {
        float x[D / 32], most = 0.0f;
        const uint32_t token = (row0 + r) / group, head = (row0 + r) - token * group;
        const T* src = static_cast<const T*>(a.q) + size_t(first_row + token) * a.q_stride + size_t(kv * group + head) * D;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            x[j] = r < rows ? to_float(src[lane + 32 * j]) : 0.0f;
            most = fmaxf(most, fabsf(x[j]));
        }
        most = warp_max(most);
        const int exponent = int(__float_as_uint(most) >> 23) - 127, up = most < INFINITY ? min(10 - exponent, 100) : 0;
        const uint32_t byte = lane & 15;
        const bool sixteenth = !kTwo && lane >= 16;
        const float by = __uint_as_float(uint32_t(127 + up - (sixteenth ? 4 : 0)) << 23) * (a.scale < 0.0f ? -1.0f : 1.0f);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const float v = x[j] * by;
            const __half high = __float2half_rn(v);
            const uint32_t step = 2 * j + (byte & 1), at = ((((r >> 3) * G::kSteps + step) * 32 + (r & 7) * 4 + (byte >> 2)) * 2 + (lane >> 4)) * 2 + ((byte >> 1) & 1);
            __half* dst = reinterpret_cast<__half*>(q_frag);
            dst[at] = high;
            if (kTwo) {
                dst[at + NT * G::kSteps * 128] = __float2half_rn(v - __half2float(high));
            } else {
                const float sum = warp_sum(__half2float(high) * (sixteenth ? 16.0f : 1.0f));
                if (lane == 0) offset[j * kRows + r] = sum * -0x1p-21f;  // -8 times it, in units of 2^-24
            }
        }
        if (lane == 0) {
            // (a query of 2^113 would take this past 32 bits: then scores are as large as they can be, and one position has the weight)
            row_scale[r] = fminf(fabsf(a.scale) * 1.4426950408889634f * __uint_as_float(uint32_t(127 - up) << 23) * (kTwo ? 1.0f : 0x1p24f), 3e38f);
            row_last[r] = last_of(token);
            row_first[r] = first_of(token);
        }
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

    const uint2* frag = reinterpret_cast<const uint2*>(q_frag) + lane;
    constexpr bool kHeld = G::kHeld;
    uint2 held_q[kHeld ? G::kSteps : 1];
    if (kHeld) {
#pragma unroll
        for (int i = 0; i < G::kSteps; ++i) held_q[kHeld ? i : 0] = frag[i * 32];
        __syncthreads();
    }
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
            constexpr int kBlocks = D / 32;
            float da[kBlocks], db[kBlocks];
#pragma unroll
            for (int i = 0; i < kBlocks / 2; ++i) {
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(st + G::kKs + pa * G::kScales + i * 4));
                const float2 y = __half22float2(*reinterpret_cast<const __half2*>(st + G::kKs + pb * G::kScales + i * 4));
                da[2 * i] = x.x; da[2 * i + 1] = x.y;
                db[2 * i] = y.x; db[2 * i + 1] = y.y;
            }
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) {
                uint32_t va[4], vb[4];
                const uint32_t wa = *reinterpret_cast<const uint32_t*>(st + G::kK + pa * G::kRow + chunk_of<D>(pa, k) * 16 + t * 4);
                const uint32_t wb = *reinterpret_cast<const uint32_t*>(st + G::kK + pb * G::kRow + chunk_of<D>(pb, k) * 16 + t * 4);
                if (kTwo) {
                    centred(wa, va);
                    centred(wb, vb);
                } else {
                    as_they_are(wa, va);
                    as_they_are(wb, vb);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float2 begin_at = kTwo ? make_float2(0.0f, 0.0f) : *reinterpret_cast<const float2*>(offset + k * kRows + n * 8 + 2 * t);
                    float y[4];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint2 q = kHeld ? held_q[kHeld ? 2 * k + u : 0] : frag[(n * G::kSteps + 2 * k + u) * 32];
                        if (u == 0) mma16816(y, va[0], vb[0], va[1], vb[1], q.x, q.y, begin_at.x, begin_at.y);
                        else mma16816(y, va[2], vb[2], va[3], vb[3], q.x, q.y);
                        if (kTwo) {
                            const uint2 r = frag[((NT + n) * G::kSteps + 2 * k + u) * 32];
                            mma16816(y, va[2 * u], vb[2 * u], va[2 * u + 1], vb[2 * u + 1], r.x, r.y);
                        }
                    }
                    s[h][n][0] = fmaf(y[0], da[k], s[h][n][0]);
                    s[h][n][1] = fmaf(y[1], da[k], s[h][n][1]);
                    s[h][n][2] = fmaf(y[2], db[k], s[h][n][2]);
                    s[h][n][3] = fmaf(y[3], db[k], s[h][n][3]);
                }
            }
        }

        // scores in powers of two, hidden ones to -inf
        const bool whole = base + 31 <= whole_to && base >= whole_from;
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
                    const int last = row_last[n * 8 + 2 * t + e], first = row_first[n * 8 + 2 * t + e];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int p = base + 16 * h + 8 * u + int(position_of<D>(g));
                            if (p > last || p < first) s[h][n][2 * u + e] = -INFINITY;
                        }
                    }
                }
            }
        }
        // Values past what an f16 holds among those that the tile's rows see (see past_f16; the keys' scales are multiplied in 32 bits).
        bool large;
        {
            const __half2* d = reinterpret_cast<const __half2*>(st + G::kVs + lane * G::kScales);  // of the lane's position
            __half2 most = larger(d[0], d[D / 64 - 1]);
            if (D == 256) most = larger(most, larger(d[1], d[2 % (D / 64)]));
            large = past_f16(__hmax(__low2half(most), __high2half(most))) && (whole || (base + int(lane) >= lo && base + int(lane) <= hi));
        }
        // The level (see Level) moves only where a weight would no longer fit.
        bool above = large;
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[n][e] = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
                above = above || top[n][e] > m[n][e] + Level<kTwo>::kMost;
            }
        }
        bool fold = false;
        if (__any_sync(0xffffffffu, above)) {
            fold = __any_sync(0xffffffffu, large);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float keep[2];
                if (fold) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        m[n][e] -= kFoldBits;
                        l[n][e] *= kUnfold;
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = top[n][e];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    x = fmaxf(x - Level<kTwo>::kBelow, m[n][e]);
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

        constexpr int kWords = D / 64;
        const uint32_t value_block = D == 64 ? g >> 2 : D == 128 ? g >> 1 : g;
        // Values of 16 positions as this lane's two pairs (see position_of); what the tile's rows do not see has scale 0, whatever lies there.
        auto load_values = [&](int h, uint32_t (&w)[4][kWords], __half2 (&pair)[2]) {
            const uint32_t odd = t ^ (D == 128 ? 1 : 2), pos[4] = {16 * h + t, 16 * h + 4 + odd, 16 * h + 8 + t, 16 * h + 12 + odd};
            __half d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned char* row = st + G::kV + pos[i] * G::kRow;
                if (D == 64) {
                    w[i][0] = *reinterpret_cast<const uint32_t*>(row + chunk_of<D>(pos[i], g >> 2) * 16 + (g & 3) * 4);
                } else if (D == 128) {
                    const uint2 x = *reinterpret_cast<const uint2*>(row + chunk_of<D>(pos[i], g >> 1) * 16 + (g & 1) * 8);
                    w[i][0] = x.x; w[i][kWords - 1] = x.y;
                } else {
                    const uint4 x = *reinterpret_cast<const uint4*>(row + chunk_of<D>(pos[i], g) * 16);
                    w[i][0] = x.x; w[i][1 % kWords] = x.y; w[i][2 % kWords] = x.z; w[i][kWords - 1] = x.w;
                }
                d[i] = *reinterpret_cast<const __half*>(st + G::kVs + pos[i] * G::kScales + value_block * 2);
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int p = base + int(pos[i]);
                    if (p < lo || p > hi) d[i] = __half(0.0f);
                }
            }
            pair[0] = __halves2half2(d[0], d[1]);
            pair[1] = __halves2half2(d[2], d[3]);
            if (fold) {
                pair[0] = __hmul2(pair[0], __float2half2_rn(kFold));
                pair[1] = __hmul2(pair[1], __float2half2_rn(kFold));
            }
        };
        if constexpr (kTwo) {
            // A product cuts its sum off at 24 bits: adding to a long sum each time loses a third of a bit of it per product, all one way. The tile's
            // products make a sum of their own, and that is added with rounding.
            uint32_t w[2][4][kWords];
            __half2 pair[2][2];
            load_values(0, w[0], pair[0]);
            load_values(1, w[1], pair[1]);
#pragma unroll
            for (int x = 0; x < kWords; ++x) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    uint32_t v[2][2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        widen(__byte_perm(w[h][0][x], w[h][1][x], z ? 0x7632 : 0x5410), pair[h][0], v[h][0]);
                        widen(__byte_perm(w[h][2][x], w[h][3][x], z ? 0x7632 : 0x5410), pair[h][1], v[h][1]);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int i = x * 4 + z * 2 + u;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float y[4];
                            mma16816(y, v[0][0][2 * u], v[0][0][2 * u + 1], v[0][1][2 * u], v[0][1][2 * u + 1], p_low[0][n][0], p_low[0][n][1], 0.0f, 0.0f);
                            mma16816(y, v[1][0][2 * u], v[1][0][2 * u + 1], v[1][1][2 * u], v[1][1][2 * u + 1], p_low[1][n][0], p_low[1][n][1]);
                            mma16816(y, v[0][0][2 * u], v[0][0][2 * u + 1], v[0][1][2 * u], v[0][1][2 * u + 1], p_high[0][n][0], p_high[0][n][1]);
                            mma16816(y, v[1][0][2 * u], v[1][0][2 * u + 1], v[1][1][2 * u], v[1][1][2 * u + 1], p_high[1][n][0], p_high[1][n][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[i][n][e] += y[e];
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[4][kWords];
                __half2 pair[2];
                load_values(h, w, pair);
#pragma unroll
                for (int x = 0; x < kWords; ++x) {
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        uint32_t v0[4], v1[4];
                        widen(__byte_perm(w[0][x], w[1][x], z ? 0x7632 : 0x5410), pair[0], v0);
                        widen(__byte_perm(w[2][x], w[3][x], z ? 0x7632 : 0x5410), pair[1], v1);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma16816(o[x * 4 + z * 2 + u][n], v0[2 * u], v0[2 * u + 1], v1[2 * u], v1[2 * u + 1], p_high[h][n][0], p_high[h][n][1]);
                        }
                    }
                }
            }
        }
        if (fold) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    m[n][e] += kFoldBits;
                    l[n][e] *= kFold;
                }
            }
        }
        __syncwarp();
        slot = slot + 1 == G::kStages ? 0 : slot + 1;
    }
    copies_wait<0>();
    release_next();
    __syncthreads();  // the rings become the warps' results
    if (S > 1) cluster_arrive();  // waited for before anything is written into another CTA's

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
                warp_total[warp * kRows + r] = x;
            }
#pragma unroll
            for (int i = 0; i < G::kSteps; ++i) {  // value f = (2 i + upper) 8 + g of the row is dim (B / 16) 32 + B % 16 + 16 upper, B = g D / 16 + i
                part[r * G::kPitch + (2 * i) * 8 + g] = o[i][n][e];
                part[r * G::kPitch + (2 * i + 1) * 8 + g] = o[i][n][2 + e];
            }
        }
    }
    __syncthreads();
    if (tid < kRows) {
        float most = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) most = fmaxf(most, warp_top[w * kRows + tid]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float top = warp_top[w * kRows + tid], x = top == -INFINITY ? 0.0f : exp2_fast(top - most);
            factor[w * kRows + tid] = x;
            sum = fmaf(warp_total[w * kRows + tid], x, sum);
        }
        if (S == 1) row_scale[tid] = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
        tops[rank * kRows + tid] = most;
        totals[rank * kRows + tid] = sum;
    }
    __syncthreads();
    // value f of a row is this dim of the head (see above)
    auto dim_of = [](uint32_t f) {
        const uint32_t B = (f & 7) * (D / 16) + (f >> 4);
        return (B >> 4) * 32 + (B & 15) + ((f >> 3) & 1) * 16;
    };
    auto row_of = [&](uint32_t r) {
        const uint32_t token = (row0 + r) / group;
        return static_cast<T*>(a.out) + size_t(first_row + token) * a.out_stride + size_t(kv * group + (row0 + r) - token * group) * D;
    };
    // Where a cluster has several CTAs each sums a share of the values: the others write theirs into it, then all meet once.
    const uint32_t share_log = 31 - __clz(uint32_t(kRows * D)) - (31 - __clz(S)), share = 1u << share_log;
    if (S > 1) cluster_wait();
    for (uint32_t r = warp; r < kRows; r += W) {
        if (S == 1 && r >= rows) break;
        float by[W];
#pragma unroll
        for (int w = 0; w < W; ++w) by[w] = factor[w * kRows + r];
        T* out = row_of(r);
        const float scale_r = S == 1 ? row_scale[r] : 1.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint32_t f = i * 32 + lane;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) sum = fmaf(reinterpret_cast<const float*>(smem)[(w * kRows + r) * G::kPitch + f], by[w], sum);
            if (S == 1) {
                put(out + dim_of(f), sum * scale_r);
            } else {
                const uint32_t x = r * D + f;
                *cluster.map_shared_rank(received + rank * share + (x & (share - 1)), x >> share_log) = sum;
            }
        }
    }
    if (S == 1) return;
    for (uint32_t x = tid; x < kRows * S; x += kThreads) {
        const uint32_t r = x % kRows, k = x / kRows;
        if (k != rank) {
            *cluster.map_shared_rank(tops + rank * kRows + r, k) = tops[rank * kRows + r];
            *cluster.map_shared_rank(totals + rank * kRows + r, k) = totals[rank * kRows + r];
        }
    }
    cluster_arrive();
    cluster_wait();
    if (tid < kRows) {
        float most = -INFINITY, sum = 0.0f;
        for (uint32_t k = 0; k < S; ++k) most = fmaxf(most, tops[k * kRows + tid]);
        for (uint32_t k = 0; k < S; ++k) {
            const float top = tops[k * kRows + tid], x = top == -INFINITY ? 0.0f : exp2_fast(top - most);
            sum = fmaf(totals[k * kRows + tid], x, sum);
            tops[k * kRows + tid] = x;  // now its factor
        }
        row_scale[tid] = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
    }
    __syncthreads();
    for (uint32_t x = tid; x < share; x += kThreads) {
        const uint32_t r = (rank * share + x) / D;
        float sum = 0.0f;
        for (uint32_t k = 0; k < S; ++k) sum = fmaf(received[k * share + x], tops[k * kRows + r], sum);
        if (r < rows) put(row_of(r) + dim_of((rank * share + x) % D), sum * row_scale[r]);
    }
}

template <class T, int D, int NT, int W>
void launch_split(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, uint64_t units, uint32_t split, bool dependent, cudaStream_t s) {
    using G = Split<D, NT, W, sizeof(T) == 4>;
    const auto kernel = cache4_split_kernel<T, D, NT, W>;
    static_assert(G::kBytes <= 227 * 1024);
    static DeviceSetup setup;
    setup.once([&] {
        BK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(G::kBytes)));
        BK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    });
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(uint32_t(units / b.sequences * split), b.sequences);
    cfg.blockDim = dim3(32 * W);
    cfg.dynamicSmemBytes = G::kBytes;
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

template <class T, int D, int NT>
void attend_split(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, bool dependent, cudaStream_t s) {
    const uint64_t rows = uint64_t(b.max_tokens) * (a.heads / c.kv_heads), tiles = (rows + 8 * NT - 1) / (8 * NT);
    const uint64_t units = tiles * c.kv_heads * b.sequences;
    const uint64_t length = a.window != 0 ? std::min<uint64_t>(b.max_length, uint64_t(a.window) + 8 * NT + 31) : b.max_length;
    // Clusters grow while that gives the SMs CTAs (about four thirds for each with 8 rows; one for every second with 16, whose rings leave
    // no room for another) and every warp tiles: one, for 16 CTAs four. us at S = 1, 2, 4, 8, 16: one token of 8 key/value heads at 517
    // positions 8.0 7.8 6.5 6.5 7.5, at 32 767 192 107 56 33 27; 36 rows of 8 heads at 2064 20 15 14 19 24; 20 rows at 8000 50 30 18 16 21.
    // Four or sixteen warps a CTA are no faster at any of them.
    constexpr int kWarps = D == 256 ? 4 : 8;
    const uint64_t most = NT == 1 ? multiprocessors() * 4 / 3 : multiprocessors() / 2;
    uint32_t split = 1;
    while (split < 16 && units * split * 2 <= most && length > uint64_t(split) * kWarps * (split < 8 ? 32 : 128)) split *= 2;
    if (units / b.sequences * split > 0x7fffffffull) throw CudaError("cuda: the 4-bit cache's attention takes fewer rows than these");
    launch_split<T, D, NT, kWarps>(c, b, a, units, split, dependent, s);
}

// 8 rows to a CTA, two of which an SM holds, or 16, which share the keys and values they widen: where there are CTAs enough all the same. us
// with 8 / 16: 9 tokens of 32 heads after 2064 positions 12 / 12, 24 tokens after 8000 46 / 63, 64 after 2000 26 / 21, 128 after 4000 83 /
// 67; 600 tokens in heads of 256 41 / 53. With 32 a CTA has an SM to itself and is slower than either nearly everywhere.
template <class T, int D>
void attend_sized(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, bool dependent, cudaStream_t s) {
    const uint64_t rows = uint64_t(b.max_tokens) * (a.heads / c.kv_heads);
    if constexpr (D <= 128) {
        if (rows >= 64 && (rows + 7) / 8 * c.kv_heads * b.sequences >= 256) return attend_split<T, D, 2>(c, b, a, dependent, s);
    }
    attend_split<T, D, 1>(c, b, a, dependent, s);
}

template <class T>
void attend(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, bool dependent, cudaStream_t s) {
    if (c.dim == 64) attend_sized<T, 64>(c, b, a, dependent, s);
    else if (c.dim == 128) attend_sized<T, 128>(c, b, a, dependent, s);
    else attend_sized<T, 256>(c, b, a, dependent, s);
}

}  // namespace

void launch_cache4_attention(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, int type, bool dependent, cudaStream_t s) {
    if (cache4_prompt_takes(c, b, a, type)) launch_cache4_prompt(c, b, a, type, dependent, s);
    else if (type == T_F32) attend<float>(c, b, a, dependent, s);
    else if (type == T_F16) attend<__half>(c, b, a, dependent, s);
    else attend<__nv_bfloat16>(c, b, a, dependent, s);
}

}  // namespace bk
