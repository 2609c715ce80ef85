// Attention over the paged cache in 4 bits for many rows - prompts and their chunks - on the tensor cores of tensor memory.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache4_math.cuh"
#include "packed.cuh"
#include "pdl.cuh"
#include "tc.cuh"

namespace bk {
namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ void cluster_meet() {
    __syncwarp();  // .aligned: by whole warps
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"(uint32_t(accumulate)) : "memory");
}
// A in tensor memory: lane = row, a column holds two values of K
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t instr, bool accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(instr), "r"(uint32_t(accumulate)) : "memory");
}
// 32 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
          "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                   "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at)
                 : "memory");
}

// A whole row, zeros where there is none: every load is under way before the first value is looked at.
template <class T, int D> struct Row {
    static constexpr int kPer = 16 / sizeof(T);
    uint4 raw[D / kPer];
    __device__ __forceinline__ void load(const T* p, bool there, int wide) {
        if (!there) {
#pragma unroll
            for (int i = 0; i < D / kPer; ++i) raw[i] = make_uint4(0, 0, 0, 0);
        } else if (wide) {
#pragma unroll
            for (int i = 0; i < D / kPer; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < D / kPer; ++i) {
                alignas(16) T y[kPer];
#pragma unroll
                for (int u = 0; u < kPer; ++u) y[u] = p[i * kPer + u];
                raw[i] = *reinterpret_cast<const uint4*>(y);
            }
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return to_float(reinterpret_cast<const T*>(raw)[i]); }
};

template <int D, bool TWO> struct Prompt {
    static constexpr int kN = TWO ? 64 : 128;  // positions of a tile
    static constexpr int kParts = TWO ? 2 : 1;  // f16 parts of a query and of a weight
    static constexpr int kPanel = 128 * 128;    // 128 rows of 128 bytes
    static constexpr int kQ = D / 64 * kPanel;  // of one part of a query tile
    static constexpr int kK = D / 64 * kN * 128, kV = kN / 64 * D * 128;
    static constexpr int kKAt = 2 * kParts * kQ, kVAt = kKAt + 2 * kK, kBarriersAt = kVAt + 2 * kV;
    static constexpr int kBytes = kBarriersAt + 256 + 1024;  // the tiles start on a 1024-byte boundary
    // columns of tensor memory: the scores (which a tile of rows leaves at once for its registers, so one place does for both), each tile's
    // weights and result
    static constexpr int kW = 128, kO = 256;
    // A product cuts its sum off at 24 bits, a third of a bit lost each time, all one way: f32 results are added up over this many tiles only, and
    // those sums with rounding, in the columns of the second tile of rows, which f32 does without.
    static constexpr int kFlush = 4, kTotal = kO + D;
};
constexpr int kPromptThreads = 16 * 32, kOrdered = 128;
constexpr uint32_t kMostSplits = 4;
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

struct Bars {
    uint64_t q_full[2], k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], s_free, p_full[2], o_done[2], drained;
    uint32_t tmem;
    uint32_t large;  // a scale was past_f16; of this CTA's, and behind the cluster's last barrier of its other CTAs' as well
};

// One row by a warp, in 32 bits from the cache as it lies, a lane to a position for the scores and to D / 32 values for the result.
template <class T, int D>
__device__ __forceinline__ void attend_row(const Cache4& c, const Cache4Batch& b, uint32_t sequence, uint32_t kv, const T* q, T* out, int first, int last, float scale) {
    constexpr int kBlocks = D / 32, kBytes = D / 64;  // of a lane: kBytes of the row
    const uint32_t lane = threadIdx.x & 31, block = lane * kBytes / 16, byte = lane * kBytes % 16;
    float m = -INFINITY, l = 0.0f, o[2 * kBytes] = {};
    for (long long base = first & ~31; base <= last; base += 32) {
        const int p = int(base + lane);
        const bool sees = base + lane <= last && p >= first;
        const int32_t page = sees ? page_of(c, b, sequence, uint32_t(p) >> c.page_shift) : -1;
        const size_t at = ((size_t(max(page, 0)) * c.kv_heads + kv) * c.page_size + (uint32_t(p) & (c.page_size - 1))) * kBlocks;
        float score = 0.0f;
        if (page >= 0) {
#pragma unroll 1
            for (int x = 0; x < 4 * kBlocks; ++x) {  // words
                const uint32_t word = reinterpret_cast<const uint32_t*>(c.k_quants + at * 16)[x];
                const T* y = q + x / 4 * 32 + x % 4 * 4;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum = fmaf(float(int(word >> (8 * i) & 15) - 8), to_float(y[i]), sum);
                    sum = fmaf(float(int(word >> (8 * i + 4) & 15) - 8), to_float(y[i + 16]), sum);
                }
                score = fmaf(sum, __half2float(c.k_scales[at + x / 4]), score);
            }
        }
        score = sees ? score * scale : -INFINITY;
        const float next = fmaxf(m, warp_max(score)), less = next == -INFINITY ? 0.0f : next, keep = m == -INFINITY ? 0.0f : exp2_fast(m - less), w = exp2_fast(score - less);
        m = next;
        l = fmaf(l, keep, warp_sum(w));
#pragma unroll
        for (int i = 0; i < 2 * kBytes; ++i) o[i] *= keep;
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
            const float of = __shfl_sync(0xffffffffu, w, i);
            const int32_t there = __shfl_sync(0xffffffffu, page, i);
            const size_t place = __shfl_sync(0xffffffffu, (unsigned long long)at, i);
            if (there >= 0) {
                const float d = of * __half2float(c.v_scales[place + block]);
                const uint8_t* n = c.v_quants + (place + block) * 16 + byte;
#pragma unroll
                for (int x = 0; x < kBytes; ++x) {
                    o[2 * x] = fmaf(float(int(n[x] & 15) - 8), d, o[2 * x]);
                    o[2 * x + 1] = fmaf(float(int(n[x] >> 4) - 8), d, o[2 * x + 1]);
                }
            }
        }
    }
    const float inverse = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
    for (int x = 0; x < kBytes; ++x) {
        put(out + block * 32 + byte + x, o[2 * x] * inverse);
        put(out + block * 32 + byte + x + 16, o[2 * x + 1] * inverse);
    }
}

// softmax(q k) v for 256 rows (or 128) - tokens times the query heads of one key/value head - of one sequence, in two tiles of 128 rows that
// take turns on the tensor cores. Four warpgroups: one for each tile's softmax, a thread to a row (its maximum and sum need no other); one
// widens the 4-bit keys and values of 128 positions (64 where queries are two f16 parts) into the operand tiles of the products,
// once for both tiles of rows; a warp of the last issues the products,
//     S = Q K^T (both operands in shared memory),     O += P V (P in tensor memory).
// S is in columns 0 .. 127 for both tiles of rows: a softmax takes it into registers at once and gives it back by s_free, before it writes
// a weight. The weights of tile i are in columns kW + 64 i, written between o_done (of the last) and p_full.
// The head's values lie in Q and K in the order in which a 4-bit word yields them. V is widened with neighbouring positions side by side, as
// the product wants them: two words of two positions give pairs of one dim.
// Where rows are few for the SMs, up to four CTAs of a cluster share a row's positions and join at the end.
// The converters look at every scale. Where one was past_f16, which no model's keys and values are meant to be, the operand tiles hold infinities:
// the CTA's rows are then computed again without them (attend_row), as exactly and far slower (one such value among 512 tokens of 32 heads:
// 0.04 ms became 4.3). Folding such tiles would have to be agreed upon before each tile's keys are widened, which cost every call:
// 4096 tokens 178 us became 195 to 220, where looking costs 3.
// Every wait is bounded; one that runs out leaves NaN in the rows of its tile and sets the caller's error word, where there is one.
template <class T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1) cache4_prompt_kernel(const Cache4 c, const Cache4Batch b, const Cache4Attend a, uint32_t rows_per_cta) {
    constexpr bool kTwo = sizeof(T) == 4;
    using G = Prompt<D, kTwo>;
    constexpr int kN = G::kN;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (saddr(smem_raw) & 1023)) & 1023);
    const uint32_t smem_at = saddr(smem);
    Bars* bar = reinterpret_cast<Bars*>(smem + G::kBarriersAt);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    wait_for_previous();
    uint32_t sequence = blockIdx.y;
    if (gridDim.y > 1 && gridDim.y <= uint32_t(kOrdered)) {  // the longest sequences begin first (see cache4_attn.cu)
        int* length = reinterpret_cast<int*>(smem);
        uint32_t* chosen = reinterpret_cast<uint32_t*>(length + kOrdered);
        if (tid < gridDim.y) {
            uint32_t from, tokens;
            sequence_rows(b, tid, from, tokens);
            length[tid] = int(min((long long)b.context[tid] + tokens, 0x7fffffffll));
        }
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
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t S = cluster.num_blocks(), rank = cluster.block_rank();  // CTAs that share the positions of these rows
    const uint32_t group = a.heads / c.kv_heads, kv = blockIdx.x / S % c.kv_heads;
    const uint32_t tile = gridDim.x / S / c.kv_heads - 1 - blockIdx.x / S / c.kv_heads;  // the last rows, which see most, begin first
    const long long context = b.context[sequence], held = (long long)b.columns * c.page_size;
    uint32_t first_row, count;
    sequence_rows(b, sequence, first_row, count);
    const uint32_t total = count * group, row0 = tile * rows_per_cta;
    const uint32_t rows = row0 < total ? min(total - row0, rows_per_cta) : 0;
    if (rows == 0) return;
    if (warp == 12) {
        if (lane == 0) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&bar->q_full[i], 4);
                mbar_init(&bar->k_full[i], 4);
                mbar_init(&bar->k_free[i], 1);
                mbar_init(&bar->v_full[i], 4);
                mbar_init(&bar->v_free[i], 1);
                mbar_init(&bar->s_full[i], 1);
                mbar_init(&bar->p_full[i], 4);
                mbar_init(&bar->o_done[i], 1);
            }
            mbar_init(&bar->s_free, 4);
            mbar_init(&bar->drained, 1);
            bar->large = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(saddr(&bar->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    __syncwarp();
    tc_fence_after();
    // All 512 columns are this CTA's, so they begin at 0: as a constant the address costs the products no move between registers.
    constexpr uint32_t tmem = 0;

    auto last_of = [&](uint32_t token) { return int(max(min(context + token, held - 1), -1ll)); };
    auto first_of = [&](uint32_t token) { return a.window != 0 ? int(min(max(context + token - (long long)a.window + 1, 0ll), held)) : 0; };
    const int lo = first_of(row0 / group), hi = last_of((row0 + rows - 1) / group);
    const int all_tiles = hi >= lo ? (hi - (lo & ~(kN - 1))) / kN + 1 : 0, halves_used = rows > 128 ? 2 : 1;
    const int each = (all_tiles + int(S) - 1) / int(S), before = min(int(rank) * each, all_tiles), tiles = min(each, all_tiles - before);
    const int begin = (lo & ~(kN - 1)) + before * kN;
    const long long limit = a.bound.cycles;
    bool dead = bar->tmem != 0;

    if (warp < 8) {
        // ---- softmax: a thread to a row ----
        more_registers<184>();
        const uint32_t half = warp >> 2, r = tid & 127, row = row0 + half * 128 + r;
        const bool real = half * 128 + r < rows;
        const uint32_t token = real ? row / group : 0, head = row - token * group;
        T* out = static_cast<T*>(a.out) + size_t(first_row + token) * a.out_stride + size_t(kv * group + head) * D;
        const bool works = int(half) < halves_used && tiles != 0;
        const uint32_t lanes = tmem + ((warp & 3) << 21);  // this warp's 32 lanes
        const uint32_t o_at = lanes + G::kO + half * D;
        float m = -INFINITY, l = 0.0f;
        if (works) {
            // the row's queries: a power of two brings the largest to 2^10 (see cache4_attn.cu)
            Row<T, D> q;
            q.load(static_cast<const T*>(a.q) + size_t(first_row + token) * a.q_stride + size_t(kv * group + head) * D, real, a.wide);
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < D; ++i) most = fmaxf(most, fabsf(q[i]));
            const int exponent = int(__float_as_uint(most) >> 23) - 127, up = most < INFINITY ? min(10 - exponent, 100) : 0;
            const float by = __uint_as_float(uint32_t(127 + up) << 23) * (a.scale < 0.0f ? -1.0f : 1.0f);
            const float scale = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float(uint32_t(127 - up) << 23);
            unsigned char* q_tile = smem + half * G::kParts * G::kQ;
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {  // 16 bytes: the order of word u (see widen)
                    uint32_t high[4], low[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int dim = u * 4 + (i >> 1) + (i & 1) * 16;
                        const float y = q[k * 32 + dim] * by, z = q[k * 32 + dim + 2] * by;
                        const __half2 h = __floats2half2_rn(y, z);
                        high[i] = bits(h);
                        if (kTwo) low[i] = bits(__floats2half2_rn(y - __low2float(h), z - __high2float(h)));
                    }
                    unsigned char* dst = q_tile + (k >> 1) * G::kPanel + r * 128 + ((((k & 1) * 4 + u) ^ (r & 7)) * 16);
                    *reinterpret_cast<uint4*>(dst) = make_uint4(high[0], high[1], high[2], high[3]);
                    if (kTwo) *reinterpret_cast<uint4*>(dst + G::kQ) = make_uint4(low[0], low[1], low[2], low[3]);
                }
            }
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->q_full[half]);
            __syncwarp();

            const int last = real ? last_of(token) : -1, first = real ? first_of(token) : 0;
            const uint32_t last_row = min(row0 + half * 128 + 127, row0 + rows - 1);
            const int whole_to = last_of((row0 + half * 128) / group), whole_from = first_of(last_row / group);
            const uint32_t s_at = lanes, w_at = lanes + G::kW + half * 64;
            auto scale_columns = [&](uint32_t at, float by) {
#pragma unroll
                for (int ch = 0; ch < D / 16; ++ch) {
                    uint32_t y[16];
                    tmem_ld16(at + ch * 16, y);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * by);
                    tmem_st16(at + ch * 16, y);
                }
            };
            auto add_up = [&](bool more) {  // the total is (or has added) the result of the last tiles
#pragma unroll
                for (int ch = 0; ch < D / 16; ++ch) {
                    uint32_t y[16], z[16];
                    tmem_ld16(o_at + ch * 16, y);
                    if (more) tmem_ld16(lanes + G::kTotal + ch * 16, z);
                    tmem_wait_ld();
                    if (more) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) + __uint_as_float(z[i]));
                    }
                    tmem_st16(lanes + G::kTotal + ch * 16, y);
                }
                tmem_wait_st();
            };
            for (int j = 0; j < tiles; ++j) {
                mbar_wait_warp(&bar->s_full[half], j & 1, dead, limit);
                if (dead) break;
                tc_fence_after();
                // the last tile's scores: nobody reads these keys any more
                if (int(half) == halves_used - 1 && (tid & 127) == 0) mbar_arrive(&bar->k_free[j & 1]);
                __syncwarp();  // loads and stores of tensor memory are a whole warp's
                const int base = begin + j * kN;
                const bool whole = base + kN - 1 <= whole_to && base >= whole_from;
                // tensor memory gives a warp little more than 32 bytes a cycle: the scores are read once and stay in registers
                uint32_t x[kN / 32][32];
#pragma unroll
                for (int ch = 0; ch < kN / 32; ++ch) tmem_ld32(s_at + ch * 32, x[ch]);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->s_free);
                __syncwarp();
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < kN; ++i) {
                        if (base + i > last || base + i < first) x[i / 32][i % 32] = 0xff800000u;  // -inf
                    }
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kN; i += 2) tops[i / 2 % 4] = fmaxf(tops[i / 2 % 4], fmaxf(__uint_as_float(x[i / 32][i % 32]), __uint_as_float(x[i / 32][i % 32 + 1])));
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * scale;
                if (j > 0) {  // the last weights have been read, the result is at rest
                    mbar_wait_warp(&bar->o_done[half], (j - 1) & 1, dead, limit);
                    if (dead) break;
                    tc_fence_after();
                    if (int(half) == halves_used - 1 && (tid & 127) == 0) mbar_arrive(&bar->v_free[(j - 1) & 1]);
                    __syncwarp();
                    if (kTwo && j % G::kFlush == 0) add_up(j > G::kFlush);
                }
                // the level (see Level) moves only where a weight would no longer fit
                const bool above = top > m + Level<kTwo>::kMost;
                if (__any_sync(0xffffffffu, above)) {
                    const float next = above ? top - Level<kTwo>::kBelow : m, keep = m == next ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - next);
                    m = next;
                    l *= keep;
                    if (kTwo && j >= G::kFlush) scale_columns(lanes + G::kTotal, keep);
                    if (kTwo ? j % G::kFlush != 0 : j != 0) scale_columns(o_at, keep);
                }
                const float less = m == -INFINITY ? 0.0f : -m;
                // A fused multiply and add takes the level, rounded, from the score that is not: past 2^20 that moves the weights, in the end past f16.
                float by = scale;
                if (__any_sync(0xffffffffu, fabsf(less) > 0x1p20f)) {
#pragma unroll
                    for (int i = 0; i < kN; ++i) x[i / 32][i % 32] = __float_as_uint(__uint_as_float(x[i / 32][i % 32]) * scale);
                    by = 1.0f;
                }
                const f32x2 scale2 = pack2(by, by), less2 = pack2(less, less);
                f32x2 sum[4] = {pack2(l, 0.0f), pack2(0.0f, 0.0f), pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
#pragma unroll
                for (int ch = 0; ch < kN / 32; ++ch) {
                    uint32_t w[16], w_low[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float y, z;
                        unpack2(fma2(pack2(x[ch][2 * i], x[ch][2 * i + 1]), scale2, less2), y, z);
                        y = exp2_fast(y);
                        z = exp2_fast(z);
                        sum[i & 3] = add2(sum[i & 3], pack2(y, z));
                        const __half2 h = __floats2half2_rn(y, z);
                        w[i] = bits(h);
                        if (kTwo) w_low[i] = bits(__floats2half2_rn(y - __low2float(h), z - __high2float(h)));
                    }
                    tmem_st16(w_at + ch * 16, w);
                    if (kTwo) tmem_st16(w_at + kN / 2 + ch * 16, w_low);
                }
                float even, odd;
                unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), even, odd);
                l = even + odd;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->p_full[half]);
            }
            mbar_wait_warp(&bar->o_done[half], (tiles - 1) & 1, dead, limit);
            tc_fence_after();
            mbar_wait_warp(&bar->v_full[(tiles - 1) & 1], (tiles - 1) >> 1 & 1, dead, limit);  // long complete: what the converters wrote before it is seen
        }
        // 32 values of the row's result, before they are divided by the sum of its weights
        auto result_of = [&](int ch, uint32_t (&x)[32]) {
            tmem_ld32(o_at + ch * 32, x);
            tmem_wait_ld();
            if (kTwo && tiles > G::kFlush) {
                uint32_t y[32];
                tmem_ld32(lanes + G::kTotal + ch * 32, y);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) + __uint_as_float(y[i]));
            }
        };
        const volatile uint32_t* large = &bar->large;
        auto attend_rows = [&](uint32_t begin_at, uint32_t step) {
            for (uint32_t x = begin_at; x < rows; x += step) {
                const uint32_t of = (row0 + x) / group, h = kv * group + row0 + x - of * group;
                attend_row<T, D>(c, b, sequence, kv, static_cast<const T*>(a.q) + size_t(first_row + of) * a.q_stride + size_t(h) * D,
                                 static_cast<T*>(a.out) + size_t(first_row + of) * a.out_stride + size_t(h) * D, first_of(of), last_of(of), a.scale * 1.4426950408889634f);
            }
        };
        if (S == 1) {
            if (works && !dead && *large != 0) {
                attend_rows(warp, 4 * halves_used);
            } else if (works) {
                const float inverse = dead ? __int_as_float(0x7fc00000) : l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
                for (int ch = 0; ch < D / 32; ++ch) {
                    uint32_t x[32];
                    result_of(ch, x);
                    if (real) {
                        if (a.wide) {
                            constexpr int kPer = 16 / sizeof(T);
#pragma unroll
                            for (int i = 0; i < 32; i += kPer) {
                                alignas(16) T y[kPer];
#pragma unroll
                                for (int u = 0; u < kPer; ++u) put(y + u, __uint_as_float(x[i + u]) * inverse);
                                *reinterpret_cast<uint4*>(out + ch * 32 + i) = *reinterpret_cast<const uint4*>(y);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) put(out + ch * 32 + i, __uint_as_float(x[i]) * inverse);
                        }
                    }
                    __syncwarp();
                }
            } else if (real && tiles == 0) {  // rows that see nothing
                for (int i = 0; i < D; ++i) put(out + i, 0.0f);
            }
            __syncwarp();
        } else {
            // Every CTA sums D / S values of each row: the others write theirs, with their maximum and sum, where its operand tiles were.
            const uint32_t share = D / S, at = half * 128 + r;
            uint4* received = reinterpret_cast<uint4*>(smem);            // [S][share / 4][256]
            float2* sums = reinterpret_cast<float2*>(smem + 256 * D * 4);  // [S][256] of maximum and sum
            static_assert(256 * D * 4 + kMostSplits * 256 * 8 <= G::kBarriersAt);
            cluster_meet();  // nobody's products read operand tiles any more
            if (int(half) < halves_used) {
                for (uint32_t k = 0; k < S; ++k) *cluster.map_shared_rank(sums + rank * 256 + at, k) = dead ? make_float2(0.0f, __int_as_float(0x7fc00000)) : make_float2(m, l);
#pragma unroll
                for (int ch = 0; ch < D / 32; ++ch) {
                    uint32_t x[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = 0;
                    if (works) result_of(ch, x);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const uint32_t dim = ch * 32 + i;
                        *cluster.map_shared_rank(received + (rank * (share / 4) + dim % share / 4) * 256 + at, dim / share) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                    }
                }
            }
            if (tid == 0 && *large != 0) {
                for (uint32_t k = 0; k < S; ++k) *cluster.map_shared_rank(&bar->large, k) = 1;
            }
            cluster_meet();
            if (*large != 0) {
                attend_rows(warp * S + rank, 8 * S);
            } else if (real) {
                float most = -INFINITY, sum = 0.0f, by[kMostSplits];
                for (uint32_t k = 0; k < S; ++k) most = fmaxf(most, sums[k * 256 + at].x);
#pragma unroll
                for (uint32_t k = 0; k < kMostSplits; ++k) {
                    by[k] = 0.0f;
                    if (k < S) {
                        const float2 y = sums[k * 256 + at];
                        by[k] = y.x == -INFINITY ? 0.0f : exp2_fast(y.x - most);
                        sum = fmaf(y.y, by[k], sum);
                    }
                }
                const float inverse = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
                for (uint32_t i = 0; i < share; i += 4) {
                    float x[4] = {};
#pragma unroll
                    for (uint32_t k = 0; k < kMostSplits; ++k) {
                        if (k < S) {
                            const uint4 y = received[(k * (share / 4) + i / 4) * 256 + at];
                            x[0] = fmaf(__uint_as_float(y.x), by[k], x[0]);
                            x[1] = fmaf(__uint_as_float(y.y), by[k], x[1]);
                            x[2] = fmaf(__uint_as_float(y.z), by[k], x[2]);
                            x[3] = fmaf(__uint_as_float(y.w), by[k], x[3]);
                        }
                    }
                    alignas(16) T z[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) put(z + u, x[u] * inverse);
                    T* dst = out + rank * share + i;
                    if (a.wide) {
                        using Four = std::conditional_t<kTwo, uint4, uint2>;
                        *reinterpret_cast<Four*>(dst) = *reinterpret_cast<const Four*>(z);
                    } else {
#pragma unroll
                        for (int u = 0; u < 4; ++u) dst[u] = z[u];
                    }
                }
            }
        }
    } else if (warp < 12) {
        // ---- keys and values: 4 bits to f16 operand tiles ----
        fewer_registers<96>();
        const uint32_t p_tid = tid - 256;
        // keys: lane = position, so that eight lanes write eight rows of the swizzled tile; a thread has kKeys blocks
        constexpr int kBlocks = D / 32, kKeys = kN * kBlocks / 128;
        const uint32_t block = (p_tid >> 5) % kBlocks, key_part = (p_tid >> 5) / kBlocks;
        auto key_position = [&](int i) { return int((p_tid & 31) + 32 * (key_part + (4 / kBlocks) * i)); };
        // values: a thread has 4 kWords bytes of 8 positions; eight lanes write eight chunks of one row
        constexpr int kWords = D * kN >= 128 * 128 ? 2 : 1, kGroups = kN / 8, kPieces = D / 8 / kWords;
        const uint32_t rest = p_tid >> 3, group8 = (p_tid & 7) + 8 * (rest % (kGroups / 8)), piece = rest / (kGroups / 8);
        const bool has_values = piece < uint32_t(kPieces);
        const uint32_t value_block = piece * kWords / 4;

        auto page_at = [&](int p) { return p >= lo - int(c.page_size) && p <= hi && p >= 0 ? page_of(c, b, sequence, uint32_t(p) >> c.page_shift) : -1; };
        uint4 key[kKeys];
        __half key_scale[kKeys];
        uint32_t value[8][kWords];
        __half value_scale[8];
        int key_page[kKeys], value_page;
        auto ask_pages = [&](int j) {
            const int base = begin + j * kN;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) key_page[i] = j < tiles ? page_at(base + key_position(i)) : -1;
            value_page = j < tiles && has_values ? page_at(base + int(group8) * 8) : -1;
        };
        auto load_keys = [&](int j) {
            const int base = begin + j * kN;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
                const int p = base + key_position(i);
                const bool there = key_page[i] >= 0 && p >= lo && p <= hi;
                const size_t at = ((size_t(there ? key_page[i] : 0) * c.kv_heads + kv) * c.page_size + (uint32_t(p) & (c.page_size - 1))) * kBlocks + block;
                key[i] = *reinterpret_cast<const uint4*>(c.k_quants + at * 16);
                key_scale[i] = there ? c.k_scales[at] : __half(0.0f);
            }
        };
        auto load_values = [&](int j) {
            if (!has_values) return;
            const int p = begin + j * kN + int(group8) * 8;
            const size_t at = ((size_t(max(value_page, 0)) * c.kv_heads + kv) * c.page_size + (uint32_t(p) & (c.page_size - 1))) * kBlocks;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned char* src = c.v_quants + (at + i * kBlocks) * 16 + piece * kWords * 4;
                if (kWords == 2) {
                    const uint2 x = *reinterpret_cast<const uint2*>(src);
                    value[i][0] = x.x;
                    value[i][kWords - 1] = x.y;
                } else {
                    value[i][0] = *reinterpret_cast<const uint32_t*>(src);
                }
                const bool there = value_page >= 0 && p + i >= lo && p + i <= hi;
                value_scale[i] = there ? c.v_scales[at + i * kBlocks + value_block] : __half(0.0f);
            }
        };
        __half2 most = __half2half2(__half(0.0f));  // of the scales' magnitudes
        ask_pages(0);
        load_keys(0);
        load_values(0);
        ask_pages(1);
        for (int j = 0; j < tiles; ++j) {
            const uint32_t slot = j & 1;
            if (uint32_t(j) == a.bound.withheld) dead = true;
            if (j >= 2) mbar_wait_warp(&bar->k_free[slot], (j >> 1) - 1 & 1, dead, limit);
            if (dead) break;
            unsigned char* tile_k = smem + G::kKAt + slot * G::kK;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
                const uint32_t p = uint32_t(key_position(i)), w[4] = {key[i].x, key[i].y, key[i].z, key[i].w};
                const __half2 d = __half2half2(key_scale[i]);
                most = larger(most, d);
                unsigned char* row = tile_k + (block >> 1) * (kN * 128) + p * 128;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint32_t v[4];
                    widen(w[u], d, v);
                    *reinterpret_cast<uint4*>(row + ((((block & 1) * 4 + u) ^ (p & 7)) * 16)) = make_uint4(v[0], v[1], v[2], v[3]);
                }
            }
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->k_full[slot]);
            if (j + 1 < tiles) load_keys(j + 1);

            if (j >= 2) mbar_wait_warp(&bar->v_free[slot], (j >> 1) - 1 & 1, dead, limit);
            if (dead) break;
            unsigned char* tile_v = smem + G::kVAt + slot * G::kV;
            if (has_values) {
                __half2 d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    d[i] = __halves2half2(value_scale[2 * i], value_scale[2 * i + 1]);
                    most = larger(most, d[i]);
                }
                unsigned char* panel = tile_v + (group8 >> 3) * (D * 128);
#pragma unroll
                for (int x = 0; x < kWords; ++x) {
#pragma unroll
                    for (int z = 0; z < 2; ++z) {  // bytes 0, 1 and 2, 3 of the word
                        uint32_t v[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) widen(__byte_perm(value[2 * i][x], value[2 * i + 1][x], z ? 0x7632 : 0x5410), d[i], v[i]);
                        const uint32_t byte = (piece * kWords + x) * 4 + z * 2;  // of the row
#pragma unroll
                        for (int u = 0; u < 4; ++u) {  // (low, high) of the first byte, then of the second
                            const uint32_t of = byte + (u >> 1), dim = (of >> 4) * 32 + (of & 15) + (u & 1) * 16;
                            *reinterpret_cast<uint4*>(panel + dim * 128 + (((group8 & 7) ^ (dim & 7)) * 16)) = make_uint4(v[0][u], v[1][u], v[2][u], v[3][u]);
                        }
                    }
                }
            }
            if (past_f16(__hmax(__low2half(most), __high2half(most)))) bar->large = 1;
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->v_full[slot]);
            if (j + 1 < tiles) load_values(j + 1);
            ask_pages(j + 2);
        }
    } else {
        fewer_registers<48>();
        if (warp == 12 && tiles != 0) {
            // ---- products ----
            constexpr uint32_t kScores = instr_f16(kN), kResult = instr_f16(D);
            const bool leader = elect_one();
            // descriptors count in 16 bytes; what is added to them is a constant, or the slot's
            const uint64_t q_desc = smem_desc_swizzled(smem_at), k_desc = smem_desc_swizzled(smem_at + G::kKAt), v_desc = smem_desc_swizzled(smem_at + G::kVAt);
            auto wait = [&](uint64_t* x, uint32_t parity) { mbar_wait_warp(x, parity, dead, limit); };
            auto scores = [&](auto half, uint64_t k) {  // S = Q_i K^T
                constexpr int i = decltype(half)::value;
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int part = G::kParts - 1; part >= 0; --part) {  // the small parts first: a sum loses up to half a bit with every product
#pragma unroll
                        for (int s = 0; s < D / 16; ++s) {
                            mma_ss(tmem, q_desc + ((i * G::kParts + part) * G::kQ + (s >> 2) * G::kPanel + (s & 3) * 32) / 16, k + ((s >> 2) * (kN * 128) + (s & 3) * 32) / 16, kScores,
                                   part != G::kParts - 1 || s != 0);
                        }
                    }
                    mma_commit(&bar->s_full[i]);
                }
                __syncwarp();
            };
            auto result = [&](auto half, uint64_t v, bool first) {  // O_i += P_i V
                constexpr int i = decltype(half)::value;
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int part = 0; part < G::kParts; ++part) {
#pragma unroll
                        for (int s = 0; s < kN / 16; ++s) {
                            mma_ts(tmem + G::kO + i * D, tmem + G::kW + i * 64 + part * (kN / 2) + s * 8, v + ((s >> 2) * (D * 128) + (s & 3) * 32) / 16, kResult, part != 0 || s != 0 || !first);
                        }
                    }
                    mma_commit(&bar->o_done[i]);
                }
                __syncwarp();
            };
            // scores of tile j, then the product of the weights of tile j - 1: a tile's softmax has the products of the other for its time
            uint32_t turns = 0;
            auto turn = [&](auto half, int j) {
                constexpr int i = decltype(half)::value;
                if (j < tiles) {
                    if (i == 0) wait(&bar->k_full[j & 1], j >> 1 & 1);
                    if (j == 0) wait(&bar->q_full[i], 0);
                    if (turns != 0) wait(&bar->s_free, (turns - 1) & 1);
                    if (dead) return;
                    scores(half, k_desc + (j & 1) * (G::kK / 16));
                    ++turns;
                }
                if (j > 0) {
                    if (i == 0) wait(&bar->v_full[(j - 1) & 1], (j - 1) >> 1 & 1);
                    wait(&bar->p_full[i], (j - 1) & 1);
                    if (dead) return;
                    result(half, v_desc + ((j - 1) & 1) * (G::kV / 16), kTwo ? (j - 1) % G::kFlush == 0 : j == 1);
                }
            };
            for (int j = 0; j <= tiles && !dead; ++j) {
                turn(std::integral_constant<int, 0>{}, j);
                if (halves_used == 2 && !dead) turn(std::integral_constant<int, 1>{}, j);
            }
            if (leader) mma_commit(&bar->drained);
            __syncwarp();
            mbar_drain(&bar->drained, 0);
        }
    }
    if (warp >= 8 && S > 1) {
        __syncwarp();
        cluster_meet();
        cluster_meet();
    }
    if (dead && lane == 0 && a.bound.error != nullptr) atomicOr(a.bound.error, 1u);
    release_next();
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// How a call's rows and positions are shared out.
struct Shares {
    uint32_t rows_per_cta, split;
    uint64_t ctas, length;  // of a sequence, where one CTA has all its positions; positions that a tile of rows sees at most
};
Shares shares_of(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, bool two) {
    const uint64_t rows = uint64_t(b.max_tokens) * (a.heads / c.kv_heads), sms = multiprocessors();
    Shares x;
    // Two tiles of rows share their keys and values where there are CTAs for all SMs all the same. us with 128 / 256 rows a CTA, bf16 heads
    // of 128: 512 tokens of 32 heads (128 or 64 CTAs) 17 / 20, 3000 positions further on 68 / 79; 16 sequences of 64 tokens after 1000 (256
    // or 128) 56 / 37.
    x.rows_per_cta = !two && (rows + 127) / 128 * c.kv_heads * b.sequences > sms ? 256 : 128;
    x.ctas = (rows + x.rows_per_cta - 1) / x.rows_per_cta * c.kv_heads;
    x.length = a.window != 0 ? std::min<uint64_t>(b.max_length, uint64_t(a.window) + x.rows_per_cta) : b.max_length;
    // Positions are spread while SMs are free for it and a CTA keeps some tiles: joining costs 3 us. us with 1 / 2 / 4 CTAs, bf16 heads of 128:
    // 32 tiles of rows after 4000 positions 77 / 46 / 31, 64 of them 79 / 48 / 59 (256 CTAs are two rounds); at the start of a prompt, 512 positions
    // at most, 16.4 / 16.1 / 28.
    x.split = 1;
    while (x.split < kMostSplits && x.ctas * b.sequences * x.split * 2 <= sms && x.length > uint64_t(x.split) * (two ? 256 : 512)) x.split *= 2;
    return x;
}

template <class T, int D>
void prompt_typed(const Cache4& c, const Cache4Batch& b, const Cache4Attend& in, bool dependent, cudaStream_t s) {
    const auto kernel = cache4_prompt_kernel<T, D>;
    constexpr size_t smem = Prompt<D, sizeof(T) == 4>::kBytes;
    static_assert(smem <= 227 * 1024);
    static DeviceSetup setup;
    setup.once([&] { BK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem))); });
    Cache4Attend a = in;
    a.wide = (reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | (a.q_stride * sizeof(T)) | (a.out_stride * sizeof(T))) % 16 == 0;
    const Shares x = shares_of(c, b, a, sizeof(T) == 4);
    if (x.ctas * x.split > 0x7fffffffull) throw CudaError("cuda: the 4-bit cache's attention takes fewer rows than these");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(uint32_t(x.ctas * x.split), b.sequences);
    cfg.blockDim = dim3(kPromptThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = x.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    BK_CUDA(cudaLaunchKernelEx(&cfg, kernel, c, b, a, x.rows_per_cta));
}

}  // namespace

// The kernel of few rows takes 16 at a time and spreads their positions over all SMs; a CTA of this one takes up to 256 rows and its positions one
// after another. So this one needs rows enough, and the line is where the times of the two meet, in ns with bf16 heads of 128 (the other types and
// heads move both alike): 30 and 1 for 17 positions of every 16 rows there, 10000 and 16 for a position of each round of CTAs here. us of few / many
// rows, heads of 128 in bf16, f32, heads of 64 in bf16, f32:
//     64 times 32 rows after 2000 positions    20.6 / 20.2   26.7 / 24.9   14.8 / 15.3   18.2 / 19.2
//     the same after 8000                      60 / 41       82 / 57       42 / 32       54 / 46
//     128 times 32 after 4000                  65 / 30       88 / 38       37 / 22       49 / 30
//     256 times 32 at the start of a prompt    23 / 12       25 / 17       12.3 / 10.0   12.8 / 11.8
//     32 sequences of 36 rows after 3000       139 / 114     179 / 165     90 / 84       111 / 126
// With 32 rows or fewer most of a tile is empty: 32 sequences of 18 rows after 3000 96 / 121, f32 124 / 155. Heads of 256 have no form here.
bool cache4_prompt_takes(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, int type) {
    const uint64_t rows = uint64_t(b.max_tokens) * (a.heads / c.kv_heads);
    if (c.dim > 128 || rows <= 32) return false;
    const Shares x = shares_of(c, b, a, type == T_F32);
    const uint64_t sms = multiprocessors(), rounds = (x.ctas * x.split * b.sequences + sms - 1) / sms;
    const double few = double((rows + 15) / 16 * c.kv_heads * b.sequences) * (30.0 + double(x.length) / 17.0), many = 10000.0 + double(rounds) * double(x.length) * 16.0 / x.split;
    return many < few;
}

void launch_cache4_prompt(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, int type, bool dependent, cudaStream_t s) {
    if (c.dim == 64) {
        if (type == T_F32) prompt_typed<float, 64>(c, b, a, dependent, s);
        else if (type == T_F16) prompt_typed<__half, 64>(c, b, a, dependent, s);
        else prompt_typed<__nv_bfloat16, 64>(c, b, a, dependent, s);
    } else {
        if (type == T_F32) prompt_typed<float, 128>(c, b, a, dependent, s);
        else if (type == T_F16) prompt_typed<__half, 128>(c, b, a, dependent, s);
        else prompt_typed<__nv_bfloat16, 128>(c, b, a, dependent, s);
    }
}

}  // namespace bk
