// The paged key/value cache in 4 bits: appending a batch's keys and values with the per-head norm and the rotation on the way, reading
// rows back as values, and the C entries of include/brisk_cuda.h. The attention over it is in cache4_attn.cu.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "../../include/brisk_cuda.h"
#include "cache4.h"
#include "packed.cuh"
#include "pdl.cuh"

namespace bk {
namespace {

template <class T> struct Convert;
template <> struct Convert<float> {
    static __device__ float from(float v) { return v; }
    static __device__ float to(float v) { return v; }
};
template <> struct Convert<__half> {
    static __device__ float from(__half v) { return __half2float(v); }
    static __device__ __half to(float v) { return __float2half_rn(v); }
};
template <> struct Convert<__nv_bfloat16> {
    static __device__ float from(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __nv_bfloat16 to(float v) { return __float2bfloat16_rn(v); }
};

template <class T, int N> struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Values {
    T v[N];
};

// A lane's E values of a row.
template <class T, int E>
__device__ __forceinline__ void load_values(const T* p, int wide, float (&x)[E]) {
    Values<T, E> u;
    if (wide) {
        u = *reinterpret_cast<const Values<T, E>*>(p);
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) u.v[j] = p[j];
    }
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = Convert<T>::from(u.v[j]);
}
template <class T, int E>
__device__ __forceinline__ void store_values(T* p, int wide, const float (&x)[E]) {
    Values<T, E> u;
#pragma unroll
    for (int j = 0; j < E; ++j) u.v[j] = Convert<T>::to(x[j]);
    if (wide) {
        *reinterpret_cast<Values<T, E>*>(p) = u;
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) p[j] = u.v[j];
    }
}

__device__ __forceinline__ float root(float v) { return __fsqrt_rn(v); }
__device__ __forceinline__ double root(double v) { return sqrt(v); }
__device__ __forceinline__ float fused(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return fma(a, b, c); }

// v to 8 significant bits, to nearest, ties to even.
__device__ __forceinline__ float eight_bits(float v) {
    uint32_t u = __float_as_uint(v);
    u += 0x7fffu + ((u >> 16) & 1u);
    return __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ float eight_bits(double v) {
    unsigned long long u = (unsigned long long)__double_as_longlong(v);
    u += (1ull << 44) - 1 + ((u >> 45) & 1ull);
    return float(__longlong_as_double((long long)(u & ~((1ull << 45) - 1))));
}

// The append kernel: a lane has 8 values of a head's row, so that a row takes D / 8 lanes and a warp 32 / (D / 8) rows at a time; four lanes
// have a block of 32.
constexpr int kLane = 8;

// Four numbers of four bits, each to a byte.
__device__ __forceinline__ uint32_t spread(uint32_t v) {
    v = (v | (v << 8)) & 0x00ff00ffu;
    return (v | (v << 4)) & 0x0f0f0f0fu;
}

// What a lane's values become: numbers of four bits, and their block's scale.
struct Numbers {
    uint32_t packed;
    __half scale;
};

// The borders between two numbers, (n - 8.5) d with d of 8 significant bits, are exact in 32 bits: the number is estimated by a
// reciprocal and then put right by comparing with the two borders beside it, so it is the one that the definition floor(x / d + 8.5)
// has, whatever the estimate rounds to. NaN counts as 0 and an infinity as the largest number that a block holds, so that no row of
// the cache holds either.
// Where values may be `within` of what they stand for, *doubt says that this leaves a number or the scale open; a lane whose `within` is 0
// has the values themselves.
template <class Real>
__device__ __forceinline__ Numbers to_numbers(Real (&x)[kLane], float within = 0.0f, bool* doubt = nullptr) {
    Real high = -Real(3e38f), low = Real(3e38f);
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
        x[j] = x[j] != x[j] ? Real(0) : x[j] > Real(3e38f) ? Real(3e38f) : x[j] < -Real(3e38f) ? -Real(3e38f) : x[j];
        high = x[j] > high ? x[j] : high;
        low = x[j] < low ? x[j] : low;
    }
#pragma unroll
    for (int o = 2; o > 0; o >>= 1) {
        const Real h = __shfl_xor_sync(0xffffffffu, high, o), l = __shfl_xor_sync(0xffffffffu, low, o);
        high = h > high ? h : high;
        low = l < low ? l : low;
    }
    const Real peak = high >= -low ? high : low;
    const float wanted = peak == Real(0) ? 0.0f : eight_bits(peak * Real(-0.125));
    if (doubt != nullptr) {
        float most = within;
#pragma unroll
        for (int o = 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float p = fabsf(float(peak));
        *doubt = most != 0.0f && (eight_bits((p - most) * 0.125f) != eight_bits((p + most) * 0.125f) || fabsf(float(high + low)) <= 2.0f * most || !(p < 1e30f));
    }
    Numbers out;
    out.scale = __float2half_rn(fminf(fmaxf(wanted, -65280.0f), 65280.0f));  // 255 x 256: the largest f16 of 8 bits
    const float signed_d = __half2float(out.scale), size = fabsf(signed_d), inverse = size != 0.0f ? __fdividef(1.0f, size) : 0.0f;
    out.packed = 0;
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
        float n = 8.0f;
        if (size != 0.0f) {
            const Real r = signed_d < 0.0f ? -x[j] : x[j];
            n = fminf(fmaxf(floorf(fmaf(float(r), inverse, 8.5f)), 0.0f), 15.0f);
            if (r < Real((n - 8.5f) * size)) n = n - 1.0f;
            else if (r >= Real((n - 7.5f) * size)) n = n + 1.0f;
            n = fminf(fmaxf(n, 0.0f), 15.0f);
            if (doubt != nullptr && within != 0.0f) *doubt = *doubt || fabsf(float(r) - (n - 8.5f) * size) <= within || fabsf((n - 7.5f) * size - float(r)) <= within;
        }
        out.packed |= uint32_t(n) << (4 * j);
    }
    return out;
}

// The same in a third of the instructions where nothing is in doubt, for values that may be `within` of what they stand for: false, and
// nothing to be relied on, where a block has a scale that this leaves open (or that is too large or too small to divide by) or a
// value that lies by a border.
__device__ __forceinline__ bool quick_numbers(const float (&x)[kLane], float within, Numbers& out) {
    float high = x[0], low = x[0], nan = 0.0f;
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
        high = fmaxf(high, x[j]);
        low = fminf(low, x[j]);
        nan += x[j];  // or an infinity
    }
#pragma unroll
    for (int o = 2; o > 0; o >>= 1) {
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        within = fmaxf(within, __shfl_xor_sync(0xffffffffu, within, o));
    }
    const float peak = high >= -low ? high : low, size_of_peak = fabsf(peak), d = eight_bits(peak * -0.125f);
    const bool sure = size_of_peak < 1e5f && size_of_peak > 1e-3f && eight_bits((size_of_peak - within) * 0.125f) == eight_bits((size_of_peak + within) * 0.125f) &&
                      (within == 0.0f || fabsf(high + low) > 2.0f * within) && nan == nan;
    out.scale = __float2half_rn(d);
    const float inverse = __fdividef(1.0f, d);
    float far = 0.0f;  // of a value from the middle between two borders, in steps
    uint32_t packed[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
        const float w = fminf(fmaxf(fmaf(x[j], inverse, 8.0f), 0.0f), 15.0f), v = w + 8388608.0f;  // to the next whole number, in the lowest bits
        far = fmaxf(far, fabsf(w - (v - 8388608.0f)));
        packed[j / 4] += __float_as_uint(v) << (4 * (j % 4));
    }
    out.packed = __byte_perm(packed[0], packed[1], 0x5410);
    // reciprocal, product and sum are under 2^-18 of a step off (values are up to 8 steps), a value `within` of its own
    return sure && far < 0.5f - 0x1p-18f - within * fabsf(inverse) * 1.001f;
}

// Two lanes on are the values 16 further on, the upper half of these bytes.
__device__ __forceinline__ void store_numbers(const Numbers& y, bool there, uint8_t* quants, __half* scales) {
    const uint32_t upper = __shfl_xor_sync(0xffffffffu, y.packed, 2), in_block = threadIdx.x & 3;
    if (there && in_block < 2) {
        uint2 bytes;
        bytes.x = spread(y.packed & 0xffffu) | (spread(upper & 0xffffu) << 4);
        bytes.y = spread(y.packed >> 16) | (spread(upper >> 16) << 4);
        *reinterpret_cast<uint2*>(quants + in_block * 8) = bytes;
        if (in_block == 0) *scales = y.scale;
    }
}

// x over its root mean square, times norm; a row is D / 8 lanes. False: the row's squares leave the range of 32 bits, or so nearly that they
// lose bits which the mean would show.
template <class Real, int D>
__device__ __forceinline__ bool normed(Real (&x)[kLane], const float* norm, float eps) {
    Real sum = Real(0);
#pragma unroll
    for (int j = 0; j < kLane; ++j) sum = fused(x[j], x[j], sum);
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const Real mean = sum / Real(D) + Real(eps), scale = Real(1) / root(mean);
#pragma unroll
    for (int j = 0; j < kLane; ++j) x[j] = x[j] * scale * Real(norm[j]);
    return mean > Real(1e-27f) && mean < Real(1e38f);
}

// Queries' rows whose squares leave 32 bits, normed in 64.
template <int D>
__device__ __noinline__ void normed_wide(float* x, const float* norm, float eps) {
    double wide[kLane];
#pragma unroll
    for (int j = 0; j < kLane; ++j) wide[j] = double(x[j]);
    normed<double, D>(wide, norm, eps);
#pragma unroll
    for (int j = 0; j < kLane; ++j) x[j] = float(wide[j]);
}

// What a lane needs to turn its values of any row of the token: y = x c + other s, in pairs of values.
struct Turns {
    f32x2 c[kLane / 2], s[kLane / 2];
    uint32_t first, rope_dim, half;  // first: the lane's place in a row, in values
    int adjacent;
    int from;   // the lane that has the others of this lane's pairs, where pairs fall on whole lanes
    bool whole, turns;  // whether they do (or are side by side), and then whether this lane's values turn
};

// cosine, sine: of the token's pairs, in 32 bits.
template <int D>
__device__ __forceinline__ Turns turns_of(uint32_t rope_dim, int adjacent, const float* cosine, const float* sine) {
    Turns t;
    const uint32_t lane = threadIdx.x & 31;
    t.first = (lane & (D / 8 - 1)) * kLane;
    t.rope_dim = rope_dim;
    t.half = rope_dim / 2;
    t.adjacent = adjacent;
    t.whole = rope_dim % kLane == 0 && (adjacent || t.half % kLane == 0);
    t.turns = t.first < rope_dim;
    t.from = int(lane) + (t.first < t.half ? int(t.half / kLane) : -int(t.half / kLane));
    if (t.whole && !adjacent) {
        const bool is_first = t.first < t.half;
        const uint32_t at = t.turns ? is_first ? t.first : t.first - t.half : 0;
#pragma unroll
        for (int j = 0; j < kLane; j += 4) {
            const float4 c = *reinterpret_cast<const float4*>(cosine + at + j), s = *reinterpret_cast<const float4*>(sine + at + j);
            t.c[j / 2] = pack2(c.x, c.y);
            t.c[j / 2 + 1] = pack2(c.z, c.w);
            t.s[j / 2] = is_first ? pack2(-s.x, -s.y) : pack2(s.x, s.y);
            t.s[j / 2 + 1] = is_first ? pack2(-s.z, -s.w) : pack2(s.z, s.w);
        }
    } else if (adjacent) {
        const uint32_t at = t.turns ? t.first / 2 : 0;  // the table has kLane values more than pairs
        const float4 c = *reinterpret_cast<const float4*>(cosine + at), s = *reinterpret_cast<const float4*>(sine + at);
        t.c[0] = pack2(c.x, c.x); t.c[1] = pack2(c.y, c.y); t.c[2] = pack2(c.z, c.z); t.c[3] = pack2(c.w, c.w);
        t.s[0] = pack2(-s.x, s.x); t.s[1] = pack2(-s.y, s.y); t.s[2] = pack2(-s.z, s.z); t.s[3] = pack2(-s.w, s.w);
    } else {
        float c[kLane], s[kLane];
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            const uint32_t i = t.first + j;
            c[j] = i < t.half ? cosine[i] : i < rope_dim ? cosine[i - t.half] : 1.0f;
            s[j] = i < t.half ? -sine[i] : i < rope_dim ? sine[i - t.half] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kLane / 2; ++j) {
            t.c[j] = pack2(c[2 * j], c[2 * j + 1]);
            t.s[j] = pack2(s[2 * j], s[2 * j + 1]);
        }
    }
    return t;
}

// Turns the lane's values; `pass`: the warp's scratch of 256 values. Returns (BOUND) the lane's largest sum of the magnitudes of a pair, 0
// where its values do not turn.
template <bool BOUND>
__device__ __forceinline__ float turned(float (&x)[kLane], const Turns& t, float* pass) {
    const uint32_t lane = threadIdx.x & 31, row = lane * kLane - t.first;
    float other[kLane], most = 0.0f;
    if (t.adjacent) {
#pragma unroll
        for (int j = 0; j < kLane; ++j) other[j] = x[j ^ 1];
    } else if (t.whole) {
#pragma unroll
        for (int j = 0; j < kLane; ++j) other[j] = __shfl_sync(0xffffffffu, x[j], t.from);
    } else {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kLane; ++j) pass[lane * kLane + j] = x[j];
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            const uint32_t i = t.first + j;
            other[j] = i < t.half ? pass[row + i + t.half] : i < t.rope_dim ? pass[row + i - t.half] : 0.0f;
        }
    }
    if (t.whole) {
        if (t.turns) {
#pragma unroll
            for (int j = 0; j < kLane / 2; ++j) {
                if (BOUND) most = fmaxf(most, fmaxf(fabsf(x[2 * j]) + fabsf(other[2 * j]), fabsf(x[2 * j + 1]) + fabsf(other[2 * j + 1])));
                unpack2(fma2(pack2(x[2 * j], x[2 * j + 1]), t.c[j], mul2(pack2(other[2 * j], other[2 * j + 1]), t.s[j])), x[2 * j], x[2 * j + 1]);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            if (t.first + j < t.rope_dim) {
                float c, s, c1, s1;
                unpack2(t.c[j / 2], c, c1);
                unpack2(t.s[j / 2], s, s1);
                most = fmaxf(most, fabsf(x[j]) + fabsf(other[j]));
                x[j] = fmaf(x[j], j % 2 ? c1 : c, other[j] * (j % 2 ? s1 : s));
            }
        }
    }
    return most;
}

// Keys' or values' rows in 64 bits.
template <class T, int D>
__device__ __noinline__ Numbers exact_numbers(const T* src, int wide, const float* bias, const float* norm, float eps, uint32_t first, uint32_t rope_dim, int adjacent, const double2* turn,
                                              double* pass) {
    const uint32_t lane = threadIdx.x & 31, half = rope_dim / 2, row = lane * kLane - first;
    float in[kLane];
    double x[kLane], y[kLane];
    load_values<T, kLane>(src, wide, in);
#pragma unroll
    for (int j = 0; j < kLane; ++j) x[j] = bias != nullptr ? double(in[j]) + double(bias[j]) : double(in[j]);
    if (norm != nullptr) normed<double, D>(x, norm, eps);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kLane; ++j) pass[lane * kLane + j] = x[j];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
        const uint32_t i = first + j;
        y[j] = x[j];
        if (i < rope_dim) {
            const bool is_first = adjacent ? j % 2 == 0 : i < half;
            const double2 t = turn[adjacent ? i / 2 : is_first ? i : i - half];
            const double other = pass[row + (adjacent ? i ^ 1 : is_first ? i + half : i - half)];
            y[j] = is_first ? fma(x[j], t.x, -(other * t.y)) : fma(other, t.y, x[j] * t.x);
        }
    }
    return to_numbers<double>(y);
}

constexpr int kAppendWarps = 2;

// A CTA of two warps to some of a token's rows, so that the token's angles are made once for them, in 64 bits: a far position turns a pair
// thousands of times. A warp takes 32 / (D / 8) rows of q, of k or of v at a time. What is stored is what 64 bits give: a row is computed
// in 32, with a bound on how far its values may be off, and once more in 64 where that bound reaches a border between two numbers or
// two scales (a row in some hundreds). The bound, in half-ulps 2^-24 of the sum of a pair's magnitudes: a value with its bias 1; the
// mean of squares 2 of that, 8 + 5 of its sums and 1 of eps, halved by the root 8; root and quotient 2; products with both and the norm 2;
// cos and sin, a product and a sum 3: 16 in the first order, 18 allowed.
//
// Rows are asked for first of all, so that they arrive while the angles are made; the loop then finds them in shared memory.
template <class T, int D>
__global__ void __launch_bounds__(32 * kAppendWarps, 12) cache4_append_kernel(const Cache4 c, const Cache4Batch b, const Cache4Append a, uint32_t items_per_cta) {
    constexpr uint32_t kLanes = D / 8, kRows = 32 / kLanes;  // lanes of a row, rows of a warp
    constexpr int kPieces = int(sizeof(T)) * kLane / 16, kAhead = 4;  // 16-byte pieces of a lane's values; items asked for at a time
    __shared__ double2 turn[D / 2];
    __shared__ __align__(16) float cosine[D / 2 + kLane], sine[D / 2 + kLane];
    __shared__ double pass[kAppendWarps][256];
    __shared__ uint4 asked[kAppendWarps][kAhead][kPieces][32];
    wait_for_previous();
    release_next();
    const uint32_t row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = (lane & (kLanes - 1)) * kLane;
    const uint32_t q_items = (a.heads + kRows - 1) / kRows, kv_items = (c.kv_heads + kRows - 1) / kRows, end = min(q_items + 2 * kv_items, (blockIdx.y + 1) * items_per_cta);
    const T* q = static_cast<const T*>(a.q) + size_t(row) * a.q_stride + first;
    const T* k = static_cast<const T*>(a.k) + size_t(row) * a.k_stride + first;
    const T* v = static_cast<const T*>(a.v) + size_t(row) * a.v_stride + first;
    // The last rows of a warp may be of no head: they repeat the last one's, and store nothing.
    auto source_of = [&](uint32_t item) {
        const uint32_t which = item < q_items ? item : item < q_items + kv_items ? item - q_items : item - q_items - kv_items;
        return (item < q_items ? q : item < q_items + kv_items ? k : v) + min(which * kRows + lane / kLanes, (item < q_items ? a.heads : c.kv_heads) - 1) * D;
    };
    auto ask = [&](uint32_t item) {
        if (a.wide) {
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                const uint32_t x = item + n * kAppendWarps;
                if (x < end) {
                    const T* src = source_of(x);
#pragma unroll
                    for (int p = 0; p < kPieces; ++p) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(&asked[warp][n][p][lane]))), "l"(src + p * (kLane / kPieces)) : "memory");
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint32_t item = blockIdx.y * items_per_cta + warp;
    ask(item);
    uint32_t sequence;
    long long position;
    const bool ours = row_place(b, row, sequence, position);
    if (!ours) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        return;
    }
    for (uint32_t i = threadIdx.x; i < a.rope_dim / 2; i += 32 * kAppendWarps) {
        double angle = double(position) * a.turns[i], z, w;
        angle -= rint(angle);
        sincospi(2.0 * angle, &z, &w);
        w *= double(a.attn_factor);
        z *= double(a.attn_factor);
        turn[i] = make_double2(w, z);
        cosine[i] = float(w);
        sine[i] = float(z);
    }
    const uint32_t column = uint32_t(position >> c.page_shift), slot = uint32_t(position) & (c.page_size - 1);
    const bool held = position >= 0 && position < (long long)b.columns * c.page_size;
    const int32_t page = held ? page_of(c, b, sequence, column) : -1;
    const size_t page_block = ((size_t(max(page, 0)) * c.kv_heads) * c.page_size + slot) * (D / 32) + first / 32;
    __syncthreads();
    const Turns t = turns_of<D>(a.rope_dim, a.adjacent, cosine, sine);
    const float reach = 0x1.2p-20f * fmaxf(1.0f, fabsf(a.attn_factor));
    T* q_out = static_cast<T*>(a.q_out) + size_t(row) * a.q_out_stride + first;
    const uint32_t sub = lane / kLanes;
    // Rows of queries (kind 0), keys (1) or values (2): item `which` of its kind, the n-th that was asked for.
    auto take = [&](auto kind, uint32_t which, uint32_t n) {
        constexpr int kKind = decltype(kind)::value;
        const uint32_t heads = kKind == 0 ? a.heads : c.kv_heads, wanted = which * kRows + sub, head = min(wanted, heads - 1);
        const bool there = wanted < heads;
        const T* src = (kKind == 0 ? q : kKind == 1 ? k : v) + head * D;
        float x[kLane];
        if (a.wide) {
            Values<T, kLane> u;
#pragma unroll
            for (int p = 0; p < kPieces; ++p) reinterpret_cast<uint4*>(&u)[p] = asked[warp][n][p][lane];
#pragma unroll
            for (int j = 0; j < kLane; ++j) x[j] = Convert<T>::from(u.v[j]);
        } else {
            load_values<T, kLane>(src, 0, x);
        }
        const float* bias = kKind == 0 ? a.q_bias : kKind == 1 ? a.k_bias : a.v_bias;
        const float* norm = kKind == 0 ? a.q_norm : kKind == 1 ? a.k_norm : nullptr;
        if (bias != nullptr) {
            bias += head * D + first;
#pragma unroll
            for (int j = 0; j < kLane; ++j) x[j] = x[j] + bias[j];
        }
        bool in_range = true;
        if (kKind != 2 && norm != nullptr) {
            norm += first;
            float before[kLane];
#pragma unroll
            for (int j = 0; j < kLane; ++j) before[j] = x[j];
            in_range = normed<float, D>(x, norm, a.eps);
            if (kKind == 0 && __any_sync(0xffffffffu, !in_range)) {
                normed_wide<D>(before, norm, a.eps);
                if (!in_range) {
#pragma unroll
                    for (int j = 0; j < kLane; ++j) x[j] = before[j];
                }
            }
        }
        if constexpr (kKind == 0) {
            if (a.rope_dim != 0) turned<false>(x, t, reinterpret_cast<float*>(pass[warp]));
            if (there) store_values<T, kLane>(q_out + head * D, a.wide, x);
        } else {
            if (page < 0) return;
            float most = 0.0f;
            if (bias != nullptr || (kKind == 1 && norm != nullptr)) {
#pragma unroll
                for (int j = 0; j < kLane; ++j) most = fmaxf(most, fabsf(x[j]));
            }
            if (kKind == 1 && a.rope_dim != 0) most = fmaxf(most, turned<true>(x, t, reinterpret_cast<float*>(pass[warp])));
            // 0 where 32 bits hold the values themselves
            const float within = most * reach;
            const size_t block = page_block + size_t(head) * c.page_size * (D / 32);
            Numbers numbers;
            const bool sure = quick_numbers(x, within, numbers) && in_range;
            if (__any_sync(0xffffffffu, !sure)) {
                bool doubt;
                numbers = to_numbers<float>(x, within, &doubt);
                if (__any_sync(0xffffffffu, doubt || !in_range)) {
                    numbers = exact_numbers<T, D>(src, a.wide, bias, norm, a.eps, first, kKind == 1 ? a.rope_dim : 0, a.adjacent, turn, pass[warp]);
                }
            }
            store_numbers(numbers, there, (kKind == 1 ? c.k_quants : c.v_quants) + block * 16, (kKind == 1 ? c.k_scales : c.v_scales) + block);
        }
    };
    for (uint32_t n = 0; item < end; item += kAppendWarps) {
        if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (item < q_items) take(std::integral_constant<int, 0>{}, item, n);
        else if (item < q_items + kv_items) take(std::integral_constant<int, 1>{}, item - q_items, n);
        else take(std::integral_constant<int, 2>{}, item - q_items - kv_items, n);
        if (++n == kAhead) {
            n = 0;
            __syncwarp();
            ask(item + kAppendWarps);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A warp to a head's row.
template <class T, int E>
__global__ void __launch_bounds__(256) cache4_read_kernel(const Cache4 c, const Cache4Batch b, T* k_out, T* v_out, size_t k_stride, size_t v_stride, int wide) {
    const uint32_t row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t sequence;
    long long position;
    if (!row_place(b, row, sequence, position)) return;
    const uint32_t column = uint32_t(position >> c.page_shift), slot = uint32_t(position) & (c.page_size - 1);
    const bool held = position >= 0 && position < (long long)b.columns * c.page_size;
    const int32_t page = held ? page_of(c, b, sequence, column) : -1;
    for (uint32_t r = blockIdx.y * 8 + warp; r < 2 * c.kv_heads; r += gridDim.y * 8) {
        const bool is_k = r < c.kv_heads;
        const uint32_t head = is_k ? r : r - c.kv_heads;
        float x[E];
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = 0.0f;
        if (page >= 0) {
            const size_t stored = ((size_t(page) * c.kv_heads + head) * c.page_size + slot) * E;
            constexpr int kLanes = 32 / E;
            const uint32_t block = lane / kLanes, in_block = lane % kLanes, shift = in_block < kLanes / 2 ? 0 : 4;
            const Values<uint8_t, E> bytes =
                *reinterpret_cast<const Values<uint8_t, E>*>((is_k ? c.k_quants : c.v_quants) + stored * 16 + block * 16 + (in_block % (kLanes / 2)) * E);
            const float d = __half2float((is_k ? c.k_scales : c.v_scales)[stored + block]);
#pragma unroll
            for (int j = 0; j < E; ++j) x[j] = (float((bytes.v[j] >> shift) & 15) - 8.0f) * d;
        }
        T* out = is_k ? k_out + size_t(row) * k_stride : v_out + size_t(row) * v_stride;
        store_values<T, E>(out + size_t(head) * (32 * E) + lane * E, wide, x);
    }
}

template <class T, int D>
void append_typed(const Cache4& c, const Cache4Batch& b, const Cache4Append& a, bool dependent, cudaStream_t s) {
    // Few tokens: an item to a warp, so that a call is as short as its slowest row. Many: a CTA to a token, which makes the angles once (setting
    // up is half a row's work; 6945 tokens of 20 / 5 heads in two warps 56 us, in four 69).
    constexpr uint32_t kRows = 32 / (D / 8);
    const uint32_t items = (a.heads + kRows - 1) / kRows + 2 * ((c.kv_heads + kRows - 1) / kRows);
    const uint32_t most = (items + kAppendWarps - 1) / kAppendWarps, parts = std::max(1u, std::min(most, 2368u / b.tokens));
    const uint32_t items_per_cta = (items + parts - 1) / parts;
    const dim3 grid(b.tokens, (items + items_per_cta - 1) / items_per_cta);
    if (dependent) {
        launch_dependent(cache4_append_kernel<T, D>, grid, dim3(32 * kAppendWarps), 0, s, c, b, a, items_per_cta);
    } else {
        cache4_append_kernel<T, D><<<grid, 32 * kAppendWarps, 0, s>>>(c, b, a, items_per_cta);
        BK_CUDA(cudaGetLastError());
    }
}

template <class T>
void append_sized(const Cache4& c, const Cache4Batch& b, const Cache4Append& a, bool dependent, cudaStream_t s) {
    if (c.dim == 64) append_typed<T, 64>(c, b, a, dependent, s);
    else if (c.dim == 128) append_typed<T, 128>(c, b, a, dependent, s);
    else append_typed<T, 256>(c, b, a, dependent, s);
}

template <class T>
void read_sized(const Cache4& c, const Cache4Batch& b, void* k_out, void* v_out, size_t k_stride, size_t v_stride, cudaStream_t s) {
    const uintptr_t step = uintptr_t(c.dim / 32) * sizeof(T) > 16 ? 16 : uintptr_t(c.dim / 32) * sizeof(T);
    const int wide = (reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out) | (k_stride * sizeof(T)) | (v_stride * sizeof(T))) % step == 0;
    const dim3 grid(b.tokens, (2 * c.kv_heads + 7) / 8);
    T *k = static_cast<T*>(k_out), *v = static_cast<T*>(v_out);
    if (c.dim == 64) cache4_read_kernel<T, 2><<<grid, 256, 0, s>>>(c, b, k, v, k_stride, v_stride, wide);
    else if (c.dim == 128) cache4_read_kernel<T, 4><<<grid, 256, 0, s>>>(c, b, k, v, k_stride, v_stride, wide);
    else cache4_read_kernel<T, 8><<<grid, 256, 0, s>>>(c, b, k, v, k_stride, v_stride, wide);
    BK_CUDA(cudaGetLastError());
}

uint32_t type_bytes(int type) { return type == T_F32 ? 4 : 2; }

}  // namespace

void launch_cache4_append(const Cache4& c, const Cache4Batch& b, const Cache4Append& in, int type, bool dependent, cudaStream_t s) {
    Cache4Append a = in;
    const uintptr_t size = type_bytes(type);
    uintptr_t all = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | (a.k_stride * size) | (a.v_stride * size);
    if (a.heads != 0) all |= reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) | (a.q_stride * size) | (a.q_out_stride * size);
    a.wide = all % 16 == 0;
    if (type == T_F32) append_sized<float>(c, b, a, dependent, s);
    else if (type == T_F16) append_sized<__half>(c, b, a, dependent, s);
    else append_sized<__nv_bfloat16>(c, b, a, dependent, s);
}

void launch_cache4_read(const Cache4& c, const Cache4Batch& b, void* k_out, void* v_out, size_t k_stride, size_t v_stride, int type, cudaStream_t s) {
    if (type == T_F32) read_sized<float>(c, b, k_out, v_out, k_stride, v_stride, s);
    else if (type == T_F16) read_sized<__half>(c, b, k_out, v_out, k_stride, v_stride, s);
    else read_sized<__nv_bfloat16>(c, b, k_out, v_out, k_stride, v_stride, s);
}

namespace {

// ---- the C entries: what they are given, checked before any launch ---------------------------------------------------

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
void require(bool ok, const char* what) {
    if (!ok) throw CudaError(std::string("cuda: the 4-bit cache ") + what);
}

Cache4 checked(const brisk_cuda_cache4* in) {
    require(in != nullptr, "is missing");
    require(in->head_dim == 64 || in->head_dim == 128 || in->head_dim == 256, "takes head sizes of 64, 128 and 256");
    require(in->kv_heads != 0 && in->kv_heads <= 65535, "needs 1 to 65535 key/value heads");
    require(in->page_size >= 16 && in->page_size <= 4096 && (in->page_size & (in->page_size - 1)) == 0, "takes pages of 16 to 4096 positions, a power of two");
    require(in->pages != 0 && in->pages <= 0x7fffffffu, "needs at least one page");
    require(in->k_quants && in->k_scales && in->v_quants && in->v_scales, "needs its four planes");
    require(aligned(in->k_quants, 16) && aligned(in->k_scales, 16) && aligned(in->v_quants, 16) && aligned(in->v_scales, 16),
            "needs planes that start on 16-byte boundaries");
    Cache4 c;
    c.k_quants = static_cast<uint8_t*>(in->k_quants); c.v_quants = static_cast<uint8_t*>(in->v_quants);
    c.k_scales = static_cast<__half*>(in->k_scales); c.v_scales = static_cast<__half*>(in->v_scales);
    c.pages = in->pages; c.page_size = in->page_size; c.kv_heads = in->kv_heads; c.dim = in->head_dim;
    while ((1u << c.page_shift) < c.page_size) ++c.page_shift;
    return c;
}

Cache4Batch checked(const brisk_cuda_cache4_batch* in, const Cache4& c) {
    require(in != nullptr, "needs the description of a batch");
    require(in->tokens <= 0x7fffffffu && in->sequences <= 65535, "takes batches of up to 65535 sequences and 2^31 - 1 tokens");
    Cache4Batch b;
    b.sequences = in->sequences; b.tokens = in->tokens; b.columns = in->table_columns;
    if (b.sequences == 0 || b.tokens == 0) {
        b.tokens = 0;  // nothing to do
        return b;
    }
    require(in->context != nullptr, "needs the positions before the batch (context)");
    require(in->query_start != nullptr || in->tokens % in->sequences == 0, "needs query_start where the tokens do not split evenly over the sequences");
    require(in->table_columns != 0 && uint64_t(in->table_columns) * c.page_size <= 0x7fffffffull, "needs 1 to 2^31 - 1 positions in a sequence's columns");
    require(aligned(in->context, 4) && aligned(in->page_table, 4) && aligned(in->query_start, 4), "needs context, page_table and query_start on 4-byte boundaries");
    b.context = in->context; b.page_table = in->page_table; b.query_start = in->query_start;
    b.max_tokens = in->query_start == nullptr ? b.tokens / b.sequences : in->max_tokens != 0 && in->max_tokens < b.tokens ? in->max_tokens : b.tokens;
    const uint32_t most = b.columns * c.page_size;
    b.max_length = in->max_length != 0 && in->max_length < most ? in->max_length : most;
    return b;
}

// Before the launch: the planes are the current device's.
void check_device(const Cache4& c) {
    int device = -1;
    BK_CUDA(cudaGetDevice(&device));
    cudaPointerAttributes where{};
    BK_CUDA(cudaPointerGetAttributes(&where, c.k_quants));
    require(where.type == cudaMemoryTypeDevice || where.type == cudaMemoryTypeManaged, "is not in device memory");
    require(where.device == device, "is on another device than the current one");
}

// Whether no token's row of a touches a row of b: rows of `width` bytes, `stride` bytes apart. Rows of one stride may lie between one another, as
// the parts of a fused buffer do.
bool apart(const void* a, uint64_t a_stride, uint64_t a_width, const void* b, uint64_t b_stride, uint64_t b_width, uint64_t tokens) {
    const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (x + (tokens - 1) * a_stride + a_width <= y || y + (tokens - 1) * b_stride + b_width <= x) return true;
    if (a_stride != b_stride) return false;
    const uint64_t behind = (y >= x ? y - x : a_stride - (x - y) % a_stride) % a_stride;  // of b's rows behind a's, within a stride
    return behind >= a_width && behind + b_width <= a_stride;
}

void check_type(int type) { require(type == T_F32 || type == T_F16 || type == T_BF16, "takes activations in f32, f16 and bf16"); }

template <class Fn>
int entry(char* err, size_t errlen, Fn&& fn) {
    try {
        fn();
        return 0;
    } catch (const std::exception& e) {
        if (err != nullptr && errlen > 0) std::snprintf(err, errlen, "%s", e.what());
    } catch (...) {
        if (err != nullptr && errlen > 0) std::snprintf(err, errlen, "%s", "cuda: unknown failure");
    }
    return -1;
}

}  // namespace
}  // namespace bk

using bk::require;

extern "C" int brisk_cuda_rope_turns(uint32_t rope_dim, double base, double scale, const float* factors, double* turns, char* err, size_t errlen) {
    return bk::entry(err, errlen, [&] {
        require(turns != nullptr && rope_dim != 0 && rope_dim % 2 == 0, "needs an even rotated width and an output for its turns");
        require(base > 0.0 && std::isfinite(base) && std::isfinite(scale), "needs a positive, finite rotation base and a finite scale");
        for (uint32_t i = 0; i < rope_dim / 2; ++i) {
            require(factors == nullptr || (factors[i] != 0.0f && std::isfinite(factors[i])), "needs divisors of the angles that are finite and not 0");
            const double angle = scale * std::pow(base, -2.0 * double(i) / double(rope_dim));
            const double turn = (factors != nullptr ? angle / double(factors[i]) : angle) / 6.283185307179586476925286766559;
            require(std::isfinite(turn), "needs a rotation whose angles are finite");
            turns[i] = turn;
        }
    });
}

extern "C" int brisk_cuda_cache4_append(const brisk_cuda_cache4* cache, const brisk_cuda_cache4_batch* batch, const brisk_cuda_cache4_rows* rows, void* stream,
                                        char* err, size_t errlen) {
    return bk::entry(err, errlen, [&] {
        const bk::Cache4 c = bk::checked(cache);
        const bk::Cache4Batch b = bk::checked(batch, c);
        require(rows != nullptr, "needs the rows to append");
        bk::check_type(rows->type);
        if (b.tokens == 0) return;
        const uintptr_t size = rows->type == bk::T_F32 ? 4 : 2;
        require(rows->k != nullptr && rows->v != nullptr && bk::aligned(rows->k, size) && bk::aligned(rows->v, size), "needs keys and values on boundaries of their type");
        require(rows->heads % c.kv_heads == 0, "needs a number of query heads that is a multiple of its key/value heads");
        require(rows->heads <= 65535, "takes up to 65535 query heads");
        if (rows->heads != 0) {
            require(rows->q != nullptr && rows->q_out != nullptr && bk::aligned(rows->q, size) && bk::aligned(rows->q_out, size), "needs queries, and where they go, on boundaries of their type");
            require(rows->q_stride >= uint64_t(rows->heads) * c.dim && rows->q_out_stride >= uint64_t(rows->heads) * c.dim, "needs token strides of at least a token's heads (q, q_out)");
        }
        const uint64_t kv = uint64_t(c.kv_heads) * c.dim;
        require((rows->k_stride >= kv && rows->v_stride >= kv), "needs token strides of at least a token's heads (k, v)");
        require(rows->rope_dim <= c.dim && rows->rope_dim % 2 == 0, "rotates an even width of at most the head size");
        require(rows->rope_dim == 0 || rows->rope_turns != nullptr, "needs the turns of the pairs it rotates");
        require(bk::aligned(rows->rope_turns, 8), "needs the turns of the pairs on an 8-byte boundary");
        require(bk::aligned(rows->q_norm, 4) && bk::aligned(rows->k_norm, 4) && bk::aligned(rows->q_bias, 4) && bk::aligned(rows->k_bias, 4) && bk::aligned(rows->v_bias, 4),
                "needs norms and biases on 4-byte boundaries");
        require(rows->eps >= 0.0f && std::isfinite(rows->eps), "needs a finite epsilon of at least 0");
        require(std::isfinite(rows->rope_attn_factor), "needs a finite factor on cos and sin");
        if (rows->heads != 0) {
            const uint64_t wide = uint64_t(rows->heads) * c.dim * size, narrow = kv * size, to = rows->q_out_stride * size;
            require((rows->q == rows->q_out && rows->q_stride == rows->q_out_stride) || bk::apart(rows->q, rows->q_stride * size, wide, rows->q_out, to, wide, b.tokens),
                    "writes its queries over q itself or apart from it");
            require(bk::apart(rows->k, rows->k_stride * size, narrow, rows->q_out, to, wide, b.tokens) && bk::apart(rows->v, rows->v_stride * size, narrow, rows->q_out, to, wide, b.tokens),
                    "cannot write its queries over keys and values");
        }
        bk::Cache4Append a;
        a.q = rows->q; a.k = rows->k; a.v = rows->v; a.q_out = rows->q_out;
        a.q_stride = rows->q_stride; a.k_stride = rows->k_stride; a.v_stride = rows->v_stride; a.q_out_stride = rows->q_out_stride;
        a.q_norm = rows->q_norm; a.k_norm = rows->k_norm; a.q_bias = rows->q_bias; a.k_bias = rows->k_bias; a.v_bias = rows->v_bias;
        a.turns = rows->rope_turns; a.heads = rows->heads; a.rope_dim = rows->rope_dim; a.adjacent = rows->rope_adjacent != 0;
        a.eps = rows->eps; a.attn_factor = rows->rope_attn_factor != 0.0f ? rows->rope_attn_factor : 1.0f;
        bk::check_device(c);
        bk::launch_cache4_append(c, b, a, rows->type, false, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int brisk_cuda_cache4_read(const brisk_cuda_cache4* cache, const brisk_cuda_cache4_batch* batch, int32_t type, void* k, void* v, uint64_t k_stride,
                                      uint64_t v_stride, void* stream, char* err, size_t errlen) {
    return bk::entry(err, errlen, [&] {
        const bk::Cache4 c = bk::checked(cache);
        const bk::Cache4Batch b = bk::checked(batch, c);
        bk::check_type(type);
        if (b.tokens == 0) return;
        const uintptr_t size = type == bk::T_F32 ? 4 : 2;
        require(k != nullptr && v != nullptr && bk::aligned(k, size) && bk::aligned(v, size), "needs outputs for keys and values on boundaries of their type");
        const uint64_t kv = uint64_t(c.kv_heads) * c.dim;
        require(k_stride >= kv && v_stride >= kv, "needs token strides of at least a token's heads (k, v)");
        require(bk::apart(k, k_stride * size, kv * size, v, v_stride * size, kv * size, b.tokens), "cannot write its keys over its values");
        bk::check_device(c);
        bk::launch_cache4_read(c, b, k, v, k_stride, v_stride, type, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int brisk_cuda_cache4_attention(const brisk_cuda_cache4* cache, const brisk_cuda_cache4_batch* batch, int32_t type, const void* q, void* out, uint64_t q_stride,
                                           uint64_t out_stride, uint32_t heads, float scale, uint32_t window, void* stream, char* err, size_t errlen) {
    return bk::entry(err, errlen, [&] {
        const bk::Cache4 c = bk::checked(cache);
        const bk::Cache4Batch b = bk::checked(batch, c);
        bk::check_type(type);
        require(heads != 0 && heads <= 65535 && heads % c.kv_heads == 0, "needs a number of query heads that is a multiple of its key/value heads");
        require(std::isfinite(scale), "needs a finite scale");
        require(uint64_t(batch->tokens) * (heads / c.kv_heads) <= 0x7fffffffull, "takes up to 2^31 - 1 tokens times query heads of a key/value head");
        if (b.tokens == 0) return;
        const uintptr_t size = type == bk::T_F32 ? 4 : 2;
        require(q != nullptr && out != nullptr && bk::aligned(q, size) && bk::aligned(out, size), "needs queries, and where the result goes, on boundaries of their type");
        require(q != out, "cannot write its result over the queries");
        require(q_stride >= uint64_t(heads) * c.dim && out_stride >= uint64_t(heads) * c.dim, "needs token strides of at least a token's heads (q, out)");
        const uint64_t wide = uint64_t(heads) * c.dim * size;
        require(bk::apart(q, q_stride * size, wide, out, out_stride * size, wide, b.tokens), "cannot write its result over the queries");
        bk::Cache4Attend a;
        a.q = q; a.out = out; a.q_stride = q_stride; a.out_stride = out_stride; a.heads = heads; a.window = window;
        a.scale = scale != 0.0f ? scale : 1.0f / std::sqrt(float(c.dim));
        bk::check_device(c);
        bk::launch_cache4_attention(c, b, a, type, false, static_cast<cudaStream_t>(stream));
    });
}
