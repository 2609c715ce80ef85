// The paged key/value cache in 4 bits: appending a batch's keys and values with the per-head norm and the rotation on the way, reading
// rows back as values, and the C entries of include/brisk_cuda.h. The attention over it is in cache4_attn.cu.
#include <cuda_bf16.h>

#include <cmath>
#include <cstdio>
#include <cstring>

#include "../../include/brisk_cuda.h"
#include "cache4.h"
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

// A row of 32 E values, E to a lane, to its blocks of 32. The borders between two numbers, (n - 8.5) d with d of 8 significant bits, are
// exact in 32 bits: the number is estimated by a reciprocal and then put right by comparing with the two borders beside it, so
// it is the one that the definition floor(x / d + 8.5) has, whatever the estimate rounds to. NaN counts as 0 and an
// infinity as the largest number that a block holds, so that no row of the cache holds either.
template <class Real, int E>
__device__ __forceinline__ void store_blocks(Real (&x)[E], uint8_t* quants, __half* scales) {
    constexpr int kLanes = 32 / E;  // of a block
    const uint32_t lane = threadIdx.x & 31;
    Real high = -Real(3e38f), low = Real(3e38f);
#pragma unroll
    for (int j = 0; j < E; ++j) {
        x[j] = x[j] != x[j] ? Real(0) : x[j] > Real(3e38f) ? Real(3e38f) : x[j] < -Real(3e38f) ? -Real(3e38f) : x[j];
        high = x[j] > high ? x[j] : high;
        low = x[j] < low ? x[j] : low;
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
        const Real h = __shfl_xor_sync(0xffffffffu, high, o), l = __shfl_xor_sync(0xffffffffu, low, o);
        high = h > high ? h : high;
        low = l < low ? l : low;
    }
    const Real peak = high >= -low ? high : low;
    const float wanted = peak == Real(0) ? 0.0f : eight_bits(peak * Real(-0.125));
    const __half d = __float2half_rn(fminf(fmaxf(wanted, -65280.0f), 65280.0f));  // 255 x 256: the largest f16 of 8 bits
    const float signed_d = __half2float(d), size = fabsf(signed_d), inverse = size != 0.0f ? __fdividef(1.0f, size) : 0.0f;
    uint32_t packed = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        float n = 8.0f;
        if (size != 0.0f) {
            const Real r = signed_d < 0.0f ? -x[j] : x[j];
            n = fminf(fmaxf(floorf(fmaf(float(r), inverse, 8.5f)), 0.0f), 15.0f);
            if (r < Real((n - 8.5f) * size)) n = n - 1.0f;
            else if (r >= Real((n - 7.5f) * size)) n = n + 1.0f;
            n = fminf(fmaxf(n, 0.0f), 15.0f);
        }
        packed |= uint32_t(n) << (4 * j);
    }
    const uint32_t upper = __shfl_xor_sync(0xffffffffu, packed, kLanes / 2);  // the numbers of the values 16 further on
    const uint32_t in_block = lane % kLanes, block = lane / kLanes;
    if (in_block < kLanes / 2) {
        Values<uint8_t, E> bytes;
#pragma unroll
        for (int j = 0; j < E; ++j) bytes.v[j] = uint8_t(((packed >> (4 * j)) & 15u) | (((upper >> (4 * j)) & 15u) << 4));
        *reinterpret_cast<Values<uint8_t, E>*>(quants + block * 16 + in_block * E) = bytes;
        if (in_block == 0) scales[block] = d;
    }
}

// y = x / rms(x) * norm, then the pairs of the first rope_dim values turned by (cos, sin). `pass` is the warp's scratch of 32 E values.
template <class Real, int E>
__device__ __forceinline__ void norm_and_turn(Real (&x)[E], const float* norm, float eps, uint32_t rope_dim, int adjacent, const double2* turn, Real* pass) {
    const uint32_t lane = threadIdx.x & 31;
    if (norm != nullptr) {
        Real sum = Real(0);
#pragma unroll
        for (int j = 0; j < E; ++j) sum = fused(x[j], x[j], sum);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const Real scale = Real(1) / root(sum / Real(32 * E) + Real(eps));
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = x[j] * scale * Real(norm[lane * E + j]);
    }
    if (rope_dim == 0) return;
    const uint32_t half = rope_dim / 2;
    if (!adjacent) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < E; ++j) pass[lane * E + j] = x[j];
        __syncwarp();
    }
    Real y[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const uint32_t i = lane * E + j;
        y[j] = x[j];
        if (i < rope_dim) {
            const bool first = adjacent ? j % 2 == 0 : i < half;
            const double2 t = turn[adjacent ? i / 2 : first ? i : i - half];
            const Real c = Real(t.x), s = Real(t.y);
            const Real other = adjacent ? x[j ^ 1] : pass[first ? i + half : i - half];
            y[j] = first ? fused(x[j], c, -(other * s)) : fused(other, s, x[j] * c);
        }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = y[j];
}

// A warp to a head's row of q, k or v; a CTA of eight warps to some of a token's rows, so that the token's angles are made once for
// them. Angles, and the keys' norm, rotation and borders, are in 64 bits: a far position turns a pair thousands of times, and a
// key that lies next to the border between two numbers is stored as the definition has it, not as 32 bits happen to round.
template <class T, int E>
__global__ void __launch_bounds__(256) cache4_append_kernel(const Cache4 c, const Cache4Batch b, const Cache4Append a, uint32_t rows_per_cta) {
    __shared__ double2 turn[E * 16];
    __shared__ double pass[8][E * 32];
    wait_for_previous();
    release_next();
    const uint32_t row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t sequence;
    long long position;
    if (!row_place(b, row, sequence, position)) return;
    for (uint32_t i = threadIdx.x; i < a.rope_dim / 2; i += 256) {
        double angle = double(position) * a.turns[i], z, w;
        angle -= rint(angle);
        sincospi(2.0 * angle, &z, &w);
        turn[i] = make_double2(w * double(a.attn_factor), z * double(a.attn_factor));
    }
    __syncthreads();
    const uint32_t column = uint32_t(position >> c.page_shift), slot = uint32_t(position) & (c.page_size - 1);
    const bool held = position >= 0 && position < (long long)b.columns * c.page_size;
    const int32_t page = held ? page_of(c, b, sequence, column) : -1;
    const uint32_t all = a.heads + 2 * c.kv_heads, end = min(all, (blockIdx.y + 1) * rows_per_cta);
    for (uint32_t r = blockIdx.y * rows_per_cta + warp; r < end; r += 8) {
        const bool is_q = r < a.heads, is_k = !is_q && r < a.heads + c.kv_heads;
        const uint32_t head = is_q ? r : is_k ? r - a.heads : r - a.heads - c.kv_heads;
        if (!is_q && page < 0) continue;
        const size_t at = size_t(head) * (32 * E) + lane * E;
        const T* src = is_q ? static_cast<const T*>(a.q) + size_t(row) * a.q_stride : is_k ? static_cast<const T*>(a.k) + size_t(row) * a.k_stride
                                                                                   : static_cast<const T*>(a.v) + size_t(row) * a.v_stride;
        const float* bias = is_q ? a.q_bias : is_k ? a.k_bias : a.v_bias;
        float in[E];
        load_values<T, E>(src + at, a.wide, in);
        if (is_q) {
            if (bias != nullptr) {
#pragma unroll
                for (int j = 0; j < E; ++j) in[j] += bias[at + j];
            }
            norm_and_turn<float, E>(in, a.q_norm, a.eps, a.rope_dim, a.adjacent, turn, reinterpret_cast<float*>(pass[warp]));
            store_values<T, E>(static_cast<T*>(a.q_out) + size_t(row) * a.q_out_stride + at, a.wide, in);
            continue;
        }
        const size_t stored = ((size_t(page) * c.kv_heads + head) * c.page_size + slot) * E;  // in units of dim / E = 32 values
        double x[E];
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = bias != nullptr ? double(in[j]) + double(bias[at + j]) : double(in[j]);
        if (is_k) {
            norm_and_turn<double, E>(x, a.k_norm, a.eps, a.rope_dim, a.adjacent, turn, pass[warp]);
            store_blocks<double, E>(x, c.k_quants + stored * 16, c.k_scales + stored);
        } else if (bias != nullptr) {
            store_blocks<double, E>(x, c.v_quants + stored * 16, c.v_scales + stored);
        } else {
            store_blocks<float, E>(in, c.v_quants + stored * 16, c.v_scales + stored);
        }
    }
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

template <class T, int E>
void append_typed(const Cache4& c, const Cache4Batch& b, const Cache4Append& a, bool dependent, cudaStream_t s) {
    // Few tokens: a warp per row, so that a call is as short as its slowest row. Many: a CTA per token, which makes the angles once.
    const uint32_t all = a.heads + 2 * c.kv_heads;
    const uint32_t parts = b.tokens >= 592 ? 1 : (all + 7) / 8;
    const uint32_t rows_per_cta = (all + parts - 1) / parts;
    const dim3 grid(b.tokens, (all + rows_per_cta - 1) / rows_per_cta);
    if (dependent) {
        launch_dependent(cache4_append_kernel<T, E>, grid, dim3(256), 0, s, c, b, a, rows_per_cta);
    } else {
        cache4_append_kernel<T, E><<<grid, 256, 0, s>>>(c, b, a, rows_per_cta);
        BK_CUDA(cudaGetLastError());
    }
}

template <class T>
void append_sized(const Cache4& c, const Cache4Batch& b, const Cache4Append& a, bool dependent, cudaStream_t s) {
    if (c.dim == 64) append_typed<T, 2>(c, b, a, dependent, s);
    else if (c.dim == 128) append_typed<T, 4>(c, b, a, dependent, s);
    else append_typed<T, 8>(c, b, a, dependent, s);
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
    const uintptr_t size = type_bytes(type), lane = uintptr_t(c.dim / 32) * size, step = lane > 16 ? 16 : lane;
    uintptr_t all = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | (a.k_stride * size) | (a.v_stride * size);
    if (a.heads != 0) all |= reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) | (a.q_stride * size) | (a.q_out_stride * size);
    a.wide = all % step == 0;
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
            const double angle = scale * std::pow(base, -2.0 * double(i) / double(rope_dim));
            turns[i] = (factors != nullptr ? angle / double(factors[i]) : angle) / 6.283185307179586476925286766559;
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
        require(rows->eps >= 0.0f, "needs an epsilon of at least 0");
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
        if (b.tokens == 0) return;
        const uintptr_t size = type == bk::T_F32 ? 4 : 2;
        require(q != nullptr && out != nullptr && bk::aligned(q, size) && bk::aligned(out, size), "needs queries, and where the result goes, on boundaries of their type");
        require(q != out, "cannot write its result over the queries");
        require(q_stride >= uint64_t(heads) * c.dim && out_stride >= uint64_t(heads) * c.dim, "needs token strides of at least a token's heads (q, out)");
        bk::Cache4Attend a;
        a.q = q; a.out = out; a.q_stride = q_stride; a.out_stride = out_stride; a.heads = heads; a.window = window;
        a.scale = scale != 0.0f ? scale : 1.0f / std::sqrt(float(c.dim));
        bk::check_device(c);
        bk::launch_cache4_attention(c, b, a, type, false, static_cast<cudaStream_t>(stream));
    });
}
