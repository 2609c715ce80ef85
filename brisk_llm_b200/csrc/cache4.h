// The paged key/value cache in 4 bits (cache4.cu, cache4_attn.cu): what its kernels are given. Pages hold
//   k_quants, v_quants  [pages][kv_heads][page_size][dim / 2] bytes
//   k_scales, v_scales  [pages][kv_heads][page_size][dim / 32] f16
// a position's row of a head being dim / 32 blocks of 32 values in the byte order of Q4_0: byte j holds value j in its low and value
// j + 16 in its high four bits, a value is (n - 8) d. The scales that the append kernel writes have 8 significant bits, so that the
// product - 3 bits and a sign times 8 - is an f16 number where the scale is below 8192: kernels that multiply in f16 multiply the stored
// values themselves. For larger scales see past_f16 (cache4_math.cuh).
#pragma once

#include <mutex>

#include "kernels.h"

namespace bk {

struct Cache4 {
    uint8_t *k_quants = nullptr, *v_quants = nullptr;
    __half *k_scales = nullptr, *v_scales = nullptr;
    uint32_t pages = 0, page_size = 0, page_shift = 0, kv_heads = 0, dim = 0;
};

// Sequences of ragged length whose tokens lie one behind the other in q, k, v and out. Token i of sequence s is row
// query_start[s] + i and stands at position context[s] + i; rows from query_start[sequences] on belong to nobody.
struct Cache4Batch {
    const int32_t* context = nullptr;      // [sequences]
    const int32_t* page_table = nullptr;   // [sequences][columns]; null: column c of sequence s is page s * columns + c
    const int32_t* query_start = nullptr;  // [sequences + 1]; null: tokens / sequences each
    uint32_t sequences = 0, columns = 0, tokens = 0;
    uint32_t max_tokens = 0, max_length = 0;  // bounds over the sequences: tokens, and context + tokens
};

struct Cache4Append {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    void* q_out = nullptr;
    size_t q_stride = 0, k_stride = 0, v_stride = 0, q_out_stride = 0;  // values between two tokens
    const float *q_norm = nullptr, *k_norm = nullptr, *q_bias = nullptr, *k_bias = nullptr, *v_bias = nullptr;
    const double* turns = nullptr;  // [rope_dim / 2] turns a position, null: no rotation
    uint32_t heads = 0, rope_dim = 0;
    int adjacent = 0;
    float eps = 0.0f, attn_factor = 1.0f;
    int wide = 0;  // rows start where a lane's values can be moved at once
};

struct Cache4Attend {
    const void* q = nullptr;
    void* out = nullptr;
    size_t q_stride = 0, out_stride = 0;
    uint32_t heads = 0, window = 0;
    float scale = 0.0f;
    int wide = 0;
    WaitBound bound;  // of the waits of the many-rows kernel; error may be null: only the NaN then says that one ran out
};

// What a kernel needs set once for each device (its opt-in to shared memory and cluster sizes), before its first launch there, whichever of
// the host's threads comes first.
struct DeviceSetup {
    std::once_flag flags[64];
    template <class Fn> void once(Fn&& fn) {
        int device = 0;
        BK_CUDA(cudaGetDevice(&device));
        if (device < 0 || device >= 64) throw CudaError("cuda: device ordinal out of range");
        std::call_once(flags[device], fn);
    }
};

// type: T_F32, T_F16 or T_BF16, of q, k, v and what comes out. dependent: started by launch_dependent().
void launch_cache4_append(const Cache4& c, const Cache4Batch& b, const Cache4Append& a, int type, bool dependent, cudaStream_t s);
void launch_cache4_read(const Cache4& c, const Cache4Batch& b, void* k_out, void* v_out, size_t k_stride, size_t v_stride, int type, cudaStream_t s);
void launch_cache4_attention(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, int type, bool dependent, cudaStream_t s);
// The kernel of many rows (cache4_prompt.cu), and whether launch_cache4_attention takes it.
bool cache4_prompt_takes(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, int type);
void launch_cache4_prompt(const Cache4& c, const Cache4Batch& b, const Cache4Attend& a, int type, bool dependent, cudaStream_t s);

#ifdef __CUDACC__
// Tokens of a sequence and where they begin, whatever the arrays hold: rows are always inside [0, tokens).
__device__ __forceinline__ void sequence_rows(const Cache4Batch& b, uint32_t s, uint32_t& first, uint32_t& count) {
    if (b.query_start == nullptr) {
        count = b.tokens / b.sequences;
        first = s * count;
        return;
    }
    const int32_t total = int32_t(b.tokens);
    const int32_t lo = min(max(b.query_start[s], 0), total), hi = min(max(b.query_start[s + 1], lo), total);
    first = uint32_t(lo);
    count = uint32_t(hi - lo);
}

// The sequence and position of a row, by a whole warp; false: the row belongs to nobody.
__device__ __forceinline__ bool row_place(const Cache4Batch& b, uint32_t row, uint32_t& sequence, long long& position) {
    uint32_t first;
    if (b.query_start == nullptr) {
        const uint32_t each = b.tokens / b.sequences;
        sequence = row / each;
        first = sequence * each;
    } else {
        const uint32_t lane = threadIdx.x & 31;
        uint32_t before = 0;  // sequences that end at or before the row
#pragma unroll 4
        for (uint32_t s = 0; s < b.sequences; s += 32) {
            const bool ended = s + lane < b.sequences && b.query_start[s + lane + 1] <= int32_t(row);
            before += __popc(__ballot_sync(0xffffffffu, ended));
        }
        if (before >= b.sequences) return false;
        sequence = before;
        const int32_t start = b.query_start[sequence];
        if (start < 0 || start > int32_t(row)) return false;
        first = uint32_t(start);
    }
    position = (long long)b.context[sequence] + (row - first);
    return true;
}

// The page of a column, or -1: a number outside the pool, which reads as zeros and is never written.
__device__ __forceinline__ int32_t page_of(const Cache4& c, const Cache4Batch& b, uint32_t sequence, uint32_t column) {
    const size_t at = size_t(sequence) * b.columns + column;
    if (b.page_table == nullptr) return at < c.pages ? int32_t(at) : -1;
    const int32_t page = b.page_table[at];
    return page >= 0 && uint32_t(page) < c.pages ? page : -1;
}

#endif

}  // namespace bk
