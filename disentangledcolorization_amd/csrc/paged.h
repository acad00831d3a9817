// paged.h - internal declarations of the paged-cache operators (rotary.hip, cache_pages.hip, cache_attention.hip, api_cache.cpp).
#pragma once
#include "common.h"

namespace disco {

// the sequence that a token of the joined rows belongs to: how many sequences end at or before it (64 lanes look at 64 ends at a time, so the
// answer is the same in every lane).  `rows` when the token lies behind the last sequence.
__device__ __forceinline__ int seq_of_token(const int* __restrict__ cu_new, int rows, int token) {
    int b = 0;
    for (int i = 0; i < rows; i += 64) {
        const int j = i + (int)(threadIdx.x & 63);
        const unsigned long long ended = __ballot(j < rows && cu_new[j + 1] <= token);
        b += __popcll(ended);
        if (ended != ~0ull) break;
    }
    return b;
}

// A grid of any number of workgroups: a launch has fewer than 2^32 threads along an axis.  block_of() counts them; the last ones may lie behind the end.
inline dim3 grid_of(long blocks) {
    constexpr long AXIS = 1 << 22;
    return blocks <= AXIS ? dim3((unsigned)blocks) : dim3((unsigned)AXIS, (unsigned)((blocks + AXIS - 1) / AXIS));
}
__device__ __forceinline__ long block_of() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }

// a length as the kernels use it: never beyond what the row of the page table can name
__device__ __host__ __forceinline__ int clamp_len(int len, int capacity) { return len < 0 ? 0 : (len < capacity ? len : capacity); }

int launch_rotary(const disco_rotary_desc& d, const void* x, const void* positions, const double* inv_freq, void* out, hipStream_t s);
int launch_cache_append(const disco_cache_desc& c, const disco_append_desc& a, const void* q, const void* k, const void* v, const int* table,
                        const int* lens, const int* cu_new, const void* positions, const double* inv_freq, void* q_out, const int* info, hipStream_t s);

// args: an AttnArgs (cache_attention.hip)
int launch_cache_attention_precise(const void* args, bool half, long many_units, long large_units, hipStream_t s);
size_t cache_attention_ws_bytes(const disco_cache_desc& c, const disco_attention_desc& a);
int launch_cache_attention(const disco_cache_desc& c, const disco_attention_desc& a, const void* q, const int* table, const int* lens,
                           const int* cu_new, void* out, float* lse, void* ws, bool precise, hipStream_t s);

int launch_cache_reserve(int rows, int width, int pages, int page_shift, const int* table, const int* lens, const int* refs, const int* cu_new,
                         int* table_out, int* lens_out, int* refs_out, int* info, hipStream_t s);
size_t cache_pages_ws_bytes(int rows, int pages);
int launch_cache_select(const disco_cache_desc& c, const int* table, const int* lens, const int* parents, int* table_out, int* lens_out,
                        int* refs_out, int* info, void* ws, hipStream_t s);
int launch_cache_compact(const disco_cache_desc& c, const int* table, const int* lens, int* table_out, int* refs_out, int* info, void* ws,
                         hipStream_t s);
int launch_cache_copy_pages(const disco_cache_desc& c, const int* src, const int* dst, int count, hipStream_t s);

}  // namespace disco
