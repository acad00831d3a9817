// cache_attention.hip - attention of new tokens over a paged cache.
#include "paged.h"

namespace disco {

namespace {

struct AttnArgs {
    const char *q, *k, *v; char* out; float* lse;
    const int *table, *lens, *cu_new;
    long q_token, q_head, out_token, out_head, page_stride, head_stride, slot_stride;    // bytes
    int tokens, q_heads, kv_heads, group, dim, rows, width, pages, page_shift, causal, window;
    float scale;
};

// One wave an output row, 64 keys at a time: lane = key for the scores, lane = elements for the sums
template <typename T>
__global__ __launch_bounds__(64) void cache_attention_kernel(AttnArgs a) {
    const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
    const int b = seq_of_token(a.cu_new, a.rows, token);
    if (b >= a.rows) return;
    const int first = a.cu_new[b], n = a.cu_new[b + 1] - first;
    const int len = clamp_len(a.lens[b], a.width << a.page_shift), p = len - n + (token - first);
    const int end = a.causal ? min(len, p + 1) : len, begin = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const T* q = (const T*)(a.q + token * a.q_token + head * a.q_head);
    const long at_head = (head / a.group) * a.head_stride;
    float m = -INFINITY, l = 0, o[4] = {0, 0, 0, 0};
    for (int k0 = begin; k0 < end; k0 += 64) {
        const int key = k0 + lane;
        float s = -INFINITY;
        long at = 0;
        bool bad = false;
        if (key < end) {
            const int page = a.table[(long)b * a.width + (key >> a.page_shift)];
            bad = page < 0 || page >= a.pages;
            at = (bad ? 0 : page * a.page_stride) + (key & ((1 << a.page_shift) - 1)) * a.slot_stride + at_head;
            const T* kr = (const T*)(a.k + at);
            float d = 0;
            for (int i = 0; i < a.dim; ++i) d = fmaf((float)q[i], (float)kr[i], d);
            s = bad ? NAN : d * a.scale;
        }
        float top = s;
        for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
        const float now = fmaxf(m, top), back = now == -INFINITY ? 1.f : expf(m - now), pr = key < end ? expf(s - now) : 0.f;
        float sum = pr;
        for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
        l = l * back + sum;
        m = now;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= back;
        const int there = min(64, end - k0);
        for (int j = 0; j < there; ++j) {
            const float w = __shfl(pr, j);
            const T* vr = (const T*)(a.v + __shfl(at, j));
#pragma unroll
            for (int i = 0; i < 4; ++i) if (lane + 64 * i < a.dim) o[i] = fmaf(w, (float)vr[lane + 64 * i], o[i]);
        }
    }
    T* out = (T*)(a.out + token * a.out_token + head * a.out_head);
#pragma unroll
    for (int i = 0; i < 4; ++i) if (lane + 64 * i < a.dim) out[lane + 64 * i] = (T)(end > begin ? o[i] / l : 0.f);
    if (a.lse && lane == 0) a.lse[(long)token * a.q_heads + head] = end > begin ? m + logf(l) : -INFINITY;
}

}  // namespace

size_t cache_attention_ws_bytes(const disco_cache_desc&, const disco_attention_desc&) { return 0; }

int launch_cache_attention(const disco_cache_desc& c, const disco_attention_desc& d, const void* q, const int* table, const int* lens,
                           const int* cu_new, void* out, float* lse, void*, hipStream_t s) {
    AttnArgs a{(const char*)q, (const char*)c.d_k, (const char*)c.d_v, (char*)out, lse, table, lens, cu_new, d.q_token * 2, d.q_head * 2, d.out_token * 2,
               d.out_head * 2, c.page_stride * 2, c.head_stride * 2, c.slot_stride * 2, d.tokens, d.q_heads, c.kv_heads, d.q_heads / c.kv_heads, c.dim,
               c.rows, c.table_width, c.pages, __builtin_ctz((unsigned)c.page_size), d.causal, d.window, d.scale};
    const dim3 grid(d.tokens, d.q_heads);
    if (c.dtype == DISCO_F16) cache_attention_kernel<f16><<<grid, 64, 0, s>>>(a);
    else cache_attention_kernel<__bf16><<<grid, 64, 0, s>>>(a);
    DISCO_LAUNCH_CHECK("cache_attention_kernel");
    return DISCO_OK;
}

}  // namespace disco
