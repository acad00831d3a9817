// api_cache.cpp - the entry points of token sequences served from a paged cache: what the host can check is checked here, before any launch.
#include <cmath>
#include "ctx.h"
#include "paged.h"

namespace {

constexpr int64_t FAR = (int64_t)1 << 56;      // strides stay far from overflow in bytes

int bad_shape(const char* op, const char* what) { set_error("%s: %s", op, what); return DISCO_ESHAPE; }
int bad_value(const char* op, const char* what) { set_error("%s: %s", op, what); return DISCO_EINVAL; }

bool within(std::initializer_list<int64_t> strides) {
    for (int64_t s : strides) if (s >= FAR || s <= -FAR) return false;
    return true;
}

int check_pages(const char* op, int rows, int width, int pages, int page_size) {
    if (!positive(op, {rows, width, pages, page_size})) return DISCO_ESHAPE;
    if (page_size & (page_size - 1)) return bad_shape(op, "page_size must be a power of two");
    if ((int64_t)width * page_size > (1 << 30)) return bad_shape(op, "table_width * page_size beyond 2^30 tokens");
    if (rows > 16384) return bad_shape(op, "more than 16384 rows");
    if ((int64_t)rows * width > 0x7fffffff) return bad_shape(op, "a page table of more than 2^31 entries");
    return DISCO_OK;
}

int check_cache(const char* op, const disco_cache_desc* c, bool one_layer) {
    if (!c || !c->d_k || !c->d_v) return bad_value(op, "null argument");
    if (c->dtype != DISCO_F16 && c->dtype != DISCO_BF16) return bad_value(op, "the cache holds fp16 or bf16");
    if (!positive(op, {c->layers, c->kv_heads, c->dim})) return DISCO_ESHAPE;
    if (int rc = check_pages(op, c->rows, c->table_width, c->pages, c->page_size)) return rc;
    if (c->dim % 8 || c->dim > 256) return bad_shape(op, "dim must be a multiple of 8, at most 256");
    if (((uintptr_t)c->d_k | (uintptr_t)c->d_v) % 16) return bad_value(op, "d_k and d_v must be aligned to 16 bytes");
    if ((c->page_stride | c->head_stride | c->slot_stride | (one_layer ? 0 : c->layer_stride)) % 8) return bad_shape(op, "cache strides must be multiples of 8 elements");
    if (!within({c->page_stride, c->head_stride, c->slot_stride, c->layer_stride})) return bad_shape(op, "stride too large");
    return DISCO_OK;
}

// what copies pages: a head of a page is counted in 16-byte pieces
int check_copied_cache(const char* op, const disco_cache_desc* c) {
    if (int rc = check_cache(op, c, false)) return rc;
    if ((int64_t)c->page_size * (c->dim / 8) > 0x7fffffff) return bad_shape(op, "a head of a page of more than 2^31 pieces of 16 bytes");
    return DISCO_OK;
}

}  // namespace

extern "C" {

int disco_op_rotary_frequencies(int dim, int scaling, double base, double factor, double original_length, double low, double high,
                                double* h_inv_freq) {
    const char* op = "rotary_frequencies";
    if (!h_inv_freq) return bad_value(op, "null argument");
    if (dim < 2 || dim % 2) return bad_shape(op, "dim must be even and positive");
    if (!(base > 1) || !std::isfinite(base)) return bad_value(op, "base must be above 1");
    if (scaling < DISCO_ROTARY_PLAIN || scaling > DISCO_ROTARY_PARTS) return bad_value(op, "unknown scaling");
    if (scaling != DISCO_ROTARY_PLAIN && (!(factor > 0) || !std::isfinite(factor))) return bad_value(op, "factor must be positive");
    if (scaling == DISCO_ROTARY_NTK && dim < 4) return bad_shape(op, "a changed base needs at least two pairs");
    if (scaling == DISCO_ROTARY_PARTS && !(original_length > 0 && std::isfinite(original_length) && high > low && low >= 0 && std::isfinite(high)))
        return bad_value(op, "original_length must be positive and 0 <= low < high");
    if (scaling == DISCO_ROTARY_NTK) base *= std::pow(factor, (double)dim / (dim - 2));
    for (int i = 0; i < dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / dim);
        if (scaling == DISCO_ROTARY_LINEAR) f /= factor;
        if (scaling == DISCO_ROTARY_PARTS) {
            double kept = (original_length * f / 6.283185307179586 - low) / (high - low);
            kept = kept < 0 ? 0 : (kept > 1 ? 1 : kept);
            f = (1 - kept) * f / factor + kept * f;
        }
        h_inv_freq[i] = f;
    }
    return DISCO_OK;
}

int disco_op_rotary(const disco_rotary_desc* d, const void* d_x, const void* d_positions, const double* d_inv_freq, void* d_out, void* stream) {
    const char* op = "rotary";
    if (!d) return bad_value(op, "null argument");
    if (d->dtype < DISCO_F16 || d->dtype > DISCO_F32) return bad_value(op, "fp16, bf16 or fp32");
    if (d->tokens < 0) return bad_shape(op, "negative size");
    if (!positive(op, {d->heads, d->dim})) return DISCO_ESHAPE;
    if (d->heads > 1 << 16 || d->dim > 1024 || d->tokens > 1 << 30) return bad_shape(op, "more than 2^30 tokens, 65536 heads or 1024 elements a head");
    if (d->rotated < 2 || d->rotated % 2 || d->rotated > d->dim) return bad_shape(op, "rotated must be even, 2 .. dim");
    if (!within({d->x_token, d->x_head, d->out_token, d->out_head})) return bad_shape(op, "stride too large");
    if (!d->tokens) return DISCO_OK;
    if (!d_x || !d_positions || !d_inv_freq || !d_out) return bad_value(op, "null argument");
    if (d_x == d_out && (d->x_token != d->out_token || d->x_head != d->out_head)) return bad_value(op, "in place with other strides");
    return launch_rotary(*d, d_x, d_positions, d_inv_freq, d_out, (hipStream_t)stream);
}

int disco_op_cache_append(const disco_cache_desc* c, const disco_append_desc* a, const void* d_q, const void* d_k, const void* d_v,
                          const int32_t* d_page_table, const int32_t* d_lens, const int32_t* d_cu_new, const void* d_positions,
                          const double* d_inv_freq, void* d_q_out, void* stream) {
    return disco_op_cache_append_reserved(c, a, d_q, d_k, d_v, d_page_table, d_lens, d_cu_new, d_positions, d_inv_freq, d_q_out, nullptr, stream);
}

int disco_op_cache_append_reserved(const disco_cache_desc* c, const disco_append_desc* a, const void* d_q, const void* d_k, const void* d_v,
                                   const int32_t* d_page_table, const int32_t* d_lens, const int32_t* d_cu_new, const void* d_positions,
                                   const double* d_inv_freq, void* d_q_out, const int32_t* d_info, void* stream) {
    const char* op = "cache_append";
    if (int rc = check_cache(op, c, true)) return rc;
    if (!a) return bad_value(op, "null argument");
    if (a->tokens < 0 || a->q_heads < 0) return bad_shape(op, "negative size");
    if (a->q_heads > 1 << 16 || c->kv_heads > 1 << 16 || a->tokens > 1 << 30) return bad_shape(op, "more than 2^30 tokens or 65536 heads");
    if (a->rotated < 0 || a->rotated % 2 || a->rotated > c->dim) return bad_shape(op, "rotated must be even, 0 .. dim");
    if (!within({a->q_token, a->q_head, a->k_token, a->k_head, a->v_token, a->v_head, a->out_token, a->out_head})) return bad_shape(op, "stride too large");
    if (!a->tokens) return DISCO_OK;
    if (!d_k || !d_v || !d_page_table || !d_lens || !d_cu_new || (a->q_heads && (!d_q || !d_q_out)) || (a->rotated && !d_inv_freq))
        return bad_value(op, "null argument");
    if (a->q_heads && d_q == d_q_out && (a->q_token != a->out_token || a->q_head != a->out_head)) return bad_value(op, "in place with other strides");
    return launch_cache_append(*c, *a, d_q, d_k, d_v, d_page_table, d_lens, d_cu_new, d_positions, d_inv_freq, d_q_out, d_info, (hipStream_t)stream);
}

static int check_attention(const char* op, const disco_cache_desc* c, const disco_attention_desc* a) {
    if (int rc = check_cache(op, c, true)) return rc;
    if (!a) return bad_value(op, "null argument");
    if (a->tokens < 0) return bad_shape(op, "negative size");
    if (!positive(op, {a->q_heads})) return DISCO_ESHAPE;
    if (c->kv_heads > 1024) return bad_shape(op, "more than 1024 key heads");
    if (a->q_heads % c->kv_heads) return bad_shape(op, "q_heads must be a multiple of kv_heads");
    if ((int64_t)a->tokens * a->q_heads > (1 << 30)) return bad_shape(op, "more than 2^30 rows");
    if (a->window < 0 || (a->window && !a->causal)) return bad_value(op, "a window needs causal attention");
    if (a->max_new < 0 || a->max_len < 0) return bad_value(op, "negative bound");
    if (!std::isfinite(a->scale)) return bad_value(op, "scale must be finite");
    if ((a->q_token | a->q_head | a->out_token | a->out_head) % 8) return bad_shape(op, "strides of q and out must be multiples of 8 elements");
    if (!within({a->q_token, a->q_head, a->out_token, a->out_head})) return bad_shape(op, "stride too large");
    return DISCO_OK;
}

int disco_op_cache_attention_workspace_bytes(const disco_cache_desc* c, const disco_attention_desc* a, size_t* bytes) {
    if (!bytes) return bad_value("cache_attention", "null argument");
    if (int rc = check_attention("cache_attention", c, a)) return rc;
    *bytes = a->tokens ? cache_attention_ws_bytes(*c, *a) : 0;
    return DISCO_OK;
}

static int attend(const disco_cache_desc* c, const disco_attention_desc* a, const void* d_q, const int32_t* d_page_table, const int32_t* d_lens,
                  const int32_t* d_cu_new, void* d_out, float* d_lse, void* d_ws, size_t ws_bytes, bool precise, void* stream) {
    const char* op = "cache_attention";
    if (int rc = check_attention(op, c, a)) return rc;
    if (!a->tokens) return DISCO_OK;
    if (!d_q || !d_page_table || !d_lens || !d_cu_new || !d_out) return bad_value(op, "null argument");
    if (((uintptr_t)d_q | (uintptr_t)d_out) % 16) return bad_value(op, "q and out must be aligned to 16 bytes");
    const size_t need = cache_attention_ws_bytes(*c, *a);
    if (need && (!d_ws || ws_bytes < need || (uintptr_t)d_ws % 16)) { set_error("%s: workspace too small or not aligned (%zu < %zu)", op, ws_bytes, need); return DISCO_ENOMEM; }
    if (d_q == d_out) return bad_value(op, "out may not be q");
    return launch_cache_attention(*c, *a, d_q, d_page_table, d_lens, d_cu_new, d_out, d_lse, d_ws, precise, (hipStream_t)stream);
}

int disco_op_cache_attention(const disco_cache_desc* c, const disco_attention_desc* a, const void* d_q, const int32_t* d_page_table,
                             const int32_t* d_lens, const int32_t* d_cu_new, void* d_out, float* d_lse, void* d_ws, size_t ws_bytes, void* stream) {
    return attend(c, a, d_q, d_page_table, d_lens, d_cu_new, d_out, d_lse, d_ws, ws_bytes, false, stream);
}

int disco_op_cache_attention_precise(const disco_cache_desc* c, const disco_attention_desc* a, const void* d_q, const int32_t* d_page_table,
                                     const int32_t* d_lens, const int32_t* d_cu_new, void* d_out, float* d_lse, void* d_ws, size_t ws_bytes, void* stream) {
    return attend(c, a, d_q, d_page_table, d_lens, d_cu_new, d_out, d_lse, d_ws, ws_bytes, true, stream);
}

int disco_op_cache_reserve(int rows, int table_width, int pages, int page_size, const int32_t* d_page_table, const int32_t* d_lens,
                           const int32_t* d_refs, const int32_t* d_cu_new, int32_t* d_page_table_out, int32_t* d_lens_out, int32_t* d_refs_out,
                           int32_t* d_info, void* stream) {
    const char* op = "cache_reserve";
    if (int rc = check_pages(op, rows, table_width, pages, page_size)) return rc;
    if (!d_page_table || !d_lens || !d_refs || !d_cu_new || !d_page_table_out || !d_lens_out || !d_refs_out || !d_info) return bad_value(op, "null argument");
    if (d_page_table == d_page_table_out || d_lens == d_lens_out || d_refs == d_refs_out) return bad_value(op, "the new state needs buffers of its own");
    return launch_cache_reserve(rows, table_width, pages, __builtin_ctz((unsigned)page_size), d_page_table, d_lens, d_refs, d_cu_new, d_page_table_out,
                                d_lens_out, d_refs_out, d_info, (hipStream_t)stream);
}

size_t disco_op_cache_pages_workspace_bytes(int rows, int pages) { return (rows > 0 && pages > 0) ? cache_pages_ws_bytes(rows, pages) : 0; }

int disco_op_cache_select(const disco_cache_desc* c, const int32_t* d_page_table, const int32_t* d_lens, const int32_t* d_parents,
                          int32_t* d_page_table_out, int32_t* d_lens_out, int32_t* d_refs_out, int32_t* d_info, void* d_ws, size_t ws_bytes,
                          void* stream) {
    const char* op = "cache_select";
    if (int rc = check_copied_cache(op, c)) return rc;
    if (!d_page_table || !d_lens || !d_parents || !d_page_table_out || !d_lens_out || !d_refs_out || !d_info || !d_ws) return bad_value(op, "null argument");
    if (d_page_table == d_page_table_out || d_lens == d_lens_out) return bad_value(op, "the new state needs buffers of its own");
    if (ws_bytes < cache_pages_ws_bytes(c->rows, c->pages) || (uintptr_t)d_ws % 16) { set_error("%s: workspace too small or not aligned", op); return DISCO_ENOMEM; }
    return launch_cache_select(*c, d_page_table, d_lens, d_parents, d_page_table_out, d_lens_out, d_refs_out, d_info, d_ws, (hipStream_t)stream);
}

int disco_op_cache_compact(const disco_cache_desc* c, const int32_t* d_page_table, const int32_t* d_lens, int32_t* d_page_table_out,
                           int32_t* d_refs_out, int32_t* d_info, void* d_ws, size_t ws_bytes, void* stream) {
    const char* op = "cache_compact";
    if (int rc = check_copied_cache(op, c)) return rc;
    if (!d_page_table || !d_lens || !d_page_table_out || !d_refs_out || !d_info || !d_ws) return bad_value(op, "null argument");
    if (d_page_table == d_page_table_out) return bad_value(op, "the new table needs a buffer of its own");
    if (ws_bytes < cache_pages_ws_bytes(c->rows, c->pages) || (uintptr_t)d_ws % 16) { set_error("%s: workspace too small or not aligned", op); return DISCO_ENOMEM; }
    return launch_cache_compact(*c, d_page_table, d_lens, d_page_table_out, d_refs_out, d_info, d_ws, (hipStream_t)stream);
}

int disco_op_cache_copy_pages(const disco_cache_desc* c, const int32_t* d_src, const int32_t* d_dst, int count, void* stream) {
    const char* op = "cache_copy_pages";
    if (int rc = check_copied_cache(op, c)) return rc;
    if (count < 0) return bad_shape(op, "negative count");
    if (!count) return DISCO_OK;
    if (!d_src || !d_dst) return bad_value(op, "null argument");
    return launch_cache_copy_pages(*c, d_src, d_dst, count, (hipStream_t)stream);
}

}  // extern "C"
