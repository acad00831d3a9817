// cache_pages.hip - the pages of a paged cache: taken for new tokens, shared and copied when sequences fork, moved together, copied.
//
// The bookkeeping is integer work on the page table (rows x width) and one count a page; it is bound by latency, so what matters is how few
// launches it takes.  The copies are bound by memory.  Every choice is the lowest number first, so that results do not depend on timing.
#include "paged.h"

namespace disco {

namespace {

constexpr int PLAN = 1024;         // threads of the one workgroup that plans
constexpr int WAVES = PLAN / 64;

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }
__device__ __forceinline__ unsigned long long lanes_below() { return (1ull << lane_id()) - 1; }

__device__ __forceinline__ int wave_scan(int v) {              // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d);
        if (lane_id() >= d) v += u;
    }
    return v;
}

// inclusive scan over the workgroup; *total in every thread.  `part`: WAVES words of LDS that nobody else uses
__device__ __forceinline__ int block_scan(int v, int* part, int* total) {
    const int w = threadIdx.x >> 6, in_wave = wave_scan(v);
    __syncthreads();
    if (lane_id() == 63) part[w] = in_wave;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        if (i < w) before += part[i];
        all += part[i];
    }
    *total = all;
    return before + in_wave;
}

__device__ __forceinline__ int pages_of(int len, int shift) { return (len + (1 << shift) - 1) >> shift; }

// counts that this workgroup (or an earlier launch) has changed by atomics: read where the atomics were done
__device__ __forceinline__ int count_now(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Calls f(page, rank) for the first `most` pages that `is` holds for, in ascending order, over [0, pages); returns how many there are.  Every wave
// has a run of pages: counts first, then ranks from ballots.
template <typename Is, typename F>
__device__ __forceinline__ int for_ranked(int pages, int most, int* part, Is is, F f) {
    const int w = threadIdx.x >> 6, run = ((pages + WAVES * 64 - 1) / (WAVES * 64)) * 64;
    const int from = w * run, to = min(pages, from + run);
    int mine = 0;
    for (int p = from; p < to; p += 64) {
        const int page = p + lane_id();
        mine += __popcll(__ballot(page < to && is(page)));
    }
    __syncthreads();
    if (lane_id() == 0) part[w] = mine;
    __syncthreads();
    int rank = 0, all = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        if (i < w) rank += part[i];
        all += part[i];
    }
    for (int p = from; p < to && rank < most; p += 64) {
        const int page = p + lane_id();
        const unsigned long long set = __ballot(page < to && is(page));
        const int r = rank + __popcll(set & lanes_below());
        if ((set >> lane_id() & 1) && r < most) f(page, r);
        rank += __popcll(set);
    }
    return all;
}

// ---- reserve ------------------------------------------------------------------------------------------------------------------------
// Block 0 plans: the rows' needs (scanned into LDS), the free pages in ascending order, each finding its row by bisection.  The other blocks copy the
// entries that every row has already; who writes an entry depends on the input alone, so nothing waits.
struct ReserveArgs {
    const int *table, *lens, *refs, *cu_new;
    int *table_out, *lens_out, *refs_out, *info;
    int rows, width, pages, shift;
};

__device__ __forceinline__ int reserve_new(const ReserveArgs& a, int r) {
    const int n = a.cu_new[r + 1] - a.cu_new[r];
    return n > 0 ? n : 0;
}

__global__ __launch_bounds__(PLAN) void cache_reserve_kernel(ReserveArgs a) {
    extern __shared__ int upto[];                                  // [rows]: pages that the rows up to and with this one need
    __shared__ int part[WAVES], over, bad;
    const int capacity = a.width << a.shift;
    if (blockIdx.x) {
        const long total = (long)a.rows * a.width, stride = (long)(gridDim.x - 1) * PLAN;
        for (long i = (long)(blockIdx.x - 1) * PLAN + threadIdx.x; i < total; i += stride) {
            const int r = (int)(i / a.width), at = (int)(i - (long)r * a.width);
            const int len = clamp_len(a.lens[r], capacity), have = pages_of(len, a.shift);
            const long want = ((long)len + reserve_new(a, r) + (1 << a.shift) - 1) >> a.shift;
            if (at < have) a.table_out[i] = a.table[i];
            else if (at >= want || want > a.width) a.table_out[i] = -1;            // (block 0 writes the others)
        }
        return;
    }
    if (threadIdx.x == 0) { over = 0; bad = 0; }
    int base = 0;
    for (int r0 = 0; r0 < a.rows; r0 += PLAN) {
        const int r = r0 + threadIdx.x;
        int need = 0, all;
        if (r < a.rows) {
            const int len = clamp_len(a.lens[r], capacity), have = pages_of(len, a.shift);
            const long want = ((long)len + reserve_new(a, r) + (1 << a.shift) - 1) >> a.shift;
            if (want > a.width) atomicAdd(&over, (int)(want - a.width < 1 << 24 ? want - a.width : 1 << 24));
            else need = (int)want - have;
            if (len != a.lens[r] || a.cu_new[r + 1] < a.cu_new[r]) atomicAdd(&bad, 1);
        }
        const int incl = block_scan(need, part, &all) + base;
        if (r < a.rows) upto[r] = incl;
        base += all;
    }
    __syncthreads();
    const int total = base, too_long = over;
    // free pages: first how many, then - if they suffice - who gets which
    const int free_pages = for_ranked(a.pages, 0, part, [&](int p) { return a.refs[p] == 0; }, [](int, int) {});
    const bool done = total <= free_pages && too_long == 0;
    for_ranked(a.pages, done ? total : 0, part, [&](int p) { return a.refs[p] == 0; }, [&](int page, int rank) {
        int lo = 0, hi = a.rows - 1;                               // the first row with upto > rank
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (upto[mid] > rank) hi = mid; else lo = mid + 1;
        }
        const int have = pages_of(clamp_len(a.lens[lo], capacity), a.shift);
        a.table_out[(long)lo * a.width + have + rank - (lo ? upto[lo - 1] : 0)] = page;
        a.refs_out[page] = 1;
    });
    // (a page taken is the only one whose count changes; the others are copied by whoever sees them taken or not)
    int rank = 0;
    {
        const int w = threadIdx.x >> 6, run = ((a.pages + WAVES * 64 - 1) / (WAVES * 64)) * 64, from = w * run, to = min(a.pages, from + run);
#pragma unroll
        for (int i = 0; i < WAVES; ++i) if (i < w) rank += part[i];
        for (int p = from; p < to; p += 64) {
            const int page = p + lane_id(), refs = page < to ? a.refs[page] : 1;
            const unsigned long long set = __ballot(refs == 0);
            const bool taken = done && refs == 0 && rank + __popcll(set & lanes_below()) < total;
            if (page < to && !taken) a.refs_out[page] = refs;
            rank += __popcll(set);
        }
    }
    for (int r = threadIdx.x; r < a.rows; r += PLAN) {
        const int len = clamp_len(a.lens[r], capacity);
        a.lens_out[r] = done ? len + reserve_new(a, r) : len;
        if (!done) {                                               // the entries that the other blocks left
            const int have = pages_of(len, a.shift);
            const long want = ((long)len + reserve_new(a, r) + (1 << a.shift) - 1) >> a.shift;
            if (want <= a.width) for (int at = have; at < want; ++at) a.table_out[(long)r * a.width + at] = -1;
        }
    }
    if (threadIdx.x == 0) {
        a.info[0] = done ? free_pages - total : free_pages;
        a.info[1] = done ? 0 : max(total - free_pages, 0) + too_long;
        a.info[2] = bad;
        a.info[3] = 0;
    }
}

// ---- pieces of select and compact ------------------------------------------------------------------------------------------------------
__global__ void clear_kernel(int* p, int n, int* q, int m) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    for (int j = i; j < n; j += gridDim.x * blockDim.x) p[j] = 0;
    if (i < m) q[i] = 0;
}

// a copy of pages: src -> dst, the first `filled` slots
struct Copy { int src, dst, filled; };

struct PlanArgs {
    const int *table, *lens, *parents;                             // parents: select only
    int *table_out, *lens_out, *refs, *refs_out, *info;
    Copy* copies; int* copy_count;
    int* map;                                                      // compact: where a page goes
    int* bad;
    int rows, width, pages, shift;
};

// the row that row r becomes, -1: none
__device__ __forceinline__ int parent_of(const PlanArgs& a, int r) {
    const int p = a.parents[r];
    return p >= 0 && p < a.rows ? p : -1;
}

// select: the rows, gathered; counts of the pages that are full (a last page that is not is counted by the plan)
// compact: counts of all pages
template <bool SELECT>
__global__ __launch_bounds__(256) void cache_count_kernel(PlanArgs a) {
    const int capacity = a.width << a.shift;
    const long total = (long)a.rows * a.width, stride = (long)gridDim.x * 256;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const int r = (int)(i / a.width), at = (int)(i - (long)r * a.width);
        const int from = SELECT ? parent_of(a, r) : r;
        const int len = from < 0 ? 0 : clamp_len(a.lens[from], capacity);
        int page = -1;
        if (at < pages_of(len, a.shift)) {
            page = a.table[(long)from * a.width + at];
            if (page < 0 || page >= a.pages) atomicAdd(a.bad, 1);
            else if (!SELECT || (at + 1) << a.shift <= len) atomicAdd(&a.refs[page], 1);
        }
        if (SELECT) a.table_out[i] = page;
        if (at == 0 && from >= 0 && len != a.lens[from]) atomicAdd(a.bad, 1);
        if (SELECT && at == 0 && from != a.parents[r]) {           // a parent that is no row (-1 says none)
            if (a.parents[r] != -1) atomicAdd(a.bad, 1);
        }
    }
}

__global__ __launch_bounds__(PLAN) void cache_select_plan_kernel(PlanArgs a) {
    extern __shared__ int keeper[];                                // [rows]: which of a parent's rows keeps its last page
    __shared__ int part[WAVES];
    const int capacity = a.width << a.shift, tid = threadIdx.x;
    for (int r = tid; r < a.rows; r += PLAN) keeper[r] = 1 << 30;
    __syncthreads();
    for (int r = tid; r < a.rows; r += PLAN) {
        const int p = parent_of(a, r);
        if (p >= 0) atomicMin(&keeper[p], p == r ? -1 : r);
    }
    __syncthreads();
    // the kept last pages are in use as well
    auto tail_of = [&](int r, int& len) {                          // the table index of row r's last page if it is not full, else -1
        const int p = parent_of(a, r);
        len = p < 0 ? 0 : clamp_len(a.lens[p], capacity);
        return len & ((1 << a.shift) - 1) ? (long)r * a.width + (len >> a.shift) : -1l;
    };
    auto keeps = [&](int r) { const int p = parent_of(a, r); return keeper[p] == (p == r ? -1 : r); };
    for (int r = tid; r < a.rows; r += PLAN) {
        int len;
        const long t = tail_of(r, len);
        if (t >= 0 && keeps(r)) {
            const int page = a.table_out[t];
            if (page >= 0 && page < a.pages) atomicAdd(&a.refs_out[page], 1);
        }
    }
    __threadfence();
    __syncthreads();
    const int free_pages = for_ranked(a.pages, 0, part, [&](int p) { return count_now(&a.refs_out[p]) == 0; }, [](int, int) {});
    // the rows that need a copy, ascending; their number first
    int need_total = 0;
    for (int r0 = 0; r0 < a.rows; r0 += PLAN) {
        const int r = r0 + tid;
        int len, all;
        const bool need = r < a.rows && tail_of(r, len) >= 0 && !keeps(r);
        const int rank = need_total + block_scan(need, part, &all) - 1;
        if (need) {
            a.copies[rank].src = r;                                // (the row for now)
            a.copies[rank].filled = len & ((1 << a.shift) - 1);
        }
        need_total += all;
    }
    __threadfence();
    __syncthreads();
    const bool done = need_total <= free_pages;
    if (done) {
        for_ranked(a.pages, need_total, part, [&](int p) { return count_now(&a.refs_out[p]) == 0; }, [&](int page, int rank) {
            a.copies[rank].dst = page;
        });
        __threadfence();
        __syncthreads();
        for (int i = tid; i < need_total; i += PLAN) {
            const int r = __hip_atomic_load(&a.copies[i].src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const int page = __hip_atomic_load(&a.copies[i].dst, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            int len;
            const long t = tail_of(r, len);
            a.copies[i].src = a.table_out[t];                      // (one outside the cache is left out by the copy)
            a.table_out[t] = page;
            a.refs_out[page] = 1;
        }
        for (int r = tid; r < a.rows; r += PLAN) {
            const int p = parent_of(a, r);
            a.lens_out[r] = p < 0 ? 0 : clamp_len(a.lens[p], capacity);
        }
    } else {                                                       // too few free pages: the old state once more
        for (int p = tid; p < a.pages; p += PLAN) a.refs_out[p] = 0;
        __threadfence();
        __syncthreads();
        for (long i = tid; i < (long)a.rows * a.width; i += PLAN) {
            const int r = (int)(i / a.width), at = (int)(i - (long)r * a.width);
            const int page = at < pages_of(clamp_len(a.lens[r], capacity), a.shift) ? a.table[i] : -1;
            a.table_out[i] = page;
            if (page >= 0 && page < a.pages) atomicAdd(&a.refs_out[page], 1);
        }
        for (int r = tid; r < a.rows; r += PLAN) a.lens_out[r] = clamp_len(a.lens[r], capacity);
        __threadfence();
        __syncthreads();
    }
    int left = 0;
    if (!done) left = for_ranked(a.pages, 0, part, [&](int p) { return count_now(&a.refs_out[p]) == 0; }, [](int, int) {});
    if (tid == 0) {
        *a.copy_count = done ? need_total : 0;
        a.info[0] = done ? free_pages - need_total : left;
        a.info[1] = done ? 0 : need_total - free_pages;
        a.info[2] = *a.bad;
        a.info[3] = done ? need_total : 0;
    }
}

__global__ __launch_bounds__(PLAN) void cache_compact_plan_kernel(PlanArgs a) {
    __shared__ int part[WAVES];
    const int tid = threadIdx.x, pages = a.pages;
    const int live = for_ranked(pages, 0, part, [&](int p) { return a.refs[p] > 0; }, [](int, int) {});
    const int moved = for_ranked(live, live, part, [&](int p) { return a.refs[p] == 0; }, [&](int page, int rank) {
        a.copies[rank].dst = page;
        a.copies[rank].filled = 1 << a.shift;
    });
    for_ranked(pages, pages, part, [&](int p) { return p >= live && a.refs[p] > 0; }, [&](int page, int rank) { a.copies[rank].src = page; });
    for (int p = tid; p < pages; p += PLAN) if (p >= live || a.refs[p] > 0) a.refs_out[p] = p < live ? a.refs[p] : 0;
    for (int p = tid; p < live; p += PLAN) a.map[p] = p;
    __threadfence();
    __syncthreads();
    for (int i = tid; i < moved; i += PLAN) {
        const int src = __hip_atomic_load(&a.copies[i].src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int dst = __hip_atomic_load(&a.copies[i].dst, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        a.map[src] = dst;
        a.refs_out[dst] = a.refs[src];
    }
    if (tid == 0) {
        *a.copy_count = moved;
        a.info[0] = pages - live;
        a.info[1] = 0;
        a.info[2] = *a.bad;
        a.info[3] = moved;
    }
}

// ---- copies, and the compacted table --------------------------------------------------------------------------------------------------
struct CopyArgs {
    char *k, *v;
    const Copy* copies; const int* count;                          // or
    const int *src, *dst; int given;                               // page lists of the caller
    long layer_stride, page_stride, head_stride, slot_stride;      // bytes
    int layers, heads, dim, page_size, pages;                      // dim: 16-byte pieces
    const int *table, *lens, *map; int* table_out;                 // compact: the table is rewritten on the way
    int rows, width, shift;
};

// One wave copies the filled slots of one head of a page; every 16 bytes once in, once out: bound by memory
__global__ __launch_bounds__(256) void cache_copy_kernel(CopyArgs a) {
    if (a.table) {
        const int capacity = a.width << a.shift;
        const long total = (long)a.rows * a.width;
        for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
            const int r = (int)(i / a.width), at = (int)(i - (long)r * a.width);
            int page = -1;
            if (at < pages_of(clamp_len(a.lens[r], capacity), a.shift)) {
                page = a.table[i];
                if (page >= 0 && page < a.pages) page = a.map[page];
            }
            a.table_out[i] = page;
        }
    }
    const int lane = threadIdx.x & 63;
    const long units = (long)(a.copies ? *a.count : a.given) * a.layers * 2 * a.heads, waves = (long)gridDim.x * 4;
    for (long u = (long)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += waves) {
        const int h = (int)(u % a.heads);
        const long rest = u / a.heads;
        const int side = (int)(rest & 1), layer = (int)((rest >> 1) % a.layers);
        const long i = (rest >> 1) / a.layers;
        const int src = a.copies ? a.copies[i].src : a.src[i], dst = a.copies ? a.copies[i].dst : a.dst[i];
        const int filled = a.copies ? a.copies[i].filled : a.page_size;
        if (src < 0 || src >= a.pages || dst < 0 || dst >= a.pages) continue;
        char* base = (side ? a.v : a.k) + layer * a.layer_stride + h * a.head_stride;
        const char* from = base + src * a.page_stride;
        char* to = base + dst * a.page_stride;
        for (int x = lane; x < filled * a.dim; x += 64) {
            const int slot = x / a.dim;
            const long at = slot * a.slot_stride + (long)(x - slot * a.dim) * 16;
            *(uint4*)(to + at) = *(const uint4*)(from + at);
        }
    }
}

int run_copy(CopyArgs& a, const disco_cache_desc& c, long most, hipStream_t s) {
    a.k = (char*)c.d_k; a.v = (char*)c.d_v;
    a.layer_stride = c.layer_stride * 2; a.page_stride = c.page_stride * 2; a.head_stride = c.head_stride * 2; a.slot_stride = c.slot_stride * 2;
    a.layers = c.layers; a.heads = c.kv_heads; a.dim = c.dim / 8; a.page_size = c.page_size; a.pages = c.pages;
    const long units = most * c.layers * 2 * c.kv_heads;
    const long blocks = units / 4 + 1;
    cache_copy_kernel<<<(unsigned)(blocks < 2048 ? blocks : 2048), 256, 0, s>>>(a);
    DISCO_LAUNCH_CHECK("cache_copy_kernel");
    return DISCO_OK;
}

int blocks_for(long items, int threads, int most) {
    const long b = (items + threads - 1) / threads;
    return (int)(b < 1 ? 1 : (b < most ? b : most));
}

// LDS beyond 64 KB has to be asked for (once a device)
template <typename K>
int allow_lds(K kernel, size_t bytes) {
    DISCO_HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return DISCO_OK;
}

struct Scratch { Copy* copies; int *count, *bad, *map, *refs; };

Scratch scratch(void* ws, int pages) {
    int* p = (int*)ws;
    Scratch s;
    s.bad = p; s.count = p + 1;
    s.refs = p + 4;
    s.map = s.refs + pages;
    s.copies = (Copy*)(s.map + pages);
    return s;
}

}  // namespace

size_t cache_pages_ws_bytes(int rows, int pages) {
    const size_t copies = (size_t)(rows > pages ? rows : pages);
    return 16 + 8 * (size_t)pages + sizeof(Copy) * copies;
}

int launch_cache_reserve(int rows, int width, int pages, int page_shift, const int* table, const int* lens, const int* refs, const int* cu_new,
                         int* table_out, int* lens_out, int* refs_out, int* info, hipStream_t s) {
    ReserveArgs a{table, lens, refs, cu_new, table_out, lens_out, refs_out, info, rows, width, pages, page_shift};
    const size_t lds = (size_t)rows * 4;
    if (lds > 32768) if (int rc = allow_lds(cache_reserve_kernel, lds)) return rc;
    cache_reserve_kernel<<<1 + blocks_for((long)rows * width, PLAN * 4, 256), PLAN, lds, s>>>(a);
    DISCO_LAUNCH_CHECK("cache_reserve_kernel");
    return DISCO_OK;
}

int launch_cache_select(const disco_cache_desc& c, const int* table, const int* lens, const int* parents, int* table_out, int* lens_out,
                        int* refs_out, int* info, void* ws, hipStream_t s) {
    const Scratch w = scratch(ws, c.pages);
    PlanArgs a{table, lens, parents, table_out, lens_out, refs_out, refs_out, info, w.copies, w.count, w.map, w.bad, c.rows, c.table_width, c.pages,
               __builtin_ctz((unsigned)c.page_size)};
    const size_t lds = (size_t)c.rows * 4;
    if (lds > 32768) if (int rc = allow_lds(cache_select_plan_kernel, lds)) return rc;
    clear_kernel<<<blocks_for(c.pages, 256, 256), 256, 0, s>>>(refs_out, c.pages, w.bad, 2);
    cache_count_kernel<true><<<blocks_for((long)c.rows * c.table_width, 256, 1024), 256, 0, s>>>(a);
    cache_select_plan_kernel<<<1, PLAN, lds, s>>>(a);
    DISCO_LAUNCH_CHECK("cache_select_plan_kernel");
    CopyArgs p{};
    p.copies = w.copies; p.count = w.count;
    return run_copy(p, c, c.rows, s);
}

int launch_cache_compact(const disco_cache_desc& c, const int* table, const int* lens, int* table_out, int* refs_out, int* info, void* ws,
                         hipStream_t s) {
    const Scratch w = scratch(ws, c.pages);
    PlanArgs a{table, lens, nullptr, table_out, nullptr, w.refs, refs_out, info, w.copies, w.count, w.map, w.bad, c.rows, c.table_width, c.pages,
               __builtin_ctz((unsigned)c.page_size)};
    clear_kernel<<<blocks_for(c.pages, 256, 256), 256, 0, s>>>(w.refs, c.pages, w.bad, 2);
    cache_count_kernel<false><<<blocks_for((long)c.rows * c.table_width, 256, 1024), 256, 0, s>>>(a);
    cache_compact_plan_kernel<<<1, PLAN, 0, s>>>(a);
    DISCO_LAUNCH_CHECK("cache_compact_plan_kernel");
    CopyArgs p{};
    p.copies = w.copies; p.count = w.count;
    p.table = table; p.lens = lens; p.map = w.map; p.table_out = table_out;
    p.rows = c.rows; p.width = c.table_width; p.shift = __builtin_ctz((unsigned)c.page_size);
    return run_copy(p, c, c.pages / 2 + 1, s);
}

int launch_cache_copy_pages(const disco_cache_desc& c, const int* src, const int* dst, int count, hipStream_t s) {
    CopyArgs p{};
    p.src = src; p.dst = dst; p.given = count;
    return run_copy(p, c, count, s);
}

}  // namespace disco
