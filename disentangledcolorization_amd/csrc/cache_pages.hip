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

// Looks at every page once, in runs of a wave each: calls look(page) -> bool, then - when all threads know how many pages it holds for - then(total), and then
// rank(page, it held, how many pages below it held).  Four loads of a lane under way at a time; what look said is kept in a register where a run is
// no longer than 4096 pages.  Returns the total.
template <typename Look, typename Then, typename Rank>
__device__ __forceinline__ int scan_pages(int pages, int* part, Look look, Then then, Rank rank) {
    const int w = threadIdx.x >> 6, run = ((pages + WAVES * 64 - 1) / (WAVES * 64)) * 64;
    const int from = min(pages, w * run), to = min(pages, from + run), steps = (to - from + 63) / 64;
    const bool kept = steps <= 64;
    unsigned long long bits = 0;
    int mine = 0;
    for (int i = 0; i < steps; i += 4) {
        bool set[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int page = from + (i + j) * 64 + lane_id();
            set[j] = page < to && look(page);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mine += __popcll(__ballot(set[j]));
            if (kept && set[j]) bits |= 1ull << ((i + j) & 63);
        }
    }
    __syncthreads();
    if (lane_id() == 0) part[w] = mine;
    __syncthreads();
    int below = 0, all = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        if (i < w) below += part[i];
        all += part[i];
    }
    then(all);
    for (int i = 0; i < steps; ++i) {
        const int page = from + i * 64 + lane_id();
        const bool set = page < to && (kept ? bits >> i & 1 : look(page));
        const unsigned long long here = __ballot(set);
        if (page < to) rank(page, set, below + __popcll(here & lanes_below()));
        below += __popcll(here);
    }
    return all;
}

// ---- reserve ------------------------------------------------------------------------------------------------------------------------
// Block 0 plans: the rows' needs (scanned into LDS), the free pages in ascending order, each finding its row by bisection.  The other blocks copy the
// entries that every row has already; who writes an entry depends on the input alone, so nothing waits.  Bound by latency: one launch of 5 us (five rows
// that take 80 pages each) to 8 (64 that take a token each, over tables of 4 096 tokens).
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
    __shared__ int part[WAVES], bad, shared;
    __shared__ unsigned long long over;                            // pages beyond the table's width
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
    if (threadIdx.x == 0) { over = 0; bad = 0; shared = 0; }
    __syncthreads();                                               // (every wave counts into them)
    int base = 0;
    for (int r0 = 0; r0 < a.rows; r0 += PLAN) {
        const int r = r0 + threadIdx.x;
        int need = 0, all;
        if (r < a.rows) {
            const int len = clamp_len(a.lens[r], capacity), have = pages_of(len, a.shift);
            const long want = ((long)len + reserve_new(a, r) + (1 << a.shift) - 1) >> a.shift;
            if (want > a.width) atomicAdd(&over, (unsigned long long)(want - a.width));
            else need = (int)want - have;
            if (len != a.lens[r] || a.cu_new[r + 1] < a.cu_new[r]) atomicAdd(&bad, 1);
            if (len & ((1 << a.shift) - 1) && reserve_new(a, r)) { // the first new token goes into a page that is there: no other row may name it
                const int page = a.table[(long)r * a.width + (len >> a.shift)];
                if (page >= 0 && page < a.pages && a.refs[page] > 1) atomicAdd(&shared, 1);
            }
        }
        const int incl = block_scan(need, part, &all) + base;
        if (r < a.rows) upto[r] = incl;
        base += all;
    }
    __syncthreads();
    const int total = base;
    const unsigned long long short_of = over + shared;
    bool done = false;
    const int free_pages = scan_pages(a.pages, part,
        [&](int p) {
            const int refs = a.refs[p];
            a.refs_out[p] = refs;
            return refs == 0;
        },
        [&](int free) { done = total <= free && short_of == 0; },
        [&](int page, bool free, int rank) {
            if (!free || !done || rank >= total) return;
            int lo = 0, hi = a.rows - 1;                           // the first row with upto > rank
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (upto[mid] > rank) hi = mid; else lo = mid + 1;
            }
            const int have = pages_of(clamp_len(a.lens[lo], capacity), a.shift);
            a.table_out[(long)lo * a.width + have + rank - (lo ? upto[lo - 1] : 0)] = page;
            a.refs_out[page] = 1;
        });
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
        const unsigned long long missing = max(total - free_pages, 0) + short_of;
        a.info[1] = done ? 0 : (int)(missing < 0x7fffffff ? missing : 0x7fffffff);
        a.info[2] = bad;
        a.info[3] = shared;
    }
}

// ---- pieces of select and compact ------------------------------------------------------------------------------------------------------
// A plan of one workgroup (new table, counts, a list of copies), then the copies.  A plan is a chain of passes over the table and the pages with the
// workgroup's barriers between them: 13 us for 64 rows of 63 entries over 2 400 pages, 15 us for the compaction of 32 rows over 3 200.
__global__ void clear_kernel(int* p, int n, int* q, int m) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    for (int j = i; j < n; j += gridDim.x * blockDim.x) p[j] = 0;
    if (i < m) q[i] = 0;
}

// a copy of pages: src -> dst, the first `filled` slots; `extra`: the plan's own
struct Copy { int src, dst, filled, extra; };

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

// How many rows name each page.  LOCAL: in LDS, for tables and pools that one workgroup looks through while two more launches would only start.
template <bool LOCAL> struct Counts {
    int* at;
    __device__ __forceinline__ int get(int p) const { return LOCAL ? at[p] : count_now(at + p); }
    __device__ __forceinline__ void add(int p) const { atomicAdd(at + p, 1); }
    __device__ __forceinline__ void lower(int p, int n) const { atomicMin(at + p, n); }
    __device__ __forceinline__ void set(int p, int n) const {
        if (LOCAL) at[p] = n;
        else __hip_atomic_store(at + p, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
};
// what one thread of the workgroup wrote is there for the others
__device__ __forceinline__ void settle() {
    __threadfence();
    __syncthreads();
}

// entry `at` of row r, SELECT: of the gathered rows.  Counts pages (select: those that are full; a last page that is not is counted by the plan), and what
// is out of range
template <bool SELECT, bool LOCAL>
__device__ __forceinline__ void count_entry(const PlanArgs& a, Counts<LOCAL> counts, int* bad, int r, int at) {
    const int from = SELECT ? parent_of(a, r) : r;
    const int given = from < 0 ? 0 : a.lens[from], len = clamp_len(given, a.width << a.shift);
    int page = -1;
    if (at < pages_of(len, a.shift)) {
        page = a.table[(long)from * a.width + at];
        if (page < 0 || page >= a.pages) atomicAdd(bad, 1);
        else if (!SELECT || (at + 1) << a.shift <= len) counts.add(page);
    }
    if (SELECT) a.table_out[(long)r * a.width + at] = page;
    if (at == 0 && given != len) atomicAdd(bad, 1);
    if (SELECT && at == 0 && from < 0 && a.parents[r] != -1) atomicAdd(bad, 1);       // a parent that is no row
}

template <bool SELECT>
__global__ __launch_bounds__(256) void cache_count_kernel(PlanArgs a) {
    const long total = (long)a.rows * a.width, stride = (long)gridDim.x * 256;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const int r = (int)(i / a.width);
        count_entry<SELECT, false>(a, Counts<false>{a.refs}, a.bad, r, (int)(i - (long)r * a.width));
    }
}

// the same by the planning workgroup, a wave a row
template <bool SELECT>
__device__ __forceinline__ void count_here(const PlanArgs& a, Counts<true> counts, int* bad) {
    for (int p = threadIdx.x; p < a.pages; p += PLAN) counts.at[p] = 0;
    __syncthreads();
    for (int r = threadIdx.x >> 6; r < a.rows; r += WAVES)
        for (int at = lane_id(); at < a.width; at += 64) count_entry<SELECT, true>(a, counts, bad, r, at);
    settle();
}

template <bool LOCAL>
__global__ __launch_bounds__(PLAN) void cache_select_plan_kernel(PlanArgs a) {
    extern __shared__ int keeper[];                                // [rows]: which of a parent's rows keeps its last page; LOCAL: [pages] counts
    __shared__ int part[WAVES], bad;
    const int capacity = a.width << a.shift, tid = threadIdx.x;
    const Counts<LOCAL> counts{LOCAL ? keeper + a.rows : a.refs_out};
    if (tid == 0) bad = LOCAL ? 0 : *a.bad;
    for (int r = tid; r < a.rows; r += PLAN) keeper[r] = 1 << 30;
    // what row r becomes: its parent, its length, how much of a last page that is not full, and that page (the thread's first row is looked up once)
    struct Last { int parent, len, filled, page; };
    auto last_of = [&](int r) {
        Last x{r < a.rows ? parent_of(a, r) : -1, 0, 0, -1};
        if (x.parent >= 0) x.len = clamp_len(a.lens[x.parent], capacity);
        x.filled = x.len & ((1 << a.shift) - 1);
        if (x.filled) x.page = a.table[(long)x.parent * a.width + (x.len >> a.shift)];
        return x;
    };
    const Last first = last_of(tid);
    __syncthreads();
    if constexpr (LOCAL) count_here<true>(a, counts, &bad);
    for (int r = tid; r < a.rows; r += PLAN) {
        const int p = parent_of(a, r);
        if (p >= 0) atomicMin(&keeper[p], p == r ? -1 : r);
    }
    __syncthreads();
    // Last pages that are not full.  The rows that end in one ask for it, below 0 in its count; a row that is its own parent goes first, then the lowest.
    // A page that is full for some row (whose neighbours have been cut back into it) has a count and stays that row's: all that end in it need copies.
    auto asked = [&](int r, int p) { return (p == r ? r : a.rows + r) - (1 << 30); };
    for (int r = tid; r < a.rows; r += PLAN) {
        const Last x = r == tid ? first : last_of(r);
        if (x.filled && x.page >= 0 && x.page < a.pages && counts.get(x.page) <= 0) counts.lower(x.page, asked(r, x.parent));
    }
    if (LOCAL) __syncthreads();
    else settle();
    // the keeper's is in use, the others need copies, numbered by row
    int need = 0;
    for (int r0 = 0; r0 < a.rows; r0 += PLAN) {
        const int r = r0 + tid;
        const Last x = r0 ? last_of(r) : first;
        bool keeps = x.parent >= 0 && keeper[x.parent] == (x.parent == r ? -1 : r);     // (of a page outside the cache)
        if (x.filled && x.page >= 0 && x.page < a.pages) {
            keeps = counts.get(x.page) == asked(r, x.parent);      // (who finds 1 there comes behind the keeper)
            if (keeps) counts.set(x.page, 1);
        }
        int all;
        const bool asks = x.filled && !keeps;
        const int rank = need + block_scan(asks, part, &all) - 1;
        if (asks) a.copies[rank] = Copy{x.page, -1, x.filled, r};  // (a page outside the cache is left out by the copy)
        if (r < a.rows) a.lens_out[r] = x.len;
        need += all;
    }
    settle();
    bool done = false;
    int free_pages = scan_pages(a.pages, part, [&](int p) { return counts.get(p) == 0; }, [&](int free) { done = need <= free; },
        [&](int page, bool free, int rank) {
            if (!free || !done || rank >= need) return;
            Copy* c = a.copies + rank;
            const int r = __hip_atomic_load(&c->extra, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            c->dst = page;
            a.table_out[(long)r * a.width + (clamp_len(a.lens[parent_of(a, r)], capacity) >> a.shift)] = page;
            counts.set(page, 1);
        });
    if (!done) {                                                   // too few free pages: the old state once more
        const int missing = need - free_pages;
        __syncthreads();
        for (int p = tid; p < a.pages; p += PLAN) counts.set(p, 0);
        settle();
        for (int r = tid >> 6; r < a.rows; r += WAVES) {
            const int len = clamp_len(a.lens[r], capacity);
            for (int at = lane_id(); at < a.width; at += 64) {
                const int page = at < pages_of(len, a.shift) ? a.table[(long)r * a.width + at] : -1;
                a.table_out[(long)r * a.width + at] = page;
                if (page >= 0 && page < a.pages) counts.add(page);
            }
            if (lane_id() == 0) a.lens_out[r] = len;
        }
        settle();
        free_pages = scan_pages(a.pages, part, [&](int p) { return counts.get(p) == 0; }, [](int) {}, [](int, bool, int) {});
        if (tid == 0) a.info[1] = missing;
    }
    if (LOCAL) {
        __syncthreads();
        for (int p = tid; p < a.pages; p += PLAN) a.refs_out[p] = counts.get(p);
    }
    if (tid == 0) {
        *a.copy_count = done ? need : 0;
        a.info[0] = done ? free_pages - need : free_pages;
        if (done) a.info[1] = 0;
        a.info[2] = bad;
        a.info[3] = done ? need : 0;
    }
}

template <bool LOCAL>
__global__ __launch_bounds__(PLAN) void cache_compact_plan_kernel(PlanArgs a) {
    extern __shared__ int counted[];                               // LOCAL: [pages] counts
    __shared__ int part[WAVES], bad, kept;
    const int tid = threadIdx.x, pages = a.pages;
    const Counts<LOCAL> counts{LOCAL ? counted : a.refs};
    if (tid == 0) bad = LOCAL ? 0 : *a.bad;
    __syncthreads();
    if constexpr (LOCAL) count_here<false>(a, counts, &bad);
    // of the `live` pages in use, those from `live` on move into the holes below it: `kept` pages in use lie below
    int live = 0;
    scan_pages(pages, part, [&](int p) { return counts.get(p) > 0; },
        [&](int total) {
            live = total;
            if (tid == 0) kept = total;                            // (when no page lies at or above it)
            __syncthreads();
        },
        [&](int page, bool used, int below) {
            if (page == live) kept = below;
            if (page < live) a.map[page] = page;
            if (used && page >= live) a.copies[below].extra = page;
            if (!used && page < live) a.copies[page - below].dst = page;
            if (used || page >= live) a.refs_out[page] = page < live ? counts.get(page) : 0;
        });
    settle();
    const int moved = live - kept;
    for (int i = tid; i < moved; i += PLAN) {
        const int src = __hip_atomic_load(&a.copies[kept + i].extra, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int dst = __hip_atomic_load(&a.copies[i].dst, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        a.copies[i].src = src;
        a.copies[i].filled = 1 << a.shift;
        a.map[src] = dst;
        a.refs_out[dst] = counts.get(src);
    }
    if (tid == 0) {
        *a.copy_count = moved;
        a.info[0] = pages - live;
        a.info[1] = 0;
        a.info[2] = bad;
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

// One wave copies the filled slots of one head of a page; every 16 bytes once in, once out: bound by memory (409 MB in and out: 80 us, 5.1 TB/s, what a large
// copy reaches)
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

// Tables of up to 64 K entries over up to 32 K pages (and 4 K rows: 144 KB of LDS): one workgroup counts while it plans (64 beams: 17 us a call, with two
// more launches 24); beyond, its passes over the table would take longer than the launches
bool local(const disco_cache_desc& c) { return (long)c.rows * c.table_width <= 65536 && c.pages <= 32768 && c.rows <= 4096; }

struct Scratch { Copy* copies; int *count, *bad, *map, *refs; };

Scratch scratch(void* ws, int pages) {
    int* p = (int*)ws;
    Scratch s;
    s.bad = p; s.count = p + 1;
    s.refs = p + 4;
    s.map = s.refs + pages;
    s.copies = (Copy*)((char*)s.refs + (8 * (size_t)pages + 15) / 16 * 16);
    return s;
}

}  // namespace

size_t cache_pages_ws_bytes(int rows, int pages) {
    const size_t copies = (size_t)(rows > pages ? rows : pages);
    return 16 + (8 * (size_t)pages + 15) / 16 * 16 + sizeof(Copy) * copies;
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
    const size_t lds = ((size_t)c.rows + (local(c) ? c.pages : 0)) * 4;
    if (local(c)) {
        if (lds > 32768) if (int rc = allow_lds(cache_select_plan_kernel<true>, lds)) return rc;
        cache_select_plan_kernel<true><<<1, PLAN, lds, s>>>(a);
    } else {
        if (lds > 32768) if (int rc = allow_lds(cache_select_plan_kernel<false>, lds)) return rc;
        clear_kernel<<<blocks_for(c.pages, 256, 256), 256, 0, s>>>(refs_out, c.pages, w.bad, 2);
        cache_count_kernel<true><<<blocks_for((long)c.rows * c.table_width, 256, 1024), 256, 0, s>>>(a);
        cache_select_plan_kernel<false><<<1, PLAN, lds, s>>>(a);
    }
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
    if (local(c)) {
        const size_t lds = (size_t)c.pages * 4;
        if (lds > 32768) if (int rc = allow_lds(cache_compact_plan_kernel<true>, lds)) return rc;
        cache_compact_plan_kernel<true><<<1, PLAN, lds, s>>>(a);
    } else {
        clear_kernel<<<blocks_for(c.pages, 256, 256), 256, 0, s>>>(w.refs, c.pages, w.bad, 2);
        cache_count_kernel<false><<<blocks_for((long)c.rows * c.table_width, 256, 1024), 256, 0, s>>>(a);
        cache_compact_plan_kernel<false><<<1, PLAN, 0, s>>>(a);
    }
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
