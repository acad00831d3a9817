// rotary.hip - positions as rotations of pairs of a head's elements, alone and on the way into a paged cache.
//
//   (a, b) -> g (a cos t - b sin t, a sin t + b cos t),   t = position * f_i
//
// Memory-bound: every element is read once and written once.  The angle is what needs care: at position 10^6 an fp32 product is off by
// 0.06 rad, so t / 2 pi is formed in fp64 and only its fraction is kept, as 32 bits of a turn (6e-10 rad); sine and cosine are then Taylor sums
// over [-pi/4, pi/4] in fp32 (next term below 3e-8).  That is ~45 instructions a pair, so a lane computes its angles once and
// uses them for several heads of one token; a wave handles one token (or a slice of its heads where tokens are few).
#include <type_traits>
#include "paged.h"

namespace disco {

namespace {

template <typename T> __device__ __forceinline__ float widen(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T narrow(float x) { return (T)x; }

// cos and sin of 2 pi p / 2^32
__device__ __forceinline__ void turn_sincos(uint32_t p, float& c, float& s) {
    const uint32_t quad = (p + 0x20000000u) >> 30;                 // the nearest quarter turn
    const float x = (float)(int32_t)(p - (quad << 30)) * 1.46291807926715968e-9f;     // 2 pi / 2^32: within +-pi/4
    const float y = x * x;
    float ps = fmaf(y, 2.75573192e-6f, -1.98412698e-4f);           // 1/9!, 1/7!, ...
    ps = fmaf(y, ps, 8.33333333e-3f);
    ps = fmaf(y, ps, -1.66666667e-1f);
    const float sx = fmaf(x * y, ps, x);
    float pc = fmaf(y, -2.75573192e-7f, 2.48015873e-5f);           // 1/10!, 1/8!, ...
    pc = fmaf(y, pc, -1.38888889e-3f);
    pc = fmaf(y, pc, 4.16666667e-2f);
    pc = fmaf(y, pc, -0.5f);
    const float cx = fmaf(y, pc, 1.0f);
    const bool swap = quad & 1;
    c = swap ? sx : cx;
    s = swap ? cx : sx;
    if ((quad + 1) & 2) c = -c;                                    // quarters 1 and 2
    if (quad & 2) s = -s;                                          // quarters 2 and 3
}

__device__ __forceinline__ uint32_t turns(double position, double inv_freq) {
    const double t = position * (inv_freq * 0.15915494309189535);  // 1 / 2 pi
    return (uint32_t)(unsigned long long)((t - floor(t)) * 4294967296.0);     // 2^32 itself wraps to 0
}

// A unit is what a lane handles of a head: V pairs (two runs of V elements, or 2 V elements where pairs lie side by side), or behind the
// rotated part 2 V elements that are copied.  V: the widest for which every run is aligned to its size.
template <typename T, int V> struct alignas(sizeof(T) * V) Run { T e[V]; };

template <typename T, int V, bool INTER>
__device__ __forceinline__ void turn_unit(const T* __restrict__ src, T* __restrict__ dst, int unit, int pair_units, int rotated, int dim, const float (&c)[V],
                                          const float (&s)[V], bool turn) {
    typedef Run<T, V> R;
    int lo, hi;
    if (unit < pair_units) {
        lo = INTER ? 2 * V * unit : V * unit;
        hi = INTER ? lo + V : lo + rotated / 2;
    } else {
        lo = rotated + 2 * V * (unit - pair_units);
        hi = lo + V;
        turn = false;
    }
    const bool two = hi < dim;                                     // an odd number of copied runs ends with one alone
    const R x = *(const R*)(src + lo), y = two ? *(const R*)(src + hi) : x;
    R u = x, w = y;
    if (turn) {
        if (INTER) {
#pragma unroll
            for (int i = 0; i < V; ++i) {                          // pair i: elements 2 i and 2 i + 1 of the 2 V
                const float a = widen(2 * i < V ? x.e[(2 * i) % V] : y.e[(2 * i) % V]), b = widen(2 * i + 1 < V ? x.e[(2 * i + 1) % V] : y.e[(2 * i + 1) % V]);
                const T p = narrow<T>(a * c[i] - b * s[i]), q = narrow<T>(a * s[i] + b * c[i]);
                if (2 * i < V) u.e[(2 * i) % V] = p; else w.e[(2 * i) % V] = p;
                if (2 * i + 1 < V) u.e[(2 * i + 1) % V] = q; else w.e[(2 * i + 1) % V] = q;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float a = widen(x.e[i]), b = widen(y.e[i]);
                u.e[i] = narrow<T>(a * c[i] - b * s[i]);
                w.e[i] = narrow<T>(a * s[i] + b * c[i]);
            }
        }
    }
    *(R*)(dst + lo) = u;
    if (two) *(R*)(dst + hi) = w;
}

struct RotaryArgs {
    const char *x, *k, *v; char *out;
    const void* positions; const double* inv_freq;
    long x_token, x_head, k_token, k_head, v_token, v_head, out_token, out_head;     // bytes
    float gain;
    int tokens, heads, dim, rotated, inverse, wide;
    int slices;                                                    // a token's heads are dealt to this many waves
    // append: the cache
    char *ck, *cv;
    const int *table, *lens, *cu_new;
    long page_stride, head_stride, slot_stride;                    // bytes
    int kv_heads, pages, page_shift, rows, width;
};

// APPEND: the wave's heads are the queries' (to out), the keys' and the values' (to their page); else the heads of x
template <typename T, int V, bool INTER, bool APPEND>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    const int wave = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int token = wave / a.slices, slice = wave - token * a.slices;
    if (token >= a.tokens) return;
    long page_at = -1;                                             // where the token's slot lies in a cache, bytes
    long position = 0;
    if (APPEND) {
        const int b = seq_of_token(a.cu_new, a.rows, token);
        if (b >= a.rows) return;                                   // behind the last sequence
        const int first = a.cu_new[b], n = a.cu_new[b + 1] - first;
        const int len = clamp_len(a.lens[b], a.width << a.page_shift), p = len - n + (token - first);
        position = p;
        if (p >= 0 && p < len) {
            const int page = a.table[(long)b * a.width + (p >> a.page_shift)];
            if (page >= 0 && page < a.pages) page_at = page * a.page_stride + (p & ((1 << a.page_shift) - 1)) * a.slot_stride;
        }
    }
    if (!APPEND || a.positions) position = a.wide ? ((const long long*)a.positions)[token] : ((const int*)a.positions)[token];
    const int pair_units = a.rotated / (2 * V), units = pair_units + (a.dim - a.rotated + 2 * V - 1) / (2 * V);
    const int across = units < 64 ? units : 64;                    // lanes that share a head
    const int lane_head = lane / across, step = 64 / across;       // heads that a wave handles at a time
    if (lane_head >= step) return;
    const int heads = APPEND ? a.heads + 2 * a.kv_heads : a.heads;
    for (int unit = lane - lane_head * across; unit < units; unit += across) {
        float c[V], s[V];
        if (unit < pair_units) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                turn_sincos(turns((double)position, a.inv_freq[unit * V + i]), c[i], s[i]);
                c[i] *= a.gain;
                s[i] *= a.inverse ? -a.gain : a.gain;
            }
        }
        for (int h = slice * step + lane_head; h < heads; h += a.slices * step) {
            const char* src; char* dst;
            bool turn = true;
            if (!APPEND || h < a.heads) {
                src = a.x + token * a.x_token + h * a.x_head;
                dst = a.out + token * a.out_token + h * a.out_head;
            } else {
                if (page_at < 0) continue;
                const bool key = h < a.heads + a.kv_heads;
                const int kh = h - a.heads - (key ? 0 : a.kv_heads);
                src = key ? a.k + token * a.k_token + kh * a.k_head : a.v + token * a.v_token + kh * a.v_head;
                dst = (key ? a.ck : a.cv) + page_at + kh * a.head_stride;
                turn = key;
            }
            turn_unit<T, V, INTER>((const T*)src, (T*)dst, unit, pair_units, a.rotated, a.dim, c, s, turn);
        }
    }
}

// how many elements every run may have: the largest power of two that divides all of `of` (elements or bytes / size), at most `most`
int widest(int most, std::initializer_list<unsigned long long> of) {
    int v = most;
    for (unsigned long long x : of) while (x % v) v >>= 1;
    return v;
}

template <bool APPEND>
int run_rotary(RotaryArgs& a, int dtype, int v, bool inter, hipStream_t s) {
    const int heads = APPEND ? a.heads + 2 * a.kv_heads : a.heads;
    const int units = a.rotated / (2 * v) + (a.dim - a.rotated + 2 * v - 1) / (2 * v);
    const int passes = cdiv(heads, 64 / (units < 64 ? units : 64));        // of a token's heads, for one wave
    // tokens alone fill the GPU from about 8 waves a SIMD's worth; below that a token's heads are dealt to several waves, which compute
    // its angles again
    a.slices = 1;
    while (a.slices * 2 <= passes && (long)a.tokens * a.slices < 4096) a.slices *= 2;
    if (a.tokens < 512) a.slices = passes;
    const long waves = (long)a.tokens * a.slices;
    const dim3 grid((unsigned)((waves + 3) / 4));
#define DISCO_ROTARY(T, V) do { if (inter) rotary_kernel<T, V, true, APPEND><<<grid, 256, 0, s>>>(a); else rotary_kernel<T, V, false, APPEND><<<grid, 256, 0, s>>>(a); } while (0)
#define DISCO_ROTARY_V(T) do { if (v == 8) DISCO_ROTARY(T, 8); else if (v == 4) DISCO_ROTARY(T, 4); else if (v == 2) DISCO_ROTARY(T, 2); else DISCO_ROTARY(T, 1); } while (0)
    if (dtype == DISCO_F16) DISCO_ROTARY_V(f16);
    else if (dtype == DISCO_BF16) DISCO_ROTARY_V(__bf16);
    else if constexpr (!APPEND) { if (v >= 4) DISCO_ROTARY(float, 4); else if (v == 2) DISCO_ROTARY(float, 2); else DISCO_ROTARY(float, 1); }
    DISCO_LAUNCH_CHECK("rotary_kernel");
    return DISCO_OK;
}

}  // namespace

int launch_rotary(const disco_rotary_desc& d, const void* x, const void* positions, const double* inv_freq, void* out, hipStream_t s) {
    const int size = d.dtype == DISCO_F32 ? 4 : 2;
    RotaryArgs a{};
    a.x = (const char*)x; a.out = (char*)out; a.positions = positions; a.inv_freq = inv_freq;
    a.x_token = d.x_token * size; a.x_head = d.x_head * size; a.out_token = d.out_token * size; a.out_head = d.out_head * size;
    a.gain = (float)d.gain; a.tokens = d.tokens; a.heads = d.heads; a.dim = d.dim; a.rotated = d.rotated; a.inverse = d.inverse; a.wide = d.wide_positions;
    const int v = widest(16 / size, {(unsigned long long)d.rotated / 2, (unsigned long long)d.dim, (unsigned long long)d.x_token, (unsigned long long)d.x_head,
                                     (unsigned long long)d.out_token, (unsigned long long)d.out_head, (unsigned long long)(uintptr_t)x / size,
                                     (unsigned long long)(uintptr_t)out / size});
    return run_rotary<false>(a, d.dtype, v, d.interleaved, s);
}

int launch_cache_append(const disco_cache_desc& c, const disco_append_desc& d, const void* q, const void* k, const void* v, const int* table,
                        const int* lens, const int* cu_new, const void* positions, const double* inv_freq, void* q_out, hipStream_t s) {
    RotaryArgs a{};
    a.x = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.out = (char*)q_out; a.positions = positions; a.inv_freq = inv_freq;
    a.x_token = d.q_token * 2; a.x_head = d.q_head * 2; a.k_token = d.k_token * 2; a.k_head = d.k_head * 2; a.v_token = d.v_token * 2; a.v_head = d.v_head * 2;
    a.out_token = d.out_token * 2; a.out_head = d.out_head * 2;
    a.gain = (float)d.gain; a.tokens = d.tokens; a.heads = d.q_heads; a.dim = c.dim; a.rotated = d.rotated; a.wide = d.wide_positions;
    a.ck = (char*)c.d_k; a.cv = (char*)c.d_v; a.table = table; a.lens = lens; a.cu_new = cu_new;
    a.page_stride = c.page_stride * 2; a.head_stride = c.head_stride * 2; a.slot_stride = c.slot_stride * 2;
    a.kv_heads = c.kv_heads; a.pages = c.pages; a.page_shift = __builtin_ctz((unsigned)c.page_size); a.rows = c.rows; a.width = c.table_width;
    unsigned long long qs = 0;
    if (d.q_heads) qs = (unsigned long long)(d.q_token | d.q_head | d.out_token | d.out_head | (int64_t)((uintptr_t)q / 2) | (int64_t)((uintptr_t)q_out / 2));
    // the cache's strides are multiples of 8 elements and its pointers of 16 bytes
    const int w = widest(8, {(unsigned long long)d.rotated / 2, qs, (unsigned long long)d.k_token, (unsigned long long)d.k_head, (unsigned long long)d.v_token,
                             (unsigned long long)d.v_head, (unsigned long long)(uintptr_t)k / 2, (unsigned long long)(uintptr_t)v / 2});
    return run_rotary<true>(a, c.dtype, w, d.interleaved, s);
}

}  // namespace disco
