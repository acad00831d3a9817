// rotary.hip - positions as rotations of pairs of a head's elements, alone and on the way into a paged cache.
//
//   (a, b) -> g (a cos t - b sin t, a sin t + b cos t),   t = position * f_i
//
// Memory-bound: every element is read once and written once.  The angle is what needs care: at position 10^6 an fp32 product is off by
// 0.06 rad, and at 2^40 an fp64 one still by 1e-4, so t / 2 pi is formed as a sum of two fp64 numbers and only its fraction is kept, to the nearest
// 2^-32 of a turn (off by 7e-10 rad at most, whatever the position); sine and cosine are then Taylor sums
// over [-pi/4, pi/4] in fp32 (next term below 3e-8).  That is ~50 instructions a pair, ten of them in fp64: a wave handles one token (or a slice of
// its heads where tokens are few), each pair's angle is computed by one lane, and the heads read it from LDS (16 384 tokens of 32 heads of
// 128, bf16: 45 us, 5.9 TB/s, what copying the tensor takes).
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

// position * inv_freq / 2 pi, its fraction in 2^-32.  Products and 1 / 2 pi are carried with what their rounding leaves (fma gives that of a product).
__device__ __forceinline__ uint32_t turns(double position, double inv_freq) {
#pragma clang fp contract(off)                                     // (t - floor(t) is of the rounded product)
    constexpr double PER = 0x1.45f306dc9c883p-3, PER_REST = -0x1.6b01ec5417056p-57;            // 1 / 2 pi
    const double f = inv_freq * PER, f_rest = fma(inv_freq, PER, -f) + inv_freq * PER_REST;
    const double t = position * f, t_rest = fma(position, f, -t) + position * f_rest;
    return (uint32_t)(long long)rint(((t - floor(t)) + t_rest) * 4294967296.0);                 // whole turns, either way, wrap to 0
}

// What a lane handles of a head, in runs of V elements (the widest that dimensions, strides and addresses allow).  A run a lane, so that a wave reads whole
// lines: with two runs a lane, half a head or half the rotated part apart, 16 384 tokens of 32 heads of 128 take 54 us, and 78 us where half of each
// head is rotated; with one 45 us, what copying the tensor takes.
//   WITHIN    pairs side by side: turned inside the run
//   EXCHANGE  pairs apart: the other ends of the run's pairs come from the lane that holds them
//   ACROSS    two runs, both ends of V pairs, or two runs of the part that is copied: what neither of the others can do - runs of one element with pairs
//             side by side, pairs apart in heads of more than 64 runs
enum Mode { WITHIN, EXCHANGE, ACROSS };
template <typename T, int V> struct alignas(sizeof(T) * V) Run { T e[V]; };

// one end of V pairs turned: x c + (the other end) s, the sine's sign being the end's
template <typename T, int V>
__device__ __forceinline__ Run<T, V> turn_end(const Run<T, V>& x, const Run<T, V>& other, const float (&c)[V], const float (&s)[V]) {
    Run<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = narrow<T>(widen(x.e[i]) * c[i] + widen(other.e[i]) * s[i]);
    return r;
}
// the V / 2 pairs inside a run, `pairs` of them turned
template <typename T, int V>
__device__ __forceinline__ void turn_within(Run<T, V>& x, int pairs, const float (&c)[V], const float (&s)[V]) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const float a = widen(x.e[2 * i]), b = widen(x.e[2 * i + 1]);
        const T p = narrow<T>(a * c[i] - b * s[i]), q = narrow<T>(a * s[i] + b * c[i]);
        if (i < pairs) { x.e[2 * i] = p; x.e[2 * i + 1] = q; }
    }
}
template <typename T, int V>
__device__ __forceinline__ Run<T, V> run_of_lane(const Run<T, V>& x, int lane) {
    constexpr int WORDS = (sizeof(T) * V + 3) / 4;
    union { Run<T, V> r; int w[WORDS]; } a;
    a.w[WORDS - 1] = 0;
    a.r = x;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) a.w[i] = __shfl(a.w[i], lane);
    return a.r;
}

constexpr int MOST_PAIRS = 512;

struct RotaryArgs {
    const char *x, *k, *v; char *out;
    const void* positions; const double* inv_freq;
    long x_token, x_head, k_token, k_head, v_token, v_head, out_token, out_head;     // bytes
    float gain;
    int tokens, heads, dim, rotated, inverse, wide;
    int slices;                                                    // a token's heads are dealt to this many waves
    // append: the cache
    char *ck, *cv;
    const int *table, *lens, *cu_new, *info;
    long page_stride, head_stride, slot_stride;                    // bytes
    int kv_heads, pages, page_shift, rows, width;
};

// APPEND: the wave's heads are the queries' (to out), the keys' and the values' (to their page); else the heads of x
template <typename T, int V, int MODE, bool INTER, bool APPEND>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    const int wave = (int)block_of() * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;       // (below 2^31: 2^30 tokens, or 2^9 of 2^17 heads)
    const int token = wave / a.slices, slice = wave - token * a.slices;
    if (token >= a.tokens) return;
    long page_at = -1;                                             // where the token's slot lies in a cache, bytes
    long position = 0;
    if (APPEND) {
        const int b = seq_of_token(a.cu_new, a.rows, token);
        if (b >= a.rows) return;                                   // behind the last sequence
        const int first = a.cu_new[b], n = a.cu_new[b + 1] - first;
        if (token < first) return;                                 // ahead of the first one
        const int len = clamp_len(a.lens[b], a.width << a.page_shift), p = len - n + (token - first);
        position = p;
        const bool reserved = !a.info || a.info[1] == 0;           // (else the length does not count the new tokens: their places are other tokens')
        if (reserved && p >= 0 && p < len) {
            const int page = a.table[(long)b * a.width + (p >> a.page_shift)];
            if (page >= 0 && page < a.pages) page_at = page * a.page_stride + (p & ((1 << a.page_shift) - 1)) * a.slot_stride;
        }
    }
    if (!APPEND || a.positions) position = a.wide ? ((const long long*)a.positions)[token] : ((const int*)a.positions)[token];
    const int pair_units = a.rotated / (2 * V), rest_units = ((a.dim - a.rotated) / V + 1) / 2;      // (ACROSS)
    const int units = MODE == ACROSS ? pair_units + rest_units : a.dim / V;
    const int across = units < 64 ? units : 64;                    // lanes that share a head
    const int lane_head = lane / across, step = 64 / across;       // heads that a wave handles at a time
    const int heads = lane_head < step ? (APPEND ? a.heads + 2 * a.kv_heads : a.heads) : 0, stride = a.slices * step;
    typedef Run<T, V> R;
    int unit = lane - lane_head * across, lo, hi;
    auto place = [&] {
        lo = V * unit;
        hi = MODE == ACROSS ? lo + a.rotated / 2 : a.dim;          // (no second run)
        if (MODE == ACROSS) {
            if (INTER) { lo = 2 * unit; hi = lo + 1; }             // (V = 1)
            if (unit >= pair_units) {
                lo = a.rotated + V * (unit - pair_units);
                hi = lo + V * rest_units;
            }
        }
    };
    // four heads at a time, all of their loads ahead of the first store - and the first four's ahead of the angles
    R x[4], y[4];
    char* dst[4];
    auto load = [&](int h0) {
        const bool two = hi < a.dim;                               // an odd number of copied runs ends with one alone
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int h = h0 + j * stride;
            dst[j] = nullptr;
            if (h >= heads) continue;
            const char* src;
            if (!APPEND || h < a.heads) {
                src = a.x + token * a.x_token + h * a.x_head;
                dst[j] = a.out + token * a.out_token + h * a.out_head;
            } else {
                if (page_at < 0) continue;
                const bool key = h < a.heads + a.kv_heads;
                const int kh = h - a.heads - (key ? 0 : a.kv_heads);
                src = key ? a.k + token * a.k_token + kh * a.k_head : a.v + token * a.v_token + kh * a.v_head;
                dst[j] = (key ? a.ck : a.cv) + page_at + kh * a.head_stride;
            }
            x[j] = *(const R*)((const T*)src + lo);
            y[j] = two ? *(const R*)((const T*)src + hi) : x[j];
        }
    };
    const int first = slice * step + lane_head;
    place();
    load(first);
    // the angles, each computed once
    __shared__ __align__(16) float cosines[4][MOST_PAIRS], sines[4][MOST_PAIRS];
    float *cw = cosines[threadIdx.x >> 6], *sw = sines[threadIdx.x >> 6];
    for (int p = lane; p < a.rotated / 2; p += 64) {
        float c, s;
        turn_sincos(turns((double)position, a.inv_freq[p]), c, s);
        cw[p] = c * a.gain;
        sw[p] = s * (a.inverse ? -a.gain : a.gain);
    }
    __builtin_amdgcn_wave_barrier();                               // (a wave's LDS operations take place in order)
    for (;;) {
        const bool two = hi < a.dim;
        const bool turn = MODE == ACROSS ? unit < pair_units : lo < a.rotated, second = lo >= a.rotated / 2;
        float c[V], s[V];                                          // (WITHIN: of V / 2 pairs)
#pragma unroll
        for (int i = 0; i < (MODE == WITHIN ? V / 2 : V); ++i) {
            int p = MODE == WITHIN ? lo / 2 + i : (MODE == EXCHANGE ? lo + i - (second ? a.rotated / 2 : 0) : unit * V + i);
            if (p >= a.rotated / 2) p = 0;                         // (not used)
            c[i] = cw[p];
            s[i] = MODE == EXCHANGE && !second ? -sw[p] : sw[p];
        }
        const int other = lane + (second ? -pair_units : pair_units);
        for (int h0 = first; h0 < heads; h0 += 4 * stride) {
            if (h0 != first) load(h0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!dst[j]) continue;
                if (turn && (!APPEND || h0 + j * stride < a.heads + a.kv_heads)) {
                    if constexpr (MODE == WITHIN) turn_within<T, V>(x[j], a.rotated / 2 - lo / 2, c, s);
                    else if constexpr (MODE == EXCHANGE) x[j] = turn_end<T, V>(x[j], run_of_lane<T, V>(x[j], other), c, s);
                    else {
                        const R u = x[j];
                        float minus[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) minus[i] = -s[i];
                        x[j] = turn_end<T, V>(u, y[j], c, minus);
                        y[j] = turn_end<T, V>(y[j], u, c, s);
                    }
                }
                *(R*)((T*)dst[j] + lo) = x[j];
                if (two) *(R*)((T*)dst[j] + hi) = y[j];
            }
        }
        unit += across;
        if (unit >= units) break;
        place();
        load(first);
    }
}

// how many elements every run may have: the largest power of two that divides all of `of` (elements or bytes / size), at most `most`
int widest(int most, std::initializer_list<unsigned long long> of) {
    int v = most;
    for (unsigned long long x : of) while (x % v) v >>= 1;
    return v;
}

template <typename T, int V, bool APPEND>
int run_rotary(RotaryArgs& a, bool inter, hipStream_t s) {
    const bool exchange = !inter && a.dim / V <= 64 && a.rotated % (2 * V) == 0;
    const int heads = APPEND ? a.heads + 2 * a.kv_heads : a.heads;
    const int units = (inter && V > 1) || exchange ? a.dim / V : a.rotated / (2 * V) + ((a.dim - a.rotated) / V + 1) / 2;
    const int passes = cdiv(heads, 64 / (units < 64 ? units : 64));        // of a token's heads, for one wave
    // tokens alone fill the GPU from about 4 waves a SIMD; below that a token's heads are dealt to several waves, which compute its angles again
    a.slices = 1;
    while (a.slices * 2 <= passes && (long)a.tokens * a.slices < 4096) a.slices *= 2;
    if (a.tokens < 512) a.slices = passes;
    const dim3 grid = grid_of(((long)a.tokens * a.slices + 3) / 4);
    if (inter) rotary_kernel<T, V, (V > 1 ? WITHIN : ACROSS), true, APPEND><<<grid, 256, 0, s>>>(a);
    else if (exchange) rotary_kernel<T, V, EXCHANGE, false, APPEND><<<grid, 256, 0, s>>>(a);
    else rotary_kernel<T, V, ACROSS, false, APPEND><<<grid, 256, 0, s>>>(a);
    DISCO_LAUNCH_CHECK("rotary_kernel");
    return DISCO_OK;
}

template <bool APPEND>
int run_rotary(RotaryArgs& a, int dtype, int v, bool inter, hipStream_t s) {
#define DISCO_ROTARY(T) (v == 8 ? run_rotary<T, 8, APPEND>(a, inter, s) : v == 4 ? run_rotary<T, 4, APPEND>(a, inter, s) \
                         : v == 2 ? run_rotary<T, 2, APPEND>(a, inter, s) : run_rotary<T, 1, APPEND>(a, inter, s))
    if (dtype == DISCO_F16) return DISCO_ROTARY(f16);
    if (dtype == DISCO_BF16) return DISCO_ROTARY(__bf16);
#undef DISCO_ROTARY
    if constexpr (!APPEND) {
        if (v >= 4) return run_rotary<float, 4, false>(a, inter, s);
        return v == 2 ? run_rotary<float, 2, false>(a, inter, s) : run_rotary<float, 1, false>(a, inter, s);
    }
    return DISCO_EINVAL;
}

}  // namespace

int launch_rotary(const disco_rotary_desc& d, const void* x, const void* positions, const double* inv_freq, void* out, hipStream_t s) {
    const int size = d.dtype == DISCO_F32 ? 4 : 2;
    RotaryArgs a{};
    a.x = (const char*)x; a.out = (char*)out; a.positions = positions; a.inv_freq = inv_freq;
    a.x_token = d.x_token * size; a.x_head = d.x_head * size; a.out_token = d.out_token * size; a.out_head = d.out_head * size;
    a.gain = (float)d.gain; a.tokens = d.tokens; a.heads = d.heads; a.dim = d.dim; a.rotated = d.rotated; a.inverse = d.inverse; a.wide = d.wide_positions;
    const int v = widest(16 / size, {d.interleaved ? 0ull : (unsigned long long)d.rotated / 2, (unsigned long long)d.dim, (unsigned long long)d.x_token, (unsigned long long)d.x_head,
                                     (unsigned long long)d.out_token, (unsigned long long)d.out_head, (unsigned long long)(uintptr_t)x / size,
                                     (unsigned long long)(uintptr_t)out / size});
    return run_rotary<false>(a, d.dtype, v, d.interleaved, s);
}

int launch_cache_append(const disco_cache_desc& c, const disco_append_desc& d, const void* q, const void* k, const void* v, const int* table,
                        const int* lens, const int* cu_new, const void* positions, const double* inv_freq, void* q_out, const int* info, hipStream_t s) {
    RotaryArgs a{};
    a.x = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.out = (char*)q_out; a.positions = positions; a.inv_freq = inv_freq;
    a.x_token = d.q_token * 2; a.x_head = d.q_head * 2; a.k_token = d.k_token * 2; a.k_head = d.k_head * 2; a.v_token = d.v_token * 2; a.v_head = d.v_head * 2;
    a.out_token = d.out_token * 2; a.out_head = d.out_head * 2;
    a.gain = (float)d.gain; a.tokens = d.tokens; a.heads = d.q_heads; a.dim = c.dim; a.rotated = d.rotated; a.wide = d.wide_positions;
    a.ck = (char*)c.d_k; a.cv = (char*)c.d_v; a.table = table; a.lens = lens; a.cu_new = cu_new; a.info = info;
    a.page_stride = c.page_stride * 2; a.head_stride = c.head_stride * 2; a.slot_stride = c.slot_stride * 2;
    a.kv_heads = c.kv_heads; a.pages = c.pages; a.page_shift = __builtin_ctz((unsigned)c.page_size); a.rows = c.rows; a.width = c.table_width;
    unsigned long long qs = 0;
    if (d.q_heads) qs = (unsigned long long)(d.q_token | d.q_head | d.out_token | d.out_head | (int64_t)((uintptr_t)q / 2) | (int64_t)((uintptr_t)q_out / 2));
    // the cache's strides are multiples of 8 elements and its pointers of 16 bytes
    const int w = widest(8, {d.interleaved ? 0ull : (unsigned long long)d.rotated / 2, qs, (unsigned long long)d.k_token, (unsigned long long)d.k_head, (unsigned long long)d.v_token,
                             (unsigned long long)d.v_head, (unsigned long long)(uintptr_t)k / 2, (unsigned long long)(uintptr_t)v / 2});
    return run_rotary<true>(a, c.dtype, w, d.interleaved, s);
}

}  // namespace disco
