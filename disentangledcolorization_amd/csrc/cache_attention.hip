// cache_attention.hip - attention of new tokens over a paged cache.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q.k_j - m),   c = scale log2 e,   m: a maximum of the row so far
//
// One pass over the keys.  The rows that share a key head - the queries of its group, for all new tokens of a sequence - form the rows of one
// matrix (row = token * group + head in group), so that keys and values are read once for all of them.  Both products run on the matrix cores
// in transposed form: S^T = K Q^T puts one row's scores into one lane's registers, where maximum, exponential and sum need no exchange
// but that between the lanes of a column, and the registers that hold the probabilities are in place the operand of O^T = V^T P^T (their key order
// is the accumulator's; V^T is read in the same order by the transposing LDS read).
//
// Three forms, chosen by a sequence's own rows (new tokens * group), so that its result does not depend on what else is in the call (rows of no sequence
// included, unless the caller has said that there are none):
//   few (up to 16 rows)    cache_attention_few_kernel: 16 rows a workgroup, its four waves deal 32-key tiles; bound by reading the cache
//   many                   cache_attention_many_kernel, 128 rows a workgroup, 32 a wave, keys and values staged in LDS for all of them; two workgroups
//                          a CU, bound by what L2 delivers into LDS (7 TB/s over the chip) and, at short ranges, by latency
//   large (above 1 024 rows of heads of 72 .. 128)
//                          the same with 256 rows, which halves what is delivered; bound by the matrix cores and the exponentials, which overlap in part.
//                          32 heads of 128 on 8: 2 048 tokens behind 16 384 keys 595 us (128 rows: 649), 1 024 of them 336 (370), 8 192 tokens
//                          583 (631), but 4 prompts of 1 024 tokens 120 (108); below 1 024 rows a CU has nothing to do beside one workgroup's start
//                          and end.  Heads of 64 stay with 128 rows, there the exponentials bound both: 5 000 tokens of 16 heads 92 us (256 rows: 105),
//                          4 x 2 048 tokens over 8 192 360 (410), 2 048 behind 16 384 220 (205); heads above 128 do not fit the registers.
// Where a sequence alone does not fill the GPU its keys are split; the parts (m, sum, o in fp32) are joined by cache_attention_join_kernel.
//
// A tile that some row sees only in part, or that has a page outside the cache, takes the masked path: scores of unseen keys are replaced (never
// added to), and values that are not finite are kept out of the product and given to the rows that see them.
#include <algorithm>
#include <type_traits>
#include "paged.h"

namespace disco {

namespace {

typedef __bf16 bf16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Mat;
template <> struct Mat<f16> {
    typedef f16x8 x8;
    static constexpr uint32_t INF = 0x7c00, ONE = 0x3c00;
    // probabilities below 2^-14 lose bits in fp16, so all of a row are 2^6 larger (at most 2^15: Run::LIMIT)
    static constexpr float BIAS = 6.f;
    static __device__ __forceinline__ f32x16 mul(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mul(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<bf16> {
    typedef bf16 x8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t INF = 0x7f80, ONE = 0x3f80;
    static constexpr float BIAS = 0.f;
    static __device__ __forceinline__ f32x16 mul(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mul(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

struct AttnArgs {
    const char *q, *k, *v; char* out; float* lse;
    float *part_o; float2* part_ml;                                // by part_at()
    const int *table, *lens, *cu_new;
    long q_token, q_head, out_token, out_head, page_stride, head_stride, slot_stride;    // bytes
    int tokens, q_heads, kv_heads, group, dim, rows, width, pages, page_shift, causal, window;
    // parts of a row that there may be, and where they are: by token, or by sequence
    int few_splits, many_splits, few_by_sequence;
    int few_fold, many_fold;                                       // a workgroup computes 2^fold parts of its rows and keeps their sum (0 or FOLD)
    int many_room;                                                 // of a sequence; 0: by token
    long many_from;
    int few, many;                                                 // sequences of at most so many rows take the form of few, of many rows
    float c;                                                       // |scale| log2 e, not 0
    int negate;                                                    // scale < 0: the queries change sign instead
};

// The kernels read their arguments where they lie, piece by piece: held in registers from start to end they would not fit beside the loops.  fresh()
// makes the compiler forget what it has read.
typedef const __attribute__((address_space(4))) AttnArgs* ArgsAt;
__device__ __forceinline__ ArgsAt fresh(ArgsAt p) {
    asm volatile("" : "+s"(p));
    return p;
}

// forms, by the rows of a sequence
enum Form { FEW, MANY, LARGE };
__host__ __device__ constexpr int rows_of(int form) { return form == FEW ? 16 : (form == MANY ? 128 : 256); }      // of a workgroup
constexpr float LN2 = 0.6931471805599453f;

// The parts of a row are added up in the order of the keys, in groups of 2^FOLD, and the groups in their order: whether a workgroup computes one part and a join adds
// up the group, or computes the whole group and adds as it goes, the result has the same bits.
constexpr int FOLD = 3;
__host__ __device__ __forceinline__ int slots_of(int splits, int fold) { return (splits + (1 << fold) - 1) >> fold; }

// ---- how a sequence is cut ------------------------------------------------------------------------------------------------------------
struct Cut { int form, tiles, splits, chunk; };
__host__ __device__ __forceinline__ int min_of(int a, int b) { return a < b ? a : b; }
// the first key that a token at position p sees, of its tile of 64
__host__ __device__ __forceinline__ int begin_of(int p, int window) { return window > 0 && p - window + 1 > 0 ? (p - window + 1) & ~63 : 0; }

// parts of a sequence's keys; grows with them
// few rows: a workgroup's waves take 128 keys a round, and up to 512 keys (4 us) one workgroup is done sooner than two and a join.  Beyond, parts of 256 /
//           384 / 512 keys take 14.4 / 16.0 / 17.7 us for one sequence of 4 096 and 134 / 129 / 125 us for 64 of up to 4 096 (32 heads of 128 on 8 key
//           heads); 64 parts of 8 key heads are two workgroups a CU
// many rows: as many parts as fill the GPU, two workgroups a CU where two fit (128 rows, heads of up to 128) and the parts are long enough for that, else
//           one; of at least 1 024 keys, as a part costs a write and a read of its rows in fp32 (24 sequences of up to 257 tokens over 4 111 take
//           78 us, with parts of 512 keys 93), and of 512 for up to 64 rows and for heads above 128, whose keys take twice the time (200 tokens over
//           8 192 keys of 8 heads of 256: 79 -> 55 us, 32 sequences of 64 over 2 048 of two: 109 -> 115).
//           32 heads of 128 on 8 key heads: 8 tokens over 65 536 take 57 us, with one workgroup a CU 66, with at most 8 parts 228; 256 tokens over
//           18 432 take 117 us, with one workgroup a CU 151.  What has a workgroup a CU as it is stays whole but for long histories, 16 heads of
//           64: four sequences of 2 048 tokens over 8 192 take 360 us (in two parts 421), one over 18 432 301 (in two parts 220).
__host__ __device__ __forceinline__ int splits_of(int form, int rows, int tiles, int keys, int kv_heads, bool narrow) {
    if (form == FEW) return keys <= 512 ? 1 : (keys > 64 * 384 ? 64 : (keys + 383) / 384);
    const int units = tiles * kv_heads;
    if (units >= 256) return form == MANY && narrow && units < 512 && keys >= 16384 ? 2 : 1;
    const int least = rows <= 64 || !narrow ? 512 : 1024, by_keys = keys <= least ? 1 : (keys + least - 1) / least;
    int s = form == MANY && narrow ? 512 / units : 256 / units;
    if (s > by_keys) s = 256 / units < by_keys ? 256 / units : by_keys;
    return s < 64 ? s : 64;
}

// How the keys that a tile of rows sees are cut: they begin at begin_of() its first token and are `keys` at most, every part takes `chunk` of them, a multiple
// of 128.  (Parts of what the tile sees, not of the sequence: 701 tokens of heads of 256 that see 1 024 keys take 60 us, cut across the sequence 81.)
__host__ __device__ __forceinline__ Cut cut_of(int n, int len, int group, int kv_heads, int window, bool narrow, int few, int many, int most_few, int most_many) {
    Cut u;
    const int rows = n * group;
    u.form = rows <= few ? FEW : (rows <= many ? MANY : LARGE);
    const int tile = rows_of(u.form), across = (tile - 1) / group + 1;        // (a tile's first token and last are no further apart)
    u.tiles = (rows + tile - 1) / tile;
    const int keys = window <= 0 ? len : (u.tiles == 1 ? len - begin_of(len - n, window) : min_of(len, window + 63 + across));
    int s = splits_of(u.form, rows, u.tiles, keys, kv_heads, narrow);
    const int most = u.form == FEW ? most_few : most_many;
    if (s > most) s = most;
    u.chunk = ((keys + s - 1) / s + 127) & ~127;
    if (u.chunk < 128) u.chunk = 128;
    u.splits = (keys + u.chunk - 1) / u.chunk;
    if (u.splits < 1) u.splits = 1;
    return u;
}

// where the first slot of a row lies, `slots` being those of each of its sequence's rows: row `row` of the sequence's rows of key head `kv_head`, token t of the call, query head h
template <typename Args>
__device__ __forceinline__ long part_at(const Args& a, int form, int slots, int b, int row, int kv_head, int t, int h) {
    const long by_token = (long)t * a.q_heads + h;
    if (form == FEW) return (a.few_by_sequence ? ((long)b * a.kv_heads + kv_head) * rows_of(FEW) + row : by_token) * slots_of(a.few_splits, a.few_fold);
    return a.many_from + (a.many_room ? (long)b * a.many_room + ((long)row * a.kv_heads + kv_head) * slots : by_token * slots_of(a.many_splits, a.many_fold));
}

struct Unit { int b, n, len, first, tile, split, parts, head, begin; Cut cut; };     // parts: that the workgroup has still to compute, `split` the next

// unit number `want` of a form over all sequences (key head fastest, then split, then tile - the last, longest tiles first); false behind the last.
// Every lane of the wave calls it and gets the same.
// The cursor keeps which 64 sequences were looked at last and how many units lie before them: a workgroup asks for ever larger numbers.
struct Cursor { int b0, before; };

template <int FORM>
__device__ __forceinline__ bool find_unit(ArgsAt a, int want, Cursor& at_last, Unit& u) {
    const int lane = threadIdx.x & 63, capacity = a->width << a->page_shift, fold = FORM == FEW ? a->few_fold : a->many_fold;
    int left = want - at_last.before;
    for (int b0 = at_last.b0; b0 < a->rows; b0 += 64) {
        const int b = b0 + lane;
        int n = 0, len = 0, first = 0, units = 0;
        Cut cut{};
        if (b < a->rows) {
            first = a->cu_new[b];
            n = a->cu_new[b + 1] - first;
            len = clamp_len(a->lens[b], capacity);
            if (first < 0 || n < 0 || n > a->tokens || first > a->tokens - n) n = 0;       // (not offsets)
            if (n > 0) {
                cut = cut_of(n, len, a->group, a->kv_heads, a->window, a->dim <= 128, a->few, a->many, a->few_splits, a->many_splits);
                if (cut.form == FORM) units = cut.tiles * slots_of(cut.splits, fold) * a->kv_heads;
            }
        }
        int upto = units;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        const unsigned long long here = __ballot(upto > left);
        if (here) {
            const int at = __ffsll((long long)here) - 1;
            at_last = Cursor{b0, want - left};
            u.b = b0 + at;
            u.n = __builtin_amdgcn_readlane(n, at);
            u.len = __builtin_amdgcn_readlane(len, at);
            u.first = __builtin_amdgcn_readlane(first, at);
            u.cut.tiles = __builtin_amdgcn_readlane(cut.tiles, at);
            u.cut.splits = __builtin_amdgcn_readlane(cut.splits, at);
            u.cut.chunk = __builtin_amdgcn_readlane(cut.chunk, at);
            int x = left - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(units, at));
            u.head = x % a->kv_heads; x /= a->kv_heads;
            const int slots = slots_of(u.cut.splits, fold);
            u.split = x % slots << fold;
            u.parts = min(1 << fold, u.cut.splits - u.split);
            u.tile = u.cut.tiles - 1 - x / slots;
            u.begin = begin_of(u.len - u.n + u.tile * rows_of(FORM) / a->group, a->window) + u.split * u.cut.chunk;
            return true;
        }
        left -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// ---- pieces of both forms -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// 4 x 16 elements of LDS, transposed on the way: in each group of 16 lanes, lane i names the four elements at row i / 4, columns 4 (i % 4) .. + 3
// of the group's block and receives rows 0 .. 3 of column i
__device__ __forceinline__ s16x4 read_transposed(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}
template <typename T>
__device__ __forceinline__ typename Mat<T>::x8 join(s16x4 a, s16x4 b) {
    const s16x8 x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Mat<T>::x8, x);
}

// Halves of a word, both at once: 0x8000 where the magnitude is above `most`
__device__ __forceinline__ uint32_t above(uint32_t w, uint32_t most) { return ((w & 0x7fff7fffu) + (0x7fffu - most) * 0x10001u) & 0x80008000u; }
__device__ __forceinline__ uint32_t word(uint4 w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }

// Values that are not finite, in a tile that not every row sees whole: 0 * inf would give NaN to rows that do not see them.  The finite ones are multiplied;
// then, for each of NaN, inf and -inf, a product of indicators (which elements of V are it, which keys the row sees) counts what a row sees.
// (rest: what the rounding of p has left, where the form multiplies that as well)
template <typename T, bool REST, typename Acc>
__device__ __forceinline__ Acc multiply_seen(typename Mat<T>::x8 v, typename Mat<T>::x8 p, typename Mat<T>::x8 rest, uint32_t seen, Acc o) {
    typedef typename Mat<T>::x8 x8;
    const uint4 w = __builtin_bit_cast(uint4, v);
    uint32_t clean[4], rows[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t y = word(w, i);
        clean[i] = y & ~((above(y, Mat<T>::INF - 1) >> 15) * 0xffffu);
        rows[i] = ((seen >> (2 * i) & 1) | (seen >> (2 * i + 1) & 1) << 16) * Mat<T>::ONE;
    }
    const x8 finite = __builtin_bit_cast(x8, uint4{clean[0], clean[1], clean[2], clean[3]});
    o = Mat<T>::mul(finite, p, o);
    if (REST) o = Mat<T>::mul(finite, rest, o);
    const x8 who = __builtin_bit_cast(x8, uint4{rows[0], rows[1], rows[2], rows[3]});
#pragma unroll 1
    for (int kind = 0; kind < 3; ++kind) {
        uint32_t is[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t y = word(w, i), nan = above(y, Mat<T>::INF), inf = above(y, Mat<T>::INF - 1) & ~nan;
            is[i] = ((kind == 0 ? nan : (kind == 1 ? inf & ~y : inf & y)) >> 15) * Mat<T>::ONE;
        }
        Acc count;
#pragma unroll
        for (int r = 0; r < (int)(sizeof(Acc) / 4); ++r) count[r] = 0;
        count = Mat<T>::mul(__builtin_bit_cast(x8, uint4{is[0], is[1], is[2], is[3]}), who, count);
        const float add = kind == 0 ? __builtin_nanf("") : (kind == 1 ? INFINITY : -INFINITY);
#pragma unroll
        for (int r = 0; r < (int)(sizeof(Acc) / 4); ++r) if (count[r] > 0) o[r] += add;
    }
    __builtin_amdgcn_sched_barrier(0);                             // (one at a time: this path is rare, its registers are not)
    return o;
}

// whether a row's sums hold a NaN or an infinity: what a value that is not finite makes of a row that does not see it (0 * inf) is always one
template <typename Acc, int N>
__device__ __forceinline__ uint32_t not_numbers(const Acc (&o)[N]) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < (int)(sizeof(Acc) / 4); ++r) x = fmaf(o[i][r], 0.f, x);
    return x != x;
}

// What a wave keeps of its rows while it walks along the keys (a lane: of its own row): the maximum in use, in log2 units, and the sum over the keys that
// this lane saw.  The maximum of a tile is not looked for as long as the sum of its probabilities says that the one in use will do: up to
// LIMIT, which fp16 holds (and leaves the fp32 sums of bf16 values up to 2^100 finite).
struct Run {
    float m = -INFINITY, l = 0.f;
    static constexpr float LIMIT = 32768.f;
    __device__ __forceinline__ bool asks(float sum) const { return !(sum <= LIMIT) || m == -INFINITY; }
    // where the row asks for it, takes a new maximum over `top` (log2 units; both the same in all lanes of the row), and returns the factor of what
    // has been summed.  A row goes by its own scores alone.
    __device__ __forceinline__ float raise(bool asked, float top) {
        if (!asked) return 1.f;
        const float now = fmaxf(m, top), back = now == -INFINITY ? 1.f : exp2_of(m - now);
        m = now;
        l *= back;
        return back;
    }
    template <typename T> __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m - Mat<T>::BIAS; }
};

template <typename T> struct Quad { T e[4]; };

// the factor of a part of maximum m and sum l, `top` being the row's maximum; 0: a part that saw no key of the row, and left no numbers
__device__ __forceinline__ float weight_of(float2 ml, float top) { return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_of(ml.x - top); }

// Two parts added: the factors of each, and the sum of a number of each.  (Every rounding is written out: whoever adds rounds alike.)
struct Fold {
    float m, of_sum, of_part;
    __device__ __forceinline__ Fold(float2 sum, float2 part) {
        m = fmaxf(sum.x, part.x);
        of_sum = weight_of(sum, m);
        of_part = weight_of(part, m);
    }
    static __device__ __forceinline__ float add(float of_sum, float sum, float of_part, float part) {
        const float kept = of_sum != 0.f ? of_sum * sum : 0.f;
        return of_part != 0.f ? __builtin_fmaf(of_part, part, kept) : kept;
    }
    static __device__ __forceinline__ f32x4 add(float of_sum, f32x4 sum, float of_part, f32x4 part) {
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = add(of_sum, sum[i], of_part, part[i]);
        return y;
    }
    template <typename T> __device__ __forceinline__ T add(T sum, T part) const { return add(of_sum, sum, of_part, part); }
};

// ---- few rows -------------------------------------------------------------------------------------------------------------------------------
// A wave takes every fourth 32-key tile of the workgroup's range.  Keys go from memory straight into the operand (lane: key lane % 16, 8 elements at
// 32 ks + 8 (lane / 16)); values go through registers into the wave's own piece of LDS, from where they are read transposed.  The next tile's
// loads are in flight under the current tile.  No barrier but for the join of the four waves at the end.  What the rounding of the probabilities
// leaves is multiplied as well: the matrix cores wait for memory here, so it costs nothing, and the error is fp32's.
// Bound by reading the cache: 64 sequences of up to 4 096 keys, 8 key heads of 128, one token each: 125 us for 585 MB, 4.7 TB/s (a large copy: 5.1);
// one sequence of 130 001 keys on two key heads is 128 workgroups: 84 us, of a CU's own latency; one short sequence 9 us, its chain of loads.

// waves of a SIMD: what the registers of the loop allow (a third one at 128 elements would spill, and take twice the time)
constexpr int few_waves(int dp) { return dp <= 32 ? 4 : dp <= 64 ? 3 : dp <= 128 ? 2 : 1; }

template <typename T, int DP> struct Few {
    static constexpr int VROW = DP * 2 + 32;                       // (rows 32 bytes apart in bank phase)
    static constexpr int OROW = DP + 4;                            // floats of a row that is joined
    static constexpr int WAVE = 32 * VROW > 16 * OROW * 4 ? 32 * VROW : 16 * OROW * 4;
};

// One unit.  ODD: the form that keeps values which are not finite, and pages outside the cache, from the rows that do not see them; without it returns whether
// a row has come out not finite, or a page was outside (then the unit is done again with it).  Both add the same products in the same order.
template <typename T, int DP, bool ODD>
__device__ __forceinline__ uint32_t few_unit(ArgsAt a, const Unit& u, char* lds, float (&part_m)[4][16], float (&part_l)[4][16]) {
    typedef typename Mat<T>::x8 x8;
    constexpr int KS = DP / 32, DB = DP / 16, NV = DP / 16, VROW = Few<T, DP>::VROW, OROW = Few<T, DP>::OROW, WAVE = Few<T, DP>::WAVE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
    char* mine = lds + wave * WAVE;
    const int head_bytes = a->dim * 2;
    const int rows = u.n * a->group;
    // this lane's row: its token, its head, its position
    const int row = u.tile * rows_of(FEW) + col, row_in = row < rows ? row : rows - 1;
    const int token = row_in / a->group, head = u.head * a->group + (row_in - token * a->group);
    const int pos = a->causal ? u.len - u.n + token : u.len - 1;
    const int last_token = (min(u.tile * rows_of(FEW) + rows_of(FEW), rows) - 1) / a->group, first_token = u.tile * rows_of(FEW) / a->group;
    const int high = a->causal ? u.len - u.n + last_token : u.len - 1, low = a->causal ? u.len - u.n + first_token : u.len - 1;
    const int begin = u.begin, end = min(min(begin + u.cut.chunk, u.len), high + 1);
    // the keys that this lane's row sees here
    const int first_seen = a->window > 0 ? pos - a->window + 1 : 0;
    const uint32_t count_seen = max(0, min(pos + 1, end) - first_seen);
    x8 q[KS];
    {
        const char* p = a->q + (u.first + token) * a->q_token + head * a->q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint4 w = uint4{0, 0, 0, 0};
            if ((32 * ks + 8 * g) * 2 < head_bytes) w = *(const uint4*)(p + (32 * ks + 8 * g) * 2);
            if (a->negate) { w.x ^= 0x80008000u; w.y ^= 0x80008000u; w.z ^= 0x80008000u; w.w ^= 0x80008000u; }
            q[ks] = __builtin_bit_cast(x8, w);
        }
    }
    f32x4 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x4{0, 0, 0, 0};
    Run run;
    uint32_t odd = 0;
    const int* table = a->table + (long)u.b * a->width;
    const long head_at = u.head * a->head_stride;
    const int slots = (1 << a->page_shift) - 1;
    // pages of the 32 keys of a tile, one a lane (twice)
    auto pages_at = [&](int k0) { return table[min(k0 + (lane & 31), end - 1) >> a->page_shift]; };
    auto at = [&](int page, int key) {
        const int p = (unsigned)page < (unsigned)a->pages ? page : 0;
        return p * a->page_stride + (min(key, end - 1) & slots) * a->slot_stride + head_at;
    };
    uint4 kf[2][KS], vf[NV];
    auto fetch_k = [&](int k0, int pg) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const char* p = a->k + at(__shfl(pg, 16 * t + col), k0 + 16 * t + col);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int byte = (32 * ks + 8 * g) * 2;
                kf[t][ks] = byte < head_bytes ? *(const uint4*)(p + byte) : uint4{0, 0, 0, 0};
            }
        }
    };
    auto fetch_v = [&](int k0, int pg) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int piece = i * 64 + lane, r = piece / (DP / 8), byte = (piece - r * (DP / 8)) * 16;
            const long p = at(__shfl(pg, r), k0 + r);
            vf[i] = byte < head_bytes ? *(const uint4*)(a->v + p + byte) : uint4{0, 0, 0, 0};
        }
    };
    int k0 = begin + 32 * wave, pg = 0, pg_next = 0;
    if (k0 < end) {
        pg = pages_at(k0);
        pg_next = pages_at(k0 + 128);
        fetch_k(k0, pg);
        fetch_v(k0, pg);
    }
    const char* vt = mine + (4 * g + (col >> 2)) * VROW + (col & 3) * 8;
    auto value = [&](int i) { return join<T>(read_transposed(vt + i * 32), read_transposed(vt + 16 * VROW + i * 32)); };
    auto tile = [&](auto masked, uint32_t bad) {
        constexpr bool MASKED = decltype(masked)::value;
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[t] = Mat<T>::mul(__builtin_bit_cast(x8, kf[t][ks]), q[ks], s[t]);
        }
        const bool more = k0 + 128 < end;
        // (loads are waited for in order: the pages of the tile after the next go ahead of the next one's keys and values)
        const int pg_after = pages_at(k0 + 256);
        if (more) fetch_k(k0 + 128, pg_next);
        uint32_t seen = 0;                                         // of this lane's eight keys
        if (MASKED) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int in_tile = 16 * t + 4 * g + r;
                    const bool sees = (uint32_t)(k0 + in_tile - first_seen) < count_seen;
                    if (ODD && sees) seen |= 1u << (4 * t + r);
                    s[t][r] = !sees ? -INFINITY : (ODD && (bad >> in_tile & 1) ? __builtin_nanf("") : s[t][r]);
                }
        }
        x8 p, rest;                                                // (reading the cache bounds this form: the second product of the probabilities' rounding is free)
        float sum;
        auto weights = [&] {
            const float base = run.base<T>();
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = exp2_of(fmaf(s[i / 4][i % 4], a->c, -base));
                sum += e;
                p[i] = (T)e;
                rest[i] = (T)(e - (float)p[i]);
            }
        };
        weights();
        const bool asks = run.asks(sum);
        if (__any(asks)) {
            asm volatile("");                                      // (a branch: not to be computed ahead)
            int asked = asks;
            asked |= __shfl_xor(asked, 16);
            asked |= __shfl_xor(asked, 32);
            float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float back = run.raise(asked != 0, top * a->c);
#pragma unroll
            for (int i = 0; i < DB; ++i) o[i] *= back;
            weights();
        }
        run.l += sum;
        // the tile's values into LDS; a wave's LDS operations take place in order
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int piece = i * 64 + lane, r = piece / (DP / 8), byte = (piece - r * (DP / 8)) * 16;
            *(uint4*)(mine + r * VROW + byte) = vf[i];
        }
        if (more) fetch_v(k0 + 128, pg_next);
        pg = pg_next;
        pg_next = pg_after;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            const x8 v = value(i);
            if (ODD && MASKED) o[i] = multiply_seen<T, true>(v, p, rest, seen, o[i]);
            else o[i] = Mat<T>::mul(v, rest, Mat<T>::mul(v, p, o[i]));
        }
        __builtin_amdgcn_wave_barrier();
    };
    auto walk = [&](auto masked, int stop) {                       // tiles that begin before `stop`
        for (; k0 < stop; k0 += 128) {
            const uint32_t bad = (uint32_t)__ballot((unsigned)pg >= (unsigned)a->pages);
            if (!ODD) odd |= bad;
            tile(masked, bad);
        }
    };
    // tiles that some row sees in part lie before and behind those that all rows see whole
    for (int part = 0; part < 2; ++part) {
        walk(std::true_type(), part || ODD ? end : (a->window > 0 ? min(end, high - a->window + 1) : begin));
        if (!ODD && part == 0) walk(std::false_type(), min(end, low + 1) - 31);
    }
    run.l += __shfl_xor(run.l, 16);
    run.l += __shfl_xor(run.l, 32);
    if (!ODD) odd |= not_numbers(o);
    a = fresh(a);
    // the four waves' rows: o to LDS (over the values), then every thread joins four elements of a row at a time
    float* om = (float*)mine;
#pragma unroll
    for (int i = 0; i < DB; ++i) *(f32x4*)(om + col * OROW + 16 * i + 4 * g) = o[i];
    if (g == 0) { part_m[wave][col] = run.m; part_l[wave][col] = run.l; }
    __syncthreads();
    const bool again = u.cut.splits > 1 && (u.split & ((1 << a->few_fold) - 1));      // not the first part that this workgroup computes of its rows
    auto slot_of = [&](int rr, int t, int h) {
        return part_at(*a, FEW, slots_of(u.cut.splits, a->few_fold), u.b, rr, u.head, t, h) + (u.split >> a->few_fold);
    };
    auto sums_of = [&](int r, float& m, float& l) {
        m = fmaxf(fmaxf(part_m[0][r], part_m[1][r]), fmaxf(part_m[2][r], part_m[3][r]));
        l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = weight_of(float2{part_m[w][r], part_l[w][r]}, m);
            if (f != 0.f) l = __builtin_fmaf(f, part_l[w][r], l);  // (NaN is not 0)
        }
    };
    for (int x = threadIdx.x; x < 16 * (DP / 4); x += 256) {
        const int r = x / (DP / 4), d = (x - r * (DP / 4)) * 4, rr = u.tile * rows_of(FEW) + r;
        if (rr >= rows || d >= a->dim) continue;
        float m, l;
        sums_of(r, m, l);
        f32x4 y = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = weight_of(float2{part_m[w][r], part_l[w][r]}, m);
            if (f != 0.f) {                                        // (0: a wave that saw nothing of the row)
                const f32x4 x = *(const f32x4*)((const float*)(lds + w * WAVE) + r * OROW + d);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(f, x[i], y[i]);
            }
        }
        const int tok = rr / a->group, h = u.head * a->group + (rr - tok * a->group);
        const long t = u.first + tok, at_row = t * a->q_heads + h;
        if (u.cut.splits > 1) {
            const long slot = slot_of(rr, (int)t, h);
            f32x4* to = (f32x4*)(a->part_o + slot * a->dim + d);
            if (again) y = Fold(a->part_ml[slot], float2{m, l}).add(*to, y);
            else if (d == 0) a->part_ml[slot] = float2{m, l};
            *to = y;
        } else {
            const int p = a->causal ? u.len - u.n + tok : u.len - 1;
            const bool none = p < 0;
            const float f = none ? 0.f : 1.f / l;
            Quad<T> z;
#pragma unroll
            for (int i = 0; i < 4; ++i) z.e[i] = (T)(none ? 0.f : y[i] * f);
            *(Quad<T>*)(a->out + t * a->out_token + h * a->out_head + d * 2) = z;
            if (a->lse && d == 0) a->lse[at_row] = none ? -INFINITY : ((m == -INFINITY ? 0.f : m - Mat<T>::BIAS) + log2f(l)) * LN2;
        }
    }
    if (again) {                                                   // (all have read the sums so far)
        __syncthreads();
        const int r = threadIdx.x, rr = u.tile * rows_of(FEW) + r;
        if (r < 16 && rr < rows) {
            const int tok = rr / a->group;
            const long slot = slot_of(rr, u.first + tok, u.head * a->group + (rr - tok * a->group));
            float m, l;
            sums_of(r, m, l);
            const Fold f(a->part_ml[slot], float2{m, l});
            a->part_ml[slot] = float2{f.m, f.add(a->part_ml[slot].y, l)};
        }
    }
    return odd;
}

// The rare form as a function of its own, apart from the kernel's registers.  The kernel hands over where its arguments lie (only a kernel can ask for
// that: in a function the builtin is null).
__device__ __forceinline__ uint64_t kernel_args() { return (uint64_t)__builtin_amdgcn_kernarg_segment_ptr(); }
__device__ __forceinline__ ArgsAt args_at(uint64_t at) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at), hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
    return (ArgsAt)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }
__device__ __forceinline__ char* lds_pointer(uint32_t offset) { return (char*)(__attribute__((address_space(3))) char*)(uintptr_t)offset; }

template <typename T, int DP>
__device__ __noinline__ void few_unit_odd(uint64_t args, int want, uint32_t lds, uint32_t m, uint32_t l) {
    const ArgsAt a = args_at(args);
    Unit u;
    Cursor c{0, 0};
    if (!find_unit<FEW>(a, __builtin_amdgcn_readfirstlane(want), c, u)) return;
    for (; u.parts > 0; --u.parts, ++u.split, u.begin += u.cut.chunk) {
        few_unit<T, DP, true>(a, u, lds_pointer(lds), *(float (*)[4][16])lds_pointer(m), *(float (*)[4][16])lds_pointer(l));
        __syncthreads();
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(256, few_waves(DP)) void cache_attention_few_kernel(AttnArgs) {
    const ArgsAt a = (ArgsAt)__builtin_amdgcn_kernarg_segment_ptr();
    __shared__ __align__(16) char lds[4 * Few<T, DP>::WAVE];
    __shared__ float part_m[4][16], part_l[4][16];
    Cursor c{0, 0};
    for (int want = blockIdx.x;; want += gridDim.x) {
        Unit u;
        if (!find_unit<FEW>(fresh(a), want, c, u)) break;
        int odd = 0;
        for (; u.parts > 0; --u.parts, ++u.split, u.begin += u.cut.chunk) odd |= __syncthreads_or(few_unit<T, DP, false>(fresh(a), u, lds, part_m, part_l) != 0);
        if (odd) few_unit_odd<T, DP>(kernel_args(), want, lds_offset(lds), lds_offset(part_m), lds_offset(part_l));
    }
}

// ---- many rows ------------------------------------------------------------------------------------------------------------------------------
// 16 bytes a lane from memory to LDS at `to` + 16 * lane (of the whole wave; lanes that are off write nothing), without a register in between.  Nothing but
// dma_landed() waits for it.
__device__ __forceinline__ void dma16(const char* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(from), "s"(__builtin_amdgcn_readfirstlane(to)) : "memory", "m0");
}
__device__ __forceinline__ void dma_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Tiles lie in LDS as they come, rows of DP elements without padding (the copy writes 1 KB runs), and which 16-byte piece of a row sits where is
// exchanged instead: such that 16 rows read at one piece (keys), and 4 rows read at 64 bytes (values, transposed), meet every bank once.
template <int DP> __device__ __forceinline__ int key_piece(int row, int piece) {
    return piece ^ (DP % 128 == 0 ? row & 15 : (DP % 64 == 0 ? row >> 1 & 7 : row >> 2 & 3));
}
template <int DP> __device__ __forceinline__ int value_piece(int row, int piece) {
    return piece ^ (DP % 128 == 0 ? (row & 3) << 2 : (DP % 64 == 0 ? (row >> 1 & 1) << 2 : 0));
}

template <int DP> constexpr int tile_keys() { return DP <= 128 ? 64 : 32; }
template <int DP> constexpr int many_lds() { return 4 * tile_keys<DP>() * DP * 2; }

// REST: what the rounding of the probabilities to the cache's type leaves is multiplied as well, as in the form of few rows.  There it costs nothing, here the
// matrix cores have no time left: 2 048 tokens behind 16 384 keys (32 heads of 128 on 8) take 554 us without and 750 with it, chunks of up to 257 over 4 111
// keys (12 heads of 64 on 4) 90 and 104, a window of 1 024 (8 heads of 256 on 2) 57 and 60.  Without it a result is off by half a step of the cache's type
// at most (of the weighted |v|), which is what rounding the result takes anyway (bf16 chunk: 0.0023 instead of 0.0017 over all elements); so the caller
// asks for it.
template <typename T, int DP, int FORM, bool ODD, bool REST>
__device__ __forceinline__ uint32_t many_unit(ArgsAt a, const Unit& u, char* lds) {
    typedef typename Mat<T>::x8 x8;
    constexpr int ROWS = rows_of(FORM), KT = tile_keys<DP>(), SUB = KT / 32, KS = DP / 16, DB = DP / 32, ROW = DP * 2, BUF = KT * ROW, STEP = 32 * ROWS, NP = (BUF + STEP - 1) / STEP;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    const int head_bytes = a->dim * 2;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;      // keys, keys, values, values
    const int rows = u.n * a->group, row0 = u.tile * ROWS + wave * 32;
    const int row = row0 + col, row_in = row < rows ? row : rows - 1;
    const int token = row_in / a->group, head = u.head * a->group + (row_in - token * a->group);
    const int pos = a->causal ? u.len - u.n + token : u.len - 1;
    const bool any_row = row0 < rows;                          // of this wave
    auto pos_of = [&](int r) { return a->causal ? u.len - u.n + min(r, rows - 1) / a->group : u.len - 1; };
    const int low = pos_of(row0), high = pos_of(row0 + 31), tile_low = pos_of(u.tile * ROWS), tile_high = pos_of(u.tile * ROWS + ROWS - 1);
    const int begin = u.begin, end = min(min(begin + u.cut.chunk, u.len), tile_high + 1);
    // the keys that this lane's row sees here
    const int first_seen = a->window > 0 ? pos - a->window + 1 : 0;
    const uint32_t count_seen = max(0, min(pos + 1, end) - first_seen);
    x8 q[KS];
    {
        const char* p = a->q + (u.first + token) * a->q_token + head * a->q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint4 w = uint4{0, 0, 0, 0};
            if ((16 * ks + 8 * h) * 2 < head_bytes) w = *(const uint4*)(p + (16 * ks + 8 * h) * 2);
            if (a->negate) { w.x ^= 0x80008000u; w.y ^= 0x80008000u; w.z ^= 0x80008000u; w.w ^= 0x80008000u; }
            q[ks] = __builtin_bit_cast(x8, w);
        }
    }
    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    Run run;
    uint32_t odd = 0;
    const int* table = a->table + (long)u.b * a->width;
    const long head_at = u.head * a->head_stride;
    const int slots = (1 << a->page_shift) - 1;
    auto pages_at = [&](int k0) { return table[min(k0 + (lane & (KT - 1)), end - 1) >> a->page_shift]; };
    auto fetch = [&](int k0, int pg, int buf) {                // the wave's share of a tile: NP runs of 1 KB of keys and of values
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int at = i * STEP + wave * 1024, x = at + lane * 16, r = x / ROW, piece = (x - r * ROW) / 16;
            if (BUF % STEP && at >= BUF) break;                    // (fewer runs than waves)
            const int page = __shfl(pg, r), p = (unsigned)page < (unsigned)a->pages ? page : 0;
            const long from = p * a->page_stride + (min(k0 + r, end - 1) & slots) * a->slot_stride + head_at;
            const int kp = key_piece<DP>(r, piece) * 16, vp = value_piece<DP>(r, piece) * 16;
            if (kp < head_bytes) dma16(a->k + from + kp, lds_at + buf * BUF + at);
            if (vp < head_bytes) dma16(a->v + from + vp, lds_at + (2 + buf) * BUF + at);
        }
    };
    auto tile = [&](auto masked, int k0, const char* kb, const char* vb, unsigned long long bad) {
        constexpr bool MASKED = decltype(masked)::value;
        f32x16 s[SUB];
        x8 p[SUB][2], rest[SUB][2];                                // (rest: only with REST)
        uint32_t seen[SUB] = {};
        auto scores = [&] {
#pragma unroll
            for (int t = 0; t < SUB; ++t) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const int r = 32 * t + col;
                    s[t] = Mat<T>::mul(*(const x8*)(kb + r * ROW + key_piece<DP>(r, 2 * ks + h) * 16), q[ks], s[t]);
                }
                if (MASKED) {
                    seen[t] = 0;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int in_tile = 32 * t + (r & 3) + 8 * (r >> 2) + 4 * h;
                        const bool sees = (uint32_t)(k0 + in_tile - first_seen) < count_seen;
                        if (ODD && sees) seen[t] |= 1u << r;
                        s[t][r] = !sees ? -INFINITY : (ODD && (bad >> in_tile & 1) ? __builtin_nanf("") : s[t][r]);
                    }
                }
            }
        };
        auto weights = [&] {
            const float base = run.base<T>();
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < SUB; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float e = exp2_of(fmaf(s[t][j], a->c, -base));
                    sum += e;
                    p[t][j >> 3][j & 7] = (T)e;
                    if (REST) rest[t][j >> 3][j & 7] = (T)(e - (float)p[t][j >> 3][j & 7]);
                }
            return sum;
        };
        scores();
        float sum = weights();
        const bool asks = run.asks(sum);
        if (__any(asks)) {
            asm volatile("" ::: "memory");                         // (a branch, and the scores once more rather than kept)
            scores();
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < SUB; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
            top = fmaxf(top, __shfl_xor(top, 32));
            const float back = run.raise(asks | __shfl_xor((int)asks, 32), top * a->c);
#pragma unroll
            for (int i = 0; i < DB; ++i) o[i] *= back;
            sum = weights();
        }
        run.l += sum;
        // element block i (32 elements: 64 bytes), keys 16 m + 4 h + {0..3} and + 8 of sub-tile t
        auto value = [&](int t, int m, int i) {
            const int r = 32 * t + 16 * m + 4 * h + ((lane & 15) >> 2), in_block = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
            return join<T>(read_transposed(vb + r * ROW + value_piece<DP>(r, 4 * i) * 16 + in_block),
                           read_transposed(vb + (r + 8) * ROW + value_piece<DP>(r + 8, 4 * i) * 16 + in_block));
        };
#pragma unroll
        for (int x = 0; x < SUB * 2 * DB; ++x) {
            const int t = x / (2 * DB), m = x / DB % 2, i = x % DB;
            const x8 v = value(t, m, i);
            if (ODD && MASKED) o[i] = multiply_seen<T, REST>(v, p[t][m], rest[t][m], seen[t] >> (8 * m), o[i]);
            else o[i] = Mat<T>::mul(v, p[t][m], o[i]);
            if (REST && !(ODD && MASKED)) o[i] = Mat<T>::mul(v, rest[t][m], o[i]);
        }
    };
    int pg = 0, pg_next = 0;
    if (begin < end) {
        pg = pages_at(begin);
        pg_next = pages_at(begin + KT);
        fetch(begin, pg, 0);
    }
    dma_landed();
    __syncthreads();
    int buf = 0, k0 = begin;
    auto walk = [&](auto masked, int stop) {
        for (; k0 < stop; k0 += KT, buf ^= 1) {
            const unsigned long long bad = __ballot((unsigned)pg >= (unsigned)a->pages);
            if (!ODD) odd |= bad != 0;
            // (the pages of the tile after the next: asked for ahead of the copies, looked at behind dma_landed() - a look in between would wait for the
            // copies as well)
            const int pg_after = pages_at(k0 + 2 * KT);
            if (k0 + KT < end) fetch(k0 + KT, pg_next, buf ^ 1);
            if (any_row && (!decltype(masked)::value || (k0 <= high && (a->window == 0 || k0 + KT - 1 > low - a->window))))
                tile(masked, k0, lds + buf * BUF, lds + (2 + buf) * BUF, bad);
            dma_landed();
            pg = pg_next;
            pg_next = pg_after;
            __syncthreads();
        }
    };
    // tiles that some row of the workgroup sees in part lie before and behind those that all rows see whole
    int whole_from = begin, whole_to = begin;
    if (!ODD) {
        if (a->window > 0) whole_from = min(end, begin + (int)max(0l, ((long)tile_high - a->window - begin + KT) / KT * KT));
        whole_to = begin + max(0, min(end, tile_low + 1) - begin) / KT * KT;
    }
    for (int part = 0; part < 2; ++part) {
        walk(std::true_type(), part ? end : whole_from);
        if (!ODD && part == 0) walk(std::false_type(), whole_to);
    }
    run.l += __shfl_xor(run.l, 32);
    if (!ODD) odd |= not_numbers(o);
    a = fresh(a);
    if (row < rows) {
        const long t = u.first + token, at_row = t * a->q_heads + head;
        if (u.cut.splits > 1) {
            const long slot = part_at(*a, FORM, slots_of(u.cut.splits, a->many_fold), u.b, row, u.head, (int)t, head) + (u.split >> a->many_fold);
            const bool again = u.split & ((1 << a->many_fold) - 1);        // not the first part that this workgroup computes of its rows
            const float2 part = float2{run.m, run.l}, sum = again ? a->part_ml[slot] : float2{-INFINITY, 0.f};
            const Fold f(sum, part);
            if (h == 0) a->part_ml[slot] = again ? float2{f.m, f.add(sum.y, part.y)} : part;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int d = 32 * i + 2 * r + 4 * h;
                    if (d >= a->dim) continue;
                    f32x4* to = (f32x4*)(a->part_o + slot * a->dim + d);
                    const f32x4 y = f32x4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
                    *to = again ? f.add(*to, y) : y;
                }
        } else {
            const bool none = pos < 0;
            const float f = none ? 0.f : 1.f / run.l;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int d = 32 * i + 2 * r + 4 * h;
                    if (d >= a->dim) continue;
                    Quad<T> z;
#pragma unroll
                    for (int j = 0; j < 4; ++j) z.e[j] = (T)(none ? 0.f : o[i][r + j] * f);
                    *(Quad<T>*)(a->out + t * a->out_token + head * a->out_head + d * 2) = z;
                }
            if (a->lse && h == 0) a->lse[at_row] = none ? -INFINITY : (run.base<T>() + log2f(run.l)) * LN2;
        }
    }
    return odd;
}

template <typename T, int DP, int FORM, bool REST>
__device__ __noinline__ void many_unit_odd(uint64_t args, int want, uint32_t lds) {
    const ArgsAt a = args_at(args);
    Unit u;
    Cursor c{0, 0};
    if (!find_unit<FORM>(a, __builtin_amdgcn_readfirstlane(want), c, u)) return;
    for (; u.parts > 0; --u.parts, ++u.split, u.begin += u.cut.chunk) {
        many_unit<T, DP, FORM, true, REST>(a, u, lds_pointer(lds));
        __syncthreads();
    }
}

template <typename T, int DP, int FORM, bool REST>
__global__ __launch_bounds__(2 * rows_of(FORM), DP <= 128 ? 2 : 1) void cache_attention_many_kernel(AttnArgs) {
    const ArgsAt a = (ArgsAt)__builtin_amdgcn_kernarg_segment_ptr();
    extern __shared__ __align__(16) char lds[];
    if (a->dim < DP) {                                             // what lies behind the head's end is never copied: zeros
        for (int x = threadIdx.x * 16; x < many_lds<DP>(); x += 32 * rows_of(FORM)) *(uint4*)(lds + x) = uint4{0, 0, 0, 0};
        __syncthreads();
    }
    Cursor c{0, 0};
    for (int want = blockIdx.x;; want += gridDim.x) {
        Unit u;
        if (!find_unit<FORM>(fresh(a), want, c, u)) break;
        int odd = 0;
        for (; u.parts > 0; --u.parts, ++u.split, u.begin += u.cut.chunk) odd |= __syncthreads_or(many_unit<T, DP, FORM, false, REST>(fresh(a), u, lds) != 0);
        if (odd) many_unit_odd<T, DP, FORM, REST>(kernel_args(), want, lds_offset(lds));
    }
}

// ---- the parts of a row whose keys were split -------------------------------------------------------------------------------------------------
// Groups of eight parts are added up in the order of the keys, and then the groups in theirs, whichever of the two forms joins a row: how a row is
// joined does not depend on the parts that other rows have, nor on how many of them a workgroup has added up before.  Both are bound by latency, the loads
// of a group's parts all under way at once.
//   a few rows of many parts   four waves a row, a group a team of dim / 4 lanes (64 rows of 64 parts of 128: 7 us; 2 048 of 11: 12 us, the other form 7)
//   many rows                  dim / 4 lanes a row, a wave takes 256 / dim heads of a token (10 000 rows of five parts of 64: 12 us)
struct Joined { int b, n, len, first, form, splits, slots; };

__device__ __forceinline__ Joined joined_of(const AttnArgs& a, int t) {
    Joined j{0, 0, 0, 0, 0, 0, 0};
    const int b = j.b = seq_of_token(a.cu_new, a.rows, t);
    if (b >= a.rows) return j;
    j.first = a.cu_new[b];
    j.n = a.cu_new[b + 1] - j.first;
    j.len = clamp_len(a.lens[b], a.width << a.page_shift);
    if (j.first < 0 || j.n < 0 || j.n > a.tokens || j.first > a.tokens - j.n || t < j.first || t >= j.first + j.n) j.n = 0;
    if (j.n > 0) {
        const Cut cut = cut_of(j.n, j.len, a.group, a.kv_heads, a.window, a.dim <= 128, a.few, a.many, a.few_splits, a.many_splits);
        j.form = cut.form;
        j.splits = cut.splits;
        j.slots = slots_of(cut.splits, cut.form == FEW ? a.few_fold : a.many_fold);
    }
    return j;
}
__device__ __forceinline__ long part_at(const AttnArgs& a, const Joined& j, int t, int h) {
    const int kv_head = h / a.group;
    return part_at(a, j.form, j.slots, j.b, (t - j.first) * a.group + h - kv_head * a.group, kv_head, t, h);
}
// the parts that a slot's group has in the workspace: 2^FOLD, or one, their sum
__device__ __forceinline__ int group_of(const AttnArgs& a, const Joined& j) { return (j.form == FEW ? a.few_fold : a.many_fold) ? 1 : 1 << FOLD; }

struct Sum {
    float2 ml; f32x4 y;
    __device__ __forceinline__ void add(bool first, float2 part, f32x4 x) {
        if (first) { ml = part; y = x; return; }
        const Fold f(ml, part);
        y = f.add(y, x);
        ml = float2{f.m, f.add(ml.y, part.y)};
    }
};

template <typename T>
__device__ __forceinline__ void put_joined(const AttnArgs& a, const Joined& j, int t, int h, int d, const Sum& sum) {
    const float m = sum.ml.x, l = sum.ml.y;
    const f32x4 y = sum.y;
    const bool none = a.causal ? j.len - j.n + (t - j.first) < 0 : j.len <= 0;
    const float f = none ? 0.f : 1.f / l;
    Quad<T> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.e[i] = (T)(none ? 0.f : y[i] * f);
    *(Quad<T>*)(a.out + t * a.out_token + h * a.out_head + d * 2) = r;
    if (a.lse && d == 0) a.lse[(long)t * a.q_heads + h] = none ? -INFINITY : ((m == -INFINITY ? 0.f : m - Mat<T>::BIAS) + log2f(l)) * LN2;
}

// (heads: h0 + the lane's of the at_once that a wave takes)
template <typename T>
__device__ __forceinline__ void join_token(const AttnArgs& a, const Joined& j, int t, int h0, int at_once) {
    const int lane = threadIdx.x & 63, quads = a.dim / 4;
    const int h = h0 + lane / quads, d = lane % quads * 4;
    if (lane / quads >= at_once || h >= a.q_heads) return;
    const long slot = part_at(a, j, t, h);
    const int group = group_of(a, j);
    Sum all;
    for (int s0 = 0; s0 < j.slots; s0 += group) {
        float2 ml[8];
        f32x4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < group && s0 + i < j.slots) {
                ml[i] = a.part_ml[slot + s0 + i];
                x[i] = *(const f32x4*)(a.part_o + (slot + s0 + i) * a.dim + d);
            }
        Sum sum;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < group && s0 + i < j.slots) sum.add(i == 0, ml[i], x[i]);
        all.add(s0 == 0, sum.ml, sum.y);
    }
    put_joined<T>(a, j, t, h, d, all);
}

// A wave takes every so-manieth token and passes over all of a sequence whose keys are not split (2 048 tokens of one, nothing to join: 8 us less).
template <typename T>
__global__ __launch_bounds__(256) void cache_attention_join_kernel(AttnArgs a, int waves_a_token) {
    const int at_once = 256 / a.dim, wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int step = (int)(gridDim.x * 4 / waves_a_token), part = wave % waves_a_token;
    int t = wave / waves_a_token;
    if (t >= step) return;
    while (t < a.tokens) {
        const Joined j = joined_of(a, t);
        if (j.b >= a.rows) return;                                 // behind the last sequence
        if (j.splits > 1) join_token<T>(a, j, t, part * at_once, at_once);
        else if (j.n > 0) t += (j.first + j.n - 1 - t) / step * step;
        t += step;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void cache_attention_join_row_kernel(AttnArgs a) {
    __shared__ __align__(16) float sums[8][256];
    const int lane = threadIdx.x & 63, t = blockIdx.x / a.q_heads, h = blockIdx.x - t * a.q_heads;
    const Joined j = joined_of(a, t);
    if (j.splits <= 1) return;
    const long slot = part_at(a, j, t, h);
    const int group = group_of(a, j);
    // a team of dim / 4 lanes adds up a group's eight parts, whose loads go first
    const int quads = a.dim / 4, teams = 256 / quads < 8 ? 256 / quads : 8, team = threadIdx.x / quads, d = (threadIdx.x - team * quads) * 4;
    f32x4 x[8];
    auto load = [&](int g) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (team < teams && i < group && g * group + i < j.slots) x[i] = *(const f32x4*)(a.part_o + (slot + g * group + i) * a.dim + d);
    };
    load(team);
    const float2 ml = lane < j.slots ? a.part_ml[slot + lane] : float2{-INFINITY, 0.f};
    // the factors: a lane follows the sums of its group, and keeps those of its own part; then all follow the groups'
    const int place = group == 1 ? 0 : lane & 7;
    float2 sum = float2{__shfl(ml.x, lane - place), __shfl(ml.y, lane - place)};
    float of_sum = 0.f, of_part = 1.f;
#pragma unroll 1
    for (int i = 1; i < group && i < j.slots; ++i) {
        const float2 part = float2{__shfl(ml.x, lane - place + i), __shfl(ml.y, lane - place + i)};
        if (lane - place + i < j.slots) {
            const Fold f(sum, part);
            if (place == i) { of_sum = f.of_sum; of_part = f.of_part; }
            sum = float2{f.m, f.add(sum.y, part.y)};
        }
    }
    float2 all = float2{__shfl(sum.x, 0), __shfl(sum.y, 0)};
    float of_all[8], of_group[8];
#pragma unroll
    for (int g = 1; g < 8; ++g) {
        if (g * group < j.slots) {
            const float2 part = float2{__shfl(sum.x, g * group), __shfl(sum.y, g * group)};
            const Fold f(all, part);
            of_all[g] = f.of_sum; of_group[g] = f.of_part;
            all = float2{f.m, f.add(all.y, part.y)};
        }
    }
    for (int g0 = 0; g0 < 8; g0 += teams) {                        // (the factors are asked of all lanes: nobody leaves the loop early)
        const int g = g0 + team;
        if (g0) load(g);
        f32x4 y = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            const int s = g * group + i;
            const float fs = __shfl(of_sum, s & 63), fp = __shfl(of_part, s & 63);
            if (i < group && s < j.slots) y = Fold::add(fs, y, fp, x[i]);
        }
        if (team < teams && g < 8 && g * group < j.slots) *(f32x4*)&sums[g][d] = y;
    }
    __syncthreads();
    if ((int)threadIdx.x >= quads) return;
    f32x4 y = *(const f32x4*)&sums[0][d];
#pragma unroll
    for (int g = 1; g < 8; ++g) if (g * group < j.slots) y = Fold::add(of_all[g], y, of_group[g], *(const f32x4*)&sums[g][d]);
    put_joined<T>(a, j, t, h, d, Sum{all, y});
}

// More workgroups than are resident at once: under a causal mask tiles differ in length, and the next one, the longest that is left, goes where one has
// ended (8 192 tokens of 32 heads of 128 on 8: 657 us with 256 workgroups of the large form, 583 with 1 024, as with 2 048, of which more lie idle in
// a call of short sequences: the bound on units is the host's).
unsigned grid_for(long units, long most) { return (unsigned)(units < 1 ? 1 : (units < most ? units : most)); }

template <typename T, int DP, int FORM, bool REST>
int run_many(const AttnArgs& a, long units, hipStream_t s) {
    static_assert(many_lds<DP>() <= 65536, "more LDS has to be asked for");
    cache_attention_many_kernel<T, DP, FORM, REST><<<grid_for(units, 1024), 2 * rows_of(FORM), many_lds<DP>(), s>>>(a);
    DISCO_LAUNCH_CHECK("cache_attention_many_kernel");
    return DISCO_OK;
}
// (units: 0 is no launch)
template <typename T, int DP, bool REST>
int run_many_forms(const AttnArgs& a, long many_units, long large_units, hipStream_t s) {
    if constexpr (DP > 64 && DP <= 128) {
        if (large_units) if (int rc = run_many<T, DP, LARGE, REST>(a, large_units, s)) return rc;
    }
    if (many_units) if (int rc = run_many<T, DP, MANY, REST>(a, many_units, s)) return rc;
    return DISCO_OK;
}

#ifdef DISCO_CACHE_PRECISE
template <typename T>
int run_precise(const AttnArgs& a, long many_units, long large_units, hipStream_t s) {
    if (a.dim <= 32) return run_many_forms<T, 32, true>(a, many_units, large_units, s);
    if (a.dim <= 64) return run_many_forms<T, 64, true>(a, many_units, large_units, s);
    if (a.dim <= 96) return run_many_forms<T, 96, true>(a, many_units, large_units, s);
    if (a.dim <= 128) return run_many_forms<T, 128, true>(a, many_units, large_units, s);
    if (a.dim <= 192) return run_many_forms<T, 192, true>(a, many_units, large_units, s);
    return run_many_forms<T, 256, true>(a, many_units, large_units, s);
}

}  // namespace

int launch_cache_attention_precise(const void* args, bool half, long many_units, long large_units, hipStream_t s) {
    const AttnArgs& a = *(const AttnArgs*)args;
    return half ? run_precise<f16>(a, many_units, large_units, s) : run_precise<bf16>(a, many_units, large_units, s);
}
#else
// ---- what the host decides ----------------------------------------------------------------------------------------------------------------------
constexpr int FEW_LIMIT = 16, MANY_LIMIT = 1024;
constexpr long ROOM = 512l << 20;

struct Plan {
    bool few, many, large;             // which forms are launched
    int few_limit, many_limit;         // rows (INT_MAX: all)
    int few_splits, many_splits;       // a row's parts, at most
    int few_fold, many_fold;
    bool few_by_sequence;
    int many_room;
    long few_parts, many_parts;        // in the workspace
    long few_units, many_units, large_units;
};

Plan plan_of(const disco_cache_desc& c, const disco_attention_desc& d) {
    Plan p;
    const long capacity = (long)c.table_width * c.page_size;
    const int group = d.q_heads / c.kv_heads;
    const int len = (int)(d.max_len > 0 && d.max_len < capacity ? d.max_len : capacity);
    const int most_new = d.max_new > 0 && d.max_new < d.tokens ? d.max_new : d.tokens;
    // Every form that a sequence of up to so many rows may ask for is launched, also where there is one sequence: it may have fewer new tokens than
    // the call has rows.  Where the caller says that it has as many, one form is enough (a launch that finds nothing takes 5 us: 2 048 tokens behind 16 384
    // 553 us, with the launches of all forms and a join 566, a fresh prompt of 2 048 tokens 76 and 91, 33 tokens over 4 096 43 and 48).
    const bool narrow = c.dim <= 128, alone = c.rows == 1 && d.max_new == d.tokens;
    const long most_rows = (long)most_new * group;
    p.large = most_rows > MANY_LIMIT && c.dim > 64 && narrow;
    p.many = most_rows > FEW_LIMIT && !(alone && p.large);
    p.few = !(alone && most_rows > FEW_LIMIT);
    p.few_limit = most_rows <= FEW_LIMIT ? 0x7fffffff : (p.few ? FEW_LIMIT : 0);
    p.many_limit = !p.large ? 0x7fffffff : (p.many ? MANY_LIMIT : 0);
    p.few_splits = p.many_splits = 1;
    // (of the longest sequence: a part more or less because of the others in a call would show in the last bit)
    const long far = (long)d.window + 63 + rows_of(LARGE);
    const int keys = d.window > 0 && far < len ? (int)far : len;
    if (p.few) p.few_splits = splits_of(FEW, 1, 1, keys, c.kv_heads, narrow);
    if (p.many || p.large) {
        const int form = alone && p.large ? LARGE : MANY, tile = rows_of(form), tiles = (int)((most_rows + tile - 1) / tile);
        p.many_splits = alone ? splits_of(form, (int)most_rows, tiles, keys, c.kv_heads, narrow)
                              : std::max(splits_of(MANY, 1, 1, keys, c.kv_heads, narrow), narrow && keys >= 16384 ? 2 : 1);
    }
    // Room for the parts: of every token's rows, or where that is less of every sequence's, which has at most FEW_LIMIT rows a key head there, and here, where
    // its keys are split, at most 65 536 parts of rows (tiles * key heads * parts <= 512 of 128 rows, or 256 of 256) or two of each row of < 512 tiles.
    // Where a form would take more than ROOM bytes, and less than half of that with one slot a group, its workgroups compute whole groups of parts; there are
    // sequences enough then to fill the GPU.  32 heads of 128 on 8, tables of 32 768, no bound on the lengths: 256 sequences of 17 tokens over 2 000 keys 649 us
    // and 0.7 GB (a slot a part: 625 and 5.8), 1 000 single tokens over 1 024 983 us and 0.27 GB (929 and 2.1).  One long sequence among many pays most: 300 of
    // 500 keys and one of 65 536, 0.3 GB, 200 us as it is, in groups 287; so ROOM is not smaller.
    const long rows = (long)d.tokens * group, heads = (long)d.tokens * d.q_heads;
    p.few_by_sequence = p.few_limit == FEW_LIMIT && (long)c.rows * c.kv_heads * FEW_LIMIT < heads;
    const long bytes = (long)c.dim * 4 + 8, few_rows = p.few_by_sequence ? (long)c.rows * c.kv_heads * FEW_LIMIT : heads;
    p.few_fold = few_rows * p.few_splits * bytes > ROOM ? FOLD : 0;
    p.few_parts = p.few_splits > 1 ? few_rows * slots_of(p.few_splits, p.few_fold) : 0;
    const long twice = 2 * c.kv_heads * (p.large ? MANY_LIMIT : rows);
    const int room = twice <= 65536 ? 65536 : (twice < 131072 ? (int)twice : 131072);
    const auto many = [&](int fold) {                              // (the two parts of a row of < 512 tiles are one slot)
        return std::min((long)c.rows * (fold ? 65536 : room), heads * slots_of(p.many_splits, fold));
    };
    p.many_fold = many(0) * bytes > ROOM && 2 * many(FOLD) <= many(0) ? FOLD : 0;
    p.many_parts = p.many_splits > 1 ? many(p.many_fold) : 0;
    p.many_room = many(p.many_fold) < heads * slots_of(p.many_splits, p.many_fold) ? (p.many_fold ? 65536 : room) : 0;
    const long some = c.rows < d.tokens ? c.rows : d.tokens;
    p.few_units = (some + (p.few_limit == FEW_LIMIT ? 0 : rows / rows_of(FEW))) * p.few_splits * c.kv_heads;      // (at most FEW_LIMIT rows are one tile)
    p.many_units = (some + rows / rows_of(MANY)) * p.many_splits * c.kv_heads;
    p.large_units = (some + rows / rows_of(LARGE)) * p.many_splits * c.kv_heads;
    return p;
}

template <typename T, int DP>
int run_forms(const AttnArgs& a, const Plan& p, bool precise, hipStream_t s) {
    const long many_units = p.many ? std::max(p.many_units, 1l) : 0, large_units = p.large ? std::max(p.large_units, 1l) : 0;
    if (int rc = precise ? launch_cache_attention_precise(&a, std::is_same<T, f16>::value, many_units, large_units, s)
                         : run_many_forms<T, DP, false>(a, many_units, large_units, s)) return rc;
    if (p.few) {
        cache_attention_few_kernel<T, DP><<<grid_for(p.few_units, 256 * few_waves(DP)), 256, 0, s>>>(a);
        DISCO_LAUNCH_CHECK("cache_attention_few_kernel");
    }
    if (p.few_parts + p.many_parts > 0) {
        const long rows = (long)a.tokens * a.q_heads;
        if ((p.few_splits > 16 || p.many_splits > 16) && rows <= 2048) cache_attention_join_row_kernel<T><<<(unsigned)rows, 256, 0, s>>>(a);
        else {
            const int waves_a_token = cdiv(a.q_heads, 256 / a.dim);
            const long most = cdiv(waves_a_token, 4) > 2048 ? cdiv(waves_a_token, 4) : 2048;      // (a wave for each part of a token at least)
            cache_attention_join_kernel<T><<<grid_for(((long)a.tokens * waves_a_token + 3) / 4, most), 256, 0, s>>>(a, waves_a_token);
        }
        DISCO_LAUNCH_CHECK("cache_attention_join_kernel");
    }
    return DISCO_OK;
}

template <typename T>
int run_dims(const AttnArgs& a, const Plan& p, bool precise, hipStream_t s) {
    if (a.dim <= 32) return run_forms<T, 32>(a, p, precise, s);
    if (a.dim <= 64) return run_forms<T, 64>(a, p, precise, s);
    if (a.dim <= 96) return run_forms<T, 96>(a, p, precise, s);
    if (a.dim <= 128) return run_forms<T, 128>(a, p, precise, s);
    if (a.dim <= 192) return run_forms<T, 192>(a, p, precise, s);
    return run_forms<T, 256>(a, p, precise, s);
}

}  // namespace

size_t cache_attention_ws_bytes(const disco_cache_desc& c, const disco_attention_desc& d) {
    const Plan p = plan_of(c, d);
    return (size_t)(p.few_parts + p.many_parts) * ((size_t)c.dim * 4 + 8);
}

int launch_cache_attention(const disco_cache_desc& c, const disco_attention_desc& d, const void* q, const int* table, const int* lens,
                           const int* cu_new, void* out, float* lse, void* ws, bool precise, hipStream_t s) {
    const Plan p = plan_of(c, d);
    const size_t parts = (size_t)(p.few_parts + p.many_parts);
    const int window = d.window >= (long)c.table_width * c.page_size ? 0 : d.window;      // (no key is that far back)
    AttnArgs a{(const char*)q, (const char*)c.d_k, (const char*)c.d_v, (char*)out, lse, (float*)ws, (float2*)((char*)ws + parts * c.dim * 4),
               table, lens, cu_new, d.q_token * 2, d.q_head * 2, d.out_token * 2, d.out_head * 2, c.page_stride * 2, c.head_stride * 2, c.slot_stride * 2,
               d.tokens, d.q_heads, c.kv_heads, d.q_heads / c.kv_heads, c.dim, c.rows, c.table_width, c.pages, __builtin_ctz((unsigned)c.page_size), d.causal,
               window, p.few_splits, p.many_splits, p.few_by_sequence, p.few_fold, p.many_fold, p.many_room, p.few_parts, p.few_limit, p.many_limit, fabsf(d.scale) * 1.4426950408889634f, d.scale < 0};
    if (a.c < 1e-37f) a.c = 1e-37f;                                // 0 * -inf is not the score of a key that is not seen
    return c.dtype == DISCO_F16 ? run_dims<f16>(a, p, precise, s) : run_dims<bf16>(a, p, precise, s);
}
#endif

}  // namespace disco
