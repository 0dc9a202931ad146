// sample.hip -- one token a row from logits: temperature, top-k, top-p, min-p and a
// given random number.
//
// The row's tokens are ordered by (logit descending, index ascending); every step keeps
// a run of that order's start, and the draw inverts the summed weights exp((x - max) / T)
// along it.  Nothing sorts the row: one pass collects its largest logits, a few hundred,
// and where they do not decide, the weights of all are summed by bins and only the bins
// that a border lies in are resolved.
//
//   collect  each thread's first logits stay in registers; the k-th smallest of the
//            threads' best bounds the row's k-th logit from below, so what lies under
//            it is passed over, in registers and in the rest of the row that streams by.
//            Without top-k the passed weights are summed in 64 bits, in an order that
//            the sizes fix.
//   finish   the collected tokens sorted, their weights summed along; every border and
//            the draw are looked for there.
//   borders  where they lie below the collected ones (a flat row, a large top-k): the
//            weights as whole numbers of 2^-44 of the first's, whose sums do not depend
//            on the order of atomics.
//
// Few rows are collected by several workgroups each (k_sample_part) and finished by one.
#include "common.h"

#include <algorithm>

namespace ds3k {

constexpr int SMP_TPB = 1024;
constexpr int SMP_BINS = 2048;               // bins of 1 / 64 over 32, the last of all beyond
constexpr int SMP_LIST = 4096;               // tokens sorted at once
constexpr int SMP_HELD = 8;                  // groups of four logits that a thread holds
constexpr int SMP_TOP_K = 512;               // top_k up to which `collect` decides
constexpr int SMP_OPEN = 256;                // tokens that it looks for without top_k
constexpr double SMP_ONE = 0x1p44;           // the first token's weight in whole numbers

constexpr int PART_LIST = 1024;              // tokens that a part of a row hands on
constexpr int PART_MOST = 16;                // parts of a row

typedef unsigned long long u64;

// Ascending order of these 32 bits is descending order of values; -0 is 0.
__device__ __forceinline__ uint32_t order_key(float x)
{
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? b : 0x7fffffffu - b;
}

__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k : 0x7fffffffu - k); }
__device__ __forceinline__ float token_value(u64 token) { return key_value((uint32_t)(token >> 32)); }
__device__ __forceinline__ u64 token_of(float x, int i) { return (u64)order_key(x) << 32 | (uint32_t)i; }
__device__ __forceinline__ bool counts(float v) { return v > -INFINITY; }      // neither -inf nor NaN

struct SampleShared {
    u64 weight[SMP_BINS];                    // by bin
    uint32_t count[SMP_BINS];
    u64 list[SMP_LIST];                      // key << 32 | index
    u64 wave_w[SMP_TPB / 64];
    double wave_d[SMP_TPB / 64];
    uint32_t wave_c[SMP_TPB / 64];
    u64 best;
    uint32_t n;                              // tokens pushed, those beyond the list too
    int bin;
    u64 found[4];
    double mass;
};

// A row's settings.
struct Draw {
    float t, p, m, u;
    int k;
};

__device__ __forceinline__ Draw settings(const SampleArgs &a, int r)
{
    Draw d;
    d.t = a.temperature ? a.temperature[r] : 1.0f;
    d.p = a.top_p ? a.top_p[r] : 1.0f;
    d.m = a.min_p ? a.min_p[r] : 0.0f;
    d.k = a.top_k ? max(a.top_k[r], 0) : 0;
    if (d.k >= a.n_vocab) d.k = 0;           // (all)
    const float u = a.uniform[r];
    d.u = u > 0.0f ? u : 0.0f;
    return d;
}

// Inclusive sums over the workgroup, and those of all.
__device__ __forceinline__ void scan2(SampleShared &sh, u64 &w, uint32_t &c, u64 &w_all, uint32_t &c_all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d *= 2) {
        const u64 a = __shfl_up(w, d);
        const uint32_t b = __shfl_up(c, d);
        if (lane >= d) {
            w += a;
            c += b;
        }
    }
    __syncthreads();
    if (lane == 63) {
        sh.wave_w[wave] = w;
        sh.wave_c[wave] = c;
    }
    __syncthreads();
    w_all = 0;
    c_all = 0;
    u64 before_w = 0;
    uint32_t before_c = 0;
    for (int i = 0; i < SMP_TPB / 64; i++) {
        if (i == wave) {
            before_w = w_all;
            before_c = c_all;
        }
        w_all += sh.wave_w[i];
        c_all += sh.wave_c[i];
    }
    w += before_w;
    c += before_c;
}

__device__ __forceinline__ double scan_f64(SampleShared &sh, double &v)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d *= 2) {
        const double a = __shfl_up(v, d);
        if (lane >= d) v += a;
    }
    __syncthreads();
    if (lane == 63) sh.wave_d[wave] = v;
    __syncthreads();
    double all = 0.0, before = 0.0;
    for (int i = 0; i < SMP_TPB / 64; i++) {
        if (i == wave) before = all;
        all += sh.wave_d[i];
    }
    v += before;
    return all;
}

// A row, read in groups of four that start on multiples of 16 bytes: group q holds logits 4 q - shift .. + 3.
struct Row {
    const float *x;
    int n, shift, groups;
    double top, inv_t;                       // the largest logit, 1 / temperature

    __device__ void bind(const SampleArgs &a, int r)
    {
        x = (const float *)((const uint8_t *)a.logits + (uint64_t)r * a.stride);
        n = a.n_vocab;
        shift = (int)((uintptr_t)x >> 2 & 3);
        groups = (n + shift + 3) / 4;
    }
    __device__ float4 load(int q) const
    {
        const int i = 4 * q - shift;
        if (i >= 0 && i + 4 <= n) return *(const float4 *)(x + i);
        const float none = -INFINITY;
        float4 v = { none, none, none, none };
        if (i >= 0 && i < n) v.x = x[i];
        if (i + 1 >= 0 && i + 1 < n) v.y = x[i + 1];
        if (i + 2 >= 0 && i + 2 < n) v.z = x[i + 2];
        if (i + 3 >= 0 && i + 3 < n) v.w = x[i + 3];
        return v;
    }
    __device__ int index(int q, int j) const { return 4 * q - shift + j; }

    __device__ double depth(float v) const { return (top - (double)v) * inv_t; }
    __device__ int bin(float v) const
    {
        const double b = depth(v) * 64.0;
        return b < SMP_BINS - 1 ? (int)b : SMP_BINS - 1;
    }
    __device__ double weight(float v) const { return exp(-depth(v)); }
    __device__ u64 units(float v) const { return (u64)__double2ll_rn(weight(v) * SMP_ONE); }

    // f(value, index) of every logit of groups [q0, q1), four groups a thread in flight
    template <typename F>
    __device__ void each(int q0, int q1, F f) const
    {
        for (int q = q0 + threadIdx.x; q < q1; q += 4 * SMP_TPB) {
            float4 v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = q + i * SMP_TPB < q1 ? load(q + i * SMP_TPB) : float4{ NAN, NAN, NAN, NAN };
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int g = q + i * SMP_TPB;
                f(v[i].x, index(g, 0));
                f(v[i].y, index(g, 1));
                f(v[i].z, index(g, 2));
                f(v[i].w, index(g, 3));
            }
        }
    }
};

__device__ __forceinline__ void clear_bins(SampleShared &sh)
{
    __syncthreads();
    for (int b = threadIdx.x; b < SMP_BINS; b += SMP_TPB) {
        sh.weight[b] = 0;
        sh.count[b] = 0;
    }
    __syncthreads();
}

// In the counts by bin: the bin at which they reach `least` (sh.bin), those before it and in it (sh.found[1], [2]).
// False: all counts together do not.
__device__ __forceinline__ bool count_border(SampleShared &sh, uint32_t least)
{
    __syncthreads();
    const int b = 2 * threadIdx.x;
    const uint32_t x = sh.count[b], y = sh.count[b + 1];
    u64 w = 0, w_all;
    uint32_t c = x + y, all;
    scan2(sh, w, c, w_all, all);
    if (c >= least && c - x - y < least) {
        const bool first = c - y >= least;
        sh.bin = b + (first ? 0 : 1);
        sh.found[1] = first ? c - x - y : c - y;
        sh.found[2] = first ? x : y;
    }
    __syncthreads();
    return all >= least;
}

// A key that at least `least` of the threads' keys do not pass (22 bits of it decided; 0xffffffff: fewer
// threads have one).  Threads without a key give 0xffffffff.
__device__ uint32_t key_bound(SampleShared &sh, uint32_t key, int least)
{
    clear_bins(sh);
    if (key != 0xffffffffu) atomicAdd(&sh.count[key >> 21], 1u);
    if (!count_border(sh, (uint32_t)least)) return 0xffffffffu;
    const uint32_t high = (uint32_t)sh.bin, before = (uint32_t)sh.found[1];
    clear_bins(sh);
    if (key != 0xffffffffu && key >> 21 == high) atomicAdd(&sh.count[key >> 10 & 2047], 1u);
    count_border(sh, (uint32_t)least - before);
    return high << 21 | (uint32_t)sh.bin << 10 | 1023u;
}

__device__ __forceinline__ void push(SampleShared &sh, u64 token)
{
    const uint32_t at = atomicAdd(&sh.n, 1u);
    if (at < SMP_LIST) sh.list[at] = token;
}

// The best token of each thread, of all.
__device__ __forceinline__ u64 best_of(SampleShared &sh, u64 best)
{
    for (int d = 32; d > 0; d /= 2) best = min(best, (u64)__shfl_xor(best, d));
    __syncthreads();
    if (threadIdx.x == 0) sh.best = ~0ull;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) atomicMin(&sh.best, best);
    __syncthreads();
    return sh.best;
}

// One pass over groups [q0, q1): sh.list gets (sh.n tells how many, perhaps more than fit) at least the `least`
// best tokens, or all; returns the best.  with_rest: sum of the other tokens' weights relative to `ref`, a logit.
__device__ u64 collect(SampleShared &sh, const Row &row, int q0, int q1, int least, bool with_rest, double inv_t, double &rest,
                       float &ref)
{
    float4 held[SMP_HELD];
#pragma unroll
    for (int i = 0; i < SMP_HELD; i++) {
        const int q = q0 + threadIdx.x + i * SMP_TPB;
        held[i] = q < q1 ? row.load(q) : float4{ NAN, NAN, NAN, NAN };
    }
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < SMP_HELD; i++) most = fmaxf(fmaxf(fmaxf(most, held[i].x), fmaxf(held[i].y, held[i].z)), held[i].w);
    const uint32_t mine = counts(most) ? order_key(most) : 0xffffffffu;
    if (threadIdx.x == 0) sh.n = 0;
    // (the first of the best keys serves as reference: any of them would, near the row's largest)
    const uint32_t bound = key_bound(sh, mine, least);
    const u64 first = best_of(sh, (u64)mine << 32);
    ref = first >> 32 == 0xffffffffu ? 0.0f : token_value(first);
    u64 best = ~0ull;
    double sum = 0.0;
    const double at = (double)ref;
    const auto take = [&](float v, int i) {
        if (!counts(v)) return;
        const uint32_t key = order_key(v);
        if (key <= bound) {
            const u64 token = (u64)key << 32 | (uint32_t)i;
            best = min(best, token);
            push(sh, token);
        } else if (with_rest) sum += exp(((double)v - at) * inv_t);
    };
#pragma unroll
    for (int i = 0; i < SMP_HELD; i++) {
        const int q = q0 + threadIdx.x + i * SMP_TPB;
        take(held[i].x, row.index(q, 0));
        take(held[i].y, row.index(q, 1));
        take(held[i].z, row.index(q, 2));
        take(held[i].w, row.index(q, 3));
    }
    row.each(q0 + SMP_HELD * SMP_TPB, q1, take);
    best = best_of(sh, best);
    if (with_rest) rest = scan_f64(sh, sum);
    __syncthreads();
    return best;
}

// Tokens of sh.list[0 .. n) in order.
__device__ void sort_list(SampleShared &sh, int n)
{
    const int tid = threadIdx.x;
    int size = 64;
    while (size < n) size *= 2;
    __syncthreads();
    for (int i = n + tid; i < size; i += SMP_TPB) sh.list[i] = ~0ull;
    __syncthreads();
    if (size <= SMP_TPB) {
        // a token a thread: steps of up to 32 within the wave
        u64 v = tid < size ? sh.list[tid] : ~0ull;
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                u64 o;
                if (j >= 64) {
                    __syncthreads();
                    if (tid < size) sh.list[tid] = v;
                    __syncthreads();
                    o = tid < size ? sh.list[tid ^ j] : v;
                } else o = __shfl_xor(v, j);
                const bool low = (tid & j) == 0, up = (tid & k) == 0;
                v = (low == up) == (o < v) ? o : v;
            }
        __syncthreads();
        if (tid < size) sh.list[tid] = v;
    } else {
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                for (int i = tid; i < size / 2; i += SMP_TPB) {
                    const int a = 2 * i - (i & (j - 1)), b = a + j;      // the pairs whose bit j differs
                    const u64 x = sh.list[a], y = sh.list[b];
                    if ((x > y) == ((a & k) == 0)) {
                        sh.list[a] = y;
                        sh.list[b] = x;
                    }
                }
                __syncthreads();
            }
    }
    __syncthreads();
}

__device__ __forceinline__ void answer(const SampleArgs &a, int r, int token, float share)
{
    a.tokens[r] = token;
    if (a.probs) a.probs[r] = share;
}

// The draw from sh.list[0 .. n), n > 0: with top_k at least the k best tokens of the row, else its best n, the others'
// weights summing to `rest` of the first's.  False: they do not decide.
__device__ bool finish(SampleShared &sh, const SampleArgs &a, int r, const Draw &d, const Row &row, int n, double rest)
{
    const int tid = threadIdx.x;
    if (d.k > 0 && n > d.k + 64) {
        // only the k best need sorting: a bound for them by counts, the others dropped
        u64 held[SMP_LIST / SMP_TPB];
        uint32_t high = 0, before = 0;
#pragma unroll
        for (int i = 0; i < SMP_LIST / SMP_TPB; i++) held[i] = tid + i * SMP_TPB < n ? sh.list[tid + i * SMP_TPB] : ~0ull;
#pragma unroll
        for (int step = 0; step < 2; step++) {
            clear_bins(sh);
#pragma unroll
            for (int i = 0; i < SMP_LIST / SMP_TPB; i++) {
                const uint32_t key = (uint32_t)(held[i] >> 32);
                if (held[i] != ~0ull && (step == 0 || key >> 21 == high)) atomicAdd(&sh.count[step == 0 ? key >> 21 : key >> 10 & 2047], 1u);
            }
            count_border(sh, (uint32_t)d.k - before);
            if (step == 0) {
                high = (uint32_t)sh.bin;
                before = (uint32_t)sh.found[1];
            }
        }
        const uint32_t bound = high << 21 | (uint32_t)sh.bin << 10 | 1023u;
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SMP_LIST / SMP_TPB; i++)
            if (held[i] != ~0ull && (uint32_t)(held[i] >> 32) <= bound) push(sh, held[i]);
        __syncthreads();
        n = (int)sh.n;
    }
    sort_list(sh, n);
    if (d.k > 0) n = min(n, d.k);
    // weights, and their sums up to and with each
    constexpr int BLOCKS = SMP_LIST / SMP_TPB;
    double own[BLOCKS], upto[BLOCKS], mass = 0.0;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
        own[b] = upto[b] = 0.0;
        if (b * SMP_TPB < n) {
            const int i = b * SMP_TPB + tid;
            own[b] = i < n ? row.weight(token_value(sh.list[i])) : 0.0;
            double w = own[b];
            const double sum = scan_f64(sh, w);
            upto[b] = mass + w;
            mass += sum;
        }
    }
    const bool complete = d.k > 0 || rest == 0.0;
    if (!complete) mass += rest;
    constexpr int NONE = 0x7fffffff;
    __syncthreads();
    if (tid == 0) {
        sh.bin = NONE;                       // tokens kept, where a border decides it
        sh.n = NONE;                         // the drawn token's place
    }
    __syncthreads();
    if (d.p < 1.0f) {
        const double least = (double)fmaxf(d.p, 0.0f) * mass;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            const int i = b * SMP_TPB + tid;
            if (i < n && upto[b] >= least) atomicMin(&sh.bin, i + 1);
        }
        __syncthreads();
        if (sh.bin == NONE && !complete) return false;
    }
    if (d.m > 0.0f) {
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            const int i = b * SMP_TPB + tid;
            if (i > 0 && i < n && own[b] < (double)d.m) atomicMin(&sh.bin, i);
        }
        __syncthreads();
        if (sh.bin == NONE && !complete) return false;
    }
    const bool open = sh.bin == NONE && !complete;           // the kept ones go on below the list
    const int kept = min(sh.bin, n);
#pragma unroll
    for (int b = 0; b < BLOCKS; b++)
        if (b * SMP_TPB + tid == kept - 1) sh.mass = open ? mass : upto[b];
    __syncthreads();
    const double total = sh.mass, target = (double)d.u * total;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
        const int i = b * SMP_TPB + tid;
        if (i < kept && upto[b] > target) atomicMin(&sh.n, (uint32_t)i);
    }
    __syncthreads();
    if (sh.n == NONE && open) return false;
    const int at = min((int)sh.n, kept - 1);
#pragma unroll
    for (int b = 0; b < BLOCKS; b++)
        if (b * SMP_TPB + tid == at) answer(a, r, (int)(uint32_t)sh.list[at], (float)(own[b] / total));
    return true;
}

// ---------------------------------------------------------------------------
// Borders below the collected tokens.
// ---------------------------------------------------------------------------

// What a border is looked for by: the first token in order whose inclusive count or weight reaches `least`.
enum : int { BY_COUNT, BY_WEIGHT };

// Where a border lies: the token, and the weights up to and with it.
struct Border {
    u64 token;
    u64 mass;
};

// The token of bin `bin` at which the inclusive sum, from (w0, c0) before the bin, reaches `least`.
__device__ Border resolve(SampleShared &sh, const Row &row, int bin, u64 w0, uint32_t c0, int by, u64 least)
{
    // the bin's tokens are narrowed by digits of key << 32 | index until they can be sorted
    u64 prefix = 0, mask = 0;
    int shift = 64, n;
    for (;;) {
        __syncthreads();
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        row.each(0, row.groups, [&](float v, int i) {
            if (!counts(v) || row.bin(v) != bin) return;
            const u64 c = token_of(v, i);
            if ((c & mask) == prefix) push(sh, c);
        });
        __syncthreads();
        n = (int)sh.n;
        if (n <= SMP_LIST) break;
        const int bits = min(11, shift);
        shift -= bits;
        clear_bins(sh);
        row.each(0, row.groups, [&](float v, int i) {
            if (!counts(v) || row.bin(v) != bin) return;
            const u64 c = token_of(v, i);
            if ((c & mask) != prefix) return;
            const int d = (int)(c >> shift) & ((1 << bits) - 1);
            atomicAdd(&sh.weight[d], row.units(v));
            atomicAdd(&sh.count[d], 1u);
        });
        __syncthreads();
        const int d0 = threadIdx.x * 2;
        const u64 wa = sh.weight[d0], wb = sh.weight[d0 + 1];
        const uint32_t ca = sh.count[d0], cb = sh.count[d0 + 1];
        u64 w = wa + wb, w_all;
        uint32_t c = ca + cb, c_all;
        scan2(sh, w, c, w_all, c_all);
        w += w0;
        c += c0;
        const u64 got = by == BY_COUNT ? c : w, was = by == BY_COUNT ? c - ca - cb : w - wa - wb,
                  mid = by == BY_COUNT ? c - cb : w - wb;
        if (got >= least && was < least) {
            const bool first = mid >= least;
            sh.found[0] = d0 + (first ? 0 : 1);
            sh.found[1] = first ? w - wa - wb : w - wb;
            sh.found[2] = first ? c - ca - cb : c - cb;
        }
        __syncthreads();
        prefix |= sh.found[0] << shift;
        mask |= (u64)((1 << bits) - 1) << shift;
        w0 = sh.found[1];
        c0 = (uint32_t)sh.found[2];
    }
    sort_list(sh, n);
    for (int i0 = 0; i0 < n; i0 += SMP_TPB) {
        const int i = i0 + threadIdx.x;
        const u64 own = i < n ? row.units(token_value(sh.list[i])) : 0;
        u64 w = own, w_all;
        uint32_t c = i < n, c_all;
        scan2(sh, w, c, w_all, c_all);
        w += w0;
        c += c0;
        const u64 got = by == BY_COUNT ? c : w, was = by == BY_COUNT ? c - 1 : w - own;
        if (i < n && got >= least && was < least) {
            sh.found[0] = sh.list[i];
            sh.found[1] = w;
        }
        w0 += w_all;
        c0 += c_all;
    }
    __syncthreads();
    const Border r = { sh.found[0], sh.found[1] };
    __syncthreads();
    return r;
}

// The whole row's draw.  row.top and row.inv_t are set.
__device__ void draw_by_borders(SampleShared &sh, const SampleArgs &a, int r, const Draw &d, const Row &row)
{
    const int tid = threadIdx.x;
    const bool by_count = d.k > 0;
    clear_bins(sh);
    row.each(0, row.groups, [&](float v, int) {
        if (!counts(v)) return;
        const int b = row.bin(v);
        if (by_count) atomicAdd(&sh.count[b], 1u);
        if (b < SMP_BINS - 1) atomicAdd(&sh.weight[b], row.units(v));      // (the last bin's weights are below 2^-46)
    });
    __syncthreads();
    // two bins a thread: sums up to and with them stay in registers
    const int b0 = 2 * tid;
    const u64 wa = sh.weight[b0], wb = sh.weight[b0 + 1];
    const uint32_t ca = sh.count[b0], cb = sh.count[b0 + 1];
    u64 w1 = wa + wb, w_all;
    uint32_t c1 = ca + cb, c_all;
    scan2(sh, w1, c1, w_all, c_all);
    __syncthreads();

    // the bin in which the sums reach `least`, resolved
    const auto border = [&](int by, u64 least) {
        const u64 got = by == BY_COUNT ? c1 : w1, was = by == BY_COUNT ? c1 - ca - cb : w1 - wa - wb,
                  mid = by == BY_COUNT ? c1 - cb : w1 - wb;
        if (got >= least && was < least) {
            const bool first = mid >= least;
            sh.bin = b0 + (first ? 0 : 1);
            sh.found[0] = first ? w1 - wa - wb : w1 - wb;
            sh.found[1] = first ? c1 - ca - cb : c1 - cb;
        }
        __syncthreads();
        const int bin = sh.bin;
        const u64 w0 = sh.found[0];
        const uint32_t c0 = (uint32_t)sh.found[1];
        __syncthreads();
        return resolve(sh, row, bin, w0, c0, by, least);
    };
    u64 mass = w_all;
    if (d.k > 0 && (uint32_t)d.k < c_all) mass = border(BY_COUNT, (u64)d.k).mass;
    if (d.p < 1.0f) {
        const u64 least = max((u64)ceil((double)fmaxf(d.p, 0.0f) * (double)mass), 1ull);
        mass = border(BY_WEIGHT, min(least, mass)).mass;
    }
    if (d.m > 0.0f) {
        // the weights of at least min_p: summed, as they are a run of the order's start
        u64 w = 0, all;
        uint32_t c = 0, c_min;
        row.each(0, row.groups, [&](float v, int) {
            if (counts(v) && row.weight(v) >= (double)d.m) w += row.units(v);
        });
        scan2(sh, w, c, all, c_min);
        __syncthreads();
        mass = min(mass, max(all, (u64)SMP_ONE));
    }
    const u64 least = min((u64)floor((double)d.u * (double)mass) + 1, mass);
    const Border drawn = border(BY_WEIGHT, least);
    if (tid == 0) answer(a, r, (int)(uint32_t)drawn.token, (float)(row.weight(token_value(drawn.token)) * SMP_ONE / (double)mass));
}

// A top_k beyond `collect`: if the k best fit the list they are gathered by counts of keys, and decide.
__device__ bool draw_large_k(SampleShared &sh, const SampleArgs &a, int r, const Draw &d, const Row &row)
{
    if (d.k > SMP_LIST - 512) return false;
    uint32_t high = 0, before = 0, upto = 0;
    for (int step = 0; step < 2; step++) {
        clear_bins(sh);
        row.each(0, row.groups, [&](float v, int) {
            if (!counts(v)) return;
            const uint32_t key = order_key(v);
            if (step == 0) atomicAdd(&sh.count[key >> 21], 1u);
            else if (key >> 21 == high) atomicAdd(&sh.count[key >> 10 & 2047], 1u);
        });
        if (!count_border(sh, (uint32_t)d.k - before)) return false;      // fewer than k tokens count
        upto = before + (uint32_t)sh.found[1] + (uint32_t)sh.found[2];
        if (step == 0) {
            high = (uint32_t)sh.bin;
            before = (uint32_t)sh.found[1];
        }
    }
    if (upto > SMP_LIST) return false;
    const uint32_t bound = high << 21 | (uint32_t)sh.bin << 10 | 1023u;
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    row.each(0, row.groups, [&](float v, int i) {
        if (counts(v) && order_key(v) <= bound) push(sh, token_of(v, i));
    });
    __syncthreads();
    return finish(sh, a, r, d, row, (int)sh.n, 0.0);
}

// What the best token decides by itself.
__device__ __forceinline__ bool first_decides(const SampleArgs &a, int r, const Draw &d, u64 best)
{
    if (best != ~0ull && d.t > 0.0f && token_value(best) < INFINITY) return false;
    if (threadIdx.x == 0) answer(a, r, best == ~0ull ? -1 : (int)(uint32_t)best, best == ~0ull ? 0.0f : 1.0f);
    return true;
}

__device__ __forceinline__ int looked_for(const Draw &d)
{
    if (!(d.t > 0.0f)) return 1;
    return d.k > 0 && d.k <= SMP_TOP_K ? d.k : d.k > 0 ? 1 : SMP_OPEN;
}

__global__ void __launch_bounds__(SMP_TPB) k_sample(SampleArgs a)
{
    __shared__ SampleShared sh;
    const int r = blockIdx.x;
    const Draw d = settings(a, r);
    Row row;
    row.bind(a, r);
    const bool rest_too = d.k == 0 && d.t > 0.0f;
    row.inv_t = 1.0 / (double)d.t;
    double rest = 0.0;
    float ref;
    const u64 best = collect(sh, row, 0, row.groups, looked_for(d), rest_too, row.inv_t, rest, ref);
    if (first_decides(a, r, d, best)) return;
    row.top = (double)token_value(best);
    const uint32_t n = sh.n;
    __syncthreads();
    if (d.k > SMP_TOP_K) {
        if (draw_large_k(sh, a, r, d, row)) return;
    } else if (n <= SMP_LIST) {
        if (rest > 0.0) rest *= exp(((double)ref - row.top) * row.inv_t);
        if (finish(sh, a, r, d, row, (int)n, rest)) return;
    }
    draw_by_borders(sh, a, r, d, row);
}

// A part of a row: what it collects, for k_sample_join.
__global__ void __launch_bounds__(SMP_TPB) k_sample_part(SampleArgs a)
{
    __shared__ SampleShared sh;
    const int r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const Draw d = settings(a, r);
    Row row;
    row.bind(a, r);
    const bool rest_too = d.k == 0 && d.t > 0.0f;
    double rest = 0.0;
    float ref;
    const u64 best = collect(sh, row, (int)((int64_t)row.groups * part / a.parts), (int)((int64_t)row.groups * (part + 1) / a.parts),
                             looked_for(d), rest_too, 1.0 / (double)d.t, rest, ref);
    SamplePart *out = a.part + blockIdx.x;
    const int n = (int)min(sh.n, (uint32_t)PART_LIST);
    if (threadIdx.x == 0) {
        out->best = best;
        out->n = (int)min(sh.n, (uint32_t)PART_LIST + 1);
        out->rest = rest;
        out->ref = ref;
    }
    for (int i = threadIdx.x; i < n; i += SMP_TPB) out->list[i] = sh.list[i];
}

__global__ void __launch_bounds__(SMP_TPB) k_sample_join(SampleArgs a)
{
    __shared__ SampleShared sh;
    const int r = blockIdx.x, tid = threadIdx.x;
    const Draw d = settings(a, r);
    Row row;
    row.bind(a, r);
    row.inv_t = 1.0 / (double)d.t;
    const SamplePart *in = a.part + (int64_t)r * a.parts;
    // every token of the parts in a register, a part's list beside the others'
    u64 held[PART_MOST], best = ~0ull;
    uint32_t mine = 0xffffffffu;
    bool fits = true;
    double rest = 0.0;
#pragma unroll
    for (int i = 0; i < PART_MOST; i++) {
        const int n = i < a.parts ? in[i].n : 0;
        fits &= n <= PART_LIST;
        held[i] = tid < n && n <= PART_LIST ? in[i].list[tid] : ~0ull;
        if (i < a.parts) best = min(best, in[i].best);
        mine = min(mine, (uint32_t)(held[i] >> 32));
    }
    if (first_decides(a, r, d, best)) return;
    row.top = (double)token_value(best);
    if (d.k > SMP_TOP_K) {
        if (draw_large_k(sh, a, r, d, row)) return;
    } else if (fits) {
        if (tid == 0) sh.n = 0;
        const uint32_t bound = key_bound(sh, mine, looked_for(d));
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < PART_MOST; i++) {
            if (held[i] == ~0ull) continue;
            if ((uint32_t)(held[i] >> 32) <= bound) push(sh, held[i]);
            else if (d.k == 0) sum += row.weight(token_value(held[i]));
        }
        if (d.k == 0) {
            rest = scan_f64(sh, sum);
#pragma unroll
            for (int i = 0; i < PART_MOST; i++)
                if (i < a.parts && in[i].rest > 0.0) rest += in[i].rest * exp(((double)in[i].ref - row.top) * row.inv_t);
        }
        __syncthreads();
        const uint32_t n = sh.n;
        __syncthreads();
        if (n <= SMP_LIST && finish(sh, a, r, d, row, (int)n, rest)) return;
    }
    draw_by_borders(sh, a, r, d, row);
}

// Workgroups a row: one where the rows fill the card, else as many as do, of at least 1024 groups of four logits.
static int sample_parts(const SampleArgs &a)
{
    const int most = std::min(256 / std::max(a.n_rows, 1), (a.n_vocab / 4 + SMP_TPB - 1) / SMP_TPB);
    return std::clamp(most, 1, PART_MOST);
}

size_t sample_workspace(const SampleArgs &a)
{
    const int parts = sample_parts(a);
    return parts == 1 ? 0 : (size_t)a.n_rows * parts * sizeof(SamplePart);
}

hipError_t launch_sample(SampleArgs a, hipStream_t s)
{
    a.parts = sample_parts(a);
    if (a.parts == 1) hipLaunchKernelGGL(k_sample, dim3(a.n_rows), SMP_TPB, 0, s, a);
    else {
        hipLaunchKernelGGL(k_sample_part, dim3(a.n_rows * a.parts), SMP_TPB, 0, s, a);
        hipLaunchKernelGGL(k_sample_join, dim3(a.n_rows), SMP_TPB, 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace ds3k
