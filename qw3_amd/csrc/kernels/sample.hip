// sample.hip -- one token a row from logits: temperature, top-k, top-p, min-p and a
// given random number.
//
// The row's tokens are ordered by (logit descending, index ascending); every step keeps
// a run of that order's start, and the draw inverts the summed weights exp((x - max) / T)
// along it.  Nothing sorts the row: one pass collects its largest logits, a few hundred,
// and where they do not decide, the weights of all are summed by bins and only the bins
// that a border lies in are resolved.
//
//   collect  from the threads' best ones of the first 32,768 logits follows a bound that
//            at least k of the row's reach, so what lies under it is passed over as the
//            row streams by.  Without top-k the weights of what is passed are summed by bins
//            of (max - x) / T, a bin an 1 / 32 octave, as whole numbers of 2^-32 of the bin's
//            largest weight: exact in any order of atomics.
//   finish   the collected tokens sorted, their weights summed along; every border and
//            the draw are looked for there.
//   below    where one lies below the collected ones (a flat row), its bin's tokens are
//            gathered and sorted.
//   borders  a top-k of thousands, thousands of equal logits: counts and weights by bins
//            of the whole row, the bins of borders narrowed by digits until they can be
//            sorted.
//
// All sums but the bins' are in 64-bit floating point, in an order that the sizes fix.
//
// A workgroup has a row, few rows are collected by several workgroups each (k_sample_part)
// and finished by one (k_sample_join).  What bounds it: the passes over a row by one
// compute unit (a pass of 256 rows of 151,936 takes 30 us, 5.2 TB/s) and the chains of
// sorting, summing and looking up behind them (10 us), which no other row hides as a call
// waits for its slowest.  256 rows of 151,936 by setting: temperature 0 33 us, top-k 20
// with top-p 42, top-k 200 50, min-p 61, temperature 0.3 alone 60, 1 alone 87 (every
// logit's weight goes into a bin: some 25 vector instructions a logit, LDS atomics), top-p
// 0.9 at temperature 1 115 (the border lies below the collected: a second pass for each
// border), top-k 2000 109 (a pass that counts, one that gathers, the sort).  One row: 10
// us, 15, 24, 32, 31, 31, 57, 65.
#include "common.h"
#include "lanes.h"

#include <algorithm>
#include <cfloat>

namespace ds3k {

constexpr int SMP_TPB = 1024;
constexpr int SMP_BINS = 2048;               // bins of 1 / 64 over 32 (the whole row's), or of 1 / 32 of an octave over 64
constexpr int SMP_LIST = 4096;               // tokens sorted at once
constexpr int SMP_HALF = SMP_LIST / 2;       // of them where a second list lies behind the first
constexpr int SMP_FIRST = 8 * SMP_TPB;        // groups of four logits from which `collect` takes its bound
constexpr int SMP_TOP_K = 512;               // top_k up to which `collect` decides
constexpr int SMP_OPEN = 64;                 // tokens that it looks for without top_k
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

// exp(y), y <= 0: reduced by multiples of ln 2 in two parts (Cody and Waite), Taylor's series to the twelfth power
// on -0.35 .. 0.35 (its rest is 2e-16).
__device__ __forceinline__ double exp_below(double y)
{
    y = fmax(y, -800.0);
    const double n = rint(y * 1.4426950408889634074);
    const double r = fma(n, -1.9082149292705877e-10, fma(n, -0.6931471803691238, y));
    double e = 1.0 / 479001600.0;
    e = fma(e, r, 1.0 / 39916800.0);
    e = fma(e, r, 1.0 / 3628800.0);
    e = fma(e, r, 1.0 / 362880.0);
    e = fma(e, r, 1.0 / 40320.0);
    e = fma(e, r, 1.0 / 5040.0);
    e = fma(e, r, 1.0 / 720.0);
    e = fma(e, r, 1.0 / 120.0);
    e = fma(e, r, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    return __builtin_ldexp(e, (int)n);
}

// 2^(f / 32) in whole numbers of 2^-32, 0 <= f < 1: 1 and Taylor's series to the fourth power in 32 bits (off by 2e-9, a
// rounding that changes its sign from logit to logit).  Bins of weights hold these; the octaves' powers come in once a bin.
constexpr double STEP_ONE = 0x1p32;
__device__ __forceinline__ unsigned long long part_of_step(float f)
{
    constexpr float a = 0.021660849392498290f;        // ln 2 / 32
    const float e = f * fmaf(f, fmaf(f, fmaf(f, a * a * a * a / 24, a * a * a / 6), a * a / 2), a);
    return 0x100000000ull + (uint32_t)fmaf(e, 0x1p32f, 0.5f);
}

struct SampleShared {
    u64 weight[SMP_BINS];                    // by bin
    uint32_t count[SMP_BINS];
    u64 list[SMP_LIST];                      // key << 32 | index
    u64 wave_w[SMP_TPB / 64];
    double wave_d[SMP_TPB / 64];
    uint32_t wave_c[SMP_TPB / 64];
    uint32_t shown[7 * (SMP_TPB / 64)];
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
    d.u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;       // (the largest number below 1)
    return d;
}

// Inclusive sums over the workgroup, and those of all.
template <typename T>
__device__ __forceinline__ T scan(T *waves, T &v)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    const T sums = row_scan(waves[lane & (SMP_TPB / 64 - 1)]);
    const int before = __builtin_amdgcn_readfirstlane(max(wave - 1, 0));
    const T base = lane_of(sums, before);
    if (wave > 0) v += base;
    return lane_of(sums, SMP_TPB / 64 - 1);
}

__device__ __forceinline__ void scan2(SampleShared &sh, u64 &w, uint32_t &c, u64 &w_all, uint32_t &c_all)
{
    w_all = scan(sh.wave_w, w);
    c_all = scan(sh.wave_c, c);
}

__device__ __forceinline__ double scan_f64(SampleShared &sh, double &v) { return scan(sh.wave_d, v); }

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
    __device__ double weight(float v) const { return exp_below(-depth(v)); }
    __device__ u64 units(float v) const { return (u64)__double2ll_rn(weight(v) * SMP_ONE); }
    // v / T in steps of 1 / 32 of an octave, as whole + more + part: a grid that the parts of a row have in common.  The
    // product of 48 bits (two factors, the first product's rounding by an fma) keeps the part to 2^-25 where steps are
    // many; 64-bit instructions for it took three times as long.  hi is the rounded product wherever it stands: taken into
    // an fma, hi - whole would count its rounding twice (weights off by 0.3 % at v / T of 5e4) and the whole steps would
    // not fall with v.
    float c_hi, c_lo;
    struct Steps {
        float whole, more, part;
    };
    __device__ void set_temperature(float t)
    {
        inv_t = 1.0 / (double)t;
        const double c = inv_t * (32 * 1.4426950408889634074);
        c_hi = (float)c;
        c_lo = (float)(c - (double)c_hi);
    }
    __device__ Steps steps(float v) const
    {
#pragma clang fp contract(off)
        const float hi = v * c_hi, lo = fmaf(v, c_lo, fmaf(v, c_hi, -hi));
        Steps s;
        s.whole = floorf(hi);
        const float f = (hi - s.whole) + lo;
        s.more = floorf(f);
        s.part = f - s.more;
        return s;
    }
    // steps of b below a (NaN where one is not finite)
    static __device__ float below(const Steps &a, const Steps &b) { return (a.whole - b.whole) + (a.more - b.more); }
    // whether steps tell logits near v apart
    __device__ bool graded(float v) const { return c_hi < 1e30f && fabsf(v * c_hi) < 1e30f; }

    // f(value, index) of every logit of groups [q0, q1), AT groups a thread in flight
    template <int AT = 2, typename F>
    __device__ __forceinline__ void each(int q0, int q1, F f) const
    {
#pragma unroll 1
        for (int q = q0 + threadIdx.x; q < q1; q += AT * SMP_TPB) {
            float4 v[AT];
#pragma unroll
            for (int i = 0; i < AT; i++) v[i] = q + i * SMP_TPB < q1 ? load(q + i * SMP_TPB) : float4{ NAN, NAN, NAN, NAN };
#pragma unroll
            for (int i = 0; i < AT; i++) {
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
    uint32_t c = x + y;
    const uint32_t all = scan(sh.wave_c, c);
    if (c >= least && c - x - y < least) {
        const bool first = c - y >= least;
        sh.bin = b + (first ? 0 : 1);
        sh.found[1] = first ? c - x - y : c - y;
        sh.found[2] = first ? x : y;
    }
    __syncthreads();
    return all >= least;
}

// A key that at least `least` of the threads' keys do not pass (0xffffffff: none is found).  Every wave sorts its keys
// and shows its best, its second, fourth, ... 64th; as many waves' 2^j-th as it takes bound so many keys, and the best
// such bound over j is taken.
__device__ __forceinline__ uint32_t key_bound(SampleShared &sh, uint32_t key, int least)
{
    constexpr int WAVES = SMP_TPB / 64;
    static_assert(WAVES == 16, "rows of 16 lanes");
    const int lane = threadIdx.x & 63, row = lane >> 4;
    key = sort_lanes<64>(key);
    __syncthreads();
    if ((lane & (lane + 1)) == 0) sh.shown[__popc(lane) * WAVES + (threadIdx.x >> 6)] = key;
    __syncthreads();
    // rows of 16 lanes sort the waves' keys of one rank: ranks 1 .. 8, then 16 .. 64
    const uint32_t a = sort_lanes<16>(sh.shown[lane]), b = sort_lanes<16>(row < 3 ? sh.shown[64 + lane] : 0xffffffffu);
    const int need_a = (least + (1 << row) - 1) >> row, need_b = (least + (16 << row) - 1) >> (4 + row);
    uint32_t bound = (lane & 15) == need_a - 1 ? a : 0xffffffffu;
    if (row < 3 && (lane & 15) == need_b - 1) bound = min(bound, b);
    return lanes_join<32>(bound, [](uint32_t x, uint32_t y) { return min(x, y); });
}

__device__ __forceinline__ void push(SampleShared &sh, u64 token)
{
    const uint32_t at = atomicAdd(&sh.n, 1u);
    if (at < SMP_LIST) sh.list[at] = token;
}

// The best token of each thread, of all.
__device__ __forceinline__ u64 best_of(SampleShared &sh, u64 best)
{
    const auto least = [](u64 x, u64 y) { return x < y ? x : y; };
    best = lanes_join<32>(best, least);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave_w[threadIdx.x >> 6] = best;
    __syncthreads();
    return lanes_join<8>(sh.wave_w[threadIdx.x & 15], least);
}

// What lies under the collected tokens: none of key `bound` or less.
struct Passed {
    uint32_t bound;
    float ref;                               // weights are relative to this logit's
};

// One pass over groups [q0, q1): sh.list gets (sh.n tells how many, perhaps more than fit) the tokens up to a bound,
// at least the `least` best or all; returns the best.  by_bins: the other tokens' weights in sh.weight, by steps below
// that of `ref`.
__device__ __forceinline__ u64 collect(SampleShared &sh, const Row &row, int q0, int q1, int least, bool by_bins, Passed &passed)
{
    if (threadIdx.x == 0) sh.n = 0;
    for (int b = threadIdx.x; b < SMP_BINS; b += SMP_TPB) sh.weight[b] = 0;
    float most = -INFINITY;
    row.each<4>(q0, min(q1, q0 + SMP_FIRST), [&](float v, int) { most = fmaxf(most, v); });
    const uint32_t mine = counts(most) ? order_key(most) : 0xffffffffu;
    const uint32_t bound = key_bound(sh, mine, least);
    // (a logit near the largest; none that is passed lies above it)
    const u64 first = best_of(sh, (u64)mine << 32);
    const float ref = first >> 32 == 0xffffffffu ? 0.0f : token_value(first);
    u64 best = ~0ull;
    // two groups a thread at a time, the next two on their way: one comparison tells that none of their logits is collected
    const Row::Steps top = row.steps(ref);
    const float least_value = bound == 0xffffffffu ? -FLT_MAX : key_value(bound);
    const auto group = [&](int q) { return q < q1 ? row.load(q) : float4{ NAN, NAN, NAN, NAN }; };
    float4 x = group(q0 + threadIdx.x), y = group(q0 + threadIdx.x + SMP_TPB);
#pragma unroll 1
    for (int q = q0 + threadIdx.x; q < q1; q += 2 * SMP_TPB) {
        const float v[8] = { x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w };
        x = group(q + 2 * SMP_TPB);
        y = group(q + 3 * SMP_TPB);
        float largest = v[0];
#pragma unroll
        for (int j = 1; j < 8; j++) largest = fmaxf(largest, v[j]);
        if (largest >= least_value) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (v[j] >= least_value) {
                    const u64 token = token_of(v[j], row.index(q + j / 4 * SMP_TPB, j & 3));
                    best = min(best, token);
                    push(sh, token);
                }
        }
        if (by_bins) {
            u64 units[8];
            float bin[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const Row::Steps s = row.steps(v[j]);
                // (beyond the bins, weights are below 2^-63; -inf and NaN are no bin's)
                bin[j] = v[j] < least_value ? Row::below(top, s) : INFINITY;
                units[j] = part_of_step(s.part);
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (bin[j] < SMP_BINS) atomicAdd(&sh.weight[(int)bin[j]], units[j]);
        }
    }
    best = best_of(sh, best);
    passed = { bound, ref };
    return best;
}

// *least gets the smallest place that holds: a wave's places rise from lane to lane, so its first lane's will do (where
// thousands hold, an atomic of each took 6 us).
template <typename U>
__device__ __forceinline__ void first_place(U *least, bool holds, int place)
{
    const uint64_t those = __ballot(holds);
    if (holds && (those & ((1ull << (threadIdx.x & 63)) - 1)) == 0) atomicMin(least, (U)place);
}

// list[0 .. size) in order, E tokens a thread (places tid, tid + SMP_TPB, ...): steps of up to 32 within the wave, of up to
// 512 through the list, larger ones within the thread.
template <int E>
__device__ __forceinline__ void sort_places(u64 *list, int size)
{
    const int tid = threadIdx.x;
    u64 v[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        v[e] = E > 1 || tid < size ? list[tid + e * SMP_TPB] : ~0ull;
        v[e] = sort_merge<1>(v[e], 2);
        v[e] = sort_merge<2>(v[e], 4);
        v[e] = sort_merge<4>(v[e], 8);
        v[e] = sort_merge<8>(v[e], 16);
        v[e] = sort_merge<16>(v[e], 32);
        v[e] = sort_merge<32>(v[e], 64);
    }
#pragma unroll 1
    for (int k = 128; k <= size; k *= 2) {
        if constexpr (E > 1) {
#pragma unroll
            for (int j = E / 2; j > 0; j /= 2)
                if (j * SMP_TPB < k) {
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if ((e & j) == 0) {
                            const bool up = (e * SMP_TPB & k) == 0;
                            const u64 x = v[e], y = v[e + j];
                            v[e] = up == (x < y) ? x : y;
                            v[e + j] = up == (x < y) ? y : x;
                        }
                }
        }
#pragma unroll 1
        for (int j = min(k, SMP_TPB) / 2; j > 32; j /= 2) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; e++)
                if (E > 1 || tid < size) list[tid + e * SMP_TPB] = v[e];
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; e++) {
                const u64 o = E > 1 || tid < size ? list[(tid ^ j) + e * SMP_TPB] : v[e];
                v[e] = ((tid & j) == 0) == ((tid + e * SMP_TPB & k) == 0) ? min(v[e], o) : max(v[e], o);
            }
        }
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = sort_merge<32>(v[e], k < SMP_TPB ? k : 0, (tid + e * SMP_TPB & k) != 0 && k >= SMP_TPB);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++)
        if (E > 1 || tid < size) list[tid + e * SMP_TPB] = v[e];
}

// list[0 .. n) in order; MOST: the places that it has.
template <int MOST>
__device__ __forceinline__ void sort_list(u64 *list, int n)
{
    int size = 64;
    while (size < n) size *= 2;
    if (size > SMP_TPB) size = size <= SMP_HALF ? SMP_HALF : MOST;
    __syncthreads();
    for (int i = n + threadIdx.x; i < size; i += SMP_TPB) list[i] = ~0ull;
    __syncthreads();
    if (size <= SMP_TPB) sort_places<1>(list, size);
    else if (MOST == SMP_HALF || size <= SMP_HALF) sort_places<SMP_HALF / SMP_TPB>(list, SMP_HALF);
    else sort_places<MOST / SMP_TPB>(list, MOST);
    __syncthreads();
}

__device__ __forceinline__ void answer(const SampleArgs &a, int r, int token, float share)
{
    a.tokens[r] = token;
    if (a.probs) a.probs[r] = share;
}

// The draw of `finish` from list[0 .. n), n <= 64, with top_k: one wave does it, in registers and in the same order of sums
// (one row of 151,936 with top_k 20: the finishing launch 7.8 us in place of 11.3).
__device__ __forceinline__ void finish_few(const u64 *list, const SampleArgs &a, int r, const Draw &d, const Row &row, int n)
{
    const int i = threadIdx.x;
    if (i >= 64) return;
    const u64 token = sort_lanes<64>(i < n ? list[i] : ~0ull);
    n = min(n, d.k);
    const double own = i < n ? row.weight(token_value(token)) : 0.0, upto = wave_scan(own);
    uint64_t ends = 1ull << (n - 1);                  // a place where the kept ones may end: the first counts
    if (d.p < 1.0f) ends |= __ballot(i < n && upto >= (double)fmaxf(d.p, 0.0f) * lane_of(upto, 63));
    if (d.m > 0.0f) ends |= __ballot(i > 0 && i < n && own < (double)d.m) >> 1;
    const int last = __builtin_ctzll(ends);
    const double total = lane_of(upto, last);
    const uint64_t past = __ballot(i < last && upto > (double)d.u * total);
    if (i == (past ? __builtin_ctzll(past) : last)) answer(a, r, (int)(uint32_t)token, (float)(own / total));
}

// The draw from sh.list[0 .. n), n > 0: with top_k at least the k best tokens of the row, else its best n, the others'
// weights summing to `rest` of the first's.  False: they do not decide.
__device__ __forceinline__ bool finish(SampleShared &sh, const SampleArgs &a, int r, const Draw &d, const Row &row, int &n,
                                       double rest, double &listed)
{
    const int tid = threadIdx.x;
    if (d.k > 0 && n <= 64) {
        finish_few(sh.list, a, r, d, row, n);
        return true;
    }
    if (d.k > 0 && n > SMP_TPB && n > d.k + 64) {
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
                if (held[i] != ~0ull && (step == 0 || key >> 21 == high))
                    atomicAdd(&sh.count[step == 0 ? key >> 21 : key >> 10 & 2047], 1u);
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
    sort_list<SMP_LIST>(sh.list, n);
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
    listed = mass;
    if (!complete) mass += rest;
    constexpr int NONE = 0x7fffffff;
    __syncthreads();
    if (tid == 0) {
        sh.bin = NONE;                       // tokens kept, where a border decides it
        sh.n = NONE;                         // the drawn token's place
    }
    __syncthreads();
    if (d.p < 1.0f || d.m > 0.0f) {
        const double least = d.p < 1.0f ? (double)fmaxf(d.p, 0.0f) * mass : INFINITY;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            const int i = b * SMP_TPB + tid;
            first_place(&sh.bin, i < n && upto[b] >= least, i + 1);
            first_place(&sh.bin, i > 0 && i < n && own[b] < (double)d.m, i);
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
        first_place(&sh.n, i < kept && upto[b] > target, i);
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
// A border below the collected tokens, without top_k.
// ---------------------------------------------------------------------------

// The smallest key in [lo, hi] whose value fails `f`, or hi + 1: f holds up to some key and not beyond.
template <typename F>
__device__ __forceinline__ u64 first_key(uint32_t lo, uint32_t hi, F f)
{
    u64 a = lo, b = (u64)hi + 1;
    while (a < b) {
        const u64 mid = (a + b) / 2;
        if (f(key_value((uint32_t)mid))) a = mid + 1;
        else b = mid;
    }
    return a;
}

// The weight of a bin's whole numbers of part_of_step, `bin` steps below those of `top`.
__device__ __forceinline__ double bin_weight(const Row &row, const Row::Steps &top, int bin, u64 units)
{
    if (units == 0) return 0.0;
    const double x = (double)top.whole + (double)top.more - bin - row.top * row.inv_t * (32 * 1.4426950408889634074);
    return (double)units / STEP_ONE * exp_below(x * (1.0 / 32 * 0.6931471805599453));
}

struct Below {
    double listed;                           // weight of the collected tokens
    double w[2], upto;                       // of this thread's two bins, and of all up to and with them
    Row::Steps top;                          // the first bin's
    uint32_t bound;                          // keys above it
};

// The token below at which the weights, with `listed`, pass `least` (or the last one), and the weights up to and with it.
__device__ __forceinline__ void border_below(SampleShared &sh, const Row &row, const Below &b, double least, u64 &token, double &mass)
{
    const int tid = threadIdx.x;
    u64 *list = sh.list + SMP_HALF;
    __syncthreads();
    if (tid == 0) sh.bin = 0x7fffffff;
    __syncthreads();
    const double upto_first = b.upto - b.w[1];
    const int mine = upto_first >= least && b.w[0] > 0.0 ? 2 * tid : b.upto >= least && b.w[1] > 0.0 ? 2 * tid + 1 : 0x7fffffff;
    first_place(&sh.bin, mine != 0x7fffffff, mine);
    __syncthreads();
    if (sh.bin == 0x7fffffff) {              // rounding: the last bin with a weight
        __syncthreads();
        if (tid == 0) sh.bin = -1;
        __syncthreads();
        if (b.w[0] > 0.0 || b.w[1] > 0.0) atomicMax(&sh.bin, b.w[1] > 0.0 ? 2 * tid + 1 : 2 * tid);
        __syncthreads();
    }
    const int bin = sh.bin;
    if (tid == bin / 2) sh.mass = bin & 1 ? b.upto - b.w[1] : upto_first - b.w[0];
    __syncthreads();
    double before = sh.mass;                 // of everything above the bin
    // its keys
    const auto depth = [&](float v) { return Row::below(b.top, row.steps(v)); };
    uint32_t lo = (uint32_t)first_key(b.bound + 1, 0xff7fffffu, [&](float v) { return depth(v) < bin; }),
             hi = (uint32_t)(first_key(lo, 0xff7fffffu, [&](float v) { return depth(v) <= bin; }) - 1);
    uint32_t i0 = 0, i1 = (uint32_t)row.n;   // where one key is left: its indices
    int n;
    for (;;) {
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        // (by values first: with keys for every logit a pass took 22 us of one row in place of 17)
        const float high = key_value(lo), low = key_value(hi);
        row.each<8>(0, row.groups, [&](float v, int i) {
            if (!(v >= low && v <= high)) return;
            const uint32_t key = order_key(v);
            if (key < lo || key > hi || (uint32_t)i < i0 || (uint32_t)i >= i1) return;
            const uint32_t at = atomicAdd(&sh.n, 1u);
            if (at < SMP_HALF) list[at] = (u64)key << 32 | (uint32_t)i;
        });
        __syncthreads();
        n = (int)sh.n;
        if (n <= SMP_HALF) break;
        // too many: their weights, at least a unit each so that a slice of tokens is not empty, by 2048 slices of the keys,
        // then of the indices
        const bool by_key = lo < hi;
        const uint32_t span = by_key ? hi - lo : i1 - i0 - 1;
        const int shift = max(0, 21 - __builtin_clz(span | 1));
        clear_bins(sh);
        row.each(0, row.groups, [&](float v, int i) {
            if (!counts(v)) return;
            const uint32_t key = order_key(v);
            if (key < lo || key > hi || (uint32_t)i < i0 || (uint32_t)i >= i1) return;
            atomicAdd(&sh.weight[(by_key ? key - lo : (uint32_t)i - i0) >> shift], max(row.units(v), 1ull));
        });
        __syncthreads();
        const u64 x = sh.weight[2 * tid], y = sh.weight[2 * tid + 1];
        u64 w = x + y, w_all;
        uint32_t c = 0, c_all;
        scan2(sh, w, c, w_all, c_all);
        __syncthreads();
        if (tid == 0) sh.bin = 0x7fffffff;
        __syncthreads();
        const auto reaches = [&](u64 units) { return before + (double)units / SMP_ONE >= least; };
        const int at = x > 0 && reaches(w - y) ? 2 * tid : y > 0 && reaches(w) ? 2 * tid + 1 : 0x7fffffff;
        first_place(&sh.bin, at != 0x7fffffff, at);
        __syncthreads();
        if (sh.bin == 0x7fffffff) {
            __syncthreads();
            if (tid == 0) sh.bin = 0;
            __syncthreads();
            if (x > 0 || y > 0) atomicMax(&sh.bin, y > 0 ? 2 * tid + 1 : 2 * tid);
            __syncthreads();
        }
        const uint32_t slice = (uint32_t)sh.bin;
        if (tid == (int)slice / 2) sh.found[0] = slice & 1 ? w - y : w - y - x;
        __syncthreads();
        before += (double)sh.found[0] / SMP_ONE;
        if (by_key) {
            hi = min(hi, lo + ((slice + 1) << shift) - 1);
            lo += slice << shift;
        } else {
            i1 = min(i1, i0 + ((slice + 1) << shift));
            i0 += slice << shift;
        }
    }
    sort_list<SMP_HALF>(list, n);
    // (n <= SMP_HALF: two tokens a thread)
    __syncthreads();
    if (tid == 0) sh.n = (uint32_t)max(n - 1, 0);
    double upto[SMP_HALF / SMP_TPB];
#pragma unroll
    for (int j = 0; j < SMP_HALF / SMP_TPB; j++) {
        const int i = j * SMP_TPB + tid;
        double w = i < n ? row.weight(token_value(list[i])) : 0.0;
        const double all = scan_f64(sh, w);
        upto[j] = before + w;
        before += all;
        first_place(&sh.n, i < n && upto[j] >= least, i);
    }
    __syncthreads();
    const int at = (int)sh.n;
#pragma unroll
    for (int j = 0; j < SMP_HALF / SMP_TPB; j++)
        if (j * SMP_TPB + tid == at) {
            sh.found[0] = list[at];
            sh.mass = upto[j];
        }
    __syncthreads();
    token = sh.found[0];
    mass = sh.mass;
    __syncthreads();
}

// The draw where the sorted list [0 .. n), n <= SMP_HALF, does not decide.
__device__ __forceinline__ void draw_below(SampleShared &sh, const SampleArgs &a, int r, const Draw &d, const Row &row, int n,
                                           const Below &b)
{
    const int tid = threadIdx.x;
    double w = b.w[0] + b.w[1], mass = b.listed + scan_f64(sh, w), kept = mass;
    u64 token;
    if (d.p < 1.0f) border_below(sh, row, b, (double)d.p * mass, token, kept);
    if (d.m > 0.0f) {
        // the weights of at least min_p are a run of the order's start
        double sum = 0.0;
        row.each(0, row.groups, [&](float v, int) {
            if (!counts(v) || order_key(v) <= b.bound) return;
            const double x = row.weight(v);
            if (x >= (double)d.m) sum += x;
        });
        kept = fmin(kept, b.listed + scan_f64(sh, sum));
    }
    const double target = (double)d.u * kept;
    if (target < b.listed) {
        __syncthreads();
        if (tid == 0) sh.n = (uint32_t)n - 1;
        double before = 0.0, own[SMP_HALF / SMP_TPB];
#pragma unroll
        for (int j = 0; j < SMP_HALF / SMP_TPB; j++) {
            const int i = j * SMP_TPB + tid;
            own[j] = i < n ? row.weight(token_value(sh.list[i])) : 0.0;
            double x = own[j];
            const double all = scan_f64(sh, x);
            first_place(&sh.n, i < n && before + x > target, i);
            before += all;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SMP_HALF / SMP_TPB; j++)
            if (j * SMP_TPB + tid == (int)sh.n) answer(a, r, (int)(uint32_t)sh.list[sh.n], (float)(own[j] / kept));
        return;
    }
    // past the target: at least the next larger number; within what is kept
    double upto;
    border_below(sh, row, b, fmin(nextafter(target, INFINITY), kept), token, upto);
    if (tid == 0) answer(a, r, (int)(uint32_t)token, (float)(row.weight(token_value(token)) / kept));
}

// ---------------------------------------------------------------------------
// Borders of the whole row.
// ---------------------------------------------------------------------------

// What a border is looked for by: the first token in order whose inclusive count or weight reaches `least`.
enum : int { BY_COUNT, BY_WEIGHT };

// Where a border lies: the token, and the weights up to and with it.
struct Border {
    u64 token;
    u64 mass;
};

// The token of bin `bin` at which the inclusive sum, from (w0, c0) before the bin, reaches `least`.
__device__ __forceinline__ Border resolve(SampleShared &sh, const Row &row, int bin, u64 w0, uint32_t c0, int by, u64 least)
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
    sort_list<SMP_LIST>(sh.list, n);
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
__device__ __forceinline__ void draw_by_borders(SampleShared &sh, const SampleArgs &a, int r, const Draw &d, const Row &row)
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

// A top_k beyond `collect`, which has looked for the SMP_TOP_K best, at least as many up to `bound`: their depth below
// the largest logit, three times over, divided into bins, shows by counts where the k-th lies (bins of keys would
// be few and their counters fought over).  Where the k best fit the list they are gathered and decide.
__device__ __forceinline__ bool draw_large_k(SampleShared &sh, const SampleArgs &a, int r, const Draw &d, const Row &row, uint32_t bound)
{
    const float top = (float)row.top, depth = 3.0f * (top - key_value(bound)), scale = (float)SMP_BINS / depth;
    if (d.k > SMP_LIST - 512 || bound == 0xffffffffu || !(depth > 0.0f && depth < INFINITY && scale < INFINITY)) return false;
    const auto bin = [&](float v) { return (top - v) * scale; };          // (rises as v falls)
    clear_bins(sh);
    row.each<8>(0, row.groups, [&](float v, int) {
        const float b = bin(v);
        if (b < SMP_BINS) atomicAdd(&sh.count[(int)b], 1u);
    });
    if (!count_border(sh, (uint32_t)d.k)) return false;                   // it lies deeper
    if (sh.found[1] + sh.found[2] > SMP_LIST) return false;
    const float last = (float)(sh.bin + 1);
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    row.each<2>(0, row.groups, [&](float v, int i) {
        if (bin(v) < last) push(sh, token_of(v, i));
    });
    __syncthreads();
    int n = (int)sh.n;
    double listed;
    return finish(sh, a, r, d, row, n, 0.0, listed);
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
    return d.k > 0 ? min(d.k, SMP_TOP_K) : SMP_OPEN;
}

__global__ void __launch_bounds__(SMP_TPB) k_sample(SampleArgs a)
{
    __shared__ SampleShared sh;
    const int r = blockIdx.x, tid = threadIdx.x;
    const Draw d = settings(a, r);
    Row row;
    row.bind(a, r);
    row.set_temperature(d.t);
    Passed passed;
    const u64 best = collect(sh, row, 0, row.groups, looked_for(d), d.k == 0 && d.t > 0.0f, passed);
    if (first_decides(a, r, d, best)) return;
    row.top = (double)token_value(best);
    int n = (int)sh.n;
    if (d.k > SMP_TOP_K) {
        if (draw_large_k(sh, a, r, d, row, passed.bound)) return;
    } else if (n <= SMP_LIST && (d.k > 0 || row.graded((float)row.top))) {
        Below b = { 0.0, { 0.0, 0.0 }, 0.0, row.steps(passed.ref), passed.bound };
        double rest = 0.0;
        if (d.k == 0) {
#pragma unroll
            for (int i = 0; i < 2; i++) b.w[i] = bin_weight(row, b.top, 2 * tid + i, sh.weight[2 * tid + i]);
            b.upto = b.w[0] + b.w[1];
            rest = scan_f64(sh, b.upto);
        }
        __syncthreads();
        if (finish(sh, a, r, d, row, n, rest, b.listed)) return;
        if (n <= SMP_HALF) {
            b.upto += b.listed;
            draw_below(sh, a, r, d, row, n, b);
            return;
        }
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
    row.set_temperature(d.t);
    Passed passed;
    const bool by_bins = d.k == 0 && d.t > 0.0f;
    const u64 best = collect(sh, row, (int)((int64_t)row.groups * part / a.parts), (int)((int64_t)row.groups * (part + 1) / a.parts),
                             looked_for(d), by_bins, passed);
    SamplePart *out = a.part + blockIdx.x;
    const int n = (int)min(sh.n, (uint32_t)PART_LIST);
    if (threadIdx.x == 0) {
        out->best = best;
        out->n = (int)min(sh.n, (uint32_t)PART_LIST + 1);
        out->bound = passed.bound;
        out->ref = passed.ref;
    }
    if (threadIdx.x < n) out->list[threadIdx.x] = sh.list[threadIdx.x];
    if (by_bins)
        for (int i = threadIdx.x; i < SMP_BINS; i += SMP_TPB) out->weight[i] = sh.weight[i];
}

__global__ void __launch_bounds__(SMP_TPB) k_sample_join(SampleArgs a)
{
    static_assert(PART_MOST <= SMP_TPB / 64 && PART_LIST == 16 * 64, "a wave holds a part's tokens");
    __shared__ SampleShared sh;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const SamplePart *in = a.part + (int64_t)r * a.parts, *own = in + min(wave, a.parts - 1);
    const Draw d = settings(a, r);
    // a wave holds a part's tokens; the first 64 places are read before their number is known
    const u64 own_best = own->best;
    u64 held[PART_LIST / 64];
    uint32_t passed = own->bound;                     // the least bound of the parts: all tokens up to it are here
    const int count = wave < a.parts ? __builtin_amdgcn_readfirstlane(own->n) : 0;
    held[0] = own->list[lane];
    if (lane >= count) held[0] = ~0ull;
    bool fits = count <= PART_LIST;
    uint32_t mine = (uint32_t)(held[0] >> 32);
#pragma unroll
    for (int i = 1; i < PART_LIST / 64; i++) {
        held[i] = ~0ull;
        if (64 * i < count) {
            if (64 * i + lane < count && fits) held[i] = own->list[64 * i + lane];
            mine = min(mine, (uint32_t)(held[i] >> 32));
        }
    }
    Row row;
    row.bind(a, r);
    row.set_temperature(d.t);
    const u64 best = best_of(sh, own_best);
    if (first_decides(a, r, d, best)) return;
    row.top = (double)token_value(best);
    if (d.k > SMP_TOP_K) {
        if (draw_large_k(sh, a, r, d, row, (uint32_t)best_of(sh, passed))) return;
    } else if (__syncthreads_and(fits && (d.k > 0 || row.graded((float)row.top)))) {
        if (tid == 0) sh.n = 0;
        for (int i = tid; i < SMP_BINS; i += SMP_TPB) sh.weight[i] = 0;
        uint32_t bound = key_bound(sh, mine, looked_for(d));
        if (d.k == 0) bound = min(bound, (uint32_t)best_of(sh, passed));
        Below b = { 0.0, { 0.0, 0.0 }, 0.0, row.steps((float)row.top), bound };
#pragma unroll
        for (int i = 0; i < PART_LIST / 64; i++) {
            if (held[i] == ~0ull) continue;
            if ((uint32_t)(held[i] >> 32) <= bound) push(sh, held[i]);
            else if (d.k == 0) {
                const Row::Steps s = row.steps(token_value(held[i]));
                const float bin = Row::below(b.top, s);
                if (bin < SMP_BINS) atomicAdd(&sh.weight[(int)bin], part_of_step(s.part));
            }
        }
        __syncthreads();
        double rest = 0.0;
        if (d.k == 0) {
            u64 units[2] = { sh.weight[2 * tid], sh.weight[2 * tid + 1] };
            // a part's bins begin at its own reference, so many below the largest logit's; a part without a bound has
            // passed nothing, and its reference may be no logit of the row
            const float behind = Row::below(b.top, row.steps(own->ref));
            if (lane == 0)
                sh.shown[wave] = passed != 0xffffffffu && behind >= 0.0f && behind < SMP_BINS ? (uint32_t)(int)behind
                                                                                             : (uint32_t)SMP_BINS;
            __syncthreads();
#pragma unroll 4
            for (int i = 0; i < a.parts; i++) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int at = 2 * tid + j - (int)sh.shown[i];
                    if (at >= 0) units[j] += in[i].weight[at];
                }
            }
            for (int i = 0; i < 2; i++) b.w[i] = bin_weight(row, b.top, 2 * tid + i, units[i]);
            b.upto = b.w[0] + b.w[1];
            rest = scan_f64(sh, b.upto);
        }
        int n = (int)sh.n;
        __syncthreads();
        if (n <= SMP_LIST) {
            if (finish(sh, a, r, d, row, n, rest, b.listed)) return;
            if (n <= SMP_HALF) {
                b.upto += b.listed;
                draw_below(sh, a, r, d, row, n, b);
                return;
            }
        }
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
