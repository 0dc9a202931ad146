// sample.hip -- one token a row from logits: temperature, top-k, top-p, min-p and a
// given random number.
//
// The row's tokens are ordered by (logit descending, index ascending); every step keeps
// a run of that order's start, and the draw inverts the summed weights along it.
// Weights exp((x - max) / T) are whole numbers of 2^-44: their sums are exact in 64
// bits, so neither atomics nor the split of the work changes them.  Instead of sorting
// the row, its weights and counts are summed by bins of (max - x) / T; only the bins
// that a border lies in are resolved, from their sorted tokens.
#include "common.h"

#include <algorithm>

namespace ds3k {

constexpr int SMP_TPB = 1024;
constexpr int SMP_BINS = 2048;               // bins of 1 / 64 over 32, the last of all beyond
constexpr int SMP_LIST = 4096;               // tokens sorted at once
constexpr double SMP_ONE = 0x1p44;           // the first token's weight

typedef unsigned long long u64;

// Ascending order of these 32 bits is descending order of values; -0 is 0.
__device__ __forceinline__ uint32_t order_key(float x)
{
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? b : 0x7fffffffu - b;
}

__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k : 0x7fffffffu - k); }

struct SampleShared {
    u64 weight[SMP_BINS];                    // by bin, then summed up to and with it
    uint32_t count[SMP_BINS];
    u64 list[SMP_LIST];                      // key << 32 | index
    u64 wave_w[SMP_TPB / 64];
    uint32_t wave_c[SMP_TPB / 64];
    u64 best;
    uint32_t n;
    int bin;
    u64 found[4];
};

// Inclusive sums over the workgroup.
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

struct Row {
    const float *x;
    int n;
    double top, inv_t;                       // the largest logit, 1 / temperature

    __device__ double depth(float v) const { return (top - (double)v) * inv_t; }
    __device__ int bin(float v) const
    {
        const double b = depth(v) * 64.0;
        return b < SMP_BINS - 1 ? (int)b : SMP_BINS - 1;
    }
    __device__ double weight(float v) const { return exp(-depth(v)); }
    __device__ u64 units(float v) const { return (u64)__double2ll_rn(weight(v) * SMP_ONE); }
};

__device__ __forceinline__ bool counts(float v) { return v > -INFINITY; }      // neither -inf nor NaN

// What a border is looked for by: the first token in order whose inclusive count or
// weight reaches `least`, or the last of at least `weight` (at least the first token).
enum : int { BY_COUNT, BY_WEIGHT };

// Where a border lies: the token, and the weights up to and with it.
struct Border {
    u64 token;                               // key << 32 | index
    u64 mass;
};

// The token in the subset { bin(x) == bin } at which the inclusive sum, from (w0, c0)
// before the subset, reaches `least`.  `members` is the subset's size.
__device__ Border resolve(SampleShared &sh, const Row &row, int bin, uint32_t members, u64 w0, uint32_t c0, int by, u64 least)
{
    // the subset is narrowed by digits of key << 32 | index until it can be sorted
    u64 prefix = 0, mask = 0;
    int shift = 64;
    while (members > SMP_LIST) {
        const int bits = min(11, shift);
        shift -= bits;
        __syncthreads();
        for (int b = threadIdx.x; b < SMP_BINS; b += SMP_TPB) {
            sh.weight[b] = 0;
            sh.count[b] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < row.n; i += SMP_TPB) {
            const float v = row.x[i];
            if (!counts(v) || row.bin(v) != bin) continue;
            const u64 c = (u64)order_key(v) << 32 | (uint32_t)i;
            if ((c & mask) != prefix) continue;
            const int d = (int)(c >> shift) & ((1 << bits) - 1);
            atomicAdd(&sh.weight[d], row.units(v));
            atomicAdd(&sh.count[d], 1u);
        }
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
            sh.found[3] = first ? ca : cb;
        }
        __syncthreads();
        prefix |= sh.found[0] << shift;
        mask |= (u64)((1 << bits) - 1) << shift;
        w0 = sh.found[1];
        c0 = (uint32_t)sh.found[2];
        members = (uint32_t)sh.found[3];
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < row.n; i += SMP_TPB) {
        const float v = row.x[i];
        if (!counts(v) || row.bin(v) != bin) continue;
        const u64 c = (u64)order_key(v) << 32 | (uint32_t)i;
        if ((c & mask) == prefix) sh.list[atomicAdd(&sh.n, 1u)] = c;
    }
    __syncthreads();
    const int n = (int)sh.n;
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += SMP_TPB) sh.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int i = threadIdx.x; i < size; i += SMP_TPB) {
                const int o = i ^ j;
                if (o > i) {
                    const u64 a = sh.list[i], b = sh.list[o];
                    if ((a > b) == ((i & k) == 0)) {
                        sh.list[i] = b;
                        sh.list[o] = a;
                    }
                }
            }
            __syncthreads();
        }
    for (int i0 = 0; i0 < n; i0 += SMP_TPB) {
        const int i = i0 + threadIdx.x;
        const u64 own = i < n ? row.units(key_value((uint32_t)(sh.list[i] >> 32))) : 0;
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

__global__ void __launch_bounds__(SMP_TPB) k_sample(SampleArgs p)
{
    __shared__ SampleShared sh;
    const int r = blockIdx.x, tid = threadIdx.x;
    Row row;
    row.x = (const float *)((const uint8_t *)p.logits + (uint64_t)r * p.stride);
    row.n = p.n_vocab;
    if (tid == 0) sh.best = ~0ull;
    for (int b = tid; b < SMP_BINS; b += SMP_TPB) {
        sh.weight[b] = 0;
        sh.count[b] = 0;
    }
    __syncthreads();
    u64 best = ~0ull;
    for (int i = tid; i < row.n; i += SMP_TPB) {
        const float v = row.x[i];
        if (counts(v)) best = min(best, (u64)order_key(v) << 32 | (uint32_t)i);
    }
    for (int d = 32; d > 0; d /= 2) best = min(best, (u64)__shfl_xor(best, d));
    if ((tid & 63) == 0) atomicMin(&sh.best, best);
    __syncthreads();
    best = sh.best;
    const float top = key_value((uint32_t)(best >> 32)), t = p.temperature ? p.temperature[r] : 1.0f;
    if (best == ~0ull || !(t > 0.0f) || top == INFINITY) {
        if (tid == 0) {
            p.tokens[r] = best == ~0ull ? -1 : (int)(uint32_t)best;
            if (p.probs) p.probs[r] = best == ~0ull ? 0.0f : 1.0f;
        }
        return;
    }
    row.top = (double)top;
    row.inv_t = 1.0 / (double)t;

    for (int i = tid; i < row.n; i += SMP_TPB) {
        const float v = row.x[i];
        if (!counts(v)) continue;
        const int b = row.bin(v);
        atomicAdd(&sh.weight[b], row.units(v));
        atomicAdd(&sh.count[b], 1u);
    }
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
            sh.found[2] = first ? ca : cb;
        }
        __syncthreads();
        const int bin = sh.bin;
        const u64 w0 = sh.found[0];
        const uint32_t c0 = (uint32_t)sh.found[1], members = (uint32_t)sh.found[2];
        __syncthreads();
        return resolve(sh, row, bin, members, w0, c0, by, least);
    };
    u64 mass = w_all;
    const int k = p.top_k ? p.top_k[r] : 0;
    if (k > 0 && (uint32_t)k < c_all) mass = border(BY_COUNT, (u64)k).mass;
    const float top_p = p.top_p ? p.top_p[r] : 1.0f;
    if (top_p < 1.0f) {
        const u64 least = max((u64)ceil((double)max(top_p, 0.0f) * (double)mass), 1ull);
        mass = border(BY_WEIGHT, min(least, mass)).mass;
    }
    const float min_p = p.min_p ? p.min_p[r] : 0.0f;
    if (min_p > 0.0f) {
        // the weights of at least min_p: counted, as they are a run of the order's start
        u64 w = 0, all;
        uint32_t c = 0, c_min;
        for (int i = tid; i < row.n; i += SMP_TPB) {
            const float v = row.x[i];
            if (counts(v) && row.weight(v) >= (double)min_p) w += row.units(v);
        }
        scan2(sh, w, c, all, c_min);
        __syncthreads();
        mass = min(mass, max(all, (u64)SMP_ONE));
    }
    const float u = p.uniform[r];
    const u64 least = min((u64)floor((double)(u > 0.0f ? u : 0.0f) * (double)mass) + 1, mass);
    const Border drawn = border(BY_WEIGHT, least);
    if (tid == 0) {
        p.tokens[r] = (int)(uint32_t)drawn.token;
        if (p.probs) p.probs[r] = (float)(row.weight(key_value((uint32_t)(drawn.token >> 32))) * SMP_ONE / (double)mass);
    }
}

hipError_t launch_sample(const SampleArgs &p, hipStream_t s)
{
    hipLaunchKernelGGL(k_sample, dim3(p.n_rows), SMP_TPB, 0, s, p);
    return hipGetLastError();
}

}  // namespace ds3k
