// kv_cache.hip -- what surrounds attention over a paged cache: rotary positions
// with the heads' norms, the writing of new tokens' k and v, and the plan of a
// step's blocks, positions and slots from the requests' lengths.
#include "common.h"
#include "lanes.h"

#include <algorithm>

namespace ds3k {

// ---------------------------------------------------------------------------
// Rotary positions.  Pair j of a head turns by position * theta_j; the table holds
// theta_j / (2 pi), so the product's whole part is dropped in 64 bits (32 lose the
// angle of far positions) and sine and cosine are taken of the remaining half turn
// in 32.  They depend on the token and the pair alone: a workgroup computes those of its
// tokens into LDS, then a group of lanes holds V pairs a lane of one token and walks over
// some of its heads, those of a token's groups side by side.
// Bound by memory: 4096 tokens of 32 + 4 + 4 heads of 128 from F32 to F16 with norms
// 22 us for 126 MB, 5.7 TB/s (part of it from the last-level cache); 4001 tokens of 64
// heads, F16 to F16, 31 us for 131 MB, 4.2 TB/s, where a copy moves 4.6.  With angles in
// every group by itself 22 and 33 (the vector units are busy 78 % of the second), runs of
// heads a group besides 23 and 36; two heads a group 27 and 32, eight 22 and 31; the next
// head's loads ahead of this one's work 23 and 35; loads that pass the caches by 26 and
// 42.  One token: 3.8 us, the launch.
// ---------------------------------------------------------------------------

constexpr int ROPE_TPB = 256;

template <typename T, int V>
__device__ __forceinline__ void load_row(const T *p, float (&v)[V])
{
    typedef T vec __attribute__((ext_vector_type(V)));
    if constexpr (V == 1) v[0] = (float)*p;
    else {
        const vec x = *(const vec *)p;
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = (float)x[i];
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T *p, const float (&v)[V])
{
    typedef T vec __attribute__((ext_vector_type(V)));
    if constexpr (V == 1) *p = (T)v[0];
    else {
        vec x;
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = (T)v[i];
        *(vec *)p = x;
    }
}

// A unit is V pairs of a head: values e .. e + V - 1 and f .. f + V - 1 where the
// halves turn against each other, 2 V consecutive ones where neighbours do and
// where nothing turns.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void load_unit(const T *head, int unit, bool turns, int half, float (&a)[V], float (&b)[V])
{
    if (INTER || !turns) {
        float w[2 * V];
        load_row<T, 2 * V>(head + 2 * V * unit, w);
#pragma unroll
        for (int i = 0; i < V; i++) {
            a[i] = w[INTER && turns ? 2 * i : i];
            b[i] = w[INTER && turns ? 2 * i + 1 : V + i];
        }
    } else {
        load_row<T, V>(head + V * unit, a);
        load_row<T, V>(head + half + V * unit, b);
    }
}

template <typename T, int V, bool INTER>
__device__ __forceinline__ void store_unit(T *head, int unit, bool turns, int half, const float (&a)[V], const float (&b)[V])
{
    if (INTER || !turns) {
        float w[2 * V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            w[INTER && turns ? 2 * i : i] = a[i];
            w[INTER && turns ? 2 * i + 1 : V + i] = b[i];
        }
        store_row<T, 2 * V>(head + 2 * V * unit, w);
    } else {
        store_row<T, V>(head + V * unit, a);
        store_row<T, V>(head + half + V * unit, b);
    }
}

// V divides rotary_dim / 2; a lane takes units lane, lane + lanes, ... of a head.
template <typename TI, typename TO, int V, bool INTER>
__global__ void __launch_bounds__(ROPE_TPB) k_rope(RopeArgs p)
{
    constexpr int NU = 4 / V;
    __shared__ float2 angle[4 * ROPE_TPB];            // cosine and sine: (ROPE_TPB / lanes) tokens of half <= 4 lanes pairs
    const int lane = threadIdx.x & (p.lanes - 1), half = p.rotary / 2;
    const int groups = ROPE_TPB / p.lanes, tokens = max(groups >> p.log_chunks, 1);
    const int64_t group = (int64_t)blockIdx.x * groups + threadIdx.x / p.lanes;
    const int64_t t = group >> p.log_chunks, t0 = (int64_t)blockIdx.x * groups >> p.log_chunks;
    if (half > 0) {
        const float m = (float)p.table[half];
        for (int i = threadIdx.x; i < tokens * half; i += ROPE_TPB) {
            const int of = tokens == 1 ? 0 : i / half;
            if (t0 + of >= p.n_tokens) break;
            const double turn = (double)p.positions[t0 + of] * p.table[i - of * half];
            float s, c;
            sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
            angle[i] = make_float2(m * c, m * s);
        }
        __syncthreads();
    }
    const int heads = p.n_head + 2 * p.n_head_kv, chunks = 1 << p.log_chunks;
    const int h0 = (int)(group & (chunks - 1));
    if (t >= p.n_tokens || h0 >= heads) return;
    const int units = p.head_dim / (2 * V), turning = half / V;

    float c[NU][V], s[NU][V];
#pragma unroll
    for (int u = 0; u < NU; u++) {
        const int unit = lane + u * p.lanes;
        if (unit < turning) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float2 cs = angle[(int)(t - t0) * half + unit * V + i];
                c[u][i] = cs.x;
                s[u][i] = cs.y;
            }
        }
    }

    int64_t at = 0;                       // first value of the token's row of kv head 0 in a cache; below 0: no row
    if (p.n_head_kv > 0) {
        const int64_t slot = p.slots[t];
        at = slot < 0 || slot >= p.n_slots ? -1
           : (((slot >> p.log_block) * p.n_head_kv << p.log_block) + (slot & ((1 << p.log_block) - 1))) * p.head_dim;
    }

    for (int h = h0; h < heads; h += chunks) {
        const int kind = h < p.n_head ? 0 : h < p.n_head + p.n_head_kv ? 1 : 2;
        const int g = h - (kind == 0 ? 0 : kind == 1 ? p.n_head : p.n_head + p.n_head_kv);
        if (kind != 0 && at < 0) continue;
        const TI *src = (const TI *)((const uint8_t *)p.x[kind] + t * p.stride[kind]) + (int64_t)g * p.head_dim;
        float a[NU][V], b[NU][V];
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const int unit = lane + u * p.lanes;
            if (unit < units) load_unit<TI, V, INTER>(src, unit, unit < turning, half, a[u], b[u]);
        }
        const float *w = kind == 2 ? nullptr : p.norm[kind];
        if (w != nullptr) {
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < NU; u++)
                if (lane + u * p.lanes < units) {
#pragma unroll
                    for (int i = 0; i < V; i++) sum += a[u][i] * a[u][i] + b[u][i] * b[u][i];
                }
            for (int d = p.lanes / 2; d > 0; d /= 2) sum += __shfl_xor(sum, d);
            const float r = 1.0f / sqrtf(sum / (float)p.head_dim + p.eps);
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const int unit = lane + u * p.lanes;
                if (unit < units) {
                    float wa[V], wb[V];
                    load_unit<float, V, INTER>(w, unit, unit < turning, half, wa, wb);
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        a[u][i] = a[u][i] * r * wa[i];
                        b[u][i] = b[u][i] * r * wb[i];
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const int unit = lane + u * p.lanes;
            if (unit >= units) continue;
            if (kind != 2 && unit < turning) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float x = a[u][i], y = b[u][i];
                    a[u][i] = x * c[u][i] - y * s[u][i];
                    b[u][i] = y * c[u][i] + x * s[u][i];
                }
            }
            const bool turns = unit < turning;
            if (kind == 0) {
                TO *dst = (TO *)((uint8_t *)p.out + t * p.out_stride) + (int64_t)g * p.head_dim;
                store_unit<TO, V, INTER>(dst, unit, turns, half, a[u], b[u]);
            } else {
                _Float16 *dst = (_Float16 *)(kind == 1 ? p.k_cache : p.v_cache) + at + ((int64_t)g << p.log_block) * p.head_dim;
                store_unit<_Float16, V, INTER>(dst, unit, turns, half, a[u], b[u]);
            }
        }
    }
}

template <typename TI, typename TO, int V>
static void rope_launch(const RopeArgs &p, bool inter, dim3 grid, hipStream_t s)
{
    if (inter) hipLaunchKernelGGL((k_rope<TI, TO, V, true>), grid, ROPE_TPB, 0, s, p);
    else hipLaunchKernelGGL((k_rope<TI, TO, V, false>), grid, ROPE_TPB, 0, s, p);
}

template <typename TI, typename TO>
static void rope_width(const RopeArgs &p, bool inter, int v, dim3 grid, hipStream_t s)
{
    if (v == 4) rope_launch<TI, TO, 4>(p, inter, grid, s);
    else if (v == 2) rope_launch<TI, TO, 2>(p, inter, grid, s);
    else rope_launch<TI, TO, 1>(p, inter, grid, s);
}

constexpr int ROPE_HEADS = 5;                // that a group of lanes takes at most

static int rope_pairs(const RopeArgs &p) { return p.rotary % 8 == 0 ? 4 : p.rotary % 4 == 0 ? 2 : 1; }

static int rope_lanes(const RopeArgs &p)
{
    int lanes = 1;
    while (lanes < std::min(p.head_dim / (2 * rope_pairs(p)), WAVE)) lanes *= 2;
    return lanes;
}

// Workgroups of groups that take `per` heads each or a few less; p.lanes is set.
static int64_t rope_split(RopeArgs &p, int per)
{
    p.log_chunks = 0;
    while ((1 << p.log_chunks) * per < p.n_head + 2 * p.n_head_kv) p.log_chunks++;
    return ((p.n_tokens << p.log_chunks) * p.lanes + ROPE_TPB - 1) / ROPE_TPB;
}

bool rope_fits(RopeArgs p)
{
    p.lanes = rope_lanes(p);
    return rope_split(p, ROPE_HEADS) <= 0xffffff;
}

hipError_t launch_rope(RopeArgs p, int in_type, int out_type, bool inter, hipStream_t s)
{
    const int v = rope_pairs(p);
    p.lanes = rope_lanes(p);
    // one head a group of lanes until the card is full, then up to five
    const int64_t groups = p.n_tokens * (p.n_head + 2 * p.n_head_kv),
                  full = (int64_t)device_cu_count() * 8 * (ROPE_TPB / p.lanes);
    const int64_t wgs = rope_split(p, (int)std::clamp<int64_t>(groups / full, 1, ROPE_HEADS));
    if (wgs > 0xffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)wgs);
    if (in_type == T_F32) {
        if (out_type == T_F32) rope_width<float, float>(p, inter, v, grid, s);
        else rope_width<float, _Float16>(p, inter, v, grid, s);
    } else if (out_type == T_F32) rope_width<_Float16, float>(p, inter, v, grid, s);
    else rope_width<_Float16, _Float16>(p, inter, v, grid, s);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// The step's plan.  One workgroup sums tokens and missing blocks over the requests
// (two prefix sums) and decides; then every token finds its request by bisection of
// the offsets.  A new block's first position is a new token's, so that token enters
// the block in the table and nothing is written twice.
// Bound by latency: lengths, sums and the decision are a chain of 4 us at any size (5 with
// sums by LDS exchanges); up to 2048 rows the same workgroup writes them (8 requests: 4 us
// in all), more are a second launch of 4.7 us (1000 requests, 25,000 rows).
// ---------------------------------------------------------------------------

constexpr int PLAN_TPB = 1024;

struct PlanSums {
    long long tokens, blocks;
};

// Inclusive sums over the workgroup; `total` gets those of all.
__device__ __forceinline__ PlanSums plan_scan(PlanSums v, PlanSums *waves, PlanSums &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v.tokens = wave_scan(v.tokens);
    v.blocks = wave_scan(v.blocks);
    __syncthreads();
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    total = { 0, 0 };
    for (int w = 0; w < PLAN_TPB / 64; w++) {
        const PlanSums o = waves[w];
        if (w < wave) {
            v.tokens += o.tokens;
            v.blocks += o.blocks;
        }
        total.tokens += o.tokens;
        total.blocks += o.blocks;
    }
    return v;
}

__device__ __forceinline__ int sat32(long long v) { return (int)min(v, 0x7fffffffll); }

// Rows [row0, row1) in steps of `step`, `total` of which belong to requests: position, slot, and the table's new entries.
template <typename O>
__device__ __forceinline__ void plan_rows(const PlanArgs &p, O offsets, int total, int n_free, int64_t row0, int64_t row1, int step)
{
    for (int64_t t = row0; t < row1; t += step) {
        int position = 0, slot = -1;
        if (t < total) {
            int lo = 0, hi = p.n_seq;                 // offsets(lo) <= t < offsets(hi)
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (offsets(mid) <= t) lo = mid;
                else hi = mid;
            }
            const int cached = p.cached[lo];
            position = cached + (int)(t - offsets(lo));
            const int had = (int)(((int64_t)cached + (1 << p.log_block) - 1) >> p.log_block), at = position >> p.log_block;
            int32_t *entry = p.table + (int64_t)lo * p.max_blocks + at;
            int block;
            if (at >= had) {
                block = p.free_blocks[n_free - 1 - (p.first[lo] + at - had)];
                if ((position & ((1 << p.log_block) - 1)) == 0) *entry = block;
            } else block = *entry;
            if (block >= 0 && block < p.n_blocks) slot = (block << p.log_block) + (position & ((1 << p.log_block) - 1));
        }
        p.positions[t] = position;
        p.slots[t] = slot;
    }
}

constexpr int PLAN_HELD = 4096;              // requests whose offsets are bisected in LDS

template <bool ROWS>
__global__ void __launch_bounds__(PLAN_TPB) k_kv_plan(PlanArgs p)
{
    __shared__ PlanSums waves[PLAN_TPB / 64];
    __shared__ int too_long;
    if (threadIdx.x == 0) too_long = 0;
    __syncthreads();                                  // (before any wave counts)
    const int n_free = min(max(*p.n_free, 0), p.n_blocks);
    PlanSums sum = { 0, 0 };
    for (int i0 = 0; i0 < p.n_seq; i0 += PLAN_TPB) {  // prefix sums, kept where they are looked up
        const int i = i0 + threadIdx.x;
        long long cached = 0, fresh = 0, n = 0;
        if (i < p.n_seq) {
            cached = max(p.kv_lens[i], 0);
            n = max(p.new_lens[i], 0);
            const long long b = (1 << p.log_block) - 1, have = (cached + n + b) >> p.log_block;
            fresh = n > 0 ? have - ((cached + b) >> p.log_block) : 0;
            if (have > p.max_blocks) atomicAdd(&too_long, 1);
        }
        PlanSums total;
        const PlanSums in = plan_scan({ n, fresh }, waves, total);
        if (i < p.n_seq) {
            p.cached[i] = (int)cached;
            p.first[i] = sat32(sum.blocks + in.blocks - fresh);
            p.offsets[i + 1] = sat32(sum.tokens + in.tokens);
        }
        sum.tokens += total.tokens;
        sum.blocks += total.blocks;
    }
    __syncthreads();
    const long long lacking = max(sum.blocks - n_free, 0ll);
    const bool done = lacking == 0 && too_long == 0 && sum.tokens <= p.max_tokens;
    if (threadIdx.x == 0) {
        p.head[0] = n_free;
        p.offsets[0] = 0;
        p.status[0] = sat32(sum.tokens);
        p.status[1] = sat32(sum.blocks);
        p.status[2] = sat32(lacking);
        p.status[3] = too_long;
        const int left = done ? n_free - (int)sum.blocks : *p.n_free;
        *p.n_free_out = left;
    }
    for (int i = threadIdx.x; i < p.n_seq; i += PLAN_TPB) {
        const int had = p.kv_lens[i];
        p.kv_lens_out[i] = done ? p.cached[i] + max(p.new_lens[i], 0) : had;
        if (!done) p.offsets[i + 1] = 0;
    }
    if constexpr (ROWS) {
        __syncthreads();
        const int total = done ? (int)sum.tokens : 0;
        plan_rows(p, [&](int i) { return p.offsets[i]; }, total, n_free, threadIdx.x, p.max_tokens, PLAN_TPB);
    }
}

__global__ void __launch_bounds__(256) k_kv_plan_rows(PlanArgs p)
{
    __shared__ int held[PLAN_HELD];
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, end = min((int64_t)p.max_tokens, t + 1);
    const int total = p.offsets[p.n_seq], n_free = p.head[0];
    if (p.n_seq <= PLAN_HELD) {              // (in memory each step of the bisection is a round trip: 5.6 us in place of 4.7 for 1000)
        for (int i = threadIdx.x; i < p.n_seq; i += 256) held[i] = p.offsets[i];
        __syncthreads();
        plan_rows(p, [&](int i) { return held[i]; }, total, n_free, t, end, 1);
    } else plan_rows(p, [&](int i) { return p.offsets[i]; }, total, n_free, t, end, 1);
}

hipError_t launch_kv_plan(const PlanArgs &p, hipStream_t s)
{
    if (p.max_tokens <= 2 * PLAN_TPB) hipLaunchKernelGGL(k_kv_plan<true>, dim3(1), PLAN_TPB, 0, s, p);
    else {
        hipLaunchKernelGGL(k_kv_plan<false>, dim3(1), PLAN_TPB, 0, s, p);
        hipLaunchKernelGGL(k_kv_plan_rows, dim3((unsigned)((p.max_tokens + 255) / 256)), 256, 0, s, p);
    }
    return hipGetLastError();
}

// Blocks given back.  A thread copies a request's entries one after the other, each a round trip to memory: 64 requests of
// 2048 blocks 400 us, 1000 of 128 170, eight of 64 23.  It runs once a request, not once a step.
__global__ void __launch_bounds__(PLAN_TPB) k_kv_release(ReleaseArgs p)
{
    __shared__ PlanSums waves[PLAN_TPB / 64];
    const int n_free = min(max(*p.n_free, 0), p.n_blocks);
    const auto blocks_of = [&](int i) -> long long {
        if (i >= p.n_seq || p.done[i] == 0) return 0;
        return min(((long long)max(p.kv_lens[i], 0) + (1 << p.log_block) - 1) >> p.log_block, (long long)p.max_blocks);
    };
    long long sum = 0;
    for (int i0 = 0; i0 < p.n_seq; i0 += PLAN_TPB) {
        PlanSums total;
        plan_scan({ 0, blocks_of(i0 + threadIdx.x) }, waves, total);
        sum += total.blocks;
    }
    if (sum > p.n_blocks - n_free) return;            // the same for every thread
    long long base = n_free;
    for (int i0 = 0; i0 < p.n_seq; i0 += PLAN_TPB) {
        const int i = i0 + threadIdx.x;
        const long long n = blocks_of(i);
        PlanSums total;
        const PlanSums in = plan_scan({ 0, n }, waves, total);
        for (long long j = 0; j < n; j++)
            p.free_blocks[base + in.blocks - n + j] = p.table[(int64_t)i * p.max_blocks + j];
        if (i < p.n_seq && p.done[i] != 0) p.kv_lens[i] = 0;
        base += total.blocks;
    }
    if (threadIdx.x == 0) *p.n_free = (int)base;
}

hipError_t launch_kv_release(const ReleaseArgs &p, hipStream_t s)
{
    hipLaunchKernelGGL(k_kv_release, dim3(1), PLAN_TPB, 0, s, p);
    return hipGetLastError();
}

}  // namespace ds3k
