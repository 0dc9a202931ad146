// attention.hip -- attention of new tokens over a paged fp16 cache.
//
// Token j of a request with n cached and new tokens, m of them new, is at position
// p = n - m + j.  Its output is sum_k w_k v_k / sum_k w_k over the keys k that it sees,
// w_k = 2^(c (s_k - max s)), s_k = q . k_k, c = scale log2 e, with the maximum and the
// sums carried over the keys in one pass.  The rows of a kv head are its tokens' q heads
// side by side (row = token * group + head of the group): all share the keys.
//
// Both products run transposed on the matrix cores, S^T = K Q^T and O^T = V^T P^T: a
// lane of the S^T result holds a row's weights for just those keys that it must hand
// to the second product, so weights never cross lanes.  Weights carry a factor 2^8
// (ATT_SHIFT), which cancels, so that small ones keep F16's precision.
//
// F32 rows are scaled by a power of two to about 2^14 and split into two F16 parts, as
// are the weights: products of 22 bits with the cache's exact values.
#include "common.h"
#include "lanes.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace ds3k {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float ATT_SHIFT = 8.0f;
constexpr float ATT_LAG = 6.0f;              // a maximum may rise by 2^6 before sums are rescaled: weights stay below 2^14

// ---------------------------------------------------------------------------
// The split of the work.  A unit is one tile of rows (M of a request) with one run
// of keys; runs are of `run` keys, chosen from all requests' lengths so that about
// `target` units a kv head result, none shorter than `least`.  Every workgroup finds
// its unit from the lengths by itself, in prefix sums over the requests.
// ---------------------------------------------------------------------------

struct Unit {
    int seq, tile, chunk, run;
    int whole;                               // the first unit of the tile, chunk 0
    int first, m, kv;                        // the request's first row, new tokens, length
    int n;                                   // positions that its blocks hold
};

constexpr int ATT_TPB = 256;
constexpr int ATT_FEW_ROWS = 64;             // requests of up to so many rows take tiles of 16
constexpr int ATT_WHOLE = 0x7fff0000;        // a run that holds any request's keys

__device__ __forceinline__ long long wave_sum(long long v)
{
    return lanes_join<32>(v, [](long long x, long long y) { return x + y; });
}

// Request i's tiles of M rows and the most keys that one of them sees.
__host__ __device__ __forceinline__ void request_work(const AttnArgs &p, int M, int i, int &tiles, int &span, Unit &u)
{
    tiles = span = 0;
    if (i >= p.n_seq) return;
    const int group = p.n_head / p.n_head_kv, o0 = p.offsets[i], o1 = p.offsets[i + 1];
    if (o0 < 0 || o1 <= o0 || o1 > p.n_tokens) return;
    u.first = o0;
    u.m = o1 - o0;
    u.kv = p.lens[i];
    u.n = (int)std::min((int64_t)std::max(u.kv, 0), (int64_t)p.max_blocks << p.log_block);
    const long long rows = (long long)u.m * group;
    if (rows < p.min_rows || rows > p.max_rows) return;
    tiles = (int)((rows + M - 1) / M);
    span = p.window ? (int)std::min((long long)u.n, (long long)p.window + M / group + 130) : u.n;
    span = std::max(span, 1);
}

// Keys a unit: work / (target - tiles) or a little more, so that splitting adds at most target - tiles units.
__host__ __device__ __forceinline__ int whole_runs(const AttnArgs &p, int M, float want)
{
    const int grain = M == 16 ? 128 : 64;             // keys that a workgroup takes at a time
    return want >= 0x1p30f ? ATT_WHOLE : std::max(((int)want + grain) & -grain, p.least);
}
// (span and run up to ATT_WHOLE: their sum passes 2^31)
__host__ __device__ __forceinline__ int runs_of(int span, int run)
{
    return (int)(((unsigned)span + (unsigned)run - 1) / (unsigned)run);
}
__host__ __device__ __forceinline__ int unit_run(const AttnArgs &p, int M, long long work, long long tiles)
{
    if (tiles >= p.target) return ATT_WHOLE;
    return whole_runs(p, M, (float)work / (float)(p.target - tiles) * (1.0f + 0x1p-20f));
}
// Runs that fill `target` units if no tile's last run were short: shorter ones, to be taken where the units that result
// are no more than `target` (one chunk of 512 tokens: 16 tiles in four runs each rather than three, 45 us to 38).
__host__ __device__ __forceinline__ int tight_run(const AttnArgs &p, int M, long long work)
{
    return whole_runs(p, M, (float)work / (float)p.target * (1.0f + 0x1p-20f));
}

// A value that every lane of the wave has, in a scalar register: what follows from it branches.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The unit `id` of this workgroup's kv head, or with TILES the tile `id` (its chunk 0); false: none.
template <int TPB, bool TILES>
__device__ __forceinline__ bool search_unit(const AttnArgs &p, int M, int id, Unit &u)
{
    __shared__ long long part[2][TPB / 64];
    __shared__ int found[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (p.n_seq == 1) {
        int tiles, span;
        request_work(p, M, 0, tiles, span, u);
        u.seq = 0;
        u.run = unit_run(p, M, (long long)tiles * span, tiles);
        const int tight = tight_run(p, M, (long long)tiles * span);
        if (tight < u.run && (long long)tiles * runs_of(span, tight) <= p.target) u.run = tight;
        const int chunks = runs_of(span, u.run);
        if ((long long)id >= (long long)tiles * (TILES ? 1 : chunks)) return false;
        u.tile = TILES ? id : id / chunks;
        u.whole = u.tile * chunks;
        u.chunk = TILES ? 0 : id - u.whole;
        u.tile = tiles - 1 - u.tile;                  // (the last tiles, which see most keys, begin first)
        return true;
    }
    if (p.n_seq <= 64) {                              // every wave by itself: neither LDS nor a barrier
        int tiles, span;
        request_work(p, M, lane, tiles, span, u);
        const long long work = wave_sum((long long)tiles * span);
        u.run = unit_run(p, M, work, wave_sum((long long)tiles));
        const int tight = tight_run(p, M, work);
        if (tight < u.run && wave_sum((long long)tiles * runs_of(span, tight)) <= p.target) u.run = tight;
        const long long units = (long long)tiles * runs_of(span, u.run);
        const long long at = wave_scan(units) - units, first = TILES ? wave_scan((long long)tiles) - tiles : at;
        const uint64_t here = __ballot(id >= first && id < first + (TILES ? tiles : units));
        if (here == 0) return false;
        const int i = __builtin_ctzll(here), of = (int)(id - first), chunks = runs_of(span, u.run);
        u.seq = i;
        u.tile = TILES ? of : of / max(chunks, 1);
        u.chunk = TILES ? 0 : of - u.tile * chunks;
        u.whole = (int)at + u.tile * chunks;
        u.tile = tiles - 1 - u.tile;
        for (int *v : { &u.tile, &u.chunk, &u.whole, &u.first, &u.m, &u.kv, &u.n }) *v = __builtin_amdgcn_readlane(*v, i);
        return true;
    }
    long long work = 0, all = 0;
    for (int i0 = 0; i0 < p.n_seq; i0 += TPB) {
        int tiles, span;
        Unit r;
        request_work(p, M, i0 + tid, tiles, span, r);
        work += (long long)tiles * span;
        all += tiles;
    }
    work = wave_sum(work);
    all = wave_sum(all);
    if (lane == 0) {
        part[0][wave] = work;
        part[1][wave] = all;
    }
    if (tid == 0) found[0] = -1;
    __syncthreads();
    work = all = 0;
    for (int w = 0; w < TPB / 64; w++) {
        work += part[0][w];
        all += part[1][w];
    }
    __syncthreads();
    u.run = unit_run(p, M, work, all);
    long long before = 0, units_before = 0;           // of what `id` counts, and of units
    for (int i0 = 0; i0 < p.n_seq && before <= id; i0 += TPB) {
        int tiles, span;
        Unit r;
        request_work(p, M, i0 + tid, tiles, span, r);
        const long long units = (long long)tiles * runs_of(span, u.run);
        const long long sum = wave_scan(units), tile_sum = wave_scan((long long)tiles);
        if (lane == 63) {
            part[0][wave] = sum;
            part[1][wave] = tile_sum;
        }
        __syncthreads();
        long long total = 0, tile_total = 0, at = units_before + sum - units, tile_at = before + tile_sum - tiles;
        for (int w = 0; w < TPB / 64; w++) {
            if (w < wave) {
                at += part[0][w];
                tile_at += part[1][w];
            }
            total += part[0][w];
            tile_total += part[1][w];
        }
        const long long first = TILES ? tile_at : at, own = TILES ? tiles : units;
        if (own > 0 && id >= first && id < first + own) {
            found[0] = i0 + tid;
            found[1] = (int)(id - first);
            found[2] = (int)at;
        }
        units_before += total;
        before += TILES ? tile_total : total;
        __syncthreads();
    }
    if (found[0] < 0) return false;
    int tiles, span;
    u.seq = found[0];
    request_work(p, M, u.seq, tiles, span, u);
    const int chunks = runs_of(span, u.run);
    u.tile = TILES ? found[1] : found[1] / chunks;
    u.chunk = TILES ? 0 : found[1] - u.tile * chunks;
    u.whole = found[2] + u.tile * chunks;
    u.tile = tiles - 1 - u.tile;
    return true;
}

template <int TPB, bool TILES>
__device__ __forceinline__ bool find_unit(const AttnArgs &p, int M, int id, Unit &u)
{
    Unit v;
    const bool is = search_unit<TPB, TILES>(p, M, id, v);
    u = { uniform(v.seq), uniform(v.tile), uniform(v.chunk), uniform(v.run), uniform(v.whole), uniform(v.first), uniform(v.m),
          uniform(v.kv), uniform(v.n) };
    return is;
}

// What a unit works on: rows of the tile, the keys that any of them sees from a multiple of 32 to an end, in how
// many runs.
struct Tile {
    int row0, rows, j0, j1;                  // rows, and the tokens of the first and the last
    int64_t base;                            // the position of the request's first new token
    int start, end, chunks;
};

__device__ __forceinline__ Tile tile_of(const AttnArgs &p, int M, const Unit &u)
{
    Tile t;
    const int group = p.n_head / p.n_head_kv;
    t.row0 = u.tile * M;
    t.rows = min(u.m * group - t.row0, M);
    t.j0 = t.row0 / group;
    t.j1 = (t.row0 + t.rows - 1) / group;
    t.base = (int64_t)u.kv - u.m;
    t.end = (int)max(min(t.base + t.j1 + 1, (int64_t)u.n), (int64_t)0);
    t.start = p.window ? (int)max(t.base + t.j0 - p.window + 1, (int64_t)0) & ~31 : 0;
    t.chunks = t.end > t.start ? runs_of(t.end - t.start, u.run) : 1;
    return t;
}

// ---------------------------------------------------------------------------
// Parts
// ---------------------------------------------------------------------------

// v * 2^-e in two F16 parts, hi + lo, for |v| 2^-e below 2^15.
__device__ __forceinline__ void split(float v, _Float16 &hi, _Float16 &lo)
{
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// The power of two that brings a row's largest magnitude to 2^13 .. 2^14 (below it where that is no normal number; 1 where
// it is not finite), as its exponent.
__device__ __forceinline__ int row_exponent(float amax)
{
    const int e = (int)((__float_as_uint(amax) >> 23) & 255);
    return e == 255 ? 0 : 13 + 127 - max(e, 1);
}

__device__ __forceinline__ float mul_pow2(float v, int e) { return __builtin_ldexpf(v, e); }

// A row's power of two, held so that the scale (not 0) without it stays above 2^-123: masked scores are -inf and must not
// meet a 0.  Where it is held, the scale comes to less than 2^-98 and scores are below 2^39: all weights are alike,
// whatever bits of q are lost.
__device__ __forceinline__ int held_exponent(int e, float scale)
{
    return min(e, 100 + (int)(__float_as_uint(scale) >> 23) - 127);
}

// 16 keys x 32 values: lane l holds key (or row) l % 16, values 8 (l / 16) + 0 .. 7.
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Two values of v, those that are not finite made 0; `bad` tells of one.
__device__ __forceinline__ int finite_pair(int w, bool &bad)
{
    const int keep = ((w & 0x7c00) != 0x7c00 ? 0xffff : 0) | ((w & 0x7c000000) != 0x7c000000 ? (int)0xffff0000 : 0);
    bad |= keep != -1;
    return w & keep;
}

// Four values of a row of v where they are not finite, else 0.
__device__ __forceinline__ f32x4 odd_values(const _Float16 *v)
{
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    const f16x4 x = *(const f16x4 *)v;
    f32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = __builtin_fabsf((float)x[i]) < INFINITY ? 0.0f : (float)x[i];
    return o;
}

// A lane's row of q, NC chunks of eight values STEP apart, as F16 parts with the row's power of two taken out of `c2`;
// STEP / 8 lanes share a row.  Every load is made, of columns that are there: a branch around each
// would wait for it (41,000 cycles of a unit's 130,000).
template <typename T, bool PAD, int NC, int STEP>
__device__ __forceinline__ void load_q(const AttnArgs &p, const T *q, bool live, int h, f16x8 *hi, f16x8 *lo, float &c2)
{
    if constexpr (sizeof(T) == 4) {
        f32x4 x[2 * NC];
#pragma unroll
        for (int c = 0; c < 2 * NC; c++) {
            const int at = STEP * (c / 2) + 8 * h;
            x[c] = *(const f32x4 *)(q + (PAD && at >= p.head_dim ? 0 : at) + 4 * (c & 1));
        }
        float amax = 0.0f;
#pragma unroll
        for (int c = 0; c < 2 * NC; c++) {
            const bool in = live && (!PAD || STEP * (c / 2) + 8 * h < p.head_dim);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[c][e] = in ? x[c][e] * p.q_sign : 0.0f;
                amax = fmaxf(amax, fabsf(x[c][e]));
            }
        }
        if constexpr (STEP == 32) amax = fmaxf(amax, lane_xor<16>(amax));
        amax = fmaxf(amax, lane_xor<32>(amax));
        const int ex = held_exponent(row_exponent(amax), c2);
        c2 = fminf(mul_pow2(c2, -ex), FLT_MAX);
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                _Float16 a, b;
                split(mul_pow2(x[2 * c + e / 4][e & 3], ex), a, b);
                hi[c][e] = a;
                lo[c][e] = b;
            }
    } else {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const bool in = !PAD || STEP * c + 8 * h < p.head_dim;
            f16x8 v = *(const f16x8 *)(q + (in ? STEP * c + 8 * h : 0));
            if (!live || !in) v = f16x8{ 0, 0, 0, 0, 0, 0, 0, 0 };
            hi[c] = v * (_Float16)p.q_sign;
        }
    }
}

// The row of a cache that holds position `key` (of kv head g) in `block`: its first value's index.
__device__ __forceinline__ int64_t cache_row(const AttnArgs &p, int block, int key, int g)
{
    return ((((int64_t)block * p.n_head_kv + g) << p.log_block) + (key & ((1 << p.log_block) - 1))) * p.head_dim;
}

// ---------------------------------------------------------------------------
// Few rows: up to 16 a tile.  The four waves of a workgroup take keys 32 by 32 in
// turn, straight from the cache to registers: bound by those reads.  For the first
// product a lane reads 16 bytes of a key's row as the matrix operand wants them; for
// the second it reads the values m DP/16 .. of eight keys, m = lane % 16, so that the
// operand of output tile t is value t of each: an 8 x (DP / 16) transposition within
// the lane.  The lane of the result then holds DP / 4 consecutive values of its row.
// LDS would only pass on what one wave alone reads.  64 streams with 433,032 keys in all, F16, 32 heads over 4 of 128:
// 167 us, 5.3 TB/s (a copy on this card moves 4.6, reads alone more), and 10 of the join; F32 1 % longer.  One stream on
// 4097 keys, F32: 8 us, of which the reads are 2: launch, the chain from lengths over the table to the keys, sums over
// four waves; and 5 of the join (one launch for both ends each unit in a device-wide fence).  Heads between 64, 128 and
// 256 take the next one's products and time: 64 streams on up to 4096 keys 59 us at 80, 62 at 128, 131 at 136, 140 at 256.
// ---------------------------------------------------------------------------

constexpr int ROWS_M = 16;

struct RowsShared {
    float o[4][ROWS_M][128 + 4];
    float m[4][ROWS_M], l[4][ROWS_M];
};

template <typename T, int DP, bool PAD, bool TINY>
__global__ void __launch_bounds__(ATT_TPB, DP == 256 ? 1 : 2) k_attn_rows(AttnArgs p)
{
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int NC = DP / 32;              // operands of a key's row
    constexpr int NT = DP / 16;              // output tiles; values of a key that a lane reads for the second product
    __shared__ RowsShared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), r = lane & 15, h = lane >> 4;
    const int g = blockIdx.x % p.n_head_kv, id = blockIdx.x / p.n_head_kv, group = p.n_head / p.n_head_kv;
    Unit u;
    if (!find_unit<ATT_TPB, false>(p, ROWS_M, id, u)) return;
    const Tile tile = tile_of(p, ROWS_M, u);
    if (u.chunk >= tile.chunks) return;
    const int row0 = tile.row0, rows = tile.rows, j0 = tile.j0, j1 = tile.j1, chunks = tile.chunks;
    const int64_t base = tile.base;
    const int k0 = (int)min((int64_t)tile.start + (int64_t)u.chunk * u.run, (int64_t)tile.end),
              k1 = (int)min((int64_t)k0 + u.run, (int64_t)tile.end);

    const int32_t *table = p.table + (int64_t)u.seq * p.max_blocks;
    // Blocks of the keys of step kb: for the first product keys r and 16 + r, for the second 4 h .. 4 h + 3 and 16 + those
    // (one entry each where a block holds at least four rows).  They are looked up one step ahead of the rows.
    constexpr int NV = TINY ? 8 : 2;
    int kblock[2], vblock[NV];
    const auto look_up = [&](int kb) {
#pragma unroll
        for (int t = 0; t < 2; t++) kblock[t] = table[min(kb + 16 * t + r, k1 - 1) >> p.log_block];
#pragma unroll
        for (int e = 0; e < NV; e++)
            vblock[e] = table[min(TINY ? kb + 16 * (e / 4) + 4 * h + (e & 3) : kb + 16 * e + 4 * h, k1 - 1) >> p.log_block];
    };
    int kb = k0 + 32 * wave;
    if (kb < k1) look_up(kb);

    // this lane's row: its position, its first key, its q
    const bool live = r < rows;
    const int my_j = (row0 + (live ? r : 0)) / group, my_h = (row0 + (live ? r : 0)) % group;
    const int pos = live ? (int)(base + my_j) : -1;
    const int low = p.window ? pos - p.window + 1 : 0;        // (a window beyond int32 has no effect below 2^31 keys)
    const T *q = (const T *)((const uint8_t *)p.q + (uint64_t)(u.first + my_j) * p.q_stride) +
                 (int64_t)(g * group + my_h) * p.head_dim;
    f16x8 qh[NC], ql[NC];
    float c2 = p.scale;                       // |scale| log2 e, times the row's power of two
    load_q<T, PAD, NC, 32>(p, q, live, h, qh, ql, c2);

    const int all_from = (int)max(p.window ? base + j1 - p.window + 1 : 0, (int64_t)0);      // keys that every row sees:
    const int64_t all_to = base + j0;                                                        // from .. to
    // Rows of one token all see the same keys: what lies before its window (the first key is a multiple of 32) is no key.
    const int lone_from = j0 == j1 ? all_from : 0;
    float m = -INFINITY, l = 0.0f;
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = { 0, 0, 0, 0 };

    for (; kb < k1; kb += 32 * (ATT_TPB / 64)) {
        f16x8 kf[2][NC];
        i32x4 vf[8][(NT + 7) / 8];
        bool seen[8];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const _Float16 *row = p.k + ((unsigned)kblock[t] < (unsigned)p.n_blocks ? cache_row(p, kblock[t], kb + 16 * t + r, g) : 0);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                f16x8 v = { 0, 0, 0, 0, 0, 0, 0, 0 };
                if (!PAD || 32 * c + 8 * h < p.head_dim) v = *(const f16x8 *)(row + 32 * c + 8 * h);
                kf[t][c] = v;
            }
        }
        bool whole = true;                    // every key of the 32 is there
        const _Float16 *first_v = nullptr;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int key = kb + 16 * (e / 4) + 4 * h + (e & 3), block = vblock[TINY ? e : e / 4];
            seen[e] = key < k1 && (unsigned)block < (unsigned)p.n_blocks;
            whole &= seen[e];
            if (TINY || e % 4 == 0)           // (the other three lie behind the first)
                first_v = p.v + ((unsigned)block < (unsigned)p.n_blocks ? cache_row(p, block, key, g) : 0);
            const _Float16 *row = first_v + (TINY ? 0 : (e % 4) * (PAD ? p.head_dim : DP));
            if constexpr (NT == 4) {
                vf[e][0] = { 0, 0, 0, 0 };
                if (!PAD || NT * r < p.head_dim) {
                    const int2 w = *(const int2 *)(row + NT * r);
                    vf[e][0].x = w.x;
                    vf[e][0].y = w.y;
                }
            } else {
#pragma unroll
                for (int x = 0; x < NT / 8; x++) {
                    vf[e][x] = { 0, 0, 0, 0 };
                    if (!PAD || NT * r + 8 * x < p.head_dim) vf[e][x] = *(const i32x4 *)(row + NT * r + 8 * x);
                }
            }
        }
        look_up(kb + 32 * (ATT_TPB / 64));

        f32x4 s[2] = { { 0, 0, 0, 0 }, { 0, 0, 0, 0 } };
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                s[t] = mfma16(kf[t][c], qh[c], s[t]);
                if constexpr (SPLIT) s[t] = mfma16(kf[t][c], ql[c], s[t]);
            }

        const bool plain = __all(whole) && kb >= all_from && kb + 31 <= all_to;
        if (!plain) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = kb + 16 * (e / 4) + 4 * h + (e & 3);
                if (!(seen[e] && key <= pos && key >= low)) s[e / 4][e & 3] = -INFINITY;
                if (!seen[e] || key < lone_from) {
#pragma unroll
                    for (int x = 0; x < (NT + 7) / 8; x++) vf[e][x] = { 0, 0, 0, 0 };
                }
            }
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))) * c2;
        top = fmaxf(top, lane_xor<16>(top));
        top = fmaxf(top, lane_xor<32>(top));
        // (the first keys always pass, as m is then -inf)
        if (__any(top > m + ATT_LAG)) {
            const float m2 = fmaxf(m, top), keep = m2 == -INFINITY ? 1.0f : fast_exp2(m - m2);
            m = m2;
            l *= keep;
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] *= keep;
        }
        const float less = m == -INFINITY ? 0.0f : m - ATT_SHIFT;
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            w[e] = fast_exp2(__builtin_fmaf(s[e / 4][e & 3], c2, -less));
            l += w[e];
        }
        f16x8 ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            _Float16 a, b;
            split(w[e], a, b);
            ph[e] = a;
            if constexpr (SPLIT) pl[e] = b;
        }
        if (!plain && j1 > j0) {
            // Keys that some rows see and others do not: an infinity or NaN of theirs must not meet a weight 0.  It is
            // left out of the product and added to the rows that see it.
            uint32_t odd = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                bool bad = false;
#pragma unroll
                for (int x = 0; x < (NT + 7) / 8; x++)
#pragma unroll
                    for (int d = 0; d < (NT == 4 ? 2 : 4); d++) vf[e][x][d] = finite_pair(vf[e][x][d], bad);
                const uint64_t any = __ballot(bad);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (any >> (16 * i) & 0xffff) odd |= 1u << (16 * (e / 4) + 4 * i + (e & 3));
            }
            for (; odd != 0; odd &= odd - 1) {
                const int key = kb + __builtin_ctz(odd);
                const _Float16 *row = p.v + cache_row(p, table[key >> p.log_block], key, g) + h * (DP / 4);
                if (key > pos || key < low) continue;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int t = 0; t < NT; t += 4) {
                        if (PAD && h * (DP / 4) + i * NT + t >= p.head_dim) continue;
                        const f32x4 o = odd_values(row + i * NT + t);
#pragma unroll
                        for (int j = 0; j < 4; j++) acc[t + j][i] += o[j];
                    }
            }
        }
        // operand of output tile t: value t of the lane's eight keys
#pragma unroll
        for (int t = 0; t < NT; t++) {
            i32x4 a;
            const unsigned pick = t & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
            for (int e = 0; e < 4; e++)
                a[e] = __builtin_amdgcn_perm(vf[2 * e + 1][t / 8][t / 2 % 4], vf[2 * e][t / 8][t / 2 % 4], pick);
            acc[t] = mfma16(__builtin_bit_cast(f16x8, a), ph, acc[t]);
            if constexpr (SPLIT) acc[t] = mfma16(__builtin_bit_cast(f16x8, a), pl, acc[t]);
        }
    }

    // the waves' sums, brought to one maximum
    l += lane_xor<16>(l);
    l += lane_xor<32>(l);
    if (h == 0) {
        sh.m[wave][r] = m;
        sh.l[wave][r] = l;
    }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) top = fmaxf(top, sh.m[w][r]);
    const float part = m == -INFINITY ? 1.0f : fast_exp2(m - top);       // (of nothing, or of NaN)
    // a unit's partial result: [rows][DP] sums, then each row's maximum and sum of weights
    float *ws = p.partial + (int64_t)(g + (int64_t)id * p.n_head_kv) * (ROWS_M * (DP + 2));
    constexpr int COLS = DP < 128 ? DP : 128;
#pragma unroll
    for (int c0 = 0; c0 < DP; c0 += COLS) {
        if (c0) __syncthreads();
        if (DP <= 128 || h * (DP / 4) / 128 == c0 / 128) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int t = 0; t < NT; t++) sh.o[wave][r][(4 * h + i) * NT + t - c0] = acc[t][i] * part;
        }
        __syncthreads();
        for (int x = tid; x < rows * COLS; x += ATT_TPB) {
            const int n = x / COLS, d = x % COLS;
            float o = 0.0f, top_n = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                o += sh.o[w][n][d];
                top_n = fmaxf(top_n, sh.m[w][n]);
            }
#pragma unroll
            for (int w = 0; w < 4; w++) sum += sh.m[w][n] == -INFINITY ? sh.l[w][n] : sh.l[w][n] * fast_exp2(sh.m[w][n] - top_n);
            if (chunks == 1) {
                if (c0 + d < p.head_dim) {
                    const int j = (row0 + n) / group, a = (row0 + n) % group;
                    T *out = (T *)((uint8_t *)p.out + (uint64_t)(u.first + j) * p.out_stride) +
                             (int64_t)(g * group + a) * p.head_dim;
                    out[c0 + d] = (T)(sum == 0.0f ? 0.0f : o / sum);
                }
            } else {
                ws[n * DP + c0 + d] = o;
                if (c0 == 0 && d == 0) {
                    ws[ROWS_M * DP + n] = top_n;
                    ws[ROWS_M * DP + ROWS_M + n] = sum;
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Many rows: tiles of 32 a wave.  The workgroup stages KT keys at a time in LDS, twice; a wave multiplies them with its
// 32 rows on 32 x 32 x 16 matrix products.  Rows of both tiles lie DP values apart in chunks of 16 bytes whose index is
// xored with bits of the key, so that eight lanes that read one chunk of eight keys (k), and 32 that read 64 bytes of
// four keys (v), meet no bank twice.  V is transposed on its way from LDS (ds_read_b64_tr_b16: a lane gets one value of
// four keys).
//
// A step's K is of one tile, its V of the tile before: weights come from scores already there, and one barrier a step,
// between weights and the products, is enough.  Waves drift apart by most of a step, so that one's weights (vector units)
// and staging run beside the other's products on its SIMD.  Two chunks of 4096 and 2582 tokens on up to 12,288 cached,
// F16, 32 heads over 4 of 128: 1610 us, 862 TFLOP/s, where a large product reaches 1176 (F32 2820, twice the products; the
// first 30 launches on an idle card 1700, single ones more).  With a second barrier after the products 1734; with four
// waves half a step behind the others and two barriers, so that they always take turns, 1756.
// ---------------------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <typename T, int DP>
struct TileShape {
    static constexpr int WAVES = DP == 256 ? 4 : 8, M = 32 * WAVES, TPB = 64 * WAVES;
    static constexpr int KT = DP == 256 || (DP == 128 && sizeof(T) == 4) ? 32 : 64;     // keys staged at a time
};

// Where a chunk of a key's row lies: the rows' starts are 256 bytes (all banks) apart, 128 for DP 64.
template <int DP>
__device__ __forceinline__ int k_chunk(int key, int chunk) { return chunk ^ (DP == 64 ? key >> 1 & 7 : key & 15); }
template <int DP>
__device__ __forceinline__ int v_chunk(int key, int chunk)
{
    return chunk ^ (DP == 64 ? (key >> 1 & 1) << 2 | (key >> 2 & 1) << 1 : (key & 3) << 2 | (key >> 2 & 1) << 1);
}

// N operands from LDS, read(i), and their products, use(i, operand): four operands ahead, in an order that the compiler
// keeps (by itself it reads each right before its product and waits).
template <int N, typename R, typename F>
__device__ __forceinline__ void stream_operands(R read, F use)
{
    constexpr int AT = 4;
    static_assert(N % AT == 0, "whole groups");
    f16x8 a[2][AT];
#pragma unroll
    for (int i = 0; i < AT; i++) a[0][i] = read(i);
#pragma unroll
    for (int g = 0; g < N / AT; g++) {
        if (g + 1 < N / AT) {
#pragma unroll
            for (int i = 0; i < AT; i++) a[(g + 1) & 1][i] = read((g + 1) * AT + i);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < AT; i++) use(g * AT + i, a[g & 1][i]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// TINY: blocks of fewer keys than a wave reads at once (64 / CH).
template <typename T, int DP, bool PAD, bool TINY>
__global__ void __launch_bounds__((TileShape<T, DP>::TPB), DP == 256 ? 1 : 2) k_attn_tiles(AttnArgs p)
{
    using S = TileShape<T, DP>;
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int NC = DP / 16, NT = DP / 32, KT = S::KT, NS = KT / 32, CH = DP / 8;
    constexpr int NL = KT * CH / S::TPB;      // chunks of each tile a thread stages
    __shared__ __attribute__((aligned(1024))) _Float16 lk[2][KT * DP], lv[2][KT * DP];
    __shared__ uint8_t odd[2][64];            // of staged keys: values of v were left out that are not finite
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), r = lane & 31, h = lane >> 5;
    const int g = blockIdx.x % p.n_head_kv, id = blockIdx.x / p.n_head_kv, group = p.n_head / p.n_head_kv;
    Unit u;
    if (!find_unit<S::TPB, false>(p, S::M, id, u)) return;
    const Tile tile = tile_of(p, S::M, u);
    if (u.chunk >= tile.chunks) return;
    const int64_t base = tile.base;
    const int k0 = (int)min((int64_t)tile.start + (int64_t)u.chunk * u.run, (int64_t)tile.end),
              k1 = (int)min((int64_t)k0 + u.run, (int64_t)tile.end);
    const int steps = (k1 - k0 + KT - 1) / KT;
    const int32_t *table = p.table + (int64_t)u.seq * p.max_blocks;

    // Staging of pair n: v of step n and k of step n + 1, from the blocks of both.  A wave's lanes read chunks of 64 / CH
    // keys at a time, which lie in one block: its place is found in scalar registers, a lane adds its own offset (with
    // places by lane, staging took 2,300 cycles of a step's 5,300).
    // Every load is made, of a row of the cache in any case: a branch around one would wait for those before it.  What is
    // not there becomes 0 on its way into LDS.
    constexpr int KW = 64 / CH;
    int block[NL];                            // of the step after a pair's
    int64_t at_k[NL], at_v[NL];               // v of a step lies where k did
    bool has_k[NL], has_v[NL];
    i32x4 sk[NL], sv[NL];
    const bool lane_in = !PAD || 8 * (lane % CH) < p.head_dim;
    const int lane_key = lane / CH, lane_at = (TINY ? 0 : lane_key * p.head_dim) + (lane_in ? 8 * (lane % CH) : 0);
    const int64_t block_stride = (int64_t)p.n_head_kv * p.head_dim << p.log_block, head_at = (int64_t)g * p.head_dim << p.log_block;
    const _Float16 *head_k = p.k + head_at, *head_v = p.v + head_at;
    const auto first_key = [&](int n, int i) { return k0 + n * KT + i * (S::TPB / CH) + wave * KW; };
    const auto look_up = [&](int n) {
#pragma unroll
        for (int i = 0; i < NL; i++) block[i] = table[min(first_key(n, i) + (TINY ? lane_key : 0), k1 - 1) >> p.log_block];
    };
    const auto load = [&](int n, bool with_v) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            at_v[i] = at_k[i];
            has_v[i] = has_k[i];
            const int b = TINY ? block[i] : uniform(block[i]), key = first_key(n + 1, i) + (TINY ? lane_key : 0);
            const bool ok = (unsigned)b < (unsigned)p.n_blocks;
            at_k[i] = (ok ? b : 0) * block_stride + (key & ((1 << p.log_block) - 1)) * p.head_dim;
            has_k[i] = ok && first_key(n + 1, i) + lane_key < k1 && lane_in;
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            if (with_v) sv[i] = *(const i32x4 *)(head_v + at_v[i] + lane_at);
            sk[i] = *(const i32x4 *)(head_k + at_k[i] + lane_at);
        }
        look_up(n + 2);
    };
    // Steps from which on some rows see keys that others do not: there an infinity or NaN of v must not meet a weight 0
    // and is left out.
    const auto floor_step = [&](int64_t key) { return (int)min(max((key - k0) >> (KT == 64 ? 6 : 5), (int64_t)-2), (int64_t)0x7ffffff0); };
    const int edge = p.window ? 0 : max(floor_step(base + tile.j0 - KT + 1) + 1, 0);
    const auto store = [&](int n, bool with_v) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int x = tid + i * S::TPB, key = x / CH, c = x % CH;
            if (!__all(has_k[i] && (has_v[i] || !with_v))) {
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    if (!has_k[i]) sk[i][d] = 0;
                    if (!has_v[i]) sv[i][d] = 0;
                }
            }
            *(i32x4 *)&lk[(n + 1) & 1][key * DP + 8 * k_chunk<DP>(key, c)] = sk[i];
            if (!with_v) continue;
            if (n >= edge) {
                bool bad = false;
#pragma unroll
                for (int d = 0; d < 4; d++) sv[i][d] = finite_pair(sv[i][d], bad);
                const uint64_t any = __ballot(bad);           // (the CH lanes of a key lie in one wave)
                if (c == 0) odd[n & 1][key] = (any >> (lane & ~(CH - 1)) & ((1ull << CH) - 1)) != 0;
            }
            *(i32x4 *)&lv[n & 1][key * DP + 8 * v_chunk<DP>(key, c)] = sv[i];
        }
    };
    // whether the keys of a step are there, a lane each (of 64 or 32), looked up a step ahead
    int key_block = 0;
    const auto look_up_key = [&](int n) { key_block = table[min(k0 + n * KT + (lane & (KT - 1)), k1 - 1) >> p.log_block]; };

    if (steps > 0) {
        look_up(0);
        look_up_key(0);
        load(-1, false);
    }

    // this lane's row
    const int row = wave * 32 + r;
    const bool live = row < tile.rows;
    const int my_row = tile.row0 + (live ? row : 0), my_j = my_row / group, my_h = my_row % group;
    const int pos = live ? (int)(base + my_j) : -1;
    const int low = p.window ? pos - p.window + 1 : 0;
    const T *q = (const T *)((const uint8_t *)p.q + (uint64_t)(u.first + my_j) * p.q_stride) +
                 (int64_t)(g * group + my_h) * p.head_dim;
    f16x8 qh[NC], ql[SPLIT ? NC : 1];
    float c2 = p.scale;
    load_q<T, PAD, NC, 16>(p, q, live, h, qh, ql, c2);
    // the wave's rows: positions from w_first to w_last; keys that all of them see end at w_first
    const int w_rows = min(tile.rows - wave * 32, 32);
    const int64_t w_first = base + (tile.row0 + wave * 32) / group, w_last = base + (tile.row0 + wave * 32 + max(w_rows, 1) - 1) / group;
    const int64_t w_from = p.window ? w_last - p.window + 1 : 0, w_low = p.window ? w_first - p.window + 1 : 0;

    float m = -INFINITY, l = 0.0f;
    f32x16 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[t][i] = 0.0f;

    const int k_row = r * DP, s16 = lane & 15;
    const int v_row = (4 * h + (s16 >> 2)) * DP, v_in = 2 * (lane >> 4 & 1) + (s16 & 3) / 2, v_half = 4 * (s16 & 1);

    // the steps that any of them sees, and those of which all see all
    const int work_from = floor_step(w_low), work_to = w_rows > 0 ? floor_step(w_last) : -1;
    const int all_from = floor_step(w_from + KT - 1), all_to = floor_step(w_first - KT + 1);
    const auto at_work = [&](int n) { return n >= work_from && n <= work_to; };
    f32x16 s[NS];
    f16x8 ph[2 * NS], pl[SPLIT ? 2 * NS : 1];
    const auto scores = [&](int n) {          // S^T of step n
        if (!at_work(n)) return;
        const int buf = n & 1;
#pragma unroll
        for (int t = 0; t < NS; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[t][i] = 0.0f;
        stream_operands<NC * NS>(
            [&](int i) { return *(const f16x8 *)&lk[buf][32 * (i % NS) * DP + k_row + 8 * k_chunk<DP>(r, 2 * (i / NS) + h)]; },
            [&](int i, f16x8 a) {
                s[i % NS] = mfma32(a, qh[i / NS], s[i % NS]);
                if constexpr (SPLIT) s[i % NS] = mfma32(a, ql[i / NS], s[i % NS]);
            });
    };
    const auto weights = [&](int n) {         // of step n, from its scores
        if (!at_work(n)) return;
        const int kb = k0 + n * KT;
        const uint64_t seen = __ballot((unsigned)key_block < (unsigned)p.n_blocks && kb + (lane & (KT - 1)) < k1);
        if (~seen != 0 || n < all_from || n > all_to) {
            const uint64_t mine = seen >> (4 * h);
#pragma unroll
            for (int t = 0; t < NS; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int k = 32 * t + 8 * (i / 4) + (i & 3);
                    if (!((mine >> k & 1) && kb + k + 4 * h <= pos && kb + k + 4 * h >= low)) s[t][i] = -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < NS; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, s[t][i]);
        top *= c2;
        top = fmaxf(top, lane_xor<32>(top));
        if (__any(top > m + ATT_LAG)) {
            const float m2 = fmaxf(m, top), keep = m2 == -INFINITY ? 1.0f : fast_exp2(m - m2);
            m = m2;
            l *= keep;
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] *= keep;
        }
        const float less = m == -INFINITY ? 0.0f : m - ATT_SHIFT;
#pragma unroll
        for (int t = 0; t < NS; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float w = fast_exp2(__builtin_fmaf(s[t][i], c2, -less));
                l += w;
                _Float16 a, b;
                split(w, a, b);
                ph[2 * t + i / 8][i % 8] = a;
                if constexpr (SPLIT) pl[2 * t + i / 8][i % 8] = b;
            }
    };
    const auto values = [&](int n) {          // O^T += V^T P^T of step n
        if (!at_work(n)) return;
        const int kb = k0 + n * KT, buf = n & 1;
        uint64_t left_out = n >= edge ? __ballot(lane < KT ? odd[buf][lane] : 0) : 0;
        for (; left_out != 0; left_out &= left_out - 1) {
            const int key = kb + __builtin_ctzll(left_out);
            const _Float16 *v = p.v + cache_row(p, table[key >> p.log_block], key, g) + 4 * h;
            if (key > pos || key < low) continue;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    if (PAD && 32 * t + 8 * b + 4 * h >= p.head_dim) continue;
                    const f32x4 o = odd_values(v + 32 * t + 8 * b);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[t][4 * b + j] += o[j];
                }
        }
        stream_operands<2 * NS * NT>(
            [&](int i) {
                // of 16 keys a value of each of 4 h .. + 3 and 8 + 4 h .. + 3
                const int k16 = i / NT, t = i % NT,
                          at = 16 * k16 * DP + v_row + 8 * ((4 * t + v_in) ^ v_chunk<DP>(4 * h + (s16 >> 2), 0)) + v_half;
                union {
                    s16x4 part[2];
                    f16x8 whole;
                } a;
                a.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)&lv[buf][at]);
                a.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)&lv[buf][at + 8 * DP]);
                return a.whole;
            },
            [&](int i, f16x8 a) {
                acc[i % NT] = mfma32(a, ph[i / NT], acc[i % NT]);
                if constexpr (SPLIT) acc[i % NT] = mfma32(a, pl[i / NT], acc[i % NT]);
            });
    };

    // A step's one barrier: before it all have stored pair n (v of n, k of n + 1), after it they read it.  The places of
    // pair n + 1 were last read before it.
    if (steps > 0) {
        store(-1, false);
        load(0, true);
        __syncthreads();
        scores(0);
        for (int n = 0; n < steps; n++) {
            store(n, true);                  // (keys past the last are zeros)
            load(n + 1, true);
            weights(n);
            look_up_key(n + 1);
            __syncthreads();
            values(n);
            if (n + 1 < steps) scores(n + 1);
        }
    }

    l += lane_xor<32>(l);
    if (!live) return;
    if (tile.chunks == 1) {
        const float by = l == 0.0f ? 0.0f : 1.0f / l;
        T *out = (T *)((uint8_t *)p.out + (uint64_t)(u.first + my_j) * p.out_stride) + (int64_t)(g * group + my_h) * p.head_dim;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int d = 32 * t + 8 * b + 4 * h;
                if (PAD && d >= p.head_dim) continue;
                typedef T vec4 __attribute__((ext_vector_type(4)));
                vec4 v;
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = (T)(acc[t][4 * b + j] * by);
                *(vec4 *)(out + d) = v;
            }
    } else {
        float *ws = p.partial + (int64_t)(g + (int64_t)id * p.n_head_kv) * (S::M * (DP + 2));
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const f32x4 v = { acc[t][4 * b], acc[t][4 * b + 1], acc[t][4 * b + 2], acc[t][4 * b + 3] };
                *(f32x4 *)(ws + row * DP + 32 * t + 8 * b + 4 * h) = v;
            }
        if (h == 0) {
            ws[S::M * DP + row] = m;
            ws[S::M * DP + S::M + row] = l;
        }
    }
}

// ---------------------------------------------------------------------------
// Tiles of several runs: a workgroup joins the partial results of some rows, [M][DP] sums and then every row's maximum
// and sum of weights, unit after unit of a kv head.  A launch of its own: a device-wide release and acquire in each unit
// of the split kernel, for the last of a tile to join it, writes back and invalidates its XCD's whole L2 and made 1,800
// units of 64 streams wait for each other (614 us in place of 186).
//
// Small tiles have up to 512 runs, which lanes share out: four rows a workgroup, their factors by a wave each, then
// 16-byte pieces of rows, ATT_TPB in all.  Large ones have few: a thread takes a piece of four rows and all their runs,
// which needs neither LDS nor a barrier (16 tiles of 256 rows in four runs, 4 kv heads: 9 us, with factors in LDS 16; 34
// MB, 3.6 TB/s).
// ---------------------------------------------------------------------------

constexpr int rows_joined(int M) { return M == ROWS_M ? 4 : 32; }       // rows a workgroup

template <typename T, int DP, int M>
__device__ __forceinline__ void join_rows(const AttnArgs &p, int block)
{
    constexpr int ROWS = rows_joined(M), parts = M / ROWS;
    const int tid = threadIdx.x, group = p.n_head / p.n_head_kv;
    const int n0 = block % parts * ROWS, g = block / parts % p.n_head_kv, id = block / parts / p.n_head_kv;
    Unit u;
    if (!find_unit<ATT_TPB, true>(p, M, id, u)) return;
    const Tile tile = tile_of(p, M, u);
    const int chunks = tile.chunks;
    if (chunks == 1 || n0 >= tile.rows) return;
    const int64_t step = (int64_t)p.n_head_kv * (M * (DP + 2));
    const float *from = p.partial + (int64_t)(g + (int64_t)u.whole * p.n_head_kv) * (M * (DP + 2));
    constexpr int ITEMS = ROWS * (DP / 4) < ATT_TPB ? ROWS * (DP / 4) : ATT_TPB, PARTS = ATT_TPB / ITEMS, AT = ITEMS / (DP / 4);
    const int item = tid % ITEMS, part = tid / ITEMS, d = item % (DP / 4) * 4;
    const auto put = [&](int n, f32x4 o) {
        if (n >= tile.rows || d >= p.head_dim) return;
        const int j = (tile.row0 + n) / group, a = (tile.row0 + n) % group;
        T *out = (T *)((uint8_t *)p.out + (uint64_t)(u.first + j) * p.out_stride) + (int64_t)(g * group + a) * p.head_dim + d;
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] = (T)o[i];
    };
    if constexpr (M == ROWS_M) {
        __shared__ float factor[ROWS][512];
        __shared__ f32x4 sums[ATT_TPB];
        {
            // each run's factor: 2^(its maximum - the largest) / sum of weights; a wave a row
            const int lane = tid & 63, n = tid >> 6;
            const float *f = from + M * DP + n0 + n;
            float top = -INFINITY, sum = 0.0f;
            for (int c = lane; c < chunks; c += 64) top = fmaxf(top, f[c * step]);
            top = lanes_join<32>(top, [](float x, float y) { return fmaxf(x, y); });
            for (int c = lane; c < chunks; c += 64) {
                const float m = f[c * step], x = m == -INFINITY ? 1.0f : fast_exp2(m - top);
                factor[n][c] = x;
                sum += x * f[c * step + M];
            }
            sum = lanes_join<32>(sum, [](float x, float y) { return x + y; });
            const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
            for (int c = lane; c < chunks; c += 64) factor[n][c] *= by;
        }
        __syncthreads();
        const int n = item / (DP / 4);
        const float *f = from + (int64_t)(n0 + n) * DP + d;
        f32x4 o = { 0, 0, 0, 0 };
#pragma unroll 8
        for (int c = part; c < chunks; c += PARTS) o += factor[n][c] * *(const f32x4 *)(f + c * step);
        if constexpr (PARTS > 1) {
            sums[tid] = o;
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int i = 1; i < PARTS; i++) o += sums[i * ITEMS + item];
            }
        }
        if (part == 0) put(n0 + n, o);
    } else {
        constexpr int EACH = ROWS / AT;
        const float *w = from + M * DP + n0 + item / (DP / 4), *f = from + (int64_t)(n0 + item / (DP / 4)) * DP + d;
        float top[EACH], sum[EACH];
        f32x4 o[EACH];
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            top[i] = -INFINITY;
            sum[i] = 0.0f;
            o[i] = f32x4{ 0, 0, 0, 0 };
        }
        for (int c = 0; c < chunks; c++) {
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const float m = w[c * step + i * AT], l = w[c * step + M + i * AT], high = fmaxf(top[i], m);
                const f32x4 v = *(const f32x4 *)(f + c * step + i * AT * DP);
                const float x = m == -INFINITY ? 1.0f : fast_exp2(m - high);
                const float y = top[i] == -INFINITY ? 1.0f : fast_exp2(top[i] - high);
                top[i] = high;
                sum[i] = sum[i] * y + x * l;
                o[i] = o[i] * y + x * v;
            }
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) put(n0 + item / (DP / 4) + i * AT, o[i] * (sum[i] == 0.0f ? 0.0f : 1.0f / sum[i]));
    }
}

template <typename T, int DP, int M>
__global__ void __launch_bounds__(ATT_TPB) k_attn_join(AttnArgs p) { join_rows<T, DP, M>(p, blockIdx.x); }

// Both kinds of tiles, the large ones' workgroups first.
template <typename T, int DP, int M>
__global__ void __launch_bounds__(ATT_TPB) k_attn_join_both(AttnArgs many, AttnArgs few, int n_many)
{
    if ((int)blockIdx.x < n_many) join_rows<T, DP, M>(many, blockIdx.x);
    else join_rows<T, DP, ROWS_M>(few, blockIdx.x - n_many);
}

static int padded_dim(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Rows of a tile of many rows.
static int tile_rows(const AttnArgs &p)
{
    static_assert(TileShape<float, 64>::M == TileShape<float, 128>::M, "one size up to heads of 128");
    return padded_dim(p.head_dim) == 256 ? TileShape<float, 256>::M : TileShape<float, 128>::M;
}

// Units a kv head that the work is split into where there are fewer tiles: several a compute unit of few rows, one of
// many.
static int target_units(const AttnArgs &p, bool many) { return std::max(1, (many ? 256 : 2048) / p.n_head_kv); }

// Tiles of at most M rows that n_seq requests with n_tokens tokens in all can have.
static int64_t most_tiles(const AttnArgs &p, int M)
{
    return (int64_t)p.n_tokens * (p.n_head / p.n_head_kv) / M + std::min(p.n_seq, p.n_tokens);
}

// Values of the partial results of split tiles, whose units are at most `target` in all.
static size_t partial_values(const AttnArgs &p, bool many)
{
    const int rows = many ? tile_rows(p) : ROWS_M;
    return (size_t)target_units(p, many) * rows * p.n_head_kv * (padded_dim(p.head_dim) + 2);
}

size_t attention_workspace(const AttnArgs &p) { return (partial_values(p, false) + partial_values(p, true)) * sizeof(float); }

// The split of the requests of min_rows .. max_rows rows into tiles of at most 16 (many: TileShape::M): `p` is set up for
// it; workgroups of the products and of the join (0: no tile is split).
static bool attention_split(AttnArgs &p, bool many, int min_rows, int max_rows, int &wgs, int &join_wgs)
{
    const int M = many ? tile_rows(p) : ROWS_M;
    p.min_rows = min_rows;
    p.max_rows = max_rows;
    p.target = target_units(p, many);
    if (!many) p.partial += partial_values(p, true);
    // (at most 512 runs a tile, whatever the lengths)
    p.least = many ? 256 : 128;
    const int64_t longest = (int64_t)p.max_blocks << p.log_block;
    while (longest / p.least >= 512) p.least *= 2;
    // Tiles at most; units: `target` or as many as there are tiles, and no more than the runs that the longest request
    // could have.
    int64_t tiles = most_tiles(p, M);
    if (max_rows < 0x7fffffff) tiles = std::min<int64_t>(tiles, (int64_t)p.n_seq * ((max_rows + M - 1) / M));
    const int64_t runs = (longest + p.least - 1) / p.least,
                  units = std::min(std::max<int64_t>(tiles, p.target), tiles * runs) * p.n_head_kv;
    if (units > 0x7fffff) return false;
    wgs = (int)units;                         // (only fewer than `target` tiles are split)
    join_wgs = longest > p.least ? (int)(std::min<int64_t>(tiles, p.target) * p.n_head_kv * (M / rows_joined(M))) : 0;
    return true;
}

// A call's tiles of many rows and of few, each with a set of arguments, workgroups of its own (0: none are launched).  A
// step of single tokens (no more tokens than requests) needs only the second, a single request only one of them.
struct AttnLaunch {
    AttnArgs many, few;
    int many_wgs, few_wgs, many_join, few_join;
};

static bool attention_launch(const AttnArgs &p, AttnLaunch &l)
{
    const int64_t rows = (int64_t)p.n_tokens * (p.n_head / p.n_head_kv);
    const bool only_few = p.n_tokens <= p.n_seq || rows <= ATT_FEW_ROWS, only_many = !only_few && p.n_seq == 1;
    l = { p, p, 0, 0, 0, 0 };
    return (only_few || attention_split(l.many, true, only_many ? 0 : ATT_FEW_ROWS + 1, 0x7fffffff, l.many_wgs, l.many_join)) &&
           (only_many || attention_split(l.few, false, 0, only_few ? 0x7fffffff : ATT_FEW_ROWS, l.few_wgs, l.few_join));
}

bool attention_fits(const AttnArgs &p)
{
    AttnLaunch l;
    return attention_launch(p, l);
}

bool attention_units(const AttnArgs &p, AttnUnits out[2])
{
    AttnLaunch l;
    if (!attention_launch(p, l)) return false;
    for (int k = 0; k < 2; k++) {
        const AttnArgs &a = k == 0 ? l.many : l.few;
        const int M = k == 0 ? tile_rows(p) : ROWS_M, wgs = k == 0 ? l.many_wgs : l.few_wgs,
                  join = k == 0 ? l.many_join : l.few_join;
        AttnUnits &o = out[k];
        o = {};
        if (wgs == 0) continue;
        const auto sum = [&](auto f) {
            int64_t n = 0;
            for (int i = 0; i < p.n_seq; i++) {
                int tiles, span;
                Unit u;
                request_work(a, M, i, tiles, span, u);
                n += tiles * (int64_t)f(span);
            }
            return n;
        };
        const int64_t work = sum([](int span) { return span; });
        o.tiles = sum([](int) { return 1; });
        int run = unit_run(a, M, work, o.tiles);
        const int tight = tight_run(a, M, work);
        if (p.n_seq <= 64 && tight < run && sum([&](int span) { return runs_of(span, tight); }) <= a.target) run = tight;
        o.run = run;
        o.units = sum([&](int span) { return runs_of(span, run); });
        o.grid = wgs / p.n_head_kv;
        o.joined = join / (p.n_head_kv * (M / rows_joined(M)));
        o.partial = (int64_t)(partial_values(p, k == 0) / ((size_t)M * p.n_head_kv * (padded_dim(p.head_dim) + 2)));
    }
    return true;
}

template <typename T, int DP>
static void attention_tiles(const AttnArgs &p, int wgs, hipStream_t s)
{
    constexpr int TPB = TileShape<T, DP>::TPB;
    if (1 << p.log_block < 512 / DP) hipLaunchKernelGGL((k_attn_tiles<T, DP, true, true>), dim3(wgs), TPB, 0, s, p);
    else if (p.head_dim != DP) hipLaunchKernelGGL((k_attn_tiles<T, DP, true, false>), dim3(wgs), TPB, 0, s, p);
    else hipLaunchKernelGGL((k_attn_tiles<T, DP, false, false>), dim3(wgs), TPB, 0, s, p);
}

template <typename T, int DP>
static void attention_few(const AttnArgs &p, int wgs, hipStream_t s)
{
    if (p.log_block < 2) hipLaunchKernelGGL((k_attn_rows<T, DP, true, true>), dim3(wgs), ATT_TPB, 0, s, p);
    else if (p.head_dim != DP) hipLaunchKernelGGL((k_attn_rows<T, DP, true, false>), dim3(wgs), ATT_TPB, 0, s, p);
    else hipLaunchKernelGGL((k_attn_rows<T, DP, false, false>), dim3(wgs), ATT_TPB, 0, s, p);
}

// Few rows and many rows are a launch each, the choice a request's own, and one joins both.
template <typename T, int DP>
static hipError_t attention_dim(const AttnArgs &p, hipStream_t s)
{
    constexpr int M = TileShape<T, DP>::M;
    AttnLaunch l;
    if (!attention_launch(p, l)) return hipErrorInvalidValue;
    if (l.many_wgs > 0) attention_tiles<T, DP>(l.many, l.many_wgs, s);
    if (l.few_wgs > 0) attention_few<T, DP>(l.few, l.few_wgs, s);
    if (l.many_join > 0 && l.few_join > 0)
        hipLaunchKernelGGL((k_attn_join_both<T, DP, M>), dim3(l.many_join + l.few_join), ATT_TPB, 0, s, l.many, l.few,
                           l.many_join);
    else if (l.many_join > 0) hipLaunchKernelGGL((k_attn_join<T, DP, M>), dim3(l.many_join), ATT_TPB, 0, s, l.many);
    else if (l.few_join > 0) hipLaunchKernelGGL((k_attn_join<T, DP, ROWS_M>), dim3(l.few_join), ATT_TPB, 0, s, l.few);
    return hipGetLastError();
}

template <typename T>
static hipError_t attention_type(const AttnArgs &p, hipStream_t s)
{
    if (p.head_dim <= 64) return attention_dim<T, 64>(p, s);
    if (p.head_dim <= 128) return attention_dim<T, 128>(p, s);
    return attention_dim<T, 256>(p, s);
}

hipError_t launch_attention(AttnArgs p, int type, hipStream_t s)
{
    // S = q . k takes |scale|; its sign goes to q, and scale 0 makes q 0
    p.q_sign = p.scale > 0.0f ? 1.0f : p.scale < 0.0f ? -1.0f : 0.0f;
    p.scale = p.scale == 0.0f ? 1.0f : std::fabs(p.scale) * 1.44269504088896340736f;
    return type == T_F32 ? attention_type<float>(p, s) : attention_type<_Float16>(p, s);
}

}  // namespace ds3k
