// mx_matmul.hip -- products of MXINT8 rows with MXFP4 weights (mx.h): dense,
// grouped by expert, and the grouped gate/up pair with SwiGLU and rounding.
//
//   C[m][n] = sum over blocks b of 32:  2^(ex + ew - 254) sum_i q_i / 64 * f_i
//
// Every product is exact and the sums are held in fp32 (mx.h), so the result
// differs from a 64-bit sum by fp32 rounding alone.
#include "mx.h"

#include <algorithm>

namespace ds3k {

// A step's number as a type: the scale byte a product takes is an immediate.
template <int I> struct Int {
    static constexpr int value = I;
};

// ---------------------------------------------------------------------------
// Row tiles of the groups.  Group g owns the rows offsets[g] .. offsets[g + 1]
// - 1; tiles of BM rows are numbered through the groups in order.  The offsets
// are device data: each is taken into 0 .. n_rows, a group that ends before it
// begins is empty.
// ---------------------------------------------------------------------------
struct RowTile {
    int group, row, rows;       // rows = 0: no such tile
};

// Inclusive prefix sum over the wavefront (DPP row shifts, then rows 1 and 3
// add lane 15 of the row below, rows 2 and 3 lane 31).
__device__ __forceinline__ int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// Four groups a lane, so that 256 groups take one round of loads: their bounds,
// tiles, and the sum and its prefix over the wave.
template <int BM> struct GroupTiles {
    int at[5], tiles[4], sum, incl;

    __device__ __forceinline__ void load(const int32_t *offsets, int n_group, int n_rows, int g0)
    {
        const int lane = threadIdx.x & (WAVE - 1);
        sum = 0;
#pragma unroll
        for (int i = 0; i < 5; i++) at[i] = min(max(offsets[min(g0 + 4 * lane + i, n_group)], 0), n_rows);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            tiles[i] = (int)(((uint32_t)max(at[i + 1] - at[i], 0) + BM - 1) / BM);
            sum += tiles[i];
        }
        incl = wave_scan(sum);
    }
    __device__ __forceinline__ uint32_t total() const { return (uint32_t)__builtin_amdgcn_readlane(incl, WAVE - 1); }
    // Tile `left` of these (left < total()).
    __device__ __forceinline__ RowTile find(uint32_t left, int g0) const
    {
        const int src = __builtin_ctzll(__ballot((uint32_t)incl > left));
        left -= (uint32_t)(__builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane(sum, src));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t n = (uint32_t)__builtin_amdgcn_readlane(tiles[i], src);
            if (left < n || i == 3) {
                // (offsets that decrease can make more tiles than 32 bits count)
                const int from = __builtin_amdgcn_readlane(at[i], src), row = (int)((uint32_t)from + left * BM);
                const int rows = min(BM, __builtin_amdgcn_readlane(at[i + 1], src) - row);
                return { g0 + 4 * src + i, row, row < from ? 0 : max(rows, 0) };
            }
            left -= n;
        }
        return { 0, 0, 0 };
    }
};

// Row tile `item`; uniform over the wave.
template <int BM>
__device__ __forceinline__ RowTile row_tile(const int32_t *offsets, int n_group, int n_rows, uint32_t item)
{
    if (offsets == nullptr) {
        const int64_t row = (int64_t)item * BM;
        return { 0, (int)row, row < n_rows ? (int)min((int64_t)BM, n_rows - row) : 0 };
    }
    for (int g0 = 0; g0 < n_group; g0 += 4 * WAVE) {
        GroupTiles<BM> t;
        t.load(offsets, n_group, n_rows, g0);
        if (item < t.total()) return t.find(item, g0);
        item -= t.total();
    }
    return { 0, 0, 0 };
}

// How many there are.
template <int BM>
__device__ __forceinline__ uint32_t row_tiles(const int32_t *offsets, int n_group, int n_rows)
{
    if (offsets == nullptr) return (uint32_t)(((int64_t)n_rows + BM - 1) / BM);
    uint32_t n = 0;
    for (int g0 = 0; g0 < n_group; g0 += 4 * WAVE) {
        GroupTiles<BM> t;
        t.load(offsets, n_group, n_rows, g0);
        n += t.total();
    }
    return n;
}

// Work is numbered by row tile, then by tile of output columns.  (All in 32
// bits: a 64-bit division takes a wave over 0.4 us.)
struct Job {
    uint32_t item, tile;
};

__device__ __forceinline__ Job job_of(uint32_t job, uint32_t n_tiles)
{
    const uint32_t item = job / n_tiles;
    return { item, job - item * n_tiles };
}

// ---------------------------------------------------------------------------
// Few rows: a workgroup takes 16 rows of x and NT blocks of 16 weight rows (GU:
// half of them gate rows, half the same up rows); its waves take the chunks of
// 512 columns in turn, straight from memory, and their sums meet in LDS.  Two to
// three waves a SIMD hide each other's loads.  Bound by memory where the weights
// are many (1 x 2048 . 151936 34.1 us, 4.9 TB/s), else by the chain of offsets,
// ids, rows and weights (in a graph 27 x 2048 . 768 4.6 us, 1 x 2048 . 2048 3.4,
// gate/up of one token in 8 of 128 experts, with the values of h, 8.3).
// ---------------------------------------------------------------------------
template <int WAVES, int NT, bool GU>
__global__ void __launch_bounds__(WAVES * WAVE, NT == 4 ? 2 : 3) k_mx_few(MxProduct p, uint32_t n_jobs, uint32_t n_tiles)
{
    static_assert(!GU || NT == 4, "the gate/up tile is two blocks of each matrix");
    constexpr int BM = 16, NW = GU ? 32 : 16 * NT;       // output columns a workgroup
    __shared__ f32x4 red[WAVES][NT][WAVE];
    const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
    const int r = lane & 15, g = lane >> 4;              // a lane's place in the products
    const int lb = 4 * g + (lane & 3);                   // and its block in loads
    const int nb = p.K / 32, n_chunk = (nb + CHUNK_BLOCKS - 1) / CHUNK_BLOCKS;

    for (uint32_t at = blockIdx.x; at < n_jobs; at += gridDim.x) {
        const Job job = job_of(at, n_tiles);
        const int64_t n0 = (int64_t)job.tile * NW;
        const RowTile tile = row_tile<BM>(p.offsets, p.n_group, p.n_rows, job.item);
        if (tile.rows == 0) continue;                    // uniform over the workgroup
        // row i of the tile in x, or -1
        const auto x_row = [&](int i) {
            const int64_t at = tile.row + min(i, tile.rows - 1);
            const int64_t id = p.ids ? (int64_t)p.ids[at] : at;
            return id >= 0 && id < p.n_x ? id : (int64_t)-1;
        };
        const bool ok = r < tile.rows && x_row(r) >= 0;  // this lane's outputs exist
        // The weight rows of block t: n_of(t) .. + 15, moved down where they would pass the
        // end (those below n0 + 16 t are then not stored).
        const auto n_of = [&](int t) {
            return max((int64_t)0, min(n0 + 16 * (GU ? t & 1 : t), (int64_t)p.N - 16));
        };
        uint32_t c_row[4];
#pragma unroll
        for (int j = 0; j < 4; j++) c_row[j] = (uint32_t)min((r & 12) + j, p.N - 1) * (p.K / 2);
        const uint32_t s_row = (uint32_t)min(lane >> 2, p.N - 1) * nb + 4 * (lane & 3);
        const uint8_t *wc[NT], *ws[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const bool up = GU && t >= 2;
            const int64_t n = (int64_t)tile.group * p.N + n_of(t);
            wc[t] = (up ? p.uc : p.wc) + n * (p.K / 2);
            ws[t] = (up ? p.us : p.ws) + n * nb;
        }
        f32x4 acc[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = f32x4{ 0.f, 0.f, 0.f, 0.f };
        // Up to 4 PER rows: a lane splits PER blocks, lanes 16 g + 4 / PER R .. the four blocks
        // 4 g + 0..3 of row R, and step k takes them from there through the LDS crossbar.  More
        // rows (PER = 4): a lane splits the four blocks that it multiplies (for one row of
        // 151936 outputs 38.4 us, not 34.1: the vector units were busy two thirds of it; for
        // eight rows, K = 4096, 4096 outputs 6.7, not 5.5).
        const auto chunks = [&](auto per) {
            constexpr int PER = decltype(per)::value, LANES = 4 / PER;
            const uint8_t *xc[4], *xs;                   // of one row, PER = 4: as the loads take them
            if constexpr (PER < 4) {
                const int64_t row = max(x_row(r / LANES), (int64_t)0);
                xc[0] = p.xc + row * p.K;
                xs = p.xs + row * nb;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) xc[j] = p.xc + max(x_row((r & 12) + j), (int64_t)0) * p.K;
                xs = p.xs + max(x_row(lane >> 2), (int64_t)0) * nb + 4 * (lane & 3);
            }
            for (int c = wave; c < n_chunk; c += WAVES) {
                // Blocks behind the last are read as the last (their x becomes zero); scales up to
                // 15 bytes on, which every allocation has.
                const int b0 = c * CHUNK_BLOCKS, b = min(b0 + lb, nb - 1);
                i32x4 x0[4], x1[4], w[NT][4];
                uint32_t sx, sw[NT];
                const int own = b0 + 4 * g + PER * (r % LANES);
                RawBlock raw[PER];
                if constexpr (PER < 4) {
#pragma unroll
                    for (int i = 0; i < PER; i++) raw[i] = raw_block(xc[0], xs, min(own + i, nb - 1));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        x0[j] = *(const i32x4 *)(xc[j] + (int64_t)b * 32);
                        x1[j] = *(const i32x4 *)(xc[j] + (int64_t)b * 32 + 16);
                    }
                    sx = *(const u32_any *)(xs + b0);
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) w[t][j] = *(const i32x4 *)(wc[t] + c_row[j] + (uint32_t)b * 16);
                    sw[t] = *(const u32_any *)(ws[t] + s_row + b0);
                }
                XFrag mine[PER];
                if constexpr (PER < 4) {
#pragma unroll
                    for (int i = 0; i < PER; i++) mine[i] = x_frag(raw[i], own + i < nb);
                } else {
                    quad_transpose(x0);
                    quad_transpose(x1);
                    sx = scales_to_place(sx);
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    quad_transpose(w[t]);
                    sw[t] = scales_within(scales_to_place(sw[t]), b0 + 4 * g, nb);
                }
                const auto step = [&](auto kc) {
                    constexpr int k = decltype(kc)::value;
                    XFrag f;
                    if constexpr (PER < 4) {
                        f = frag_from(mine[k % PER], 16 * g + ((LANES * r + k / PER) & 15));
                    } else {
                        RawBlock q;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            q.w[i] = (uint32_t)x0[k][i];
                            q.w[4 + i] = (uint32_t)x1[k][i];
                        }
                        q.sc = byte_of(sx, k);
                        f = x_frag(q, b0 + 4 * g + k < nb);
                    }
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[t] = mx_mfma_hi<k>(w[t][k], sw[t], f, acc[t]);
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[t] = mx_mfma_lo<k>(w[t][k], sw[t], f, acc[t]);
                };
                step(Int<0>{});
                step(Int<1>{});
                step(Int<2>{});
                step(Int<3>{});
            }
        };
        if (tile.rows <= 4) chunks(Int<1>{});
        else if (tile.rows <= 8) chunks(Int<2>{});
        else chunks(Int<4>{});
#pragma unroll
        for (int t = 0; t < NT; t++) red[wave][t][lane] = acc[t];
        __syncthreads();
        if constexpr (!GU) {
            for (int t = wave; t < NT; t += WAVES) {
                f32x4 s = red[0][t][lane];
#pragma unroll
                for (int w = 1; w < WAVES; w++) s += red[w][t][lane];
                if (ok) {
                    const int64_t n = n_of(t) + 4 * g, first = n0 + 16 * t;
                    float *c = p.c + (int64_t)(tile.row + r) * p.N + n;
                    if (p.c_vec && first + 16 <= p.N) {
                        *(f32x4 *)c = s;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (n + i >= first && n + i < p.N) c[i] = s[i];
                    }
                }
            }
        } else {
            // eight neighbouring lanes take the 32 columns of one row
            for (int i = threadIdx.x; i < BM * 8; i += WAVES * WAVE) {
                const int m = i >> 3, s = i & 7, src = (s & 3) * 16 + m;
                if (m >= tile.rows || x_row(m) < 0) continue;
                f32x4 gt = red[0][s >> 2][src], up = red[0][2 + (s >> 2)][src];
#pragma unroll
                for (int w = 1; w < WAVES; w++) {
                    gt += red[w][s >> 2][src];
                    up += red[w][2 + (s >> 2)][src];
                }
                float h[4];
#pragma unroll
                for (int e = 0; e < 4; e++) h[e] = swiglu(gt[e], up[e]);
                uint32_t mx = abs_bits(h[0]);
#pragma unroll
                for (int e = 1; e < 4; e++) mx = max(mx, abs_bits(h[e]));
                const uint32_t c = mx_scale<T_MXINT8>(max8(mx));
                const int64_t row = tile.row + m;
                *(uint32_t *)(p.hc + row * p.N + n0 + 4 * s) = mx_round4<T_MXINT8>(h, c);
                if (s == 0) p.hs[row * (p.N / 32) + n0 / 32] = (uint8_t)c;
            }
        }
        __syncthreads();                                 // red is written again
    }
}

// ---------------------------------------------------------------------------
// More rows: a workgroup takes 16 MT rows of x and `span` tiles of output
// columns, which its waves share out (a tile: 16 NT rows of weights; GU: 8 NT
// gate rows and the same up rows).
//
// The rows of x are split into digits once and stay in LDS, in the matrix
// cores' lane order, for all columns.  After that a wave runs by itself, with no
// barrier: its weights go from memory to its registers a chunk of 512 columns
// ahead, over the end of a tile into its next one.  Two waves a SIMD.
//
// 16384 rows in 128 groups of 768 x 2 outputs, K = 2048: 116 us, 0.9 PFLOP/s; the
// vector units are busy 60 % of the waves' time (a third of that the exchange of the
// weights between lanes, a quarter the epilogue, as much the split of x), the
// matrix cores 33 %.  296 rows in those groups: 43 us, memory at 4.4 TB/s.  512 x
// 4096: 15.3 us, of which 4.4 the split of x and 5 the launch and the last stores.
// ---------------------------------------------------------------------------
constexpr int FRAG_LO = 0, FRAG_HI = 1024, FRAG_HI2 = 2048, FRAG_SC = 2560, FRAG_BYTES = 2688;
// 32 bytes between the steps' fragments: the four lanes that write a row's
// neighbouring blocks write to four steps.
constexpr int step_bytes(int mt) { return mt * FRAG_BYTES + 32; }

// Place `at` (a lane of the products) of a fragment.
__device__ __forceinline__ void frag_store(uint8_t *frag, int at, const XFrag &f)
{
    *(i32x4 *)(frag + FRAG_LO + 16 * at) = f.lo;
    *(i32x4 *)(frag + FRAG_HI + 16 * at) = i32x4{ (int)f.hi[0], (int)f.hi[1], (int)f.hi[2], (int)f.hi[3] };
    *(u32x2 *)(frag + FRAG_HI2 + 8 * at) = u32x2{ f.hi[4], f.hi[5] };
    *(uint16_t *)(frag + FRAG_SC + 2 * at) = (uint16_t)f.sc;
}

__device__ __forceinline__ XFrag frag_load(const uint8_t *frag, int at)
{
    XFrag f;
    f.lo = *(const i32x4 *)(frag + FRAG_LO + 16 * at);
    const i32x4 h = *(const i32x4 *)(frag + FRAG_HI + 16 * at);
    const u32x2 t = *(const u32x2 *)(frag + FRAG_HI2 + 8 * at);
    f.hi = u32x6{ (uint32_t)h[0], (uint32_t)h[1], (uint32_t)h[2], (uint32_t)h[3], t[0], t[1] };
    f.sc = *(const uint16_t *)(frag + FRAG_SC + 2 * at);
    return f;
}

template <int WAVES, int NT, int MT, int LEAD, bool GU, bool BESIDE>
__global__ void __launch_bounds__(WAVES * WAVE, 2) k_mx_tile(MxProduct p, uint32_t n_jobs, uint32_t n_tiles, int span,
                                                             int spread)
{
    static_assert(!GU || NT % 4 == 0, "a wave's gate and up rows make whole blocks of 32 outputs");
    constexpr int BM = 16 * MT, OUT = GU ? 8 * NT : 16 * NT, STEP = step_bytes(MT);
    extern __shared__ __align__(16) uint8_t lds[];       // n_chunk x 4 steps
    const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane & 15, g = lane >> 4;              // a lane's place in the products
    const int rl = lane >> 2, gl = lane & 3;             // and in loads of four blocks of 16 rows
    const int nb = p.K / 32, n_chunk = (nb + CHUNK_BLOCKS - 1) / CHUNK_BLOCKS;
    const int col_tiles = (int)(((uint32_t)p.N + OUT - 1) / OUT);
    const uint32_t n_items = spread ? row_tiles<BM>(p.offsets, p.n_group, p.n_rows) : 0;

    for (uint32_t at = blockIdx.x; at < n_jobs; at += gridDim.x) {
        // Consecutive workgroups run on different XCDs, each with its own L2.  An XCD takes a
        // run of row tiles with all their columns: those share their rows of x, and the row
        // tiles of a group its weights.  With too few row tiles for that, consecutive
        // columns.
        Job job;
        if (spread) {
            const uint32_t per = (n_items + 7) / 8;
            job = job_of(at >> 3, n_tiles);
            if (job.item >= per) continue;               // the grid is for the most row tiles there can be
            job.item += (at & 7) * per;
            if (job.item >= n_items) continue;
        } else {
            job = job_of(at, n_tiles);
        }
        const RowTile tile = row_tile<BM>(p.offsets, p.n_group, p.n_rows, job.item);
        if (tile.rows == 0) continue;                    // uniform over the workgroup
        const int first = (int)job.tile * span, last = min(first + span, col_tiles) - 1;

        // The weight rows of block t of tile q: n_of(q, t) .. + 15, moved down where they
        // would pass the end (those below the block's place are then not stored).  The base
        // addresses are the same for the wave; a lane adds 32-bit offsets.
        const auto n_of = [&](int q, int t) {
            return max((int64_t)0, min((int64_t)q * OUT + 16 * (GU ? t % (NT / 2) : t), (int64_t)p.N - 16));
        };
        uint32_t c_row[4];
#pragma unroll
        for (int j = 0; j < 4; j++) c_row[j] = (uint32_t)min((r & 12) + j, p.N - 1) * (p.K / 2);
        const uint32_t s_row = (uint32_t)min(rl, p.N - 1) * nb + 4 * gl;

        // A chunk's weights in place, and the next chunk's as loaded.  Blocks behind the last
        // are read as the last, their x is zero; scales up to 15 bytes on, which every
        // allocation has.
        i32x4 w[NT][4], wn[NT][4];
        uint32_t sw[NT], swn[NT];
        const uint8_t *wc[NT], *ws[NT];                  // of the tile that is being loaded
        const auto at_tile = [&](int q) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const bool up = GU && t >= NT / 2;
                const int64_t n = (int64_t)tile.group * p.N + n_of(q, t);
                wc[t] = (up ? p.uc : p.wc) + n * (p.K / 2);
                ws[t] = (up ? p.us : p.ws) + n * nb;
            }
        };
        const auto load_w = [&](int chunk, int j) {
            const uint32_t co = c_row[j] + (uint32_t)min(chunk * CHUNK_BLOCKS + 4 * g + gl, nb - 1) * 16;
#pragma unroll
            for (int t = 0; t < NT; t++) wn[t][j] = *(const i32x4 *)(wc[t] + co);
        };
        const auto load_sw = [&](int chunk) {
#pragma unroll
            for (int t = 0; t < NT; t++) swn[t] = *(const u32_any *)(ws[t] + s_row + (uint32_t)(chunk * CHUNK_BLOCKS));
        };
        const auto place_w = [&](int t, int chunk, auto beside) {
#pragma unroll
            for (int j = 0; j < 4; j++) w[t][j] = wn[t][j];
            if constexpr (decltype(beside)::value != 0) quad_transpose_beside(w[t]);
            else quad_transpose(w[t]);
            sw[t] = scales_within(scales_to_place(swn[t]), chunk * CHUNK_BLOCKS + 4 * g, nb);
        };
        // x: a wave splits units of 16 rows x 4 blocks, one for each step of a chunk.  Blocks
        // behind the last become zeros, whatever their weights (the last block's, whose NaN
        // scale the row has anyway).  Its first loads go before those of the weights: loads
        // return in order.
        // (A wave keeps to one block of 16 rows where the waves divide by them.)
        constexpr bool ONE = WAVES % MT == 0;
        constexpr int MS = ONE ? 1 : MT, EACH = ONE ? WAVES / MT : WAVES, AT_ONCE = ONE ? 4 : MT;
        const uint8_t *xc[MS], *xs[MS];
#pragma unroll
        for (int i = 0; i < MS; i++) {
            int64_t xr = tile.row + min(16 * (ONE ? wave % MT : i) + rl, tile.rows - 1);
            if (p.ids) xr = p.ids[xr];
            if (xr < 0 || xr >= p.n_x) xr = 0;
            xc[i] = p.xc + xr * p.K;
            xs[i] = p.xs + xr * nb;
        }
        RawBlock raw[AT_ONCE];
        const auto load_x = [&](int u) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++)
                raw[i] = raw_block(xc[i % MS], xs[i % MS], min(4 * (u + i / MS * EACH) + gl, nb - 1));
        };
        const int u0 = ONE ? wave / MT : wave;
        load_x(u0);
        int q = min(first + wave, last);
        at_tile(q);
        load_sw(0);
#pragma unroll
        for (int j = 0; j < 4; j++) load_w(0, j);
        for (int u = u0; u < 4 * n_chunk; u += AT_ONCE / MS * EACH) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++) {
                const int v = u + i / MS * EACH;
                if (v < 4 * n_chunk)
                    frag_store(lds + (4 * (v / 4) + gl) * STEP + (ONE ? wave % MT : i % MS) * FRAG_BYTES, 16 * (v % 4) + rl,
                               x_frag(raw[i], 4 * v + gl < nb));
            }
            load_x(u + AT_ONCE / MS * EACH);
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++) place_w(t, 0, Int<0>{});

        for (q = first + wave; q <= last; q += WAVES) {
            f32x4 acc[NT][MT];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int m = 0; m < MT; m++) acc[t][m] = f32x4{ 0.f, 0.f, 0.f, 0.f };
            for (int c = 0; c < n_chunk; c++) {
                // the chunk that comes next; after the wave's last one this one again, for nothing
                int next_c = c + 1;
                if (next_c == n_chunk) {
                    if (q + WAVES <= last) {
                        next_c = 0;
                        at_tile(q + WAVES);
                    } else {
                        next_c = c;
                    }
                }
                // One block of straight code, in which everything comes ahead of its use:
                // fragments of x by one of 16 rows, weights by a chunk.
                const uint8_t *frags = lds + c * 4 * STEP;
                XFrag f = frag_load(frags, lane);
                load_sw(next_c);
#pragma unroll
                for (int j = 0; j < LEAD; j++) load_w(next_c, j);
                const auto step = [&](auto kc) {
                    constexpr int k = decltype(kc)::value;
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        XFrag next;
                        if (m + 1 < MT) next = frag_load(frags + k * STEP + (m + 1) * FRAG_BYTES, lane);
                        else if (k + 1 < 4) next = frag_load(frags + (k + 1) * STEP, lane);
#pragma unroll
                        for (int t = 0; t < NT; t++) acc[t][m] = mx_mfma_hi<k>(w[t][k], sw[t], f, acc[t][m]);
                        __builtin_amdgcn_sched_barrier(0x7f6);   // no product passes: lo waits for its own hi
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            acc[t][m] = mx_mfma_lo<k>(w[t][k], sw[t], f, acc[t][m]);
                            if (k == 3 && m == MT - 1) place_w(t, next_c, Int<BESIDE>{});
                        }
                        if (m == MT - 1 && k == 1) {             // the registers of two steps are free
#pragma unroll
                            for (int j = LEAD; j < 4; j++) load_w(next_c, j);
                        }
                        f = next;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                };
                step(Int<0>{});
                step(Int<1>{});
                step(Int<2>{});
                step(Int<3>{});
            }

            const int64_t n0 = (int64_t)q * OUT;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const int i = 16 * m + r;
                if (i >= tile.rows) continue;
                const int64_t row = tile.row + i;
                const int64_t id = p.ids ? (int64_t)p.ids[row] : row;
                if (id < 0 || id >= p.n_x) continue;     // four lanes of one row together
                if constexpr (!GU) {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const int64_t n = n_of(q, t) + 4 * g, place = n0 + 16 * t;
                        float *c = p.c + row * p.N + n;
                        if (p.c_vec && place + 16 <= p.N) {
                            *(f32x4 *)c = acc[t][m];
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                if (n + j >= place && n + j < p.N) c[j] = acc[t][m][j];
                        }
                    }
                } else {
                    // 32 columns of a row: eight values in each of four lanes
#pragma unroll
                    for (int e = 0; e < NT / 4; e++) {
                        const int64_t n = n0 + 32 * e;
                        if (n >= p.N) continue;          // uniform
                        float h[2][4];
                        uint32_t mx = 0;
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int i4 = 0; i4 < 4; i4++) {
                                h[j][i4] = swiglu(acc[2 * e + j][m][i4], acc[NT / 2 + 2 * e + j][m][i4]);
                                mx = max(mx, abs_bits(h[j][i4]));
                            }
                        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, WAVE));
                        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, WAVE));
                        const uint32_t sc = mx_scale<T_MXINT8>(mx);
#pragma unroll
                        for (int j = 0; j < 2; j++)
                            *(uint32_t *)(p.hc + row * p.N + n + 16 * j + 4 * g) = mx_round4<T_MXINT8>(h[j], sc);
                        if (g == 0) p.hs[row * (p.N / 32) + n / 32] = (uint8_t)sc;
                    }
                }
            }
        }
        __syncthreads();                                 // x is written again
    }
}

constexpr int CUS = 256, LDS_BYTES = 160 * 1024;

// Row tiles of bm: the most that n_rows rows in n_group groups can make, and about
// as many as groups of unlike sizes make (half of the last one empty in each, or one
// a group where rows are few).
static int64_t most_tiles(const MxProduct &p, int bm)
{
    return std::min<int64_t>(p.n_rows, ((int64_t)p.n_rows + bm - 1) / bm + p.n_group - 1);
}

static int64_t usual_tiles(const MxProduct &p, int bm)
{
    const int64_t rows = p.n_rows;
    return std::max(std::min<int64_t>(rows, (rows + bm - 1) / bm + p.n_group / 2), std::min<int64_t>(rows, p.n_group));
}

// Row tiles times tiles of `cols` output columns; false beyond 32 bits, which
// no operands that a device holds reach.
static bool count_jobs(const MxProduct &p, int bm, int64_t cols, uint32_t &n_jobs, uint32_t &n_tiles)
{
    const int64_t tiles = (p.N + cols - 1) / cols, jobs = tiles * most_tiles(p, bm);
    n_tiles = (uint32_t)tiles;
    n_jobs = (uint32_t)jobs;
    return jobs <= 0x7fffffff;
}

static dim3 job_grid(uint32_t n_jobs) { return dim3(std::min(n_jobs, 1u << 20)); }

static int tile_lds(const MxProduct &p, int mt)
{
    const int64_t n = (int64_t)((p.K / 32 + CHUNK_BLOCKS - 1) / CHUNK_BLOCKS) * 4 * step_bytes(mt);
    return (int)std::min<int64_t>(n, 1 << 30);
}

// How many column tiles a workgroup takes, and for how long it all runs.  With
// `parts` workgroups for a row tile, they run in rounds of as many as the CUs hold,
// each for its rows of x to be split (about as long as six of its tiles with eight
// waves a workgroup, four with four) and its tiles, one a SIMD at a time.  4096 x
// 1536, K = 2048: 24 tiles in two parts 25.5 us, in three 35; 16384 rows in 128 groups, 32
// a workgroup, 24 tiles in one part 142, in two 142, in three 153; 296 rows in 128 groups,
// in three parts 47.5, in four 44.5.
//
// (Equal shares of all tiles for every workgroup, that end within row tiles, were no
// faster: 128 against 131 us for those 16384 rows, 32 a workgroup, 144 against 135 for groups of equal
// sizes, 62 against 57 for 8000 rows, K = 768.  Nor were two halves of the columns for
// the waves that have no tile: 512 x 4096 15.9 us with and without.)
struct Span {
    int64_t span, cost;         // the cost in 1/20 of a tile of 32 rows
};

template <int WAVES, int NT, int MT, bool GU>
static Span tile_span(const MxProduct &p)
{
    constexpr int OUT = GU ? 8 * NT : 16 * NT;
    // workgroups a CU holds: eight waves' registers
    const int at_once = WAVES == 8 || 2 * tile_lds(p, MT) > LDS_BYTES ? CUS : 2 * CUS;
    const int64_t tiles = ((int64_t)p.N + OUT - 1) / OUT, rows = usual_tiles(p, 16 * MT);
    // (48 rows: the split takes half as long again, a tile a tenth)
    const int64_t split = (at_once == CUS ? 6 : 4) * (MT == 3 ? 30 : 20), tile = MT == 3 ? 22 : 20;
    Span best{ tiles, INT64_MAX };
    // by the number q of tiles a SIMD, the shortest span of each number of parts
    for (int64_t q = (tiles + 3) / 4; q > 0; q--) {
        const int64_t parts = (tiles + 4 * q - 1) / (4 * q);
        q = (tiles + 4 * parts - 1) / (4 * parts);
        const int64_t rounds = (rows * parts + at_once - 1) / at_once, cost = rounds * (split + 4 * q * tile);
        if (cost < best.cost) {
            // as many more workgroups as the last round has room for, with a tile for each
            // SIMD: they share the end
            const int64_t most = q > 1 ? (tiles - 1) / (4 * (q - 1)) : std::max(parts, tiles / 4);
            const int64_t more = std::max(parts, std::min(most, rounds * at_once / rows));
            best = { (tiles + more - 1) / more, cost };
        }
    }
    return best;
}

template <int WAVES, int NT, int MT, int LEAD, bool GU>
static hipError_t launch_tile(const MxProduct &p, const MxPlan &plan, hipStream_t s)
{
    const int lds = tile_lds(p, MT);
    if (lds > LDS_BYTES) return hipErrorInvalidValue;
    const auto kernel = plan.beside ? k_mx_tile<WAVES, NT, MT, LEAD, GU, true> : k_mx_tile<WAVES, NT, MT, LEAD, GU, false>;
    if (lds > 64 * 1024) {
        const hipError_t e =
            hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
        if (e != hipSuccess) return e;
    }
    uint32_t n_jobs, n_tiles;
    if (!count_jobs(p, 16 * MT, plan.outputs * plan.span, n_jobs, n_tiles)) return hipErrorInvalidValue;
    const uint32_t items = n_jobs / n_tiles;
    const int spread = items >= 32 ? 1 : 0;
    if (spread) n_jobs = (items + 7) / 8 * 8 * n_tiles;          // row tiles past the last are empty
    hipLaunchKernelGGL(kernel, job_grid(n_jobs), dim3(WAVES * WAVE), (size_t)lds, s, p, n_jobs, n_tiles, (int)plan.span,
                       spread);
    return hipGetLastError();
}

template <int WAVES, int NT, bool GU>
static hipError_t launch_few(const MxProduct &p, hipStream_t s)
{
    uint32_t n_jobs, n_tiles;
    if (!count_jobs(p, 16, GU ? 32 : 16 * NT, n_jobs, n_tiles)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_mx_few<WAVES, NT, GU>), job_grid(n_jobs), dim3(WAVES * WAVE), 0, s, p, n_jobs, n_tiles);
    return hipGetLastError();
}

template <int WAVES, int NT, bool GU>
static MxPlan few_of(const MxProduct &p)
{
    const int64_t outputs = GU ? 32 : 16 * NT;
    return { 0, WAVES, 16, (int)outputs, 0, ((int64_t)p.N + outputs - 1) / outputs, 1 };
}

template <int WAVES, int NT, int MT, bool GU>
static MxPlan tile_of(const MxProduct &p)
{
    constexpr int64_t outputs = GU ? 8 * NT : 16 * NT;
    const int64_t tiles = ((int64_t)p.N + outputs - 1) / outputs;
    // Whether every SIMD has two waves with a tile each (K = 2048: 512 x 4096, 1024 tiles,
    // 16.9 us with the transposition for that, 16.0 without; 768 x 4096, 1536 tiles, 19.25,
    // 18.9; 1024 x 4096, 2048 tiles, 20.15, 20.5).
    const int beside = usual_tiles(p, 16 * MT) * tiles >= 8 * CUS;
    return { 1, WAVES, 16 * MT, (int)outputs, beside, tiles, tile_span<WAVES, NT, MT, GU>(p).span };
}

// The variant, by the number of 16 x 64 blocks of products and the rows a group.
// Both sides of each line, in us, K = 2048 unless said:
//  - k_mx_few below 512 blocks, where the CUs are not full and splitting x in
//    every workgroup costs less than a prologue: 64 x 4096, 256 blocks, 7.1
//    against 9.7; at 512 blocks (128 x 4096) 11.3 against 10.0.  Beyond, too, with few
//    rows to split, at most one a group: 128 rows in 128 groups of 768 x 2 outputs 32.0
//    against 39, K = 768 and 2048 outputs 17.9 against 18.6 (with two a group 23.8
//    against 21.3); or eight rows of one matrix: one of 65536 outputs, K = 768, 7.8
//    against 10.7, K = 4096, 27.6 against 34, eight 30.3 against 34.4; nor do digits of
//    16 rows fit the LDS above K = 7680 (4096 outputs of 64 rows 19.5 us at 7680, 20.4 at
//    8192, of 512 rows 46.8 and 91.4, of 2048 rows 127 and 282);
//  - in it, one block of weight rows a workgroup below 128 blocks (64 blocks 5.1, two
//    5.3; 128 blocks 6.5 against 5.6), two below 512 and four waves (64 x 4096: 7.1,
//    with four by two waves 8.4), or with the two chunks of K = 768 below 256 (128 x
//    2048: 6.9 against 6.0);
//  - 32 rows instead of 16 from 16 rows a group (16: 54 against 65, gate/up; 8: 62
//    against 51) or, for one matrix, 2048 blocks (512 x 4096: 15.3 against 17.7; 256 x
//    4096: 13.3 against 11.6), as long as they fit the LDS; 48 where their plan is the
//    shorter one (16384 rows in 128 groups, gate/up: 119 against 139; 4096 rows 81 against
//    68; K = 768: 16000 rows 87 against 96, 4096 rows 40.8 against 44.2, 2048 rows 33
//    against 30; 2048 x 16384: 101 against 113, 2048 x 4096: 34 against 31);
//  - four waves instead of eight where two such workgroups fit a CU: for 16 rows 128 x
//    4096: 10.0 against 10.5 (at K = 4096, where they do not, 2048 x 2048: 45.9 against
//    41.2); for 32 rows of groups of unequal sizes, 16000 rows in 128 groups x 2048, K =
//    768: 98 against 108 (2048 rows of one matrix: 15.1 against 13.6).
template <bool GU>
static MxPlan product_plan(const MxProduct &p)
{
    const int64_t blocks = usual_tiles(p, 16) * (((int64_t)p.N * (GU ? 2 : 1) + 63) / 64);
    if (blocks < 512 || p.n_rows <= (p.offsets ? p.n_group : 8) || tile_lds(p, 1) > LDS_BYTES) {
        if constexpr (GU) return blocks < 512 ? few_of<4, 4, true>(p) : few_of<2, 4, true>(p);
        else if (blocks < 128) return few_of<4, 1, false>(p);
        else if (blocks < (p.K > 1024 ? 512 : 256)) return few_of<4, 2, false>(p);
        else return few_of<2, 4, false>(p);
    }
    const bool wide = p.offsets ? (int64_t)p.n_rows >= 16 * (int64_t)p.n_group : blocks >= 2048;
    if (wide && tile_lds(p, 2) <= LDS_BYTES) {
        if (p.offsets && 2 * tile_lds(p, 2) <= LDS_BYTES) {
            if (2 * tile_lds(p, 3) <= LDS_BYTES && tile_span<4, 4, 3, GU>(p).cost < tile_span<4, 4, 2, GU>(p).cost)
                return tile_of<4, 4, 3, GU>(p);
            return tile_of<4, 4, 2, GU>(p);
        }
        if (tile_lds(p, 3) <= LDS_BYTES && tile_span<8, 4, 3, GU>(p).cost < tile_span<8, 4, 2, GU>(p).cost)
            return tile_of<8, 4, 3, GU>(p);
        return tile_of<8, 4, 2, GU>(p);
    }
    if (2 * tile_lds(p, 1) <= LDS_BYTES) return tile_of<4, 4, 1, GU>(p);
    return tile_of<8, 4, 1, GU>(p);
}

template <bool GU>
static hipError_t launch_product(const MxProduct &p, hipStream_t s)
{
    const MxPlan f = product_plan<GU>(p);
    if (f.kernel == 0) {
        if constexpr (GU) return f.waves == 4 ? launch_few<4, 4, true>(p, s) : launch_few<2, 4, true>(p, s);
        else if (f.waves == 2) return launch_few<2, 4, false>(p, s);
        else return f.outputs == 16 ? launch_few<4, 1, false>(p, s) : launch_few<4, 2, false>(p, s);
    }
    if (f.rows == 48) return f.waves == 4 ? launch_tile<4, 4, 3, 0, GU>(p, f, s) : launch_tile<8, 4, 3, 0, GU>(p, f, s);
    if (f.rows == 32) return f.waves == 4 ? launch_tile<4, 4, 2, 2, GU>(p, f, s) : launch_tile<8, 4, 2, 2, GU>(p, f, s);
    return f.waves == 4 ? launch_tile<4, 4, 1, 4, GU>(p, f, s) : launch_tile<8, 4, 1, 4, GU>(p, f, s);
}

MxPlan mx_product_plan(const MxProduct &p, bool gate_up) { return gate_up ? product_plan<true>(p) : product_plan<false>(p); }

hipError_t launch_mx_product(const MxProduct &p0, hipStream_t s)
{
    MxProduct p = p0;
    p.c_vec = p.N % 4 == 0 && ((uintptr_t)p.c & 15) == 0;
    return p.hc != nullptr ? launch_product<true>(p, s) : launch_product<false>(p, s);
}

}  // namespace ds3k
