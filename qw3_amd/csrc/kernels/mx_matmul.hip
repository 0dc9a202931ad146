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

// ---------------------------------------------------------------------------
// Row tiles of the groups.  Group g owns the rows offsets[g] .. offsets[g + 1]
// - 1; tiles of BM rows are numbered through the groups in order.  The offsets
// are device data: each is taken into 0 .. n_rows, a group that ends before it
// begins is empty.
// ---------------------------------------------------------------------------
struct RowTile {
    int group, row, rows;       // rows = 0: no such tile
};

__device__ __forceinline__ int wave_scan(int v)
{
    const int lane = threadIdx.x & (WAVE - 1);
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const int u = __shfl_up(v, o, WAVE);
        if (lane >= o) v += u;
    }
    return v;
}

// Uniform over the wave.
template <int BM>
__device__ __forceinline__ RowTile row_tile(const int32_t *offsets, int n_group, int n_rows, int64_t item)
{
    if (offsets == nullptr) {
        const int64_t row = item * BM;
        return { 0, (int)row, row < n_rows ? (int)min((int64_t)BM, n_rows - row) : 0 };
    }
    const int lane = threadIdx.x & (WAVE - 1);
    int64_t before = 0;
    for (int g0 = 0; g0 < n_group; g0 += WAVE) {
        const int g = g0 + lane;
        int begin = 0, end = 0;
        if (g < n_group) {
            begin = min(max(offsets[g], 0), n_rows);
            end = min(max(offsets[g + 1], begin), n_rows);
        }
        const int tiles = (end - begin + BM - 1) / BM;
        const int incl = wave_scan(tiles);
        const int total = __builtin_amdgcn_readlane(incl, WAVE - 1);
        if (item < before + total) {
            const int at = (int)(item - before);
            const int src = __builtin_ctzll(__ballot(incl > at));
            const int b = __builtin_amdgcn_readlane(begin, src), e = __builtin_amdgcn_readlane(end, src);
            const int row = b + (at - (__builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane(tiles, src))) * BM;
            return { g0 + src, row, min(BM, e - row) };
        }
        before += total;
    }
    return { 0, 0, 0 };
}

// ---------------------------------------------------------------------------
// Few rows: a workgroup takes 16 rows of x and NT blocks of 16 weight rows (GU:
// two blocks of the gate and two of the up matrix, 32 outputs); its waves take
// the K steps of 128 in turn, straight from memory, and their sums meet in LDS.
// ---------------------------------------------------------------------------
constexpr int FEW_WAVES = 4;

template <int NT, bool GU>
__global__ void __launch_bounds__(FEW_WAVES * WAVE) k_mx_few(MxProduct p, int64_t n_items, int64_t n_tiles)
{
    static_assert(!GU || NT == 4, "the gate/up tile is two blocks of each matrix");
    constexpr int BM = 16, NW = GU ? 32 : 16 * NT;       // output columns a workgroup
    __shared__ f32x4 red[FEW_WAVES][NT][WAVE];
    const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
    const int r = lane & 15, g = lane >> 4;
    const int nb = p.K / 32, nk = (nb + 3) / 4;

    for (int64_t job = blockIdx.x; job < n_items * n_tiles; job += gridDim.x) {
        const int64_t item = job / n_tiles;
        const int64_t n0 = (job - item * n_tiles) * NW;
        const RowTile tile = row_tile<BM>(p.offsets, p.n_group, p.n_rows, item);
        if (tile.rows == 0) continue;                    // uniform over the workgroup
        // this lane's row of x, and whether its outputs exist
        int64_t xr = tile.row + min(r, tile.rows - 1);
        if (p.ids) xr = p.ids[xr];
        const bool ok = r < tile.rows && xr >= 0 && xr < p.n_x;
        if (xr < 0 || xr >= p.n_x) xr = 0;
        const uint8_t *xc = p.xc + xr * p.K, *xs = p.xs + xr * nb;
        const uint8_t *wc[NT], *ws[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const bool up = GU && t >= 2;
            const int64_t n = (int64_t)tile.group * p.N + min(n0 + 16 * (GU ? t & 1 : t) + r, (int64_t)p.N - 1);
            wc[t] = (up ? p.uc : p.wc) + n * (p.K / 2);
            ws[t] = (up ? p.us : p.ws) + n * nb;
        }
        f32x4 acc[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = f32x4{ 0.f, 0.f, 0.f, 0.f };
        for (int kk = wave; kk < nk; kk += FEW_WAVES) {
            const int b = 4 * kk + g;
            uint32_t x[8] = { 0, 0, 0, 0, 0, 0, 0, 0 };
            uint32_t sx = 127, sw[NT];
            i32x4 w[NT];
            if (b < nb) {                                // a row's last step may have fewer than four blocks
                const uint4 x0 = *(const uint4 *)(xc + b * 32), x1 = *(const uint4 *)(xc + b * 32 + 16);
                x[0] = x0.x; x[1] = x0.y; x[2] = x0.z; x[3] = x0.w;
                x[4] = x1.x; x[5] = x1.y; x[6] = x1.z; x[7] = x1.w;
                sx = xs[b];
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                w[t] = i32x4{ 0, 0, 0, 0 };
                sw[t] = 127;
                if (b < nb) {
                    w[t] = *(const i32x4 *)(wc[t] + b * 16);
                    sw[t] = ws[t][b];
                }
            }
            const XFrag f = x_frag(x, sx);
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] = mx_mfma(w[t], sw[t], f, acc[t]);
        }
#pragma unroll
        for (int t = 0; t < NT; t++) red[wave][t][lane] = acc[t];
        __syncthreads();
        if constexpr (!GU) {
            for (int t = wave; t < NT; t += FEW_WAVES) {
                f32x4 s = red[0][t][lane];
#pragma unroll
                for (int w = 1; w < FEW_WAVES; w++) s += red[w][t][lane];
                if (ok) {
                    const int64_t n = n0 + 16 * t + 4 * g;
                    float *c = p.c + (int64_t)(tile.row + r) * p.N + n;
                    if (p.c_vec && n + 4 <= p.N) {
                        *(f32x4 *)c = s;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (n + i < p.N) c[i] = s[i];
                    }
                }
            }
        } else {
            // eight neighbouring lanes take the 32 columns of one row
            const int m = threadIdx.x >> 3, s = threadIdx.x & 7, src = (s & 3) * 16 + m;
            if (threadIdx.x < BM * 8 && m < tile.rows) {
                f32x4 gt = red[0][s >> 2][src], up = red[0][2 + (s >> 2)][src];
#pragma unroll
                for (int w = 1; w < FEW_WAVES; w++) {
                    gt += red[w][s >> 2][src];
                    up += red[w][2 + (s >> 2)][src];
                }
                float h[4];
#pragma unroll
                for (int i = 0; i < 4; i++) h[i] = swiglu(gt[i], up[i]);
                const int64_t row = tile.row + m;
                const int64_t id = p.ids ? (int64_t)p.ids[row] : row;
                if (id >= 0 && id < p.n_x) {
                    uint32_t mx = abs_bits(h[0]);
#pragma unroll
                    for (int i = 1; i < 4; i++) mx = max(mx, abs_bits(h[i]));
                    const uint32_t c = mx_scale<T_MXINT8>(max8(mx));
                    *(uint32_t *)(p.hc + row * p.N + n0 + 4 * s) = mx_round4<T_MXINT8>(h, c);
                    if (s == 0) p.hs[row * (p.N / 32) + n0 / 32] = (uint8_t)c;
                }
            }
        }
        __syncthreads();                                 // red is written again
    }
}

// The most row tiles of BM that n_rows rows in n_group groups can make.
static int64_t most_tiles(int64_t n_rows, int64_t n_group, int bm)
{
    return std::min(n_rows, (n_rows + bm - 1) / bm + n_group - 1);
}

hipError_t launch_mx_product(const MxProduct &p, hipStream_t s)
{
    const bool gu = p.hc != nullptr;
    const int64_t items = most_tiles(p.n_rows, p.n_group, 16);
    const int64_t n_tiles = (p.N + 31) / 32;
    const dim3 grid((unsigned)std::min<int64_t>(items * n_tiles, (int64_t)1 << 20)), tpb(FEW_WAVES * WAVE);
    if (gu) hipLaunchKernelGGL((k_mx_few<4, true>), grid, tpb, 0, s, p, items, n_tiles);
    else hipLaunchKernelGGL((k_mx_few<2, false>), grid, tpb, 0, s, p, items, n_tiles);
    return hipGetLastError();
}

}  // namespace ds3k
