// mx_rows.hip -- rows to and from the microscaled formats (mx.h): rounding of
// F32 / F16 / GGUF-quantised rows, its inverse, and the FFN block's prologue
// (residual addition, RMS norm, rounding) in one pass.
#include "mx.h"

#include <algorithm>

namespace ds3k {

constexpr int MXR_TPB = 256;

// ---------------------------------------------------------------------------
// Rounding.  One pass, bound by its reads: eight lanes take a block, four
// values each (16-byte loads of F32), so that a wave reads 1 KiB and writes
// whole lines.  98304 x 2048 F32 to MXFP4 163 us, 5.6 TB/s; F16, 8 bytes a lane, 125, 4.1.
// ---------------------------------------------------------------------------

// Four consecutive values; VEC: the address is a multiple of their size.
template <bool F16, bool VEC>
__device__ __forceinline__ void load4(const uint8_t *p, float (&v)[4])
{
    if constexpr (F16) {
        if constexpr (VEC) {
            const half4_t h = *(const half4_t *)p;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = (float)h[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = (float)((const _Float16 *)p)[i];
        }
    } else if constexpr (VEC) {
        const float4 f = *(const float4 *)p;
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = ((const float *)p)[i];
    }
}

// The eight lanes of a block: values v of lane s = lane % 8, block `b` of the
// matrix (row major).
template <int MX>
__device__ __forceinline__ void store_block8(const float (&v)[4], int64_t b, int s, uint8_t *codes, uint8_t *scales)
{
    uint32_t m = abs_bits(v[0]);
#pragma unroll
    for (int i = 1; i < 4; i++) m = max(m, abs_bits(v[i]));
    const uint32_t c = mx_scale<MX>(max8(m));
    const uint32_t w = mx_round4<MX>(v, c);
    if constexpr (MX == T_MXINT8) *(uint32_t *)(codes + b * 32 + 4 * s) = w;
    else *(uint16_t *)(codes + b * 16 + 2 * s) = (uint16_t)w;
    if (s == 0) scales[b] = (uint8_t)c;
}

// nb blocks a row, rows `stride` bytes apart (dense rows are given as one).
template <int MX, bool F16, bool VEC>
__global__ void __launch_bounds__(MXR_TPB) k_mx_round(const uint8_t *src, uint64_t stride, int64_t n_blocks, int64_t nb,
                                                      uint8_t *codes, uint8_t *scales)
{
    const int s = threadIdx.x & 7;
    const int64_t step = (int64_t)gridDim.x * (MXR_TPB / 8);
    for (int64_t b = (int64_t)blockIdx.x * (MXR_TPB / 8) + (threadIdx.x >> 3); b < n_blocks; b += step) {
        const int64_t row = nb == n_blocks ? 0 : b / nb;
        const int64_t col = (b - row * nb) * 32 + 4 * s;
        float v[4];
        load4<F16, VEC>(src + row * stride + col * (F16 ? 2 : 4), v);
        store_block8<MX>(v, b, s, codes, scales);
    }
}

// The largest magnitude's bits.  The values have one scale in common: one that is
// not finite makes all of them infinite or NaN, the first too, while the maximum
// itself passes over NaN.
template <int N>
__device__ __forceinline__ uint32_t amax_of(const float *v)
{
    float m = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < N; i++) m = __builtin_fmaxf(m, fabsf(v[i]));
    return max(__float_as_uint(m), abs_bits(v[0]));
}

// The codes of N values, in dwords.
template <int MX, int N>
__device__ __forceinline__ void round_dwords(const float *v, uint32_t c, int *out)
{
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
        const float x[4] = { v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3] };
        const uint32_t q = mx_round4<MX>(x, c);
        if constexpr (MX == T_MXINT8) out[i] = (int)q;
        else if (i % 2 == 0) out[i / 2] = (int)q;
        else out[i / 2] |= (int)(q << 16);
    }
}

// GGUF blocks: a thread decodes one 32-weight unit (common.h) and rounds it with
// the scales of the blocks of 32 that its parts lie in.  A Q4_K unit is 16 weights
// each of two blocks that it shares with the next lane, a Q6_K unit 8 each of four
// that a quad shares; their codes are exchanged so that every lane stores the
// whole of one block.  98304 x 2048 weights to MXFP4: Q4_K 55 us (4.0 TB/s read and
// written; 72 with the weights themselves exchanged through LDS), Q6_K 77, Q8_0 65
// (its 34-byte blocks are read as dwords in halves); a copy of as much would take 42, 53
// and 62.  Q4_K's and Q6_K's decoding and rounding keep the vector units busy all the time.
template <int MX, int TYPE>
__global__ void __launch_bounds__(MXR_TPB) k_mx_round_gguf(const uint8_t *src, uint64_t stride, int64_t n_blocks,
                                                           int64_t nb, uint8_t *codes, uint8_t *scales)
{
    constexpr int D = MX == T_MXINT8 ? 8 : 4;            // dwords of a block's codes
    const int64_t step = (int64_t)gridDim.x * MXR_TPB;
    // rows are whole GGUF blocks of eight units (Q8_0: one), which stay together
    for (int64_t b = (int64_t)blockIdx.x * MXR_TPB + threadIdx.x; b < n_blocks; b += step) {
        const int64_t row = b / nb;
        float w[32];
        int k0[4], q[D];
        unit_decode<TYPE>(src + row * stride, (int)(b - row * nb), w, k0);
        uint32_t c;
        if constexpr (TYPE == T_Q4_K) {
            int lo[D / 2], hi[D / 2];
            uint32_t ml = amax_of<16>(w), mh = amax_of<16>(w + 16);
            ml = max(ml, (uint32_t)quad_xor<1>((int)ml));
            mh = max(mh, (uint32_t)quad_xor<1>((int)mh));
            const uint32_t cl = mx_scale<MX>(ml), ch = mx_scale<MX>(mh);
            round_dwords<MX, 16>(w, cl, lo);
            round_dwords<MX, 16>(w + 16, ch, hi);
            const bool odd = threadIdx.x & 1;            // of the two blocks the even lane stores the first
#pragma unroll
            for (int i = 0; i < D / 2; i++) {
                const int got = quad_xor<1>(odd ? lo[i] : hi[i]);
                q[i] = odd ? got : lo[i];
                q[D / 2 + i] = odd ? hi[i] : got;
            }
            c = odd ? ch : cl;
        } else if constexpr (TYPE == T_Q6_K) {
            const int p = threadIdx.x & 3;               // of the four blocks lane p stores the p-th
            c = 0;
            int part[D / 4][4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                uint32_t m = amax_of<8>(w + 8 * t);
                m = max(m, (uint32_t)quad_xor<1>((int)m));
                m = max(m, (uint32_t)quad_xor<2>((int)m));
                const uint32_t ct = mx_scale<MX>(m);
                int d[D / 4];
                round_dwords<MX, 8>(w + 8 * t, ct, d);
#pragma unroll
                for (int i = 0; i < D / 4; i++) part[i][t] = d[i];
                c = p == t ? ct : c;
            }
#pragma unroll
            for (int i = 0; i < D / 4; i++) {
                quad_transpose(part[i]);
#pragma unroll
                for (int t = 0; t < 4; t++) q[D / 4 * t + i] = part[i][t];
            }
        } else {
            c = mx_scale<MX>(amax_of<32>(w));
            round_dwords<MX, 32>(w, c, q);
        }
        uint4 *out = (uint4 *)(codes + b * (4 * D));
#pragma unroll
        for (int i = 0; i < D / 4; i++)
            out[i] = make_uint4((uint32_t)q[4 * i], (uint32_t)q[4 * i + 1], (uint32_t)q[4 * i + 2], (uint32_t)q[4 * i + 3]);
        scales[b] = (uint8_t)c;
    }
}

// The workgroups of a grid-stride kernel over n units of `per` a workgroup.
static unsigned strided_grid(int64_t n, int per)
{
    const int64_t wg = (n + per - 1) / per;
    return (unsigned)std::min<int64_t>(wg, (int64_t)1 << 20);
}

template <int MX>
static hipError_t launch_round(int type, const uint8_t *src, uint64_t stride, int64_t n_rows, int64_t n_cols,
                               uint8_t *codes, uint8_t *scales, hipStream_t s)
{
    const int64_t n_blocks = n_rows * (n_cols / 32);
    int64_t nb = n_cols / 32;
    if (type == T_F32 || type == T_F16) {
        const int size = type == T_F32 ? 4 : 2;
        if (stride == (uint64_t)n_cols * size) nb = n_blocks;                   // one long row
        const bool vec = ((uintptr_t)src | (nb == n_blocks ? 0 : stride)) % (4 * size) == 0;
        const dim3 grid(strided_grid(n_blocks, MXR_TPB / 8)), tpb(MXR_TPB);
        if (type == T_F32) {
            if (vec) hipLaunchKernelGGL((k_mx_round<MX, false, true>), grid, tpb, 0, s, src, stride, n_blocks, nb, codes, scales);
            else hipLaunchKernelGGL((k_mx_round<MX, false, false>), grid, tpb, 0, s, src, stride, n_blocks, nb, codes, scales);
        } else {
            if (vec) hipLaunchKernelGGL((k_mx_round<MX, true, true>), grid, tpb, 0, s, src, stride, n_blocks, nb, codes, scales);
            else hipLaunchKernelGGL((k_mx_round<MX, true, false>), grid, tpb, 0, s, src, stride, n_blocks, nb, codes, scales);
        }
        return hipGetLastError();
    }
    const dim3 grid(strided_grid(n_blocks, MXR_TPB)), tpb(MXR_TPB);
    switch (type) {
    case T_Q8_0: hipLaunchKernelGGL((k_mx_round_gguf<MX, T_Q8_0>), grid, tpb, 0, s, src, stride, n_blocks, nb, codes, scales); break;
    case T_Q4_K: hipLaunchKernelGGL((k_mx_round_gguf<MX, T_Q4_K>), grid, tpb, 0, s, src, stride, n_blocks, nb, codes, scales); break;
    case T_Q6_K: hipLaunchKernelGGL((k_mx_round_gguf<MX, T_Q6_K>), grid, tpb, 0, s, src, stride, n_blocks, nb, codes, scales); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_mx_quantize(int type, const uint8_t *src, uint64_t stride, int64_t n_rows, int64_t n_cols, int mx,
                              uint8_t *codes, uint8_t *scales, hipStream_t s)
{
    return mx == T_MXFP4 ? launch_round<T_MXFP4>(type, src, stride, n_rows, n_cols, codes, scales, s)
                         : launch_round<T_MXINT8>(type, src, stride, n_rows, n_cols, codes, scales, s);
}

// ---------------------------------------------------------------------------
// The values of a matrix.  Four a thread; every product is exact in fp32 but
// for those of 2^128 and more, which overflow to infinity.  98304 x 2048 MXFP4 in F32
// 187 us, 4.9 TB/s; in F16, 8 bytes a lane, 174, 2.9.
// ---------------------------------------------------------------------------
template <int MX, bool F16, bool VEC>
__global__ void __launch_bounds__(MXR_TPB) k_mx_values(const uint8_t *codes, const uint8_t *scales, int64_t n4, void *dst)
{
    const int64_t step = (int64_t)gridDim.x * MXR_TPB;
    for (int64_t i = (int64_t)blockIdx.x * MXR_TPB + threadIdx.x; i < n4; i += step) {
        const int c = scales[i >> 3];
        float v[4];
        if constexpr (MX == T_MXINT8) {
            const uint32_t w = ((const uint32_t *)codes)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __builtin_amdgcn_ldexpf((float)(int8_t)byte_of(w, j), c - 133);
        } else {
            const uint32_t w = ((const uint16_t *)codes)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                // twice the magnitudes, as bytes 0, 1, 2, 3 and 4, 6, 8, 12
                const uint32_t n = (w >> (4 * j)) & 15u, k = n & 7u;
                const float m = (float)byte_of(k < 4u ? 0x03020100u : 0x0c080604u, (int)(k & 3u));
                v[j] = __builtin_amdgcn_ldexpf(n & 8u ? -m : m, c - 128);
            }
        }
        if (c == 255)
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __uint_as_float(0x7fc00000u);
        if constexpr (F16) {
            const half4_t h = { (_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3] };
            if constexpr (VEC) ((half4_t *)dst)[i] = h;
            else
#pragma unroll
                for (int j = 0; j < 4; j++) ((_Float16 *)dst)[4 * i + j] = h[j];
        } else if constexpr (VEC) {
            ((float4 *)dst)[i] = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) ((float *)dst)[4 * i + j] = v[j];
        }
    }
}

template <int MX, bool F16>
static void values(const uint8_t *codes, const uint8_t *scales, int64_t n4, void *dst, hipStream_t s)
{
    const dim3 grid(strided_grid(n4, MXR_TPB)), tpb(MXR_TPB);
    if ((uintptr_t)dst % (F16 ? 8 : 16) == 0)
        hipLaunchKernelGGL((k_mx_values<MX, F16, true>), grid, tpb, 0, s, codes, scales, n4, dst);
    else
        hipLaunchKernelGGL((k_mx_values<MX, F16, false>), grid, tpb, 0, s, codes, scales, n4, dst);
}

hipError_t launch_mx_dequantize(int mx, const uint8_t *codes, const uint8_t *scales, int64_t n, int dst_type, void *dst,
                                hipStream_t s)
{
    if (mx == T_MXFP4) dst_type == T_F16 ? values<T_MXFP4, true>(codes, scales, n / 4, dst, s)
                                         : values<T_MXFP4, false>(codes, scales, n / 4, dst, s);
    else dst_type == T_F16 ? values<T_MXINT8, true>(codes, scales, n / 4, dst, s)
                           : values<T_MXINT8, false>(codes, scales, n / 4, dst, s);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// y = s / sqrt(mean(s^2) + eps) * g of s = x + delta (the reference's RMSNorm,
// src/ds3_reference.c:329-342), rounded to MXINT8.  s (when delta is given) and y
// are also written where asked for.
//
// The s that is written is rounded once; y comes from the unrounded sum, in 64
// bits, and is rounded once: a factor rounded to 32 bits would move a whole row the
// same way, and squares in 32 bits would overflow from 1.8e19 on.  Memory bounds the
// kernel (6001 x 4096 with delta and sum 64 us, 5.0 TB/s; in 32 bits 68.5 where this took 67), and the
// vector units have the time.
//
// A row is read once and stays in registers between the sum of squares and the
// rounding: TPR threads a row, four columns a thread and chunk, so a block of
// 32 is eight neighbouring lanes.  Rows of more than CH chunks (CH = 0) are
// read a second time, from the cache.
// ---------------------------------------------------------------------------
struct NormArgs {
    const float *x, *delta, *g;
    float *sum, *y;
    uint8_t *codes, *scales;
    float eps;
    int n;
    int64_t n_rows;
};

template <bool VEC>
__device__ __forceinline__ void store4f(float *p, const float (&v)[4])
{
    if constexpr (VEC) {
        *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = v[i];
    }
}

// Four columns' x and delta.
struct Terms {
    float x[4], d[4];

    __device__ __forceinline__ double sum(int i) const { return (double)x[i] + (double)d[i]; }
};

template <bool VEC>
__device__ __forceinline__ void load_terms(const NormArgs &a, int64_t at, Terms &v)
{
    load4<false, VEC>((const uint8_t *)(a.x + at), v.x);
    if (a.delta) {
        load4<false, VEC>((const uint8_t *)(a.delta + at), v.d);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v.d[i] = -0.f;           // x + -0 is x, for -0 too
    }
}

template <bool VEC>
__device__ __forceinline__ void finish4(const NormArgs &a, int64_t row, int col, double rms, const Terms &v)
{
    const int64_t at = row * a.n + col;
    float g[4], y[4];
    load4<false, VEC>((const uint8_t *)(a.g + col), g);
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = (float)(v.sum(i) * rms * (double)g[i]);
    if (a.sum) {
        const float s[4] = { v.x[0] + v.d[0], v.x[1] + v.d[1], v.x[2] + v.d[2], v.x[3] + v.d[3] };
        store4f<VEC>(a.sum + at, s);
    }
    if (a.y) store4f<VEC>(a.y + at, y);
    store_block8<T_MXINT8>(y, at / 32, (col / 4) & 7, a.codes, a.scales);
}

// v + v of the lane that DPP takes, in both halves.
template <int CTRL>
__device__ __forceinline__ double add_dpp(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return v + __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ double lane_of(double v, int lane)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// The sum over the wavefront: neighbours, quads, halves and rows of 16, then the
// four rows.
__device__ __forceinline__ double wave_sum64(double v)
{
    v = add_dpp<0xb1>(v);
    v = add_dpp<0x4e>(v);
    v = add_dpp<0x141>(v);
    v = add_dpp<0x140>(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// Eight lanes hold a block, and columns come in 32s, so a block's lanes are in
// or out together.  y is rounded to 32 bits before its block is: a value that 64 bits
// put a hair below a power of two would else halve its block's scale and saturate.
template <int TPR, int CH, bool VEC>
__global__ void __launch_bounds__(MXR_TPB) k_add_rms_norm_mx(NormArgs a)
{
    constexpr int ROWS = MXR_TPB / TPR, WPR = TPR / WAVE;
    __shared__ double part[MXR_TPB / WAVE];
    const int t = threadIdx.x % TPR;
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + threadIdx.x / TPR;
    if (row >= a.n_rows) return;                            // whole waves; WPR > 1 has one row a workgroup
    Terms v[CH > 0 ? CH : 1];
    double ss = 0.0;
    const int64_t base = row * a.n;
    if constexpr (CH > 0) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (c * TPR + t) * 4;
            if (col < a.n) {
                load_terms<VEC>(a, base + col, v[c]);
            } else {
                v[c] = Terms{};
            }
        }
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) ss = fma(v[c].sum(i), v[c].sum(i), ss);
    } else {
        for (int col = 4 * t; col < a.n; col += 4 * TPR) {
            load_terms<VEC>(a, base + col, v[0]);
#pragma unroll
            for (int i = 0; i < 4; i++) ss = fma(v[0].sum(i), v[0].sum(i), ss);
        }
    }
    ss = wave_sum64(ss);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & (WAVE - 1)) == 0) part[threadIdx.x / WAVE] = ss;
        __syncthreads();
        ss = part[0];
#pragma unroll
        for (int w = 1; w < WPR; w++) ss += part[w];
    }
    const double rms = 1.0 / sqrt(ss / a.n + a.eps);
    if constexpr (CH > 0) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (c * TPR + t) * 4;
            if (col < a.n) finish4<VEC>(a, row, col, rms, v[c]);
        }
    } else {
        for (int col = 4 * t; col < a.n; col += 4 * TPR) {
            load_terms<VEC>(a, base + col, v[0]);
            finish4<VEC>(a, row, col, rms, v[0]);
        }
    }
}

template <int TPR, int CH>
static hipError_t norm_launch(const NormArgs &a, bool vec, hipStream_t s)
{
    // a launch takes fewer than 2^32 threads in x
    const int64_t wg = (a.n_rows + MXR_TPB / TPR - 1) / (MXR_TPB / TPR), gx = std::min<int64_t>(wg, 1 << 20);
    const dim3 grid((unsigned)gx, (unsigned)((wg + gx - 1) / gx)), tpb(MXR_TPB);
    if (vec) hipLaunchKernelGGL((k_add_rms_norm_mx<TPR, CH, true>), grid, tpb, 0, s, a);
    else hipLaunchKernelGGL((k_add_rms_norm_mx<TPR, CH, false>), grid, tpb, 0, s, a);
    return hipGetLastError();
}

hipError_t launch_add_rms_norm_mx(const float *x, const float *delta, const float *g, float eps, float *sum, float *y,
                                  uint8_t *codes, uint8_t *scales, int n, int64_t n_rows, hipStream_t s)
{
    const NormArgs a{ x, delta, g, sum, y, codes, scales, eps, n, n_rows };
    const bool vec = (((uintptr_t)x | (uintptr_t)delta | (uintptr_t)g | (uintptr_t)sum | (uintptr_t)y) & 15) == 0;
    if (n <= 256) return norm_launch<WAVE, 1>(a, vec, s);
    if (n <= 1024) return norm_launch<WAVE, 4>(a, vec, s);
    if (n <= 2048) return norm_launch<MXR_TPB, 2>(a, vec, s);
    if (n <= 4096) return norm_launch<MXR_TPB, 4>(a, vec, s);
    if (n <= 8192) return norm_launch<MXR_TPB, 8>(a, vec, s);
    return norm_launch<MXR_TPB, 0>(a, vec, s);
}

}  // namespace ds3k
