// mx.h -- device helpers of the microscaled (MX) formats on gfx950.
//
// An MX matrix is two planes.  For every 32 consecutive values of a row the
// scale plane [rows][cols / 32] holds one E8M0 byte c: 2^(c - 127), 255 for
// NaN.  The code plane holds
//   MXFP4   4 bits a value (E2M1): bit 3 the sign, bits 0..2 the magnitudes
//           0, .5, 1, 1.5, 2, 3, 4, 6; value 2j of a row in the low half of
//           byte j, value 2j + 1 in the high half; [rows][cols / 2] bytes
//   MXINT8  one signed byte q a value, for q / 64; [rows][cols] bytes
//
// Products run on the block-scaled matrix cores, and exactly: the 8-bit format
// of those is FP8, whose sums drop what lies more than about 13 bits below the
// largest product of a group (relative L2 error 4e-6 on normal data, 4.5e-5 on
// values of many magnitudes), while products of 4-bit with 4- or 6-bit
// operands keep every bit down to the fp32 sum (no difference from a 64-bit
// sum over 10^5 random tiles of equal scales, 2^-22 of the sum of magnitudes
// with scales 2^30 apart).  So a row byte q is split as
//   q = 8 hi + lo,  hi = the nearest integer to q / 8 (ties to even), |lo| <= 4
// hi / 8 is an E2M3 value (6 bits: steps of 1/8 up to 2) and lo / 2 an E2M1
// value, both exactly, and q / 64 = hi / 8 + 2^-5 (lo / 2): two matrix
// instructions at the 4-bit rate (8.4 PFLOP/s measured, 4.2 for the pair; one
// FP8 x FP4 instruction measured 4.46) against the same weight operand, the
// second with the scale lowered by 2^5.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace ds3k {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half32_t __attribute__((ext_vector_type(32)));

// ---------------------------------------------------------------------------
// Rounding to a block
// ---------------------------------------------------------------------------

// |v| as bits: ordered like the magnitudes, with NaN above infinity, so an
// integer maximum keeps a block's NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Maximum over the 8 lanes of an aligned group.
__device__ __forceinline__ uint32_t max8(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));    // lanes 1, 0, 3, 2
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));    // lanes 2, 3, 0, 1
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true)); // mirrored in 8
}

// The scale byte of a block whose largest magnitude has the bits `amax`.
// MXINT8: 2^floor(log2 amax), so q stays below 128.  MXFP4: the smallest power
// of two with at most seven of it in amax: up to 7 the largest value rounds to
// 6 with no more error than a value between 4 and 6 can have, and 5 to 6 %
// less squared error comes out on normal weights than with floor(log2 amax) - 2,
// whose blocks reach 8.  A block of zeros (or of magnitudes below 2^-126) gets
// the lowest scale, one with an infinity or a NaN gets 255.
template <int MX>
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax)
{
    if (amax >= 0x7f800000u) return 255u;
    if constexpr (MX == T_MXINT8) return amax >> 23;
    const uint32_t c = (amax + 0x1fffffu) >> 23;      // one more above 1.75 = 7/4
    return c > 2u ? c - 2u : 0u;
}

// Four values of a block with scale byte c, rounded to nearest (ties to even):
// MXINT8: four signed bytes, at most 127 in magnitude; MXFP4: four nibbles in
// the low 16 bits.  The power of two is applied exactly (ldexp).
template <int MX>
__device__ __forceinline__ uint32_t mx_round4(const float (&v)[4], uint32_t c)
{
    if (c == 255u) return 0u;
    if constexpr (MX == T_MXINT8) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float y = __builtin_amdgcn_ldexpf(v[i], 133 - (int)c);
            const int q = (int)rintf(fminf(fmaxf(y, -127.f), 127.f));
            w |= (uint32_t)(q & 0xff) << (8 * i);
        }
        return w;
    } else {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = __builtin_amdgcn_ldexpf(v[i], 127 - (int)c);
        uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.0f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1);
        return w & 0xffffu;
    }
}

// ---------------------------------------------------------------------------
// Matrix-core operands
//
// v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds row (A) or column (B) l % 16
// and, for 4- and 6-bit operands, the values 32 (l / 16) .. + 31 of the 128;
// its scale byte is that block's.  D: lane l, register i is row
// 4 (l / 16) + i, column l % 16.  The weights are A and the rows of x B, so a
// lane ends with four consecutive outputs of one row of x.
// ---------------------------------------------------------------------------

// 32 values of an MXINT8 row as operand B.
struct XFrag {
    u32x6 hi;          // E2M3 digits
    i32x4 lo;          // E2M1 digits
    uint32_t sc;       // byte 0: scale of hi, byte 1: of lo
};

// Splits 32 signed bytes (w, in order) with scale byte c.  A block whose scale
// is below 2^-122 (c < 5), for which lo would need one below 2^-127, is first
// rounded to multiples of 2^-128: what is lost lies under the smallest normal
// fp32 number.
__device__ __forceinline__ XFrag x_frag(const uint32_t (&w)[8], uint32_t c)
{
    half32_t q;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        // byte + 128 in the mantissa of 1024 = 0x6400, less 1152
        const uint32_t b = w[i] ^ 0x80808080u;
        const half2_t k = { (_Float16)1152.f, (_Float16)1152.f };
        const half2_t a = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - k;
        const half2_t d = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - k;
        q[4 * i] = a[0];
        q[4 * i + 1] = a[1];
        q[4 * i + 2] = d[0];
        q[4 * i + 3] = d[1];
    }
    if (__builtin_expect(c < 5u, 0)) {
        q = q * (_Float16)__builtin_amdgcn_ldexpf(1.0f, (int)c - 5);
        c = 5u;
    }
    XFrag f;
    f.hi = __builtin_bit_cast(u32x6, __builtin_amdgcn_cvt_scalef32_pk32_fp6_f16(q, 64.f));
    q = q - __builtin_amdgcn_cvt_scalef32_pk32_f16_fp6(f.hi, 64.f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t o = 0;
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, half2_t{ q[8 * i], q[8 * i + 1] }, 2.f, 0);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, half2_t{ q[8 * i + 2], q[8 * i + 3] }, 2.f, 1);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, half2_t{ q[8 * i + 4], q[8 * i + 5] }, 2.f, 2);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, half2_t{ q[8 * i + 6], q[8 * i + 7] }, 2.f, 3);
        f.lo[i] = (int)o;
    }
    f.sc = c | ((c - 5u) << 8);
    return f;
}

// acc += weights (32 E2M1 codes a lane, scale byte 0 of wsc) . x
__device__ __forceinline__ f32x4 mx_mfma(i32x4 w, uint32_t wsc, const XFrag &x, f32x4 acc)
{
    const i32x8 a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
    const i32x8 h = { (int)x.hi[0], (int)x.hi[1], (int)x.hi[2], (int)x.hi[3], (int)x.hi[4], (int)x.hi[5], 0, 0 };
    const i32x8 l = __builtin_shufflevector(x.lo, x.lo, 0, 1, 2, 3, -1, -1, -1, -1);
    // formats: 4 = E2M1, 2 = E2M3
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, h, acc, 4, 2, 0, (int)wsc, 0, (int)x.sc);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, l, acc, 4, 4, 0, (int)wsc, 1, (int)x.sc);
}

}  // namespace ds3k
