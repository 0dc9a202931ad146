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
//   q = 8 hi + lo,  hi = floor((q + 4) / 8),  -4 <= lo <= 3
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
typedef int i32x6 __attribute__((ext_vector_type(6)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef uint32_t u32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32_any __attribute__((aligned(1)));     // at any address
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
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

// 32 bytes of a row of x with their scale byte, as loaded.
struct RawBlock {
    uint32_t w[8], sc;
};

__device__ __forceinline__ RawBlock raw_block(const uint8_t *xc, const uint8_t *xs, int b)
{
    RawBlock q;
    const uint4 x0 = *(const uint4 *)(xc + (int64_t)b * 32), x1 = *(const uint4 *)(xc + (int64_t)b * 32 + 16);
    q.w[0] = x0.x; q.w[1] = x0.y; q.w[2] = x0.z; q.w[3] = x0.w;
    q.w[4] = x1.x; q.w[5] = x1.y; q.w[6] = x1.z; q.w[7] = x1.w;
    q.sc = xs[b];
    return q;
}

// The digits of 32 signed bytes; `in` false: of zeros.  With b = q + 128 the
// digits are hi = floor((b + 4) / 8) - 16 and lo = (b + 4) % 8 - 4.  b is put in
// the mantissa of 1024 = 0x6400: 8 (hi + 16) is it with 4 added and the low bits
// cleared, so that one conversion finds hi with nothing to round, and lo's code
// is looked up by the low three bits, four at a time.  (By the way of hi rounded
// and subtracted again it took one more conversion of 90 cycles and 16 of 10.)
//
// lo's scale byte is 5 less than hi's, so a block with a byte below 5 (values
// under 2^-121) is first taken to the nearest multiples of 2^-128, what its bytes
// stand for with scale byte 5: 1024 + b' = (1024 + b) s + 1152 (1 - s), rounded
// once, as f16 holds 1152 (1 - s) for every s = 2^0 .. 2^-5 and 0.  Without a
// branch: one in the loop of k_mx_few keeps the loads behind it from being issued
// early (37 tokens in 8 of 128 experts each: 78 us with it, 48 without).
__device__ __forceinline__ XFrag x_frag(const RawBlock &raw, bool in)
{
    const uint32_t s1 = in ? 0x3c00u - (uint32_t)(5 - min((int)raw.sc, 5)) * 0x400u : 0u;
    const half2_t s = __builtin_bit_cast(half2_t, s1 * 0x10001u);
    const half2_t m = { (_Float16)1152.f, (_Float16)1152.f }, k = m - m * s;
    u32x16 q;
    uint32_t n[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t b = raw.w[i] ^ 0x80808080u;
        const uint32_t u0 = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
        const uint32_t v0 = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
        const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2_t, u0), s, k));
        const uint32_t v = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2_t, v0), s, k));
        const uint32_t u8 = (u + 0x00040004u) & 0xfff8fff8u, v8 = (v + 0x00040004u) & 0xfff8fff8u;
        const half2_t a = __builtin_bit_cast(half2_t, u8) - m, d = __builtin_bit_cast(half2_t, v8) - m;
        q[2 * i] = __builtin_bit_cast(uint32_t, a);
        q[2 * i + 1] = __builtin_bit_cast(uint32_t, d);
        // 0, 1, 2, 3, -4, -3, -2, -1 for the low bits 0 .. 7
        const uint32_t c = __builtin_amdgcn_perm(0x090a0b0cu, 0x03020100u,
                                                 __builtin_amdgcn_perm(v, u, 0x06040200u) & 0x07070707u);
        n[i] = c | (c >> 4);
    }
    const uint32_t sc = in ? max(raw.sc, 5u) : 127u;
    XFrag f;
    f.hi = __builtin_bit_cast(u32x6, __builtin_amdgcn_cvt_scalef32_pk32_fp6_f16(__builtin_bit_cast(half32_t, q), 64.f));
#pragma unroll
    for (int i = 0; i < 4; i++) f.lo[i] = (int)__builtin_amdgcn_perm(n[2 * i + 1], n[2 * i], 0x06040200u);
    f.sc = sc | ((sc - 5u) << 8);
    return f;
}

// Lane `from`'s.
__device__ __forceinline__ XFrag frag_from(const XFrag &x, int from)
{
    XFrag f;
#pragma unroll
    for (int i = 0; i < 6; i++) f.hi[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * from, (int)x.hi[i]);
#pragma unroll
    for (int i = 0; i < 4; i++) f.lo[i] = __builtin_amdgcn_ds_bpermute(4 * from, x.lo[i]);
    f.sc = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * from, (int)x.sc);
    return f;
}

// acc += weights (32 E2M1 codes a lane, scale byte S of wsc) . x, in two parts.
// The second waits for the first's sum, so several of the first go before.
template <int S>
__device__ __forceinline__ f32x4 mx_mfma_hi(i32x4 w, uint32_t wsc, const XFrag &x, f32x4 acc)
{
    const i32x8 a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
    const i32x6 t = __builtin_bit_cast(i32x6, x.hi);
    const i32x8 h = __builtin_shufflevector(t, t, 0, 1, 2, 3, 4, 5, -1, -1);
    // formats: 4 = E2M1, 2 = E2M3
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, h, acc, 4, 2, S, (int)wsc, 0, (int)x.sc);
}

template <int S>
__device__ __forceinline__ f32x4 mx_mfma_lo(i32x4 w, uint32_t wsc, const XFrag &x, f32x4 acc)
{
    const i32x8 a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
    const i32x8 l = __builtin_shufflevector(x.lo, x.lo, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, l, acc, 4, 4, S, (int)wsc, 1, (int)x.sc);
}

// ---------------------------------------------------------------------------
// From memory to the operands' places
//
// A load is fast when four neighbouring lanes read 64 bytes in a row, and
// fastest on whole lines: 16 rows x 64 bytes with neighbouring lanes on
// neighbouring rows reach 15 B/clk a CU from L2, 4 rows x 256 bytes 52.  An
// operand wants neighbouring lanes on neighbouring rows.  So 16 rows of a chunk
// of 16 blocks (512 columns) are loaded as four times 4 rows x 16 blocks: in
// load j, lane 16 g + 4 R + p takes block 4 g + p of row 4 R + j, and a 4 x 4
// transposition among the four lanes of a quad (two exchanges between
// neighbouring lanes, one instruction a register each) leaves lane 16 g + r
// with the blocks 4 g + 0..3 of row r.  Step k of a chunk thus multiplies the
// blocks 4 g + k, and the scale bytes of a lane's four steps are one dword.
// ---------------------------------------------------------------------------
constexpr int CHUNK_BLOCKS = 16;

template <int XOR>
__device__ __forceinline__ int quad_xor(int v)
{
    return __builtin_amdgcn_mov_dpp(v, XOR == 1 ? 0xb1 : 0x4e, 0xf, 0xf, true);
}

// v[j] of lane p of each quad <-> v[p] of lane j: an exchange and a choice a
// register and stage.
__device__ __forceinline__ void quad_transpose(int (&v)[4])
{
    const bool b0 = threadIdx.x & 1, b1 = threadIdx.x & 2;
    // every exchange before the choices: under a branch it would miss the other lanes
    const int x0 = quad_xor<1>(v[0]), x1 = quad_xor<1>(v[1]), x2 = quad_xor<1>(v[2]), x3 = quad_xor<1>(v[3]);
    const int a0 = b0 ? x1 : v[0], a1 = b0 ? v[1] : x0, a2 = b0 ? x3 : v[2], a3 = b0 ? v[3] : x2;
    const int y0 = quad_xor<2>(a0), y1 = quad_xor<2>(a1), y2 = quad_xor<2>(a2), y3 = quad_xor<2>(a3);
    v[0] = b1 ? y2 : a0;
    v[2] = b1 ? a2 : y0;
    v[1] = b1 ? y3 : a1;
    v[3] = b1 ? a3 : y1;
}

__device__ __forceinline__ void quad_transpose(i32x4 (&v)[4])
{
#pragma unroll
    for (int d = 0; d < 4; d++) {
        int t[4] = { v[0][d], v[1][d], v[2][d], v[3][d] };
        quad_transpose(t);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j][d] = t[j];
    }
}

// The same beside matrix products: v_cndmask_b32 takes its exchange as a DPP
// operand, half the instructions, but its mask from VCC.  Where the SIMD's other wave
// and the matrix cores have work meanwhile, the instructions count (16384 rows in 128
// groups of 768 x 2 outputs: 120.2 us, 125.6 as above; 2048 x 4096, K = 2048: 32.7,
// 34.6); where a SIMD has one wave, the waits for VCC do (512 x 4096: 16.1, 15.0), and
// the transposition above serves.
//
// The masks are constants that scalar instructions write: a vector instruction may
// read a VCC that a scalar one wrote in the very next place, one that a comparison
// wrote two places later (such waits in place of them: 16.5, 121.8).  The compiler does
// not look inside, so the block keeps the distances itself: two places from a vector
// write to a DPP read of it and three from a product that reads a register as its sum to
// the register's next write (before the block by s_nop and two s_mov, inside by four
// selections), two from its last write to a product that reads it (products of other
// weights or the next turn's first loads).
__device__ __forceinline__ void quad_transpose_beside(i32x4 (&v)[4])
{
#define QUAD_XOR1 " quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf bound_ctrl:0\n"
#define QUAD_XOR2 " quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf bound_ctrl:0\n"
#pragma unroll
    for (int d = 0; d < 4; d += 2) {
        int s0, s1, s2, s3, t0, t1, t2, t3;              // after the first exchange
        int o0, o1, o2, o3, q0, q1, q2, q3;
        asm("s_nop 0\n"
            "s_mov_b32 vcc_lo, 0x55555555\n"            // the even lanes
            "s_mov_b32 vcc_hi, 0x55555555\n"
            "v_cndmask_b32_dpp %[s0], %[a1], %[a0], vcc" QUAD_XOR1
            "v_cndmask_b32_dpp %[s2], %[a3], %[a2], vcc" QUAD_XOR1
            "v_cndmask_b32_dpp %[t0], %[c1], %[c0], vcc" QUAD_XOR1
            "v_cndmask_b32_dpp %[t2], %[c3], %[c2], vcc" QUAD_XOR1
            "s_not_b64 vcc, vcc\n"
            "v_cndmask_b32_dpp %[s1], %[a0], %[a1], vcc" QUAD_XOR1
            "v_cndmask_b32_dpp %[s3], %[a2], %[a3], vcc" QUAD_XOR1
            "v_cndmask_b32_dpp %[t1], %[c0], %[c1], vcc" QUAD_XOR1
            "v_cndmask_b32_dpp %[t3], %[c2], %[c3], vcc" QUAD_XOR1
            "s_mov_b32 vcc_lo, 0x33333333\n"            // the first two of each quad
            "s_mov_b32 vcc_hi, 0x33333333\n"
            "v_cndmask_b32_dpp %[o0], %[s2], %[s0], vcc" QUAD_XOR2
            "v_cndmask_b32_dpp %[o1], %[s3], %[s1], vcc" QUAD_XOR2
            "v_cndmask_b32_dpp %[q0], %[t2], %[t0], vcc" QUAD_XOR2
            "v_cndmask_b32_dpp %[q1], %[t3], %[t1], vcc" QUAD_XOR2
            "s_not_b64 vcc, vcc\n"
            "v_cndmask_b32_dpp %[o2], %[s0], %[s2], vcc" QUAD_XOR2
            "v_cndmask_b32_dpp %[o3], %[s1], %[s3], vcc" QUAD_XOR2
            "v_cndmask_b32_dpp %[q2], %[t0], %[t2], vcc" QUAD_XOR2
            "v_cndmask_b32_dpp %[q3], %[t1], %[t3], vcc" QUAD_XOR2
            : [s0] "=&v"(s0), [s1] "=&v"(s1), [s2] "=&v"(s2), [s3] "=&v"(s3), [t0] "=&v"(t0), [t1] "=&v"(t1),
              [t2] "=&v"(t2), [t3] "=&v"(t3), [o0] "=&v"(o0), [o1] "=&v"(o1), [o2] "=&v"(o2), [o3] "=&v"(o3),
              [q0] "=&v"(q0), [q1] "=&v"(q1), [q2] "=&v"(q2), [q3] "=&v"(q3)
            : [a0] "v"(v[0][d]), [a1] "v"(v[1][d]), [a2] "v"(v[2][d]), [a3] "v"(v[3][d]), [c0] "v"(v[0][d + 1]),
              [c1] "v"(v[1][d + 1]), [c2] "v"(v[2][d + 1]), [c3] "v"(v[3][d + 1])
            : "vcc", "scc");
        v[0][d] = o0, v[1][d] = o1, v[2][d] = o2, v[3][d] = o3;
        v[0][d + 1] = q0, v[1][d + 1] = q1, v[2][d + 1] = q2, v[3][d + 1] = q3;
    }
#undef QUAD_XOR1
#undef QUAD_XOR2
}

// The scale dwords of 16 rows are loaded with lane 4 r + g on dword g of row r;
// one pass through the LDS crossbar takes them to lane 16 g + r.
__device__ __forceinline__ uint32_t scales_to_place(uint32_t v)
{
    const int lane = threadIdx.x & (WAVE - 1);
    return (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (4 * (lane & 15) + (lane >> 4)), (int)v);
}

// 127 in the bytes of blocks b .. b + 3 that are nb or more.
__device__ __forceinline__ uint32_t scales_within(uint32_t v, int b, int nb)
{
    const int n = min(max(nb - b, 0), 4);
    const uint32_t m = n == 4 ? ~0u : (1u << (8 * n)) - 1u;
    return (v & m) | (0x7f7f7f7fu & ~m);
}

}  // namespace ds3k
