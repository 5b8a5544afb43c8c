// nt_mx4.cuh -- the 4-bit microscaled form (NtMx4Matrix): scales, codes, addresses.
#pragma once

#include "nt_layer_common.cuh"

namespace nt {
namespace mx4 {

constexpr int kTileRows = 128;   // rows of one 512-byte scale tile
constexpr int kTileBytes = 512;  // 128 rows x 4 blocks

__host__ __device__ constexpr int tiles_per_row(int cols, int block) { return (int)(((int64_t)cols + 4 * block - 1) / (4 * block)); }
__host__ __device__ constexpr int64_t row_pitch(int cols) { return ((int64_t)cols + 31) / 32 * 16; }

// Byte of scale tile `tile` of a row of tiles: a row of 2^31 columns has 16 GB of them.
__host__ __device__ constexpr int64_t tile_offset(int tile) { return (int64_t)tile * kTileBytes; }
static_assert(tile_offset(1 << 22) == (int64_t)1 << 31, "no 32-bit product");

// Byte of the scale of row r, block k.
__device__ __forceinline__ int64_t scale_at(int64_t r, int k, int tiles)
{
    return ((r >> 7) * tiles + (k >> 2)) * kTileBytes + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (k & 3);
}

// Largest magnitude of a block (as the bits of a non-negative fp32) -> scale byte.
template <int BLOCK>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits)
{
    if (BLOCK == 32) {
        const int e = (int)(amax_bits >> 23);  // floor(log2) + 127; 255: NaN or infinity
        return e == 255 ? 0xffu : (uint32_t)max(e - 2, 0);
    }
    if (amax_bits >= 0x7f800000u) return 0x7fu;
    const float s = __fdiv_rn(__uint_as_float(amax_bits), 6.f);
    uint16_t pair;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(0.f), "f"(s));
    return pair & 0xffu;
}

template <int BLOCK>
__device__ __forceinline__ float scale_value(uint32_t byte)
{
    if (BLOCK == 32) {
        if (byte == 0xffu) return __uint_as_float(0x7fffffffu);
        return __uint_as_float(byte ? byte << 23 : 0x00400000u);  // 2^-127 is subnormal
    }
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)byte));
    return __half2float(__ushort_as_half((unsigned short)(h2 & 0xffffu)));
}

// Eight codes from eight scaled values, value i in nibble i: nearest, ties to even, at most 6.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8])
{
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// The values of eight codes, in pairs of fp16 (every E2M1 value is exact).
__device__ __forceinline__ void values8(uint32_t codes, uint32_t (&h2)[4])
{
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h2[0]), "=r"(h2[1]), "=r"(h2[2]), "=r"(h2[3])
        : "r"(codes));
}

// What a value is multiplied by before rounding to a code, given its block's scale.  Block 32: the
// scale is a power of two, so the product is exact (it only loses digits far below the smallest
// code).  Block 16: see `scaled`.
template <int BLOCK>
__device__ __forceinline__ float inverse_scale(uint32_t byte)
{
    if (BLOCK == 32) return __uint_as_float((254u - byte) << 23);  // byte 0xff is handled by the NaN scale
    const float s = scale_value<16>(byte);
    return s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
}

// x / s of two values, near enough to round to the code of the exact quotient.  A code changes at quotients
// t = 1/4 .. 5, and there t * s is exact in 7 bits.
//  - 16-bit x: x has at most 11 bits, so |x| is t * s or at least 2^-11 of it away.  x times the
//    rounded 1 / s is within 2^-22 of the quotient: rounding it to a multiple of 2^-16 (adding and
//    subtracting 192) makes ties exact again and moves no other quotient across its t.
//  - fp32 x (`kExact`): x can be one rounding step beside t * s.  The quotient is corrected once with its
//    remainder x - q s (exact: s has 4 bits), truncated by the sign of the new remainder, and its last bit set
//    when that is not zero: enough to order it against t.
template <int BLOCK, bool kExact>
__device__ __forceinline__ float2 scaled2(float2 x, float inv, float s)
{
    const float2 i2 = make_float2(inv, inv);
    if (BLOCK == 32) return __fmul2_rn(x, i2);
    if (!kExact) {
        const float2 q = __fadd2_rn(__ffma2_rn(x, i2, make_float2(192.f, 192.f)), make_float2(-192.f, -192.f));
        return make_float2(copysignf(q.x, x.x), copysignf(q.y, x.y));
    }
    const float2 a = make_float2(fabsf(x.x), fabsf(x.y)), n = make_float2(-s, -s);
    float2 q = __fmul2_rn(a, i2);
    q = __ffma2_rn(__ffma2_rn(q, n, a), i2, q);
    const float2 r = __ffma2_rn(q, n, a);
    const int lo = __float_as_int(q.x) + (__float_as_int(r.x) >> 31) | (r.x != 0.f);
    const int hi = __float_as_int(q.y) + (__float_as_int(r.y) >> 31) | (r.y != 0.f);
    return make_float2(copysignf(__int_as_float(lo), x.x), copysignf(__int_as_float(hi), x.y));
}

}  // namespace mx4
}  // namespace nt
