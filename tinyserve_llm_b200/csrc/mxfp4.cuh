// Microscaled 4-bit floating point.  A row of K numbers is cut into blocks of 32; a block has one scale, the power of two
// 2^(s - 127) held in the byte s (255: the block is NaN), and 32 codes of four bits: sign, two bits of exponent, one of mantissa,
// which stand for 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Two codes a byte, the lower four bits the earlier one: a block is 16 bytes of codes,
// a row's codes are its blocks one behind the other, and its scales lie in a matrix of their own whose rows start 16-byte aligned.
#pragma once

#include "common.cuh"

constexpr int MX_BLOCK = 32;
constexpr int MX_MOST = 0x3fffffff;              // columns of a matrix, rows of a product: counted in 32 bits, with room for a block or a doubling

// 2^(s - 127) as float32; NaN for s = 255.
__device__ __forceinline__ float mx_scale(uint32_t s) {
    return s == 0 ? __uint_as_float(0x00400000u) : s == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(s << 23);
}

// Eight codes as bfloat16 numbers.  The exponent and mantissa bits of a code, put at the low end of a bfloat16's exponent and the high
// end of its mantissa, are a bfloat16 that is the code's value times 2^-126 (code 1 becomes a subnormal, as it is in four bits), so one
// multiplication by 2^126 times the block's scale makes the number, exactly: a mask and shifts instead of a table.  p[i] holds codes i
// (low half) and i + 4 (high half): one shift serves both halves.
__device__ __forceinline__ void mx_spread(uint32_t w, uint32_t (&p)[4]) {
    constexpr uint32_t SIGN = 0x80008000u, REST = 0x01c001c0u;
    p[0] = ((w << 12) & SIGN) | ((w << 6) & REST);
    p[1] = ((w << 8) & SIGN) | ((w << 2) & REST);
    p[2] = ((w << 4) & SIGN) | ((w >> 2) & REST);
    p[3] = (w & SIGN) | ((w >> 6) & REST);
}

// The same with neighbours together, p[i] = codes 2 i (low half) and 2 i + 1: a byte times a number of two bits lands in both halves at once.
// Products run on another pipe than shifts and masks, whose 16 lanes a cycle bound whoever spreads codes.
__device__ __forceinline__ void mx_spread_neighbours(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = __byte_perm(w, 0, 0x4440 | i);
        p[i] = ((b * 0x01001000u) & 0x80008000u) | ((b * 0x00040040u) & 0x01c001c0u);
    }
}

// The multiplication takes a factor that a bfloat16 can hold: 2^(s - 1) up to s = 128 (scales up to 2), beyond that 2^127 times `more`.
struct MxFactor {
    uint32_t first, more;       // both halves alike
};
__device__ __forceinline__ uint32_t mx_factor(uint32_t s) {                  // s <= 128
    return s * 0x00800080u + 0x3f003f00u;                                     // exponent field s + 126
}
__device__ __forceinline__ bool mx_large(uint32_t s) { return s > 128; }
__device__ __forceinline__ MxFactor mx_factor_large(uint32_t s) {
    if (s <= 128) return MxFactor{mx_factor(s), 0x3f803f80u};
    // 2^(s - 128): exponent field s - 1; 255 is NaN
    return MxFactor{0x7f007f00u, s == 255 ? 0x7fff7fffu : (s - 1) * 0x00800080u};
}
__device__ __forceinline__ uint32_t mx_mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// The codes of two numbers, the first in the lower four bits: the nearest, ties to the even code, magnitudes over 6 to 6.
__device__ __forceinline__ uint32_t mx_codes_of_two(float low, float high) {
    uint32_t d;
    asm("{\n\t.reg .b8 c;\n\tcvt.rn.satfinite.e2m1x2.f32 c, %1, %2;\n\tcvt.u32.u8 %0, c;\n\t}" : "=r"(d) : "f"(high), "f"(low));
    return d;
}
// The value of a code, by the same bits as above in a float32.
__device__ __forceinline__ float mx_code_value(uint32_t code) { return __uint_as_float((code & 8) << 28 | (code & 7) << 22) * 0x1p126f; }
