// The 8-bit cache: what a page holds and how its numbers are made and read.
//
// A page [2, kv_heads, page_size, head_dim + 1] of bytes holds, per part (keys, values) and kv head, a block of
// page_size rows of head_dim codes and behind them one scale byte per row. A code is an 8-bit float (e4m3: sign, four bits
// of exponent, three of fraction, largest magnitude 448, one NaN per sign); scale byte b stands for 2^(b - 127). The scale of
// a row is the smallest power of two that brings its largest finite magnitude to 448 or below. A power of two costs a
// floating code nothing against a 32-bit scale, and makes every number read back one that bfloat16 holds exactly.
// Page sizes and head sizes are multiples of 16, so that rows, blocks and the scales of 16 keys start on 16 bytes.
#pragma once
#include "common.cuh"

#define C8_LOW -64                    // the least exponent of a scale: rows whose largest magnitude is below 2^-55 lose bits
#define C8_HIGH 120

// The exponent of the scale of a row whose largest finite magnitude is `largest`.
__device__ __forceinline__ int c8_exponent(float largest) {
    const uint32_t bits = __float_as_uint(largest);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);      // 448 = 1.75 * 2^8
    return min(max(e, C8_LOW), C8_HIGH);
}
// |x| for the largest magnitude of a row: numbers that are not finite do not count.
__device__ __forceinline__ float c8_magnitude(float x) {
    const float a = fabsf(x);
    return a <= 3.4028234663852886e38f ? a : 0.f;
}
__device__ __forceinline__ float c8_power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Codes of a (low byte) and b, already divided by their scale; NaN stays NaN. c8_pack2: infinities become NaN, too.
__device__ __forceinline__ uint32_t c8_pack2_finite(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t c8_pack4_finite(float a, float b, float c, float d) { return c8_pack2_finite(a, b) | c8_pack2_finite(c, d) << 16; }
__device__ __forceinline__ uint32_t c8_pack2(float a, float b) {
    if (fabsf(a) == INFINITY) a = __uint_as_float(0x7fc00000u);
    if (fabsf(b) == INFINITY) b = __uint_as_float(0x7fc00000u);
    return c8_pack2_finite(a, b);
}
__device__ __forceinline__ uint32_t c8_pack4(float a, float b, float c, float d) { return c8_pack2(a, b) | c8_pack2(c, d) << 16; }

// Two codes (the low 16 bits) as two halves; every code is a half exactly.
__device__ __forceinline__ uint32_t c8_halves(uint32_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"((uint16_t)codes));
    return r;
}
// Two codes times a power of two as a pair of bfloat16 (exact: four significant bits).
__device__ __forceinline__ uint32_t c8_bf16x2(uint32_t codes, float scale) {
    const uint32_t h = c8_halves(codes);
    float lo, hi;
    asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}\n" : "=f"(lo), "=f"(hi) : "r"(h));
    __nv_bfloat162 p = __floats2bfloat162_rn(lo * scale, hi * scale);
    return *(uint32_t*)&p;
}
// Sixteen codes as sixteen bfloat16.
__device__ __forceinline__ void c8_unpack16(const uint4& codes, float scale, uint4& a, uint4& b) {
    a.x = c8_bf16x2(codes.x, scale); a.y = c8_bf16x2(codes.x >> 16, scale);
    a.z = c8_bf16x2(codes.y, scale); a.w = c8_bf16x2(codes.y >> 16, scale);
    b.x = c8_bf16x2(codes.z, scale); b.y = c8_bf16x2(codes.z >> 16, scale);
    b.z = c8_bf16x2(codes.w, scale); b.w = c8_bf16x2(codes.w >> 16, scale);
}
