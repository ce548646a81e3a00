// The 8-bit key/value cache, as every kernel that touches it sees it.
//
// A row is the key (or value) of one position and one key/value head: hd numbers of type e4m3 (4 exponent bits, 3 of
// mantissa, largest 448, no infinity) times one power of two 2^e.  Pages of 64 positions:
//   codes      [pages, nkv, 64, hd]      keys; the same of values
//   exponents  [pages, nkv, 2, 64]       bytes e + 127: of the 64 keys, then of the 64 values
// e is the smallest whole number from KV8_LOWEST on for which the row's largest magnitude is at most 448 * 2^e.  A power of
// two takes nothing from a floating format but a part of a bit of its range, scaling by it is exact, and a code times
// 2^e is a bfloat16 number, so a kernel may work on codes and exponents or on bfloat16 and means the same.
// A row that holds a NaN, an infinity or a magnitude above 448 * 2^KV8_HIGHEST is stored as codes 0 and the byte KV8_NAN:
// whoever sees such a position gets NaN, whoever's mask hides it gets nothing of it.
// Where a sequence's table names no page, attention gives the page's keys no weight (a row without keys is zeros) and the status says so.
#pragma once
#include "common.cuh"

constexpr int KV8_PAGE = 64, KV8_LOWEST = -100, KV8_HIGHEST = 100, KV8_NAN = 255;

// (a, b) -> two e4m3 codes, a in the low byte; to nearest, ties to even
__device__ __forceinline__ unsigned kv8_pack2(float a, float b) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
// two e4m3 codes (the low byte first) as two halfs: exact
__device__ __forceinline__ unsigned kv8_half2(unsigned short two) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"(two));
    return r;
}
// 2^e, e in -126 .. 127
__device__ __forceinline__ float kv8_pow2(int e) { return __int_as_float((e + 127) << 23); }

// The exponent byte of a row whose largest magnitude is ``amax`` (all of its numbers finite): amax = (1 + f) 2^x is at most
// 448 * 2^e = 1.75 * 2^(8 + e) iff e >= x - 8, or x - 7 where 1 + f > 1.75.  KV8_NAN beyond the highest exponent.
__device__ __forceinline__ int kv8_exponent_byte(float amax) {
    const unsigned bits = __float_as_uint(amax);
    const int e = max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), KV8_LOWEST);
    return e > KV8_HIGHEST ? KV8_NAN : e + 127;
}
