// Activations kept in 8 bits: 32 channels of a row (the last of a row may be fewer) in units of a power of two 2^e, the least with
// -126 <= e <= 121 in which the largest rounds to at most 127; the byte e + 127 beside them, 255 where a value is not finite (they come back as NaN).
// x / 2^e is exact, so that rounding to the nearest whole number (ties to even) is the only one: half a unit at most, 1/128
// of the group's largest.  (From 127.5 * 2^121 = 3.39e38 on, 128 * 2^121 being no number: 127 units.)  A value of 7 bits and a sign
// times a power of two is exact in BF16.
#pragma once

#include "pairs.cuh"

namespace mgpt {

constexpr int KEPT_GROUP = 32;      // channels that share an exponent
__host__ __device__ constexpr int kept_groups(int C) { return (C + KEPT_GROUP - 1) / KEPT_GROUP; }

// The byte for a group whose largest magnitude has these bits.  (127.5 units and more would round to 128: the carry takes the next power.)
__device__ __forceinline__ uint32_t kept_exponent(uint32_t largest)
{
    const uint32_t e = (largest + 0x10000u) >> 23;
    return largest >= 0x7f800000u ? 255u : min(max(e, 7u), 254u) - 6u;
}
__device__ __forceinline__ float kept_units(uint32_t byte) { return __uint_as_float(byte == 255u ? 0u : (254u - byte) << 23); }     // 2^-e
__device__ __forceinline__ float kept_unit(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fffffffu : byte << 23); }     // 2^e, or NaN

__device__ __forceinline__ float at_most(float v, uint32_t top) { return copysignf(fminf(fabsf(v), __uint_as_float(top)), v); }

// N values of one lane (8 or 4), all of a group in 32 / N neighbouring lanes, which all call it (with zeros beyond the row's end):
// the group's byte, and the values packed.
template <int N> __device__ __forceinline__ uint32_t kept_pack(const F2 (&v)[N / 2], uint32_t (&packed)[N / 4])
{
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        const uint32_t a = __float_as_uint(v[j].lo()) & 0x7fffffffu, b = __float_as_uint(v[j].hi()) & 0x7fffffffu;
        m = max(m, max(a, b));
    }
#pragma unroll
    for (int o = KEPT_GROUP / N / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t byte = kept_exponent(m);
    const uint32_t top = byte == 248u ? 0x7f7e0000u : 0xffffffffu;      // 127 * 2^121
    const F2 units(kept_units(byte)), magic(12582912.0f);       // 1.5 * 2^23: the sum's last byte is the whole number in two's complement
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
        F2 a = fma2(v[2 * j], units, magic), b = fma2(v[2 * j + 1], units, magic);
        if (__builtin_expect(m > top, 0)) {
            a = F2(at_most(v[2 * j].lo(), top), at_most(v[2 * j].hi(), top)) * units + magic;
            b = F2(at_most(v[2 * j + 1].lo(), top), at_most(v[2 * j + 1].hi(), top)) * units + magic;
        }
        const uint32_t lo = __byte_perm(__float_as_uint(a.lo()), __float_as_uint(a.hi()), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(b.lo()), __float_as_uint(b.hi()), 0x0040);
        packed[j] = __byte_perm(lo, hi, 0x5410);
    }
    return byte;
}
// four values of a word
__device__ __forceinline__ void kept_unpack(uint32_t w, F2 unit, F2& a, F2& b)
{
    w ^= 0x80808080u;                                           // q + 128 as the last byte of 2^23 + q + 128
    const F2 off(-8388736.0f);
    a = (F2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7651))) + off) * unit;
    b = (F2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7652)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7653))) + off) * unit;
}

}  // namespace mgpt
