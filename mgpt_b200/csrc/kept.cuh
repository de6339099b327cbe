// Activations kept in 8 bits: 32 channels of a row (the last of a row may be fewer) in units of a power of two 2^e, the least with
// -126 <= e <= 121 in which the largest rounds to at most 127; the byte e + 127 beside them, 255 where a value is not finite (they come back as NaN).
// x / 2^e is exact, so that rounding to the nearest whole number (ties to even) is the only one: half a unit at most, which is 1/127
// of the group's largest where that is 2^-120 or more; below, the unit stays 2^-126 (2^-127 and less comes back as 0).  (From
// 127.5 * 2^121 = 3.39e38 on, 128 * 2^121 being no number: 127 units, up to a whole one off.)  A value of 7 bits and a sign times a power of
// two is exact in BF16.
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
__device__ __forceinline__ float kept_unit(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fffffffu : byte << 23); }     // 2^e, or NaN
__device__ __forceinline__ float at_most(float v, uint32_t top) { return copysignf(fminf(fabsf(v), __uint_as_float(top)), v); }

// The larger of two magnitudes (NaN: that), BF16: of two pairs of them.
__device__ __forceinline__ uint32_t kept_larger(uint32_t a, uint32_t b, bf16)
{
    uint32_t c;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    return c;
}
__device__ __forceinline__ uint32_t kept_larger(uint32_t a, uint32_t b, float) { return max(a, b); }
// of 16 bytes, as they lie in registers
template <typename T> __device__ __forceinline__ uint32_t kept_largest(const uint4& u)
{
    constexpr uint32_t M = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
    return kept_larger(kept_larger(u.x & M, u.y & M, T()), kept_larger(u.z & M, u.w & M, T()), T());
}
template <typename T> __device__ __forceinline__ uint32_t kept_largest_of_lanes(uint32_t m)
{
#pragma unroll
    for (int o = KEPT_GROUP * (int)sizeof(T) / 32; o > 0; o >>= 1) m = kept_larger(m, __shfl_xor_sync(0xffffffffu, m, o), T());
    return m;
}

// 16 bytes of T in the units of a group whose largest magnitude has the bits m: the group's byte, and the values packed.
template <typename T> __device__ __forceinline__ uint32_t kept_round(uint32_t m, const F2 (&v)[8 / sizeof(T)], uint32_t (&packed)[4 / sizeof(T)])
{
    uint32_t e = max((m + 0x10000u) >> 23, 7u);                     // 6 more than the byte, but for the largest numbers
    F2 units(__uint_as_float((260u - e) << 23)), magic(12582912.0f);       // 2^-e; 1.5 * 2^23: a sum's last byte is the whole number in two's complement
    F2 a[8 / sizeof(T)];
#pragma unroll
    for (int j = 0; j < 8 / (int)sizeof(T); ++j) a[j] = fma2(v[j], units, magic);
    if (__builtin_expect(m >= 0x7f7f0000u, 0)) {
        e = kept_exponent(m) + 6u;
        if (e == 254u) units = F2(0x1p-121f);
#pragma unroll
        for (int j = 0; j < 8 / (int)sizeof(T); ++j) a[j] = F2(at_most(v[j].lo(), 0x7f7e0000u), at_most(v[j].hi(), 0x7f7e0000u)) * units + magic;      // 127 * 2^121
    }
#pragma unroll
    for (int j = 0; j < 4 / (int)sizeof(T); ++j) {
        const uint32_t lo = __byte_perm(__float_as_uint(a[2 * j].lo()), __float_as_uint(a[2 * j].hi()), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(a[2 * j + 1].lo()), __float_as_uint(a[2 * j + 1].hi()), 0x0040);
        packed[j] = __byte_perm(lo, hi, 0x5410);
    }
    return e - 6u;
}
// 16 bytes of one lane (u, and as numbers v), all of a group in neighbouring lanes, which all call it (with zeros beyond the row's end).
template <typename T> __device__ __forceinline__ uint32_t kept_pack(const uint4& u, const F2 (&v)[8 / sizeof(T)], uint32_t (&packed)[4 / sizeof(T)])
{
    const uint32_t m = kept_largest_of_lanes<T>(kept_largest<T>(u));
    return kept_round<T>(sizeof(T) == 2 ? max(m & 0xffff0000u, m << 16) : m, v, packed);
}
// Two of them, whose groups are not one.  (BF16: both maxima in a word.)
template <typename T>
__device__ __forceinline__ void kept_pack_two(const uint4& u, const F2 (&v)[8 / sizeof(T)], const uint4& u2, const F2 (&v2)[8 / sizeof(T)],
                                              uint32_t (&packed)[4 / sizeof(T)], uint32_t (&packed2)[4 / sizeof(T)], uint32_t& byte, uint32_t& byte2)
{
    uint32_t m = kept_largest<T>(u), m2 = kept_largest<T>(u2);
    if constexpr (sizeof(T) == 2) {
        m = kept_largest_of_lanes<T>(kept_larger(__byte_perm(m, m2, 0x5410), __byte_perm(m, m2, 0x7632), T()));
        m2 = m & 0xffff0000u;
        m <<= 16;
    } else {
        m = kept_largest_of_lanes<T>(m);
        m2 = kept_largest_of_lanes<T>(m2);
    }
    byte = kept_round<T>(m, v, packed);
    byte2 = kept_round<T>(m2, v2, packed2);
}
// the four whole numbers of a word
__device__ __forceinline__ void kept_unpack(uint32_t w, F2& a, F2& b)
{
    w ^= 0x80808080u;                                           // q + 128 as the last byte of 2^23 + q + 128
    const F2 off(-8388736.0f);
    a = F2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7651))) + off;
    b = F2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7652)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7653))) + off;
}

}  // namespace mgpt
