// Two FP32 operations per instruction, on values that lie side by side, and copies that run beside the arithmetic.
#pragma once

#include "common.cuh"

namespace mgpt {

// Each half is rounded as the operation alone would round it.  (A product and a sum of two F2 are compiled to one operation
// with one rounding; where that matters the sum is written as fma2(product, 1, x) with a 1 that the compiler does not know.)
struct F2 {
    uint64_t r;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit F2(float a) : F2(a, a) {}
    __device__ __forceinline__ float lo() const { float a, b; get(a, b); return a; }
    __device__ __forceinline__ float hi() const { float a, b; get(a, b); return b; }
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
};
__device__ __forceinline__ F2 operator+(F2 a, F2 b) { F2 c; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.r) : "l"(a.r), "l"(b.r)); return c; }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) { F2 c; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.r) : "l"(a.r), "l"(b.r)); return c; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 d) { F2 c; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(c.r) : "l"(a.r), "l"(b.r), "l"(d.r)); return c; }
// the two bf16 of a word, and back
__device__ __forceinline__ F2 widen(uint32_t w) { return F2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t narrow(F2 v)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.lo(), v.hi());
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Asynchronous copies to shared memory (addresses of the shared space), in groups.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy8(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
// the first `bytes` (0 to 4) of a word, zeros behind them
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, uint32_t bytes) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory"); }
template <int BYTES> __device__ __forceinline__ void copy_piece8(uint32_t dst, const void* src)
{
    static_assert(BYTES == 8 || BYTES == 4, "");
    if constexpr (BYTES == 8) copy8(dst, src);
    else copy4(dst, src);
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }
template <typename T> __device__ __forceinline__ T taken(uint32_t src)
{
    static_assert(sizeof(T) == 16 || sizeof(T) == 8 || sizeof(T) == 4, "");
    T v;
    uint32_t* o = reinterpret_cast<uint32_t*>(&v);
    if constexpr (sizeof(T) == 16) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(src) : "memory");
    else if constexpr (sizeof(T) == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(o[0]), "=r"(o[1]) : "r"(src) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(o[0]) : "r"(src) : "memory");
    return v;
}

}  // namespace mgpt
