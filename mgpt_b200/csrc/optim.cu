// AdamW over many tensors in one launch, with moments in 32 or in 8 bits.
//
//   m' = b1 m + (1-b1) g,   v' = b2 v + (1-b2) g g
//   w' = w - lr wd w - lr (m' / (1-b1^t)) / (sqrt(v' / (1-b2^t)) + eps)
//
// (the reference's, one launch per tensor: optimisers/AdamWOptimiser.h:24-36, utils/Tensor.cpp:683-699.)
//
// Blocks of 256 elements.  Every tensor starts on a block of its own; the blocks of all tensors are numbered through, and the
// moments of block i are elements 256 i .. of the state arrays, which belong to the caller.
//
// 8 bits.  m and s = sqrt(v) are kept as codes with a sign, 4 bits of exponent and 3 of mantissa (E4M3), in units of a power of
// two per block that puts the block's largest value between 128 and 256; the scales are exact, so that a code only ever loses
// mantissa bits.  The root of v has half its range of exponents, and is what the update divides by.  Rounding is stochastic: a step
// moves v by a thousandth (1-b2), a code by an eighth, and to nearest no code would ever move.  The 16 random bits of a value come from
// the finaliser of MurmurHash3 (A. Appleby) over the element's place, the seed and the step: the same call has the same result.
//
// A root that is not zero never becomes zero: below the smallest code, 2^-9 units, it is kept as that.  m and the root are rounded by bits of
// their own, so that an element some 2^17 below its block's largest would now and then keep an m of 2^-9 units and a root of zero, and the
// next update would divide that m by sqrt(1-b2) of its own small gradient: steps of up to 1600 lr where exact moments take 1.1
// (steady gradients of 1 and 1e-5 side by side), now 2.4.  Elements further down take smaller steps than exact moments would: the
// root is at least 2^-17 of the block's largest.
//
// Elsewhere the root of v is within a factor of 0.8 to 1.3 of the exact one for nine elements in ten, and v, the square of what
// is rounded without bias, 4 % too large in the mean.
//
// An element whose new moments are not finite (its gradient is not, or overflows) keeps w, m and v, and sets the caller's flag.
#include <cmath>
#include <cstring>
#include <memory>

#include <cuda_fp8.h>

#include "pairs.cuh"

struct mgpt_moe_optim {
    int device;
    int n_tensors;
    int state_bits;
    long blocks;
    int run, grid;
    void* tables = nullptr;     // device: the tensors
};

namespace mgpt {

namespace {

constexpr int BLOCK = 256;              // elements that share a scale
constexpr int WARPS = 8;

struct OptTensor {
    float* w;
    const void* g;
    bf16* copy;
    long n;
    int block0, block1;                 // its first block, and the one after its last
    float decay;
    int g_bf16;
    int vec;                            // w and the gradient start on 16-byte boundaries, the copy on one of 8: whole blocks go in pieces
};
struct OptP {
    const OptTensor* tensors;           // those with elements, in order
    int n_tensors;
    const int* ends;                    // their block1
    const int* starts;                  // per thread block: the tensor of its first block
    int blocks;                         // of all tensors
    int run;                            // that a thread block takes at a time, a multiple of WARPS
    void *m, *v;
    float *m_scale, *v_scale;
    float b1, b2, omb1, omb2, eps, lr, one;
    float step, rvs;                    // -lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    const float* grad_scale;
    int32_t* found;
    uint32_t key;
};

// the finaliser of MurmurHash3 behind its first line
__host__ __device__ __forceinline__ uint32_t mixed_rest(uint32_t h)
{
    h *= 0x85ebca6bu;
    h ^= h >> 13;
    h *= 0xc2b2ae35u;
    return h ^ (h >> 16);
}
__host__ __device__ __forceinline__ uint32_t mixed(uint32_t h)
{
    return mixed_rest(h ^ (h >> 16));
}
__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float sqrt_fast(float x) { float y; asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp_fast(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// Values of 0 to 256 to 3 bits of mantissa, steps of 2^-9 below 2^-6: 16 random bits are added below the last kept bit, what is
// below it is dropped.
__device__ __forceinline__ F2 rounded(F2 a, uint32_t r0, uint32_t r1)
{
    const float l0 = a.lo() < 0.015625f ? 0.015625f : 0.0f, l1 = a.hi() < 0.015625f ? 0.015625f : 0.0f;
    const F2 b = a + F2(l0, l1);
    const uint32_t q0 = (__float_as_uint(b.lo()) + (r0 << 4)) & 0xfff00000u, q1 = (__float_as_uint(b.hi()) + (r1 << 4)) & 0xfff00000u;
    return F2(__uint_as_float(q0), __uint_as_float(q1)) + F2(-l0, -l1);
}

// The root's smallest code for a root that is not zero.  (2^126: the smallest quotient of a root and its unit is 2^-119.)
__device__ __forceinline__ F2 least_root(F2 s)
{
    const F2 big = s * F2(0x1p126f);
    return F2(fminf(big.lo(), 0x1p-9f), fminf(big.hi(), 0x1p-9f));
}
__device__ __forceinline__ F2 no_less(F2 a, F2 b) { return F2(fmaxf(a.lo(), b.lo()), fmaxf(a.hi(), b.hi())); }

// A thread block takes runs of blocks, its warps every eighth block of a run.  Lane's elements of a block: four from lane * 4, four
// from 128 + lane * 4, so that every access of the warp is one run of memory.  A warp's blocks are copied to shared memory some
// blocks ahead, in pieces of 16 bytes per lane.
//
// Bound by HBM: w, m and v are written where they were read, which this memory takes at 5.7 TB/s at most (the 32-bit form's rate).  With loads
// into registers, one block per warp and two tables to look up before the first load, 24 warps of 66 registers kept 3.2 TB/s going:
// 562 us for 386 tensors of 100 M elements, now 336 (5.4 TB/s).  Copies of 4 bytes per lane (the codes, the scales) cost as much
// as those of 16: 368 us without the scales' against 395.  In 8 bits an element is about 70 instructions for the 14 to 18 bytes
// that it moves, so that moments go two to an instruction, the update takes its root and quotient from the approximating
// instructions (2 ulp of an update that is itself a small part of w) and elements that are not finite are sorted out in a rare pass
// of their own; 268 M elements with BF16 gradients are 860 us, 5.0 TB/s.  Three thread blocks of 80 registers per SM spill: 921.
// m' and v' are rounded operation by operation: the scales hang on their last bits.
template <int BITS> constexpr int stages() { return BITS == 8 ? 4 : 3; }
constexpr uint32_t OFF_G = 1024, OFF_M = 2048;
template <int BITS> constexpr uint32_t off_v() { return OFF_M + BLOCK * BITS / 8; }
template <int BITS> constexpr uint32_t off_scale() { return OFF_M + 2 * BLOCK * BITS / 8; }
template <int BITS> constexpr uint32_t stage_bytes() { return off_scale<BITS>() + (BITS == 8 ? 16 : 0); }
template <int BITS> constexpr uint32_t smem_bytes() { return WARPS * stages<BITS>() * stage_bytes<BITS>(); }

template <int BITS>
__global__ void __launch_bounds__(32 * WARPS, 2) optim_kernel(const OptP p)
{
    constexpr int NS = stages<BITS>();
    extern __shared__ __align__(16) uint8_t ring[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t slots = (uint32_t)__cvta_generic_to_shared(ring) + warp * NS * stage_bytes<BITS>();
    const int b0 = (int)blockIdx.x * p.run, b1 = p.blocks;
    int ahead_left = p.run, left = p.run;
    auto after = [&](int b, int& n) {                               // the warp's block after b
        n -= WARPS;
        if (n > 0) return b + WARPS;
        n = p.run;
        return b + WARPS + (int)(gridDim.x - 1) * p.run;
    };
    pdl_wait();
    const int start = p.starts[blockIdx.x];                         // of the thread block's first block
    // The tensor of the block that is copied next, and of the block that is worked on: pointers as if its block 0 were the first of
    // all, the first block that is not taken in whole pieces (the last one, or all of them), the block after its last.
    int ahead = start, here = start;
    const float* fw;
    const uint8_t* fg;
    int fwhole, fend, fsize;
    auto to_fetch = [&](int i) {
        const OptTensor& t = p.tensors[i];
        fsize = t.g_bf16 ? 2 : 4;
        fw = t.w - (long)t.block0 * BLOCK;
        fg = (const uint8_t*)t.g - (long)t.block0 * BLOCK * fsize;
        fwhole = t.vec ? t.block0 + (int)(t.n / BLOCK) : t.block0;
        fend = t.block1;
    };
    float* tw;
    bf16* tcopy;
    int twhole, tend, tbf16;
    float lrwd;
    auto to_work = [&](int i) {
        const OptTensor& t = p.tensors[i];
        tbf16 = t.g_bf16;
        tw = t.w - (long)t.block0 * BLOCK;
        tcopy = t.copy ? t.copy - (long)t.block0 * BLOCK : nullptr;
        twhole = t.vec ? t.block0 + (int)(t.n / BLOCK) : t.block0;
        tend = t.block1;
        lrwd = p.lr * t.decay;
    };
    // the tensor of block b, at or behind tensor i
    auto find = [&](int b, int i) {
        for (;; i += 32) {
            const uint32_t in = __ballot_sync(0xffffffffu, i + lane >= p.n_tensors || b < p.ends[i + lane]);
            if (in) return i + __ffs(in) - 1;
        }
    };
    if (b0 + warp < b1) {                                           // (a run's first block and most of the others: the tensor is known)
        to_fetch(start);
        if (b0 + warp >= fend) to_fetch(ahead = here = find(b0 + warp, start + 1));
        to_work(here);
    }
    auto fetch = [&](int b, int s) {
        if (b < b1) {
            if (b >= fend) to_fetch(ahead = find(b, ahead + 1));
            const uint32_t d = slots + s * stage_bytes<BITS>();
            const long o = (long)b * BLOCK + lane * 4;
            if (BITS == 8) {
                // 256 bytes of m by half of the lanes, of v by the others; the scales by one lane each
                copy16(d + OFF_M + lane * 16, (const uint8_t*)(lane < 16 ? p.m : p.v) + (long)b * BLOCK + (lane & 15) * 16);
                if (lane < 2) copy4(d + off_scale<BITS>() + lane * 4, (lane ? p.v_scale : p.m_scale) + b);
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    copy16(d + OFF_M + i * 512 + lane * 16, (const float*)p.m + o + i * 128);
                    copy16(d + off_v<BITS>() + i * 512 + lane * 16, (const float*)p.v + o + i * 128);
                }
            }
            if (b < fwhole) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    copy16(d + i * 512 + lane * 16, fw + o + i * 128);
                    if (fsize == 4) copy16(d + OFF_G + i * 512 + lane * 16, fg + (o + i * 128) * 4);
                }
                if (fsize == 2) copy16(d + OFF_G + lane * 16, fg + (long)b * (BLOCK * 2) + lane * 16);
            }
        }
        copy_commit();
    };
    int next = b0 + warp;
#pragma unroll
    for (int s = 0; s < NS - 1; ++s, next = after(next, ahead_left)) fetch(next, s);
    int slot = 0;
    for (int block = b0 + warp; block < b1; block = after(block, left), slot = slot + 1 == NS ? 0 : slot + 1) {
        __syncwarp();                                                   // (every lane has taken what the slot held)
        fetch(next, slot == 0 ? NS - 1 : slot - 1);
        next = after(next, ahead_left);
        copy_wait<NS - 1>();
        __syncwarp();                                                   // the other lanes' copies are there
        if (block >= tend) to_work(here = find(block, here + 1));
        const long at = (long)block * BLOCK + lane * 4;
        const bool whole = block < twhole;
        const uint32_t d = slots + slot * stage_bytes<BITS>();
        F2 w[4], g[4], m[4], v[4];
        uint32_t cm[2], cv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (BITS == 32) {
                const float4 a = taken<float4>(d + OFF_M + i * 512 + lane * 16), b = taken<float4>(d + off_v<BITS>() + i * 512 + lane * 16);
                m[2 * i] = F2(a.x, a.y); m[2 * i + 1] = F2(a.z, a.w);
                v[2 * i] = F2(b.x, b.y); v[2 * i + 1] = F2(b.z, b.w);
            } else {
                cm[i] = taken<uint32_t>(d + OFF_M + i * 128 + lane * 4);
                cv[i] = taken<uint32_t>(d + off_v<BITS>() + i * 128 + lane * 4);
            }
            if (whole) {
                const float4 a = taken<float4>(d + i * 512 + lane * 16);
                w[2 * i] = F2(a.x, a.y); w[2 * i + 1] = F2(a.z, a.w);
                if (tbf16) {
                    const uint2 b = taken<uint2>(d + OFF_G + i * 256 + lane * 8);
                    g[2 * i] = F2(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u));
                    g[2 * i + 1] = F2(__uint_as_float(b.y << 16), __uint_as_float(b.y & 0xffff0000u));
                } else {
                    const float4 b = taken<float4>(d + OFF_G + i * 512 + lane * 16);
                    g[2 * i] = F2(b.x, b.y); g[2 * i + 1] = F2(b.z, b.w);
                }
            } else {
                const OptTensor& t = p.tensors[here];
                const long e = at + i * 128 - (long)t.block0 * BLOCK;
                float wi[4], gi[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool in = e + j < t.n;
                    wi[j] = in ? t.w[e + j] : 0.0f;
                    gi[j] = in ? t.g_bf16 ? __bfloat162float(((const bf16*)t.g)[e + j]) : ((const float*)t.g)[e + j] : 0.0f;
                }
                w[2 * i] = F2(wi[0], wi[1]); w[2 * i + 1] = F2(wi[2], wi[3]);
                g[2 * i] = F2(gi[0], gi[1]); g[2 * i + 1] = F2(gi[2], gi[3]);
            }
        }
        if (BITS == 8) {
            const float sm = taken<float>(d + off_scale<BITS>()), sv = taken<float>(d + off_scale<BITS>() + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(cm[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
                const __half2_raw y = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(cv[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
                const float2 fx = __half22float2(__half2(x)), fy = __half22float2(__half2(y));
                m[i] = F2(fx.x, fx.y) * F2(sm, sm);
                const F2 s = F2(fy.x, fy.y) * F2(sv, sv);
                v[i] = s * s;
            }
        }
        if (p.grad_scale) {
            const float gs = *p.grad_scale;
#pragma unroll
            for (int i = 0; i < 4; ++i) g[i] = g[i] * F2(gs, gs);
        }
        F2 m1[4], v1[4];
        uint32_t tm = 0, tv = 0;                                        // the largest; non-negative floats order as whole numbers, NaN above all
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // (sums as x * 1 + y: see F2)
            m1[i] = fma2(F2(p.b1, p.b1) * m[i], F2(p.one, p.one), F2(p.omb1, p.omb1) * g[i]);
            v1[i] = fma2(F2(p.b2, p.b2) * v[i], F2(p.one, p.one), F2(p.omb2, p.omb2) * g[i] * g[i]);
            tm = max(tm, max(__float_as_uint(m1[i].lo()) & 0x7fffffffu, __float_as_uint(m1[i].hi()) & 0x7fffffffu));
            tv = max(tv, max(__float_as_uint(v1[i].lo()), __float_as_uint(v1[i].hi())));
        }
        tm = __reduce_max_sync(0xffffffffu, tm);
        tv = __reduce_max_sync(0xffffffffu, tv);
        const bool rare = max(tm, tv) >= 0x7f800000u;                   // something is not finite
        uint32_t keep = 0;                                              // elements that keep what they are
        if (__builtin_expect(rare, 0)) {
            tm = tv = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float a[2], b[2], c[2], d[2];
                m1[i].get(a[0], a[1]); v1[i].get(b[0], b[1]); m[i].get(c[0], c[1]); v[i].get(d[0], d[1]);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (!(isfinite(a[k]) && isfinite(b[k]))) {
                        keep |= 1u << (2 * i + k);
                        a[k] = c[k];
                        b[k] = d[k];
                    }
                    tm = max(tm, __float_as_uint(a[k]) & 0x7fffffffu);
                    tv = max(tv, __float_as_uint(b[k]));
                }
                m1[i] = F2(a[0], a[1]); v1[i] = F2(b[0], b[1]);
            }
            if (keep && p.found) atomicOr(p.found, 1);
            tm = __reduce_max_sync(0xffffffffu, tm);
            tv = __reduce_max_sync(0xffffffffu, tv);
        }
        float inv_m = 1.0f, inv_v = 1.0f;
        uint32_t place = 0;
        if (BITS == 8) {
            const int em = max((int)(tm >> 23) - 127, -100), ev = ((int)(tv >> 23) - 127) >> 1;
            inv_m = power(7 - em);
            inv_v = power(7 - ev);
            if (lane == 0) {
                p.m_scale[block] = power(em - 7);
                p.v_scale[block] = power(ev - 7);
            }
            place = (uint32_t)at ^ p.key ^ ((uint32_t)(at >> 32) * 0x9e3779b1u);
            place ^= place >> 16;                                       // (what distinguishes a lane's elements are low bits)
        }
        F2 root[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const F2 o = w[i];
            if (BITS == 8) {
                root[i] = F2(sqrt_fast(v1[i].lo()), sqrt_fast(v1[i].hi()));
                const F2 d = fma2(root[i], F2(p.rvs, p.rvs), F2(p.eps, p.eps));
                w[i] = o + fma2(o, F2(-lrwd, -lrwd), m1[i] * F2(p.step, p.step) * F2(rcp_fast(d.lo()), rcp_fast(d.hi())));
            } else {
                const float n0 = o.lo() - lrwd * o.lo() + __fdiv_rn(p.step * m1[i].lo(), __fsqrt_rn(v1[i].lo()) * p.rvs + p.eps);
                const float n1 = o.hi() - lrwd * o.hi() + __fdiv_rn(p.step * m1[i].hi(), __fsqrt_rn(v1[i].hi()) * p.rvs + p.eps);
                w[i] = F2(n0, n1);
            }
            if (__builtin_expect(rare, 0)) w[i] = F2(keep >> (2 * i) & 1 ? o.lo() : w[i].lo(), keep >> (2 * i + 1) & 1 ? o.hi() : w[i].hi());
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long o = at + i * 128;
            float wi[4];
            w[2 * i].get(wi[0], wi[1]);
            w[2 * i + 1].get(wi[2], wi[3]);
            if (whole) {
                *reinterpret_cast<float4*>(tw + o) = make_float4(wi[0], wi[1], wi[2], wi[3]);
                if (tcopy) {
                    const __nv_bfloat162 a = __floats2bfloat162_rn(wi[0], wi[1]), b = __floats2bfloat162_rn(wi[2], wi[3]);
                    *reinterpret_cast<uint2*>(tcopy + o) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
                }
            } else {
                const OptTensor& t = p.tensors[here];
                const long e = o - (long)t.block0 * BLOCK;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (e + j < t.n) {
                        t.w[e + j] = wi[j];
                        if (t.copy) t.copy[e + j] = __float2bfloat16(wi[j]);
                    }
            }
            if (BITS == 32) {
                *reinterpret_cast<float4*>((float*)p.m + o) = make_float4(m1[2 * i].lo(), m1[2 * i].hi(), m1[2 * i + 1].lo(), m1[2 * i + 1].hi());
                *reinterpret_cast<float4*>((float*)p.v + o) = make_float4(v1[2 * i].lo(), v1[2 * i].hi(), v1[2 * i + 1].lo(), v1[2 * i + 1].hi());
            } else {
                uint32_t om = 0, ov = 0;
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    const F2 x = m1[2 * i + j / 2], sx = x * F2(inv_m, inv_m), sy = root[2 * i + j / 2] * F2(inv_v, inv_v);
                    const uint32_t r0 = mixed_rest(place ^ (uint32_t)(i * 128 + j)), r1 = mixed_rest(place ^ (uint32_t)(i * 128 + j + 1));    // (bits that at + lane * 4 has not)
                    const F2 a = rounded(F2(fabsf(sx.lo()), fabsf(sx.hi())), r0 & 0xffffu, r1 & 0xffffu);
                    const F2 b = no_less(rounded(sy, r0 >> 16, r1 >> 16), least_root(sy));
                    om |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(copysignf(a.lo(), x.lo()), copysignf(a.hi(), x.hi())), __NV_SATFINITE, __NV_E4M3) << (8 * j);
                    ov |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(b.lo(), b.hi()), __NV_SATFINITE, __NV_E4M3) << (8 * j);
                }
                *reinterpret_cast<uint32_t*>((uint8_t*)p.m + o) = om;
                *reinterpret_cast<uint32_t*>((uint8_t*)p.v + o) = ov;
            }
        }
    }
}

}  // namespace

}  // namespace mgpt

using namespace mgpt;

extern "C" {

int64_t mgpt_moe_optim_blocks(const mgpt_moe_optim_tensor* tensors, int n)
{
    if (!tensors || n <= 0) return 0;
    long b = 0;
    for (int i = 0; i < n; ++i) {
        if (tensors[i].n < 0) return 0;
        b += (tensors[i].n + BLOCK - 1) / BLOCK;
    }
    return b;
}

int mgpt_moe_optim_create(int device, const mgpt_moe_optim_tensor* tensors, int n, int state_bits, mgpt_moe_optim** out)
{
    if (!out) return fail(MGPT_MOE_EINVAL, "null argument");
    *out = nullptr;
    if (!tensors || n <= 0) return fail(MGPT_MOE_EINVAL, "optimiser: no tensors");
    if (state_bits != 8 && state_bits != 32) return fail(MGPT_MOE_EINVAL, "optimiser: state_bits must be 8 or 32");
    try {
        std::vector<OptTensor> ts;
        long block = 0;
        for (int i = 0; i < n; ++i) {
            const mgpt_moe_optim_tensor& s = tensors[i];
            if (s.n < 0 || s.n > (1L << 40)) return fail(MGPT_MOE_EINVAL, "optimiser: tensor size out of range");
            if (s.n && (!s.w || !s.grad)) return fail(MGPT_MOE_EINVAL, "optimiser: null tensor");
            if (s.grad_dtype != MGPT_MOE_IO_F32 && s.grad_dtype != MGPT_MOE_IO_BF16) return fail(MGPT_MOE_EINVAL, "optimiser: unknown gradient dtype");
            const bool gb = s.grad_dtype == MGPT_MOE_IO_BF16;
            MGPT_TRY(check_aligned(s.w, "optimiser: w", 4));
            MGPT_TRY(check_aligned(s.grad, "optimiser: gradient", gb ? 2 : 4));
            MGPT_TRY(check_aligned(s.w_bf16, "optimiser: BF16 copy", 2));
            const long blocks = (s.n + BLOCK - 1) / BLOCK;
            if (!blocks) continue;
            OptTensor t;
            t.w = s.w; t.g = s.grad; t.copy = (bf16*)s.w_bf16; t.n = s.n; t.block0 = (int)block; t.block1 = (int)(block + blocks); t.decay = s.weight_decay; t.g_bf16 = gb;
            t.vec = !((uintptr_t)s.w & 15) && !((uintptr_t)s.grad & 15) && !((uintptr_t)s.w_bf16 & 7);
            ts.push_back(t);
            block += blocks;
            if (block >= (1L << 31) - 65536) return fail(MGPT_MOE_EINVAL, "optimiser: too many elements");
        }
        MGPT_CUDA(cudaSetDevice(device));
        std::unique_ptr<mgpt_moe_optim> o(new mgpt_moe_optim());
        o->device = device; o->n_tensors = (int)ts.size(); o->state_bits = state_bits; o->blocks = block;
        // Two thread blocks per SM, or as many as give every warp a block, take runs of blocks in turn.  Runs of 8 keep neighbouring
        // memory on its way at the same time; 24 where such a step of all of them would pass whole tensors, which each warp then
        // has to find first.  us, runs of 8 / 24: 386 tensors of 100 M elements 401 / 337, one of 268 M 860 / 919, of 100 M 351 / 369.
        int sms = 0;
        MGPT_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        const long most = 2L * sms;
        o->run = (double)ts.size() * most * WARPS > (double)block ? 3 * WARPS : WARPS;
        if ((block + o->run - 1) / o->run < most) o->run = WARPS;
        const long runs = (block + o->run - 1) / o->run;
        o->grid = (int)(runs < most ? runs : most);
        std::vector<int> ints;
        for (const OptTensor& t : ts) ints.push_back(t.block1);
        for (int i = 0, j = 0; i < o->grid; ++i) {
            while (ts[j].block1 <= i * o->run) ++j;
            ints.push_back(j);
        }
        const size_t tb = ts.size() * sizeof(OptTensor), ib = ints.size() * sizeof(int);
        cudaError_t e = cudaMalloc(&o->tables, tb + ib + 16);
        std::vector<char> table(tb + ib);
        if (tb) memcpy(table.data(), ts.data(), tb);
        if (ib) memcpy(table.data() + tb, ints.data(), ib);
        if (e == cudaSuccess && tb + ib) e = cudaMemcpy(o->tables, table.data(), tb + ib, cudaMemcpyHostToDevice);
        if (e == cudaSuccess) e = state_bits == 8 ? cudaFuncSetAttribute(optim_kernel<8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<8>())
                                                  : cudaFuncSetAttribute(optim_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<32>());
        if (e != cudaSuccess) {
            if (o->tables) cudaFree(o->tables);
            return cuda_fail(e, "optimiser tables");
        }
        *out = o.release();
    } catch (const std::exception& e) {
        return fail(MGPT_MOE_ENOMEM, std::string("optimiser: ") + e.what());
    }
    return 0;
}

void mgpt_moe_optim_destroy(mgpt_moe_optim* o)
{
    if (!o) return;
    cudaSetDevice(o->device);
    cudaFree(o->tables);
    delete o;
}

int mgpt_moe_optim_step(mgpt_moe_optim* o, void* m, void* v, float* m_scale, float* v_scale, double lr, double beta1, double beta2, double eps,
                        int64_t t, const float* grad_scale, uint32_t seed, int32_t* found_nonfinite, mgpt_stream_t stream)
{
    if (!o) return fail(MGPT_MOE_EINVAL, "null argument");
    if (t < 1) return fail(MGPT_MOE_EINVAL, "optimiser: steps count from 1");
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return fail(MGPT_MOE_EINVAL, "optimiser: beta1 and beta2 must be in [0, 1)");
    if (o->blocks == 0) return 0;
    if (!m || !v || (o->state_bits == 8 && (!m_scale || !v_scale))) return fail(MGPT_MOE_EINVAL, "null argument");
    MGPT_TRY(check_aligned(m, "optimiser: m"));
    MGPT_TRY(check_aligned(v, "optimiser: v"));
    MGPT_CUDA(cudaSetDevice(o->device));
    cudaStreamCaptureStatus capture;
    MGPT_CUDA(cudaStreamIsCapturing((cudaStream_t)stream, &capture));
    if (capture != cudaStreamCaptureStatusNone)
        return fail(MGPT_MOE_EINVAL, "optimiser: a step is not captured in a graph, whose replays would repeat its number, its rates and its random bits");
    OptP p = {};
    p.tensors = (const OptTensor*)o->tables;
    p.n_tensors = o->n_tensors; p.blocks = (int)o->blocks;
    p.run = o->run;
    p.ends = (const int*)((const char*)o->tables + (size_t)o->n_tensors * sizeof(OptTensor));
    p.starts = p.ends + o->n_tensors;
    p.m = m; p.v = v; p.m_scale = m_scale; p.v_scale = v_scale;
    p.b1 = (float)beta1; p.b2 = (float)beta2; p.omb1 = (float)(1.0 - beta1); p.omb2 = (float)(1.0 - beta2); p.eps = (float)eps; p.lr = (float)lr; p.one = 1.0f;
    p.step = (float)(-lr / (1.0 - std::pow(beta1, (double)t)));
    p.rvs = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)t)));
    p.grad_scale = grad_scale; p.found = found_nonfinite;
    p.key = mixed(seed * 0x9e3779b1u + (uint32_t)t);
    cudaStream_t st = (cudaStream_t)stream;
    if (o->state_bits == 8) MGPT_CUDA(launch_pdl(optim_kernel<8>, o->grid, 32 * WARPS, smem_bytes<8>(), st, p));
    else MGPT_CUDA(launch_pdl(optim_kernel<32>, o->grid, 32 * WARPS, smem_bytes<32>(), st, p));
    MGPT_LAUNCHED("optim_kernel");
    return 0;
}

}  // extern "C"
