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
// An element whose new moments are not finite (its gradient is not, or overflows) keeps w, m and v, and sets the caller's flag.
#include <cmath>

#include <cuda_fp8.h>

#include "common.cuh"

struct mgpt_moe_optim {
    int device;
    int n_tensors;
    int state_bits;
    long blocks;
    long chunks;
    void* tables = nullptr;     // device: tensors, then chunks
};

namespace mgpt {

namespace {

constexpr int BLOCK = 256;              // elements that share a scale
constexpr int CHUNK = 8;                // blocks of a thread block, one per warp

struct OptTensor {
    float* w;
    const void* g;
    bf16* copy;
    long n;
    long block0;
    float decay;
    int g_bf16;
    int vec;                            // all of them start on a boundary that four elements can be moved at
};
struct OptChunk {
    int tensor;
    int first;                          // in units of CHUNK blocks from the tensor's first
};
struct OptP {
    const OptTensor* tensors;
    const OptChunk* chunks;
    void *m, *v;
    float *m_scale, *v_scale;
    float b1, b2, omb1, omb2, eps, lr, ms, vs;
    const float* grad_scale;
    int32_t* found;
    uint32_t key;
};

__host__ __device__ __forceinline__ uint32_t mixed(uint32_t h)
{
    h ^= h >> 16;
    h *= 0x85ebca6bu;
    h ^= h >> 13;
    h *= 0xc2b2ae35u;
    return h ^ (h >> 16);
}
__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }

// |a| (a block's largest below 256) to 3 bits of mantissa, steps of 2^-9 below 2^-6: 16 random bits are added below the last
// kept bit, what is below it is dropped.
__device__ __forceinline__ float rounded(float a, uint32_t random16)
{
    const float low = a < 0.015625f ? 0.015625f : 0.0f;
    const uint32_t bits = __float_as_uint(__fadd_rn(a, low)) + (random16 << 4);
    return __uint_as_float(bits & 0xfff00000u) - low;
}

template <int BITS>
__global__ void __launch_bounds__(256) optim_kernel(const OptP p)
{
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const OptChunk ch = p.chunks[blockIdx.x];
    const OptTensor t = p.tensors[ch.tensor];
    const long in_tensor = (long)ch.first * CHUNK + warp;           // this warp's block
    const long first = in_tensor * BLOCK;
    if (first >= t.n) return;
    const long block = t.block0 + in_tensor, at = block * BLOCK;
    const float gs = p.grad_scale ? *p.grad_scale : 1.0f;
    float w[8], g[8], m[8], v[8];
    // lane's elements: four from lane * 4, four from 128 + lane * 4
    int valid[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long e = first + i * 128 + lane * 4, left = t.n - e;
        valid[i] = left >= 4 ? 4 : left > 0 ? (int)left : 0;
        float *wi = w + 4 * i, *gi = g + 4 * i, *mi = m + 4 * i, *vi = v + 4 * i;
        if (t.vec && valid[i] == 4) {
            const float4 a = *reinterpret_cast<const float4*>(t.w + e);
            wi[0] = a.x; wi[1] = a.y; wi[2] = a.z; wi[3] = a.w;
            if (t.g_bf16) {
                const uint2 b = *reinterpret_cast<const uint2*>((const bf16*)t.g + e);
                gi[0] = __uint_as_float(b.x << 16); gi[1] = __uint_as_float(b.x & 0xffff0000u);
                gi[2] = __uint_as_float(b.y << 16); gi[3] = __uint_as_float(b.y & 0xffff0000u);
            } else {
                const float4 b = *reinterpret_cast<const float4*>((const float*)t.g + e);
                gi[0] = b.x; gi[1] = b.y; gi[2] = b.z; gi[3] = b.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                wi[j] = j < valid[i] ? t.w[e + j] : 0.0f;
                gi[j] = j < valid[i] ? t.g_bf16 ? __bfloat162float(((const bf16*)t.g)[e + j]) : ((const float*)t.g)[e + j] : 0.0f;
            }
        }
        const long o = at + i * 128 + lane * 4;
        if (BITS == 32) {
            const float4 a = *reinterpret_cast<const float4*>((const float*)p.m + o), b = *reinterpret_cast<const float4*>((const float*)p.v + o);
            mi[0] = a.x; mi[1] = a.y; mi[2] = a.z; mi[3] = a.w;
            vi[0] = b.x; vi[1] = b.y; vi[2] = b.z; vi[3] = b.w;
        } else {
            const uint32_t a = *reinterpret_cast<const uint32_t*>((const uint8_t*)p.m + o), b = *reinterpret_cast<const uint32_t*>((const uint8_t*)p.v + o);
            const float sm = p.m_scale[block], sv = p.v_scale[block];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(a >> (16 * j)), __NV_E4M3);
                const __half2_raw y = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(b >> (16 * j)), __NV_E4M3);
                const float2 fx = __half22float2(__half2(x)), fy = __half22float2(__half2(y));
                mi[2 * j] = fx.x * sm;
                mi[2 * j + 1] = fx.y * sm;
                const float s0 = fy.x * sv, s1 = fy.y * sv;
                vi[2 * j] = __fmul_rn(s0, s0);
                vi[2 * j + 1] = __fmul_rn(s1, s1);
            }
        }
    }
    const float lrwd = p.lr * t.decay;
    bool bad = false;
    float top_m = 0.0f, top_v = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float gj = p.grad_scale ? g[j] * gs : g[j];
        const float m1 = __fadd_rn(__fmul_rn(p.b1, m[j]), __fmul_rn(p.omb1, gj));
        const float v1 = __fadd_rn(__fmul_rn(p.b2, v[j]), __fmul_rn(__fmul_rn(p.omb2, gj), gj));
        if (isfinite(m1) && isfinite(v1)) {
            m[j] = m1;
            v[j] = v1;
            w[j] = w[j] - lrwd * w[j] - __fdiv_rn(p.lr * (m1 * p.ms), __fsqrt_rn(v1 * p.vs) + p.eps);
        } else {
            bad = true;
        }
        top_m = fmaxf(top_m, fabsf(m[j]));
        top_v = fmaxf(top_v, v[j]);
    }
    if (bad && p.found) atomicOr(p.found, 1);
    float inv_m = 1.0f, inv_v = 1.0f;
    uint32_t place = 0;
    if (BITS == 8) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            top_m = fmaxf(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
            top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
        }
        const int em = max((__float_as_int(top_m) >> 23) - 127, -100), ev = ((__float_as_int(top_v) >> 23) - 127) >> 1;
        inv_m = power(7 - em);
        inv_v = power(7 - ev);
        if (lane == 0) {
            p.m_scale[block] = power(em - 7);
            p.v_scale[block] = power(ev - 7);
        }
        place = (uint32_t)at ^ p.key ^ ((uint32_t)(at >> 32) * 0x9e3779b1u);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long e = first + i * 128 + lane * 4;
        float *wi = w + 4 * i, *mi = m + 4 * i, *vi = v + 4 * i;
        if (t.vec && valid[i] == 4) {
            *reinterpret_cast<float4*>(t.w + e) = make_float4(wi[0], wi[1], wi[2], wi[3]);
            if (t.copy) {
                const __nv_bfloat162 a = __floats2bfloat162_rn(wi[0], wi[1]), b = __floats2bfloat162_rn(wi[2], wi[3]);
                *reinterpret_cast<uint2*>(t.copy + e) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < valid[i]) {
                    t.w[e + j] = wi[j];
                    if (t.copy) t.copy[e + j] = __float2bfloat16(wi[j]);
                }
        }
        const long o = at + i * 128 + lane * 4;
        if (BITS == 32) {
            *reinterpret_cast<float4*>((float*)p.m + o) = make_float4(mi[0], mi[1], mi[2], mi[3]);
            *reinterpret_cast<float4*>((float*)p.v + o) = make_float4(vi[0], vi[1], vi[2], vi[3]);
        } else {
            uint32_t cm = 0, cv = 0;
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                float a[2], b[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t r = mixed(place ^ (uint32_t)(i * 128 + lane * 4 + j + k));       // (the block's place is a multiple of 256)
                    a[k] = copysignf(rounded(fabsf(mi[j + k]) * inv_m, r & 0xffffu), mi[j + k]);
                    b[k] = rounded(__fsqrt_rn(vi[j + k]) * inv_v, r >> 16);
                }
                cm |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a[0], a[1]), __NV_SATFINITE, __NV_E4M3) << (8 * j);
                cv |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(b[0], b[1]), __NV_SATFINITE, __NV_E4M3) << (8 * j);
            }
            *reinterpret_cast<uint32_t*>((uint8_t*)p.m + o) = cm;
            *reinterpret_cast<uint32_t*>((uint8_t*)p.v + o) = cv;
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
        std::vector<OptTensor> ts(n);
        std::vector<OptChunk> cs;
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
            OptTensor& t = ts[i];
            t.w = s.w; t.g = s.grad; t.copy = (bf16*)s.w_bf16; t.n = s.n; t.block0 = block; t.decay = s.weight_decay; t.g_bf16 = gb;
            t.vec = !((uintptr_t)s.w & 15) && !((uintptr_t)s.grad & (gb ? 7 : 15)) && !((uintptr_t)s.w_bf16 & 7);
            const long blocks = (s.n + BLOCK - 1) / BLOCK;
            for (long b = 0; b < blocks; b += CHUNK) cs.push_back({i, (int)(b / CHUNK)});
            block += blocks;
        }
        if (cs.size() > (size_t)INT32_MAX) return fail(MGPT_MOE_EINVAL, "optimiser: too many elements");
        MGPT_CUDA(cudaSetDevice(device));
        mgpt_moe_optim* o = new mgpt_moe_optim();
        o->device = device; o->n_tensors = n; o->state_bits = state_bits; o->blocks = block; o->chunks = (long)cs.size();
        const size_t tb = ts.size() * sizeof(OptTensor), cb = cs.size() * sizeof(OptChunk);
        cudaError_t e = cudaMalloc(&o->tables, tb + cb + 16);
        if (e == cudaSuccess) e = cudaMemcpy(o->tables, ts.data(), tb, cudaMemcpyHostToDevice);
        if (e == cudaSuccess && cb) e = cudaMemcpy((char*)o->tables + tb, cs.data(), cb, cudaMemcpyHostToDevice);
        if (e != cudaSuccess) {
            if (o->tables) cudaFree(o->tables);
            delete o;
            return cuda_fail(e, "optimiser tables");
        }
        *out = o;
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
    OptP p = {};
    p.tensors = (const OptTensor*)o->tables;
    p.chunks = (const OptChunk*)((const char*)o->tables + (size_t)o->n_tensors * sizeof(OptTensor));
    p.m = m; p.v = v; p.m_scale = m_scale; p.v_scale = v_scale;
    p.b1 = (float)beta1; p.b2 = (float)beta2; p.omb1 = (float)(1.0 - beta1); p.omb2 = (float)(1.0 - beta2); p.eps = (float)eps; p.lr = (float)lr;
    p.ms = (float)(1.0 / (1.0 - std::pow(beta1, (double)t)));
    p.vs = (float)(1.0 / (1.0 - std::pow(beta2, (double)t)));
    p.grad_scale = grad_scale; p.found = found_nonfinite;
    p.key = mixed(seed * 0x9e3779b1u + (uint32_t)t);
    cudaStream_t st = (cudaStream_t)stream;
    if (o->state_bits == 8) MGPT_CUDA(launch_pdl(optim_kernel<8>, (unsigned)o->chunks, 256, 0, st, p));
    else MGPT_CUDA(launch_pdl(optim_kernel<32>, (unsigned)o->chunks, 256, 0, st, p));
    MGPT_LAUNCHED("optim_kernel");
    return 0;
}

}  // extern "C"
