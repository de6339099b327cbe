// The norms around a block's output, fused with its gate and the skip connection:
//
//   y = alpha * x + gate * (h * r1 * post),   r1 = 1 / sqrt(mean(h^2) + eps)
//   u = y * r2 * pre,                         r2 = 1 / sqrt(mean(y^2) + eps)
//
// x is the residual stream, h what the block computed, u the next block's input.  post, gate and pre may each be absent.
// The gate has a row of C values for every tokens_per_gate tokens (0: one row for all).  The reference has the norm before a
// block and a plain skip connection (layers/TransformerBlock.cpp:38-46; utils/Tensor.cpp:785-800, 1674-1690).
//
// Backward, with y_hat = y*r2, h_hat = h*r1, D the gradient of y by both ways:
//   D  = dy + r2 * (du*pre - y_hat * mean(du*pre*y_hat))
//   dx = alpha * D,   dh = r1 * (D*gate*post - h_hat * mean(D*gate*post*h_hat))
//   d_pre += sum du*y_hat,   d_post += sum D*gate*h_hat,   d_gate += sum D*h_hat*post  (over the row's tokens)
// y is computed again from x and h; r1 and r2 are kept by the forward pass.
//
// Bound by HBM: every element of x, h (dy, du) is read once into registers and y, u (dx, dh) written once.
#include "common.cuh"

namespace mgpt {

namespace {

constexpr int MAX_C = 16384;
constexpr int UNITS = 592;          // blocks of the backward pass aimed at: four per SM

// Eight consecutive elements as they lie in memory.
template <typename T> struct Raw;
template <> struct Raw<bf16> {
    uint4 a;
    __device__ __forceinline__ void load(const bf16* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ float at(int i) const
    {
        const uint32_t w = i < 2 ? a.x : i < 4 ? a.y : i < 6 ? a.z : a.w;
        return i & 1 ? __uint_as_float(w & 0xffff0000u) : __uint_as_float(w << 16);
    }
};
template <> struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p)
    {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ float at(int i) const
    {
        return i == 0 ? a.x : i == 1 ? a.y : i == 2 ? a.z : i == 3 ? a.w : i == 4 ? b.x : i == 5 ? b.y : i == 6 ? b.z : b.w;
    }
};
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8])
{
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
// eight parameters, or ones
__device__ __forceinline__ void params8(const float* p, int c, float (&v)[8])
{
    if (p) {
        const float4 a = *reinterpret_cast<const float4*>(p + c), b = *reinterpret_cast<const float4*>(p + c + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 1.0f;
    }
}

// Sums of K values over the `warps` warps of a token's group; every thread of the block calls it.
template <int K> __device__ __forceinline__ void group_sum(float (&v)[K], int warps, float* sh /* [K][32] */)
{
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (warps == 1) return;
    const int warp = threadIdx.x >> 5, first = warp / warps * warps;
    __syncthreads();                                        // (the last sums have been read)
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) sh[k * 32 + warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = 0.0f;
        for (int i = 0; i < warps; ++i) v[k] += sh[k * 32 + first + i];
    }
}
__device__ __forceinline__ float inv_rms(float ss, int C, float eps) { return __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)C) + eps)); }

struct NormP {
    const void *x, *h;
    const float *post, *gate, *pre;
    float alpha, eps;
    int n, C, per_gate, warps;
    void *y, *u;
    float* stats;                   // [2][n]: r1, r2
    // backward
    const void *dy, *du;
    void *dx, *dh;
    float* part;                    // [units][2][C]: sums of D*h_hat and du*y_hat
    int splits, length;             // units per gate row, tokens per unit
};

template <typename T, int NV>
__global__ void __launch_bounds__(512) norm_fwd_kernel(const NormP p)
{
    pdl_wait();
    __shared__ float sh[32];
    const int gt = threadIdx.x % (32 * p.warps), GT = 32 * p.warps, groups = blockDim.x / GT;
    const int tok = blockIdx.x * groups + threadIdx.x / GT;
    const bool have = tok < p.n;                            // (the barriers are everyone's)
    const size_t o = (size_t)tok * p.C;
    Raw<T> h[NV], x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (gt + i * GT) * 8;
        if (have && c < p.C) {
            h[i].load((const T*)p.h + o + c);
            x[i].load((const T*)p.x + o + c);
        }
    }
    float r1 = 1.0f, s[1] = {0.0f};
    if (p.post) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (have && (gt + i * GT) * 8 < p.C)
#pragma unroll
                for (int j = 0; j < 8; ++j) s[0] = fmaf(h[i].at(j), h[i].at(j), s[0]);
        group_sum(s, p.warps, sh);
        r1 = inv_rms(s[0], p.C, p.eps);
    }
    const float* gate = p.gate && p.per_gate ? p.gate + (size_t)(tok / p.per_gate) * p.C : p.gate;
    float y[NV][8];
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (gt + i * GT) * 8;
        if (have && c < p.C) {
            float a[8], g[8];
            params8(p.post, c, a);
            params8(gate, c, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[i][j] = fmaf(p.alpha, x[i].at(j), g[j] * (h[i].at(j) * r1 * a[j]));
                s[0] = fmaf(y[i][j], y[i][j], s[0]);
            }
            store8((T*)p.y + o + c, y[i]);
        }
    }
    float r2 = 1.0f;
    if (p.u) {
        group_sum(s, p.warps, sh);
        r2 = inv_rms(s[0], p.C, p.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (gt + i * GT) * 8;
            if (have && c < p.C) {
                float b[8];
                params8(p.pre, c, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[i][j] = y[i][j] * r2 * b[j];
                store8((T*)p.u + o + c, y[i]);
            }
        }
    }
    if (have && gt == 0) {
        p.stats[tok] = r1;
        p.stats[p.n + tok] = r2;
    }
}

// One block per unit: tokens of one gate row.  The sums over a unit's tokens stay in registers, a thread's columns being
// always the same; the three sums over a token's columns are taken in one round:
//   mean(D*gp*h_hat) = mean((dy + r2*du*pre)*gp*h_hat) - r2 * mean(du*pre*y_hat) * mean(y_hat*gp*h_hat),   gp = gate*post
template <typename T, int NV>
__global__ void __launch_bounds__(512) norm_bwd_kernel(const NormP p)
{
    pdl_wait();
    extern __shared__ __align__(16) float cols[];           // [groups][C]
    __shared__ float sh[3 * 32];
    const int gt = threadIdx.x % (32 * p.warps), GT = 32 * p.warps, groups = blockDim.x / GT, group = threadIdx.x / GT;
    const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
    const int per = p.per_gate ? p.per_gate : p.n;
    const int t0 = row * per + split * p.length, t1 = min(min(t0 + p.length, (row + 1) * per), p.n);
    const float* gate = p.gate ? p.gate + (size_t)row * p.C : nullptr;
    float S1[NV][8] = {}, S2[NV][8] = {};
    for (int tok0 = t0; tok0 < t1; tok0 += groups) {
        const int tok = tok0 + group;
        const bool have = tok < t1;
        const size_t o = (size_t)tok * p.C;
        const float r1 = have ? p.stats[tok] : 0.0f, r2 = have ? p.stats[p.n + tok] : 0.0f;
        Raw<T> h[NV], x[NV], dy[NV], du[NV];
        float s[3] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (gt + i * GT) * 8;
            if (have && c < p.C) {
                h[i].load((const T*)p.h + o + c);
                x[i].load((const T*)p.x + o + c);
                dy[i].load((const T*)p.dy + o + c);
                if (p.du) du[i].load((const T*)p.du + o + c);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (gt + i * GT) * 8;
            if (have && c < p.C) {
                float a[8], g[8], b[8];
                params8(p.post, c, a);
                params8(gate, c, g);
                params8(p.pre, c, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float hh = h[i].at(j) * r1, gp = g[j] * a[j], q = gp * hh;
                    const float yh = fmaf(p.alpha, x[i].at(j), g[j] * (hh * a[j])) * r2, d = p.du ? du[i].at(j) * b[j] : 0.0f;
                    s[0] = fmaf(d, yh, s[0]);
                    s[1] = fmaf(fmaf(r2, d, dy[i].at(j)), q, s[1]);
                    s[2] = fmaf(yh, q, s[2]);
                }
            }
        }
        group_sum(s, p.warps, sh);
        const float inv = 1.0f / (float)p.C, mA = p.du ? s[0] * inv : 0.0f, mB = p.post ? (s[1] - r2 * mA * s[2]) * inv : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (gt + i * GT) * 8;
            if (have && c < p.C) {
                float a[8], g[8], b[8], dx[8], dh[8];
                params8(p.post, c, a);
                params8(gate, c, g);
                params8(p.pre, c, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float hh = h[i].at(j) * r1, gp = g[j] * a[j], w = p.du ? du[i].at(j) : 0.0f;
                    const float yh = fmaf(p.alpha, x[i].at(j), g[j] * (hh * a[j])) * r2;
                    const float D = p.du ? fmaf(r2, fmaf(-yh, mA, w * b[j]), dy[i].at(j)) : dy[i].at(j);
                    dx[j] = p.alpha * D;
                    dh[j] = r1 * fmaf(-hh, mB, D * gp);
                    S1[i][j] = fmaf(D, hh, S1[i][j]);
                    S2[i][j] = fmaf(w, yh, S2[i][j]);
                }
                store8((T*)p.dx + o + c, dx);
                store8((T*)p.dh + o + c, dh);
            }
        }
    }
    if (!p.part) return;
    float* out = p.part + (size_t)blockIdx.x * 2 * p.C;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (groups > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (gt + i * GT) * 8;
                if (c < p.C) store8(cols + group * p.C + c, k ? S2[i] : S1[i]);
            }
            __syncthreads();
            for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
                float t = 0.0f;
                for (int g = 0; g < groups; ++g) t += cols[g * p.C + c];
                out[k * p.C + c] = t;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (gt + i * GT) * 8;
                if (c < p.C) store8(out + k * p.C + c, k ? S2[i] : S1[i]);
            }
        }
    }
}

// The units' sums into the parameters' gradients: 32 columns per block, eight warps that share the units of a row, or the
// rows where there are eight or more.  Sums are taken in a fixed order.
__global__ void __launch_bounds__(256)
norm_params_kernel(const float* part, const float* post, const float* gate, int C, int n_gate, int splits, float* d_post, float* d_gate, float* d_pre)
{
    pdl_wait();
    __shared__ float sh[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const bool in = c < C, by_row = n_gate >= 8;
    const float a = post && in ? post[c] : 1.0f;
    auto joined = [&](float v) {                            // over the warps; every thread calls it
        __syncthreads();
        sh[warp][lane] = v;
        __syncthreads();
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += sh[i][lane];
        return t;
    };
    float dp = 0.0f, db = 0.0f;
    for (int row = by_row ? warp : 0; row < n_gate; row += by_row ? 8 : 1) {
        float s = 0.0f;
        if (in)
#pragma unroll 4
            for (int i = by_row ? 0 : warp; i < splits; i += by_row ? 1 : 8) {
                const float* from = part + (size_t)(row * splits + i) * 2 * C + c;
                s += from[0];
                db += from[C];
            }
        if (!by_row) s = joined(s);
        const float g = gate && in ? gate[(size_t)row * C + c] : 1.0f;
        if (in && d_gate && (by_row || warp == 0)) d_gate[(size_t)row * C + c] += s * a;
        dp = fmaf(s, g, dp);
    }
    if (by_row) dp = joined(dp);
    db = joined(db);
    if (warp == 0 && in) {
        if (d_post) d_post[c] += dp;
        if (d_pre) d_pre[c] += db;
    }
}

int gate_rows(int n, int per_gate) { return per_gate ? (n + per_gate - 1) / per_gate : 1; }
int one_row(int n, int per_gate) { return per_gate >= n ? 0 : per_gate; }

// Warps per token with NV pieces of eight elements per thread, a power of two up to 16.
int warps_of(int C, int nv)
{
    int w = 1;
    while (w < 16 && w * 32 * 8 * nv < C) w *= 2;
    return w;
}
struct Split {
    int splits, length;
};
Split split_of(int n, int per_gate)
{
    const int rows = gate_rows(n, per_gate), per = per_gate ? per_gate : n;
    int want = (UNITS + rows - 1) / rows, most = (per + 7) / 8;      // (a unit of fewer than eight tokens is not worth its sums)
    if (want > most) want = most;
    Split s;
    s.length = (per + want - 1) / want;
    s.splits = (per + s.length - 1) / s.length;
    return s;
}

int check_norm(int n, int C, int per_gate, int io)
{
    if (n < 0 || n > (1 << 30) || C <= 0 || per_gate < 0) return fail(MGPT_MOE_EINVAL, "residual norm: sizes out of range");
    if (C % 8 || C > MAX_C) return fail(MGPT_MOE_EINVAL, "residual norm: embed_dim must be a multiple of 8, at most 16384");
    if (io != MGPT_MOE_IO_F32 && io != MGPT_MOE_IO_BF16) return fail(MGPT_MOE_EINVAL, "unknown io dtype");
    return 0;
}
int check_params(const float* post, const float* gate, const float* pre)
{
    MGPT_TRY(check_aligned(post, "post_scale"));
    MGPT_TRY(check_aligned(gate, "gate"));
    MGPT_TRY(check_aligned(pre, "pre_scale"));
    return 0;
}

template <typename T> int run_fwd(NormP& p, cudaStream_t st)
{
    // few tokens: as many threads per token as it has pieces, else four pieces per thread
    const int nv = p.C > 4096 * 2 ? 4 : p.C > 4096 ? 2 : (size_t)p.n * p.C <= (size_t)148 * 2048 * 4 ? 1 : 4;
    p.warps = warps_of(p.C, nv);
    const int threads = 32 * p.warps > 256 ? 32 * p.warps : 256, groups = threads / (32 * p.warps), blocks = (p.n + groups - 1) / groups;
    if (nv == 1) MGPT_CUDA(launch_pdl(norm_fwd_kernel<T, 1>, blocks, threads, 0, st, p));
    else if (nv == 2) MGPT_CUDA(launch_pdl(norm_fwd_kernel<T, 2>, blocks, threads, 0, st, p));
    else MGPT_CUDA(launch_pdl(norm_fwd_kernel<T, 4>, blocks, threads, 0, st, p));
    MGPT_LAUNCHED("norm_fwd_kernel");
    return 0;
}
template <typename T> int run_bwd(NormP& p, int units, cudaStream_t st)
{
    const int nv = p.C > 8192 ? 4 : p.C > 4096 || sizeof(T) == 2 ? 2 : 1;
    p.warps = warps_of(p.C, nv);
    const int threads = 32 * p.warps > 256 ? 32 * p.warps : 256, groups = threads / (32 * p.warps);
    const size_t smem = groups > 1 ? (size_t)groups * p.C * 4 : 0;           // at most 256 threads * 8 * nv floats: 32 KiB
    if (nv == 1) MGPT_CUDA(launch_pdl(norm_bwd_kernel<T, 1>, units, threads, smem, st, p));
    else if (nv == 2) MGPT_CUDA(launch_pdl(norm_bwd_kernel<T, 2>, units, threads, smem, st, p));
    else MGPT_CUDA(launch_pdl(norm_bwd_kernel<T, 4>, units, threads, smem, st, p));
    MGPT_LAUNCHED("norm_bwd_kernel");
    return 0;
}

}  // namespace

}  // namespace mgpt

using namespace mgpt;

extern "C" {

int mgpt_moe_op_residual_norm(const void* x, const void* h, int io, const float* post_scale, const float* gate, int tokens_per_gate,
                              const float* pre_scale, float alpha, float eps, int n, int C, void* y, void* u, float* stats, mgpt_stream_t stream)
{
    MGPT_TRY(check_norm(n, C, tokens_per_gate, io));
    if (n == 0) return 0;
    if (!x || !h || !y || !stats) return fail(MGPT_MOE_EINVAL, "null argument");
    if (!pre_scale != !u) return fail(MGPT_MOE_EINVAL, "residual norm: u and pre_scale go together");
    const struct { const void* p; const char* what; } io_bufs[] = {{x, "x"}, {h, "h"}, {y, "y"}, {u, "u"}};
    for (const auto& b : io_bufs) MGPT_TRY(check_aligned(b.p, b.what));
    MGPT_TRY(check_params(post_scale, gate, pre_scale));
    NormP p = {};
    p.x = x; p.h = h; p.post = post_scale; p.gate = gate; p.pre = pre_scale; p.alpha = alpha; p.eps = eps; p.n = n; p.C = C;
    p.per_gate = one_row(n, tokens_per_gate); p.y = y; p.u = u; p.stats = stats;
    return io == MGPT_MOE_IO_BF16 ? run_fwd<bf16>(p, (cudaStream_t)stream) : run_fwd<float>(p, (cudaStream_t)stream);
}

size_t mgpt_moe_op_residual_norm_backward_workspace_bytes(int n, int C, int tokens_per_gate)
{
    if (check_norm(n, C, tokens_per_gate, MGPT_MOE_IO_BF16) || n == 0) return 0;
    tokens_per_gate = one_row(n, tokens_per_gate);
    return (size_t)gate_rows(n, tokens_per_gate) * split_of(n, tokens_per_gate).splits * 2 * C * sizeof(float);
}

int mgpt_moe_op_residual_norm_backward(const void* x, const void* h, int io, const float* post_scale, const float* gate, int tokens_per_gate,
                                       const float* pre_scale, float alpha, int n, int C, const float* stats, const void* dy, const void* du,
                                       void* dx, void* dh, float* d_post_scale, float* d_gate, float* d_pre_scale,
                                       void* workspace, size_t ws_bytes, mgpt_stream_t stream)
{
    MGPT_TRY(check_norm(n, C, tokens_per_gate, io));
    if (n == 0) return 0;
    if (!x || !h || !stats || !dy || !dx || !dh) return fail(MGPT_MOE_EINVAL, "null argument");
    if (!pre_scale != !du) return fail(MGPT_MOE_EINVAL, "residual norm: du and pre_scale go together");
    if ((d_post_scale && !post_scale) || (d_gate && !gate) || (d_pre_scale && !pre_scale))
        return fail(MGPT_MOE_EINVAL, "residual norm: a gradient of a parameter that is absent");
    const struct { const void* p; const char* what; } io_bufs[] = {{x, "x"}, {h, "h"}, {dy, "dy"}, {du, "du"}, {dx, "dx"}, {dh, "dh"}};
    for (const auto& b : io_bufs) MGPT_TRY(check_aligned(b.p, b.what));
    MGPT_TRY(check_params(post_scale, gate, pre_scale));
    tokens_per_gate = one_row(n, tokens_per_gate);
    const bool sums = d_post_scale || d_gate || d_pre_scale;
    const Split s = split_of(n, tokens_per_gate);
    const int rows = gate_rows(n, tokens_per_gate), units = rows * s.splits;
    if (sums) {
        if (!workspace || ((uintptr_t)workspace & 255)) return fail(MGPT_MOE_EINVAL, "workspace must be 256-byte aligned");
        if (ws_bytes < (size_t)units * 2 * C * sizeof(float))
            return fail(MGPT_MOE_ENOMEM, "workspace smaller than mgpt_moe_op_residual_norm_backward_workspace_bytes()");
    }
    NormP p = {};
    p.x = x; p.h = h; p.post = post_scale; p.gate = gate; p.pre = pre_scale; p.alpha = alpha; p.n = n; p.C = C; p.per_gate = tokens_per_gate;
    p.stats = (float*)stats; p.dy = dy; p.du = du; p.dx = dx; p.dh = dh; p.part = sums ? (float*)workspace : nullptr;
    p.splits = s.splits; p.length = s.length;
    cudaStream_t st = (cudaStream_t)stream;
    MGPT_TRY(io == MGPT_MOE_IO_BF16 ? run_bwd<bf16>(p, units, st) : run_bwd<float>(p, units, st));
    if (!sums) return 0;
    MGPT_CUDA(launch_pdl(norm_params_kernel, (C + 31) / 32, 256, 0, st, p.part, post_scale, gate, C, rows, s.splits, d_post_scale, d_gate, d_pre_scale));
    MGPT_LAUNCHED("norm_params_kernel");
    return 0;
}

}  // extern "C"
