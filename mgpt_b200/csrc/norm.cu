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
// Bound by HBM: every element of x, h (dy, du) is read once and y, u (dx, dh) written once.  A token is held by the fewest warps
// (a constant, so that addresses are immediate) and comes through a ring of two tokens per group of warps; sums take one barrier.
// us and TB/s on a B200: 32768 x 2048 BF16 forward 108 (5.0), backward with the parameters' sums 151 (5.3); 16384 x 2048 FP32
// forward 89 (6.0), backward 140 (5.7).  BF16, with twice the elements per byte, is at 56 and 60 % of the
// issue slots.  Before: loads
// into registers, four pieces per thread, 193 and 316; the ring with the number of warps at run time 116 and 190; FP32 in two
// pieces of 32 bytes side by side, half a sector per access, 137 and 227.  A third token in the ring costs more blocks than it hides.
#include "pairs.cuh"

namespace mgpt {

namespace {

constexpr int MAX_C = 16384;
__host__ __device__ constexpr int threads_of(int warps) { return warps > 8 ? 32 * warps : 256; }     // whole groups of warps, one per token
constexpr int UNITS = 296;          // blocks of the backward pass aimed at: two per SM of 148 (not asked of the device: a workspace's size is known without one)
constexpr int FWD_CTAS = 4;         // of the forward pass, per SM

// A piece: 16 bytes of a row, so that a warp's access is one run of memory whatever the type.  A thread copies its pieces to places
// of their own in shared memory, some tokens ahead, and takes them from there.
template <typename T> constexpr int piece() { return 16 / sizeof(T); }          // elements
template <typename T> struct Piece {
    F2 v[piece<T>() / 2];
};
// RING: from there, else from memory (rows too wide for a ring, which the second pass over a token finds in the caches)
template <typename T, bool RING> __device__ __forceinline__ void take(uint32_t src, const T* mem, Piece<T>& o)
{
    if constexpr (sizeof(T) == 2) {
        const uint4 u = RING ? taken<uint4>(src) : *reinterpret_cast<const uint4*>(mem);
        o.v[0] = widen(u.x); o.v[1] = widen(u.y); o.v[2] = widen(u.z); o.v[3] = widen(u.w);
    } else {
        const float4 a = RING ? taken<float4>(src) : *reinterpret_cast<const float4*>(mem);
        o.v[0] = F2(a.x, a.y); o.v[1] = F2(a.z, a.w);
    }
}
__device__ __forceinline__ void store(bf16* p, const Piece<bf16>& o)
{
    *reinterpret_cast<uint4*>(p) = make_uint4(narrow(o.v[0]), narrow(o.v[1]), narrow(o.v[2]), narrow(o.v[3]));
}
__device__ __forceinline__ void store(float* p, const Piece<float>& o)
{
    *reinterpret_cast<float4*>(p) = make_float4(o.v[0].lo(), o.v[0].hi(), o.v[1].lo(), o.v[1].hi());
}
// the same columns of FP32 sums
template <typename T> __device__ __forceinline__ void store_sums(float* p, const Piece<T>& o)
{
#pragma unroll
    for (int j = 0; j < piece<T>() / 4; ++j)
        *reinterpret_cast<float4*>(p + 4 * j) = make_float4(o.v[2 * j].lo(), o.v[2 * j].hi(), o.v[2 * j + 1].lo(), o.v[2 * j + 1].hi());
}
// a piece's parameters, or ones
template <typename T> __device__ __forceinline__ void params(const float* p, int c, Piece<T>& o)
{
#pragma unroll
    for (int j = 0; j < piece<T>() / 4; ++j) {
        const float4 a = p ? *reinterpret_cast<const float4*>(p + c + 4 * j) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        o.v[2 * j] = F2(a.x, a.y);
        o.v[2 * j + 1] = F2(a.z, a.w);
    }
}

// Sums of K values over the W warps of a token's group; every thread of the group calls it.  Two buffers in turn: who writes one
// again has met the others at the barrier of the call between, and they had read it by then.
template <int K, int W> struct __align__(16) Sums {
    float v[2][threads_of(W) / 32 / W][K][W < 4 ? 4 : W];   // [turn][group][value][warp of the group]
};
template <int K, int W> __device__ __forceinline__ void group_sum(float (&v)[K], Sums<K, W>& sh, int& turn)
{
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if constexpr (W > 1) {
        const int group = (threadIdx.x >> 5) / W;
        auto& mine = sh.v[turn][group];
        turn ^= 1;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) mine[k][(threadIdx.x >> 5) % W] = v[k];
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * W) : "memory");
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if constexpr (W == 2) {
                const float2 a = *reinterpret_cast<const float2*>(mine[k]);
                v[k] = a.x + a.y;
            } else {
                v[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < W; i += 4) {
                    const float4 a = *reinterpret_cast<const float4*>(&mine[k][i]);
                    v[k] += (a.x + a.y) + (a.z + a.w);
                }
            }
        }
    }
}
// 1 / sqrt(x): the approximation (2 ulp) and a Newton step; 0 for infinity
__device__ __forceinline__ float inv_sqrt(float x)
{
    const float r = rsqrtf(x);
    return x < INFINITY ? fmaf(fmaf(-x * r, r, 1.0f) * 0.5f, r, r) : r;
}
// A row whose squares overflow is summed again with its values at this much of their size: the largest number's square times 16384 fits, and
// the squares of what made the sum overflow are far above the smallest.
constexpr float SMALL = 0x1p-72f;

struct NormP {
    const void *x, *h;
    const float *post, *gate, *pre;
    float alpha, eps;
    int n, C, per_gate;
    void *y, *u;
    float* stats;                   // [2][n]: r1, r2
    // backward
    const void *dy, *du;
    void *dx, *dh;
    float* part;                    // [units][2][C]: sums of D*h_hat and du*y_hat
    int splits, length;             // units per gate row, tokens per unit
};

// Bytes of a block's ring: `arrays` of NV pieces per thread, STAGES tokens.
constexpr int STAGES = 2;
constexpr uint32_t ring_bytes(int arrays, int nv, int threads) { return STAGES * arrays * nv * threads * 16; }

// A group of warps per token, the groups of the grid taking tokens in turn.
template <typename T, int NV, int W, bool RING>
__global__ void __launch_bounds__(threads_of(W), RING ? 4 : 1) norm_fwd_kernel(const NormP p)
{
    extern __shared__ __align__(16) uint8_t ring[];
    constexpr int THREADS = threads_of(W), GT = 32 * W, GROUPS = THREADS / GT, E = piece<T>(), H = E / 2;
    __shared__ Sums<1, W> sh;
    const int gt = threadIdx.x % GT, step = gridDim.x * GROUPS;
    constexpr uint32_t vec = THREADS * 16, array = NV * vec;
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * 16;
    const float inv = 1.0f / (float)p.C;
    int turn = 0;
    pdl_wait();
    auto fetch = [&](int tok, int s) {
        if (RING && tok < p.n) {
            const size_t o = (size_t)tok * p.C;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (gt + i * GT) * E;
                if (c < p.C) {
                    copy16(mine + s * 2 * array + i * vec, (const T*)p.h + o + c);
                    copy16(mine + (s * 2 + 1) * array + i * vec, (const T*)p.x + o + c);
                }
            }
        }
        copy_commit();
    };
    const int tok0 = blockIdx.x * GROUPS, mine0 = threadIdx.x / GT;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(tok0 + mine0 + s * step, s);
    int slot = 0;
    for (int base = tok0; base < p.n; base += step, slot = slot + 1 == STAGES ? 0 : slot + 1) {
        const int tok = base + mine0;
        const bool have = tok < p.n;                        // (the barriers are everyone's)
        const size_t o = (size_t)tok * p.C;
        fetch(tok + (STAGES - 1) * step, slot == 0 ? STAGES - 1 : slot - 1);
        copy_wait<STAGES - 1>();
        const uint32_t from = mine + slot * 2 * array;
        float r1 = 1.0f, s[1] = {0.0f};
        if (p.post) {
            F2 t(0.0f);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (const int c = (gt + i * GT) * E; have && c < p.C) {
                    Piece<T> h;
                    take<T, RING>(from + i * vec, (const T*)p.h + o + c, h);
#pragma unroll
                    for (int j = 0; j < H; ++j) t = fma2(h.v[j], h.v[j], t);
                }
            s[0] = t.lo() + t.hi();
            group_sum<1, W>(s, sh, turn);
            r1 = inv_sqrt(fmaf(s[0], inv, p.eps));
            if (__builtin_expect(s[0] == INFINITY, 0)) {        // (the same for all of the group)
                t = F2(0.0f);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (const int c = (gt + i * GT) * E; have && c < p.C) {
                        Piece<T> h;
                        take<T, RING>(from + i * vec, (const T*)p.h + o + c, h);
#pragma unroll
                        for (int j = 0; j < H; ++j) t = fma2(h.v[j] * F2(SMALL), h.v[j] * F2(SMALL), t);
                    }
                s[0] = t.lo() + t.hi();
                group_sum<1, W>(s, sh, turn);
                r1 = inv_sqrt(s[0] * inv) * SMALL;
            }
        }
        const float* gate = p.gate && p.per_gate ? p.gate + (size_t)(tok / p.per_gate) * p.C : p.gate;
        Piece<T> y[NV];
        F2 t(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (gt + i * GT) * E;
            if (have && c < p.C) {
                Piece<T> a, g, h, x;
                params<T>(p.post, c, a);
                params<T>(gate, c, g);
                take<T, RING>(from + i * vec, (const T*)p.h + o + c, h);
                take<T, RING>(from + array + i * vec, (const T*)p.x + o + c, x);
#pragma unroll
                for (int j = 0; j < H; ++j) {
                    y[i].v[j] = fma2(F2(p.alpha), x.v[j], g.v[j] * a.v[j] * (h.v[j] * F2(r1)));
                    t = fma2(y[i].v[j], y[i].v[j], t);
                }
                store((T*)p.y + o + c, y[i]);
            }
        }
        float r2 = 1.0f;
        if (p.u) {
            s[0] = t.lo() + t.hi();
            group_sum<1, W>(s, sh, turn);
            r2 = inv_sqrt(fmaf(s[0], inv, p.eps));
            if (__builtin_expect(s[0] == INFINITY, 0)) {
                t = F2(0.0f);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if ((gt + i * GT) * E < p.C && have)
#pragma unroll
                        for (int j = 0; j < H; ++j) t = fma2(y[i].v[j] * F2(SMALL), y[i].v[j] * F2(SMALL), t);
                s[0] = t.lo() + t.hi();
                group_sum<1, W>(s, sh, turn);
                r2 = inv_sqrt(s[0] * inv) * SMALL;
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (gt + i * GT) * E;
                if (have && c < p.C) {
                    Piece<T> b;
                    params<T>(p.pre, c, b);
#pragma unroll
                    for (int j = 0; j < H; ++j) y[i].v[j] = y[i].v[j] * F2(r2) * b.v[j];
                    store((T*)p.u + o + c, y[i]);
                }
            }
        }
        if (have && gt == 0) {
            p.stats[tok] = r1;
            p.stats[p.n + tok] = r2;
        }
    }
}

// One block per unit: tokens of one gate row.  The sums over a unit's tokens stay in registers, a thread's columns being
// always the same; the three sums over a token's columns are taken in one round:
//   mean(D*gp*h_hat) = mean((dy + r2*du*pre)*gp*h_hat) - r2 * mean(du*pre*y_hat) * mean(y_hat*gp*h_hat),   gp = gate*post
template <typename T, int NV, int W, bool RING>
__global__ void __launch_bounds__(threads_of(W), RING ? 2 : 1) norm_bwd_kernel(const NormP p)
{
    extern __shared__ __align__(16) uint8_t ring[];         // at the end: [groups][C] sums
    constexpr int THREADS = threads_of(W), GT = 32 * W, GROUPS = THREADS / GT, E = piece<T>(), H = E / 2;
    __shared__ Sums<3, W> sh;
    const int gt = threadIdx.x % GT, group = threadIdx.x / GT;
    constexpr uint32_t vec = THREADS * 16, array = NV * vec;
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * 16;
    const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
    const int per = p.per_gate ? p.per_gate : p.n;
    const int t0 = row * per + split * p.length, t1 = min(min(t0 + p.length, (row + 1) * per), p.n);
    const float* gate = p.gate ? p.gate + (size_t)row * p.C : nullptr;
    int turn = 0;
    pdl_wait();
    const bool with_u = p.du != nullptr;
    float nr1 = 0.0f, nr2 = 0.0f;                           // of the token that is copied next
    auto fetch = [&](int tok, int s) {
        if (RING && tok < t1) {
            const size_t o = (size_t)tok * p.C;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (gt + i * GT) * E;
                if (c < p.C) {
                    const uint32_t d = mine + s * 4 * array + i * vec;
                    copy16(d, (const T*)p.h + o + c);
                    copy16(d + array, (const T*)p.x + o + c);
                    copy16(d + 2 * array, (const T*)p.dy + o + c);
                    if (with_u) copy16(d + 3 * array, (const T*)p.du + o + c);
                }
            }
        }
        copy_commit();
    };
    Piece<T> S1[NV], S2[NV], gp[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (gt + i * GT) * E;
        Piece<T> a, g;
        if (c < p.C) {
            params<T>(p.post, c, a);
            params<T>(gate, c, g);
        }
#pragma unroll
        for (int j = 0; j < H; ++j) {
            S1[i].v[j] = S2[i].v[j] = F2(0.0f);
            if (c < p.C) gp[i].v[j] = g.v[j] * a.v[j];
        }
    }
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(t0 + group + s * GROUPS, s);
    if (t0 + group < t1) {
        nr1 = p.stats[t0 + group];
        nr2 = p.stats[p.n + t0 + group];
    }
    const float inv = 1.0f / (float)p.C;
    int slot = 0;
    for (int tok0 = t0; tok0 < t1; tok0 += GROUPS, slot = slot + 1 == STAGES ? 0 : slot + 1) {
        const int tok = tok0 + group;
        const bool have = tok < t1;
        const size_t o = (size_t)tok * p.C;
        const float r1 = nr1, r2 = nr2;
        fetch(tok + (STAGES - 1) * GROUPS, slot == 0 ? STAGES - 1 : slot - 1);
        if (tok + GROUPS < t1) {
            nr1 = p.stats[tok + GROUPS];
            nr2 = p.stats[p.n + tok + GROUPS];
        }
        copy_wait<STAGES - 1>();
        const uint32_t from = mine + slot * 4 * array;
        F2 s0(0.0f), s1(0.0f), s2(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (gt + i * GT) * E;
            if (have && c < p.C) {
                Piece<T> h, x, dy, du, b;
                take<T, RING>(from + i * vec, (const T*)p.h + o + c, h);
                take<T, RING>(from + array + i * vec, (const T*)p.x + o + c, x);
                take<T, RING>(from + 2 * array + i * vec, (const T*)p.dy + o + c, dy);
                if (with_u) {
                    take<T, RING>(from + 3 * array + i * vec, (const T*)p.du + o + c, du);
                    params<T>(p.pre, c, b);
                }
#pragma unroll
                for (int j = 0; j < H; ++j) {
                    const F2 q = gp[i].v[j] * (h.v[j] * F2(r1)), yh = fma2(F2(p.alpha), x.v[j], q) * F2(r2);
                    if (with_u) {
                        const F2 d = du.v[j] * b.v[j];
                        s0 = fma2(d, yh, s0);
                        s1 = fma2(fma2(F2(r2), d, dy.v[j]), q, s1);
                    } else {
                        s1 = fma2(dy.v[j], q, s1);
                    }
                    s2 = fma2(yh, q, s2);
                }
            }
        }
        float s[3] = {s0.lo() + s0.hi(), s1.lo() + s1.hi(), s2.lo() + s2.hi()};
        group_sum<3, W>(s, sh, turn);
        // (without u the last sum has y itself in it, and may overflow where nothing of it is wanted)
        const float mA = s[0] * inv, mB = p.post ? (with_u ? s[1] - r2 * mA * s[2] : s[1]) * inv : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (gt + i * GT) * E;
            if (have && c < p.C) {
                Piece<T> h, x, D, du, b, dx;
                take<T, RING>(from + i * vec, (const T*)p.h + o + c, h);
                take<T, RING>(from + array + i * vec, (const T*)p.x + o + c, x);
                take<T, RING>(from + 2 * array + i * vec, (const T*)p.dy + o + c, D);
                if (with_u) {
                    take<T, RING>(from + 3 * array + i * vec, (const T*)p.du + o + c, du);
                    params<T>(p.pre, c, b);
                }
#pragma unroll
                for (int j = 0; j < H; ++j) {
                    const F2 hh = h.v[j] * F2(r1);
                    if (with_u) {
                        const F2 yh = fma2(F2(p.alpha), x.v[j], gp[i].v[j] * hh) * F2(r2);
                        D.v[j] = fma2(F2(r2), fma2(yh, F2(-mA), du.v[j] * b.v[j]), D.v[j]);
                        S2[i].v[j] = fma2(du.v[j], yh, S2[i].v[j]);
                    }
                    dx.v[j] = F2(p.alpha) * D.v[j];
                    S1[i].v[j] = fma2(D.v[j], hh, S1[i].v[j]);
                    h.v[j] = F2(r1) * fma2(hh, F2(-mB), D.v[j] * gp[i].v[j]);
                }
                store((T*)p.dx + o + c, dx);
                store((T*)p.dh + o + c, h);
            }
        }
    }
    if (!p.part) return;
    float* out = p.part + (size_t)blockIdx.x * 2 * p.C;
    float* const cols = reinterpret_cast<float*>(ring);
    copy_wait<0>();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (GROUPS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (gt + i * GT) * E;
                if (c < p.C) store_sums<T>(cols + group * p.C + c, k ? S2[i] : S1[i]);
            }
            __syncthreads();
            for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
                float t = 0.0f;
                for (int g = 0; g < GROUPS; ++g) t += cols[g * p.C + c];
                out[k * p.C + c] = t;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (gt + i * GT) * E;
                if (c < p.C) store_sums<T>(out + k * p.C + c, k ? S2[i] : S1[i]);
            }
        }
    }
}

// The units' sums into the parameters' gradients: 32 columns per block, PW warps that share the units of a row, or the rows where
// there are as many.  Sums are taken in a fixed order.
constexpr int PW = 16;
__global__ void __launch_bounds__(32 * PW)
norm_params_kernel(const float* part, const float* post, const float* gate, int C, int n_gate, int splits, float* d_post, float* d_gate, float* d_pre)
{
    pdl_wait();
    __shared__ float sh[PW][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const bool in = c < C, by_row = n_gate >= PW;
    const float a = post && in ? post[c] : 1.0f;
    auto joined = [&](float v) {                            // over the warps; every thread calls it
        __syncthreads();
        sh[warp][lane] = v;
        __syncthreads();
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < PW; ++i) t += sh[i][lane];
        return t;
    };
    float dp = 0.0f, db = 0.0f;
    for (int row = by_row ? warp : 0; row < n_gate; row += by_row ? PW : 1) {
        float s = 0.0f;
        if (in)
#pragma unroll 8
            for (int i = by_row ? 0 : warp; i < splits; i += by_row ? 1 : PW) {
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

template <typename K> int opt_in(K kernel, uint32_t bytes, bool (&done)[64])
{
    int dev = 0;
    MGPT_CUDA(cudaGetDevice(&dev));
    if (dev < 64 && done[dev]) return 0;
    MGPT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev < 64) done[dev] = true;
    return 0;
}
template <typename T, int NV, int W, bool RING> int run_fwd(const NormP& p, cudaStream_t st)
{
    constexpr int threads = threads_of(W), groups = threads / (32 * W);
    constexpr uint32_t smem = RING ? ring_bytes(2, NV, threads) : 0;
    const int most = 148 * FWD_CTAS, want = (p.n + groups - 1) / groups;
    static bool done[64];
    MGPT_TRY(opt_in(norm_fwd_kernel<T, NV, W, RING>, smem, done));
    MGPT_CUDA(launch_pdl(norm_fwd_kernel<T, NV, W, RING>, want < most ? want : most, threads, smem, st, p));
    MGPT_LAUNCHED("norm_fwd_kernel");
    return 0;
}
template <typename T, int NV, int W, bool RING> int run_bwd(const NormP& p, int units, cudaStream_t st)
{
    // (the ring is more than the sums at the end, 4 NV piece<T>() bytes per thread where there are groups)
    constexpr uint32_t smem = RING ? ring_bytes(4, NV, threads_of(W)) : 0;
    static bool done[64];
    MGPT_TRY(opt_in(norm_bwd_kernel<T, NV, W, RING>, smem, done));
    MGPT_CUDA(launch_pdl(norm_bwd_kernel<T, NV, W, RING>, units, threads_of(W), smem, st, p));
    MGPT_LAUNCHED("norm_bwd_kernel");
    return 0;
}
// NV pieces per thread: the fewest warps that hold a token, a power of two
#define MGPT_BY_WARPS(run, NV, ...)                                                               \
    (p.C <= 32 * piece<T>() * NV ? run<T, NV, 1, true>(__VA_ARGS__)                               \
     : p.C <= 64 * piece<T>() * NV ? run<T, NV, 2, true>(__VA_ARGS__)                             \
     : p.C <= 128 * piece<T>() * NV ? run<T, NV, 4, true>(__VA_ARGS__) : run<T, NV, 8, true>(__VA_ARGS__))
template <typename T> int run_fwd(const NormP& p, cudaStream_t st)
{
    constexpr int F = sizeof(T) / 2;                        // pieces that hold eight elements
    if (p.C > 8192) return run_fwd<T, 4 * F, 16, false>(p, st);
    if (p.C > 4096) return run_fwd<T, 4 * F, 8, false>(p, st);
    if (p.C > 2048) return run_fwd<T, 2 * F, 8, true>(p, st);
    // Two pieces per thread (4 of FP32: 16384 x 2048 123 us against 89); one of BF16 where the tokens are few and a thread's chain is
    // what counts (8 x 1024: 3.1 us against 4.3; 32768 x 2048: 150 against 106).
    if constexpr (sizeof(T) == 2)
        if ((size_t)p.n * p.C <= (size_t)148 * 2048 * 4) return MGPT_BY_WARPS(run_fwd, 1, p, st);
    return MGPT_BY_WARPS(run_fwd, 2, p, st);
}
template <typename T> int run_bwd(const NormP& p, int units, cudaStream_t st)
{
    constexpr int F = sizeof(T) / 2;
    if (p.C > 8192) return run_bwd<T, 4 * F, 16, false>(p, units, st);
    if (p.C > 4096) return run_bwd<T, 4 * F, 8, false>(p, units, st);
    if (p.C > 2048) return run_bwd<T, 2 * F, 8, true>(p, units, st);
    return MGPT_BY_WARPS(run_bwd, 2, p, units, st);
}
#undef MGPT_BY_WARPS

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
    MGPT_CUDA(launch_pdl(norm_params_kernel, (C + 31) / 32, 32 * PW, 0, st, p.part, post_scale, gate, C, rows, s.splits, d_post_scale, d_gate, d_pre_scale));
    MGPT_LAUNCHED("norm_params_kernel");
    return 0;
}

}  // extern "C"
