// Routing to experts from their logits, and its gradient.  Token with logits z, bias b (order only), k chosen:
//
//   s_e = 1 / (1 + exp(-z_e))   or   exp(z_e) / sum exp(z),      c_e = s_e + b_e
//   the top_groups groups of consecutive experts with the largest sums of their group_top largest c stay;
//   chosen are their k largest c in falling order, equal ones by index; without a bias the order is that of z itself
//   w_j = scale * s_j / (sum of the chosen s + 1e-20)   or   scale * s_j
//
// Gradient, with S the sum of the chosen s plus 1e-20 and A = sum dw_j s_j:
//   dg_j = scale / S * (dw_j - A / S)   or   scale * dw_j
//   sigmoid: dz_e = dg_j s_j (1 - s_j) for the chosen, 0 elsewhere;   softmax: dz_e = p_e ([chosen] dg_j - sum_j dg_j p_j)
// The reference has clamped softmax and top-k only (utils/Tensor.cpp:850-909).
//
// What is chosen is what exact arithmetic chooses (up to FP64's rounding): scores are formed in FP32 with a known bound on their
// error, and a token in which some comparison that decides is closer than that is gone through again in FP64 by its warp.
#include "common.cuh"

namespace mgpt {

namespace {

constexpr int ROUTE_MAX_E = 512, ROUTE_MAX_K = 32, ROUTE_MAX_GROUPS = 32;
constexpr int WARPS = 4;
constexpr float TINY = 1e-20f;      // beside the sum that is divided by
constexpr unsigned FULL = 0xffffffffu;

struct RouteP {
    const void* logits;
    const float* bias;
    int n, E, k;
    int softmax, groups, top_groups, group_top, renorm;
    float scale;
    int gsize;          // experts per group
    uint32_t gdiv;      // 2^20 / gsize, rounded up: e * gdiv >> 20 is e / gsize for e < 512
    uint32_t kdiv;      // 2^16 / k, rounded up: q * kdiv >> 16 is q / k for q < 256
    int32_t* idx;
    float* w;
    int32_t* counts;
    // backward
    const int32_t* top;
    const float* dw;
    void* dz;
    bf16* dz16;         // a second copy of width E8, or null
    int E8;
};

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(bf16 v) { return __bfloat162float(v); }

// Numbers as unsigned integers of the same order: minus infinity is NONE, and 0 is below every number.  (-0 and 0 are equal.)
template <typename V> struct Ordered;
template <> struct Ordered<float> {
    using U = uint32_t;
    static constexpr U NONE = 0x007fffffu;
    static __device__ __forceinline__ U key(float v)
    {
        const uint32_t u = __float_as_uint(v + 0.0f);
        return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    }
    static __device__ __forceinline__ float value(U k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
};
template <> struct Ordered<double> {
    using U = unsigned long long;
    static constexpr U NONE = 0x000fffffffffffffull;
    static __device__ __forceinline__ U key(double v)
    {
        const long long u = __double_as_longlong(v + 0.0);
        return (U)u ^ ((U)(u >> 63) | 0x8000000000000000ull);
    }
};

// over the L lanes of a token
template <int L, typename V> __device__ __forceinline__ V lanes_max(V v)
{
    if constexpr (L == 32 && sizeof(V) == 4 && (V)(-1) > (V)0) return __reduce_max_sync(FULL, v);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
        const V other = __shfl_xor_sync(FULL, v, o);
        v = other > v ? other : v;
    }
    return v;
}
template <int L, typename V> __device__ __forceinline__ V lanes_min(V v)
{
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
        const V other = __shfl_xor_sync(FULL, v, o);
        v = other < v ? other : v;
    }
    return v;
}
template <int L, typename V> __device__ __forceinline__ V lanes_sum(V v)
{
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
template <int L> __device__ __forceinline__ uint32_t lanes_or(uint32_t v)
{
    if constexpr (L == 32) return __reduce_or_sync(FULL, v);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v |= __shfl_xor_sync(FULL, v, o);
    return v;
}

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float over_one(float v) { return __fdividef(1.0f, v); }
__device__ __forceinline__ double over_one(double v) { return 1.0 / v; }
// FP32: exp to 2^-22, the sum and the reciprocal to 2^-24 and 2^-23 of themselves: at most 3.5e-7 off
template <typename V> __device__ __forceinline__ V sigmoid(V z) { return over_one((V)1 + exp_of(-z)); }

// A token's experts e = i*L + sub of its lanes, i < P.  Bit i of the masks: the expert exists / is out (its logit or bias leaves it no place).
template <int L, int P> struct Lane {
    int sub, t;         // place among the token's lanes, the token among the warp's
    uint32_t exists, out;
};

// The chosen experts of the warp's tokens into `chosen` [tokens][k].  V float: whether some comparison is too close for FP32.
// c: the warp's shared memory, [tokens][E].  top_z: largest logit that is not out; inv: 1 / sum of exp(z - top_z).
template <typename V, typename T, int L, int P>
__device__ __forceinline__ bool choose(const RouteP& p, const Lane<L, P>& a, int tok, bool have, const float (&z)[P], const float (&b)[P],
                                       float bmax, float top_z, V inv, V* c, int32_t* chosen)
{
    using O = Ordered<V>;
    using U = typename O::U;
    constexpr bool PROVE = sizeof(V) == 4;
    const V NOTHING = -(V)INFINITY;
    const bool grouped = p.top_groups < p.groups;
    bool unsure = false;
    // half of what two scores have to differ by
    const float base = p.softmax ? 2e-6f * (float)inv + 3e-8f : 3.5e-7f;
    U key[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const bool out = a.out >> i & 1;
        V v = NOTHING;
        if (!out) {
            v = p.softmax ? exp_of((V)z[i] - (V)top_z) * inv : sigmoid((V)z[i]);
            if (p.bias) v += (V)b[i];
        }
        if (grouped && (a.exists >> i & 1)) c[a.t * p.E + i * L + a.sub] = v;
        key[i] = !(a.exists >> i & 1) ? 0 : p.bias ? O::key(v) : out ? O::NONE : O::key((V)z[i]);
    }
    if (grouped) {
        __syncwarp();
        // S lanes to a group, L / S groups at a time
        int S = L;
        while (S > 1 && L / S < p.groups) S >>= 1;
        const int first = a.sub / S, part = a.sub % S, at_once = L / S;
        uint32_t kept = 0;
        // a group's two largest: its lanes take every S-th expert, each group from another one on (the banks of shared memory)
        V score = NOTHING;
        V* const scores = c + (32 / L) * p.E;                   // [tokens][groups]
        for (int g0 = 0; g0 < p.groups; g0 += at_once) {
            const int g = g0 + first;
            V m1 = NOTHING, m2 = NOTHING;
            if (g < p.groups) {
                const V* from = c + a.t * p.E + g * p.gsize;
                const int count = (p.gsize - part + S - 1) / S;
                int j = count ? g % count : 0;
                for (int i = 0; i < count; ++i, j = j + 1 == count ? 0 : j + 1) {
                    const V v = from[part + j * S];
                    m2 = v > m1 ? m1 : v > m2 ? v : m2;
                    m1 = v > m1 ? v : m1;
                }
            }
            for (int o = S / 2; o > 0; o >>= 1) {
                const V n1 = __shfl_xor_sync(FULL, m1, o), n2 = __shfl_xor_sync(FULL, m2, o);
                const V low = n1 > m1 ? m1 : n1, high = n1 > m1 ? n1 : m1;
                m2 = n2 > m2 ? n2 : m2;
                m2 = low > m2 ? low : m2;
                m1 = high;
            }
            if (p.group_top == 2 && m2 > NOTHING) m1 += m2;
            if (g < p.groups && part == 0) scores[a.t * p.groups + g] = m1;
        }
        __syncwarp();
        V least = INFINITY, most = NOTHING;     // of the kept, of the others
        for (int g = a.sub; g < p.groups; g += L) {
            score = scores[a.t * p.groups + g];
            int before = 0;
            for (int h = 0; h < p.groups; ++h) {
                const V v = scores[a.t * p.groups + h];
                before += v > score || (v == score && h < g);
            }
            if (before < p.top_groups) {
                kept |= 1u << g;
                least = score < least ? score : least;
            } else {
                most = score > most ? score : most;
            }
        }
        kept = lanes_or<L>(kept);
        if (PROVE) {
            least = lanes_min<L>(least);
            most = lanes_max<L>(most);
            // (a sum of two: twice the error, and roundings of terms of at most 1 + bmax; where nothing is left in two groups the index decides)
            const bool nothing = least == NOTHING && most == NOTHING && bmax < 1e30f;
            unsure = have && !nothing && !((float)(least - most) > 4.0f * base + 5e-7f * (1.0f + bmax));
        }
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (!(kept >> ((uint32_t)(i * L + a.sub) * p.gdiv >> 20) & 1)) key[i] = 0;
    }
    const int rounds = p.k + (PROVE && p.bias);
    U last = 0;
    int last_e = 0;
    const uint32_t mine = (L == 32 ? FULL : ((1u << (L & 31)) - 1) << (a.t * L));
    for (int j = 0; j < rounds; ++j) {
        U best = key[0];
#pragma unroll
        for (int i = 1; i < P; ++i) best = key[i] > best ? key[i] : best;
        const U m = lanes_max<L>(best);
        int e = 0x7fffffff;
#pragma unroll
        for (int i = P - 1; i >= 0; --i) e = key[i] == m ? i * L + a.sub : e;
        const uint32_t equal = __ballot_sync(FULL, best == m) & mine;
        if (__any_sync(FULL, equal & (equal - 1))) e = lanes_min<L>(e);
        else e = __shfl_sync(FULL, e, __ffs(equal) - 1);
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (e == i * L + a.sub) key[i] = 0;
        if (j < p.k && a.sub == 0) chosen[a.t * p.k + j] = e;
        if constexpr (PROVE)
            if (p.bias && j > 0) {
                const float hi = O::value(last), lo = O::value(m);
                const bool close = have && m > O::NONE && !(hi - lo > 2.0f * base + 1.3e-7f * (fabsf(hi) + fabsf(lo)));
                if (__any_sync(FULL, close))
                    if (close) {                // equal inputs have equal scores, and the index decides
                        const T* row = (const T*)p.logits + (size_t)tok * p.E;
                        unsure |= !(as_float(row[e]) == as_float(row[last_e]) && p.bias[e] == p.bias[last_e]);
                    }
            }
        last = m;
        last_e = e;
    }
    return unsure;
}

template <typename T, int L, int P>
__device__ __noinline__ void choose_again(const RouteP& p, int tok, bool have, float top_z, double* c, int32_t* chosen)
{
    const int lane = threadIdx.x & 31;
    Lane<L, P> a{lane % L, lane / L, 0, 0};
    float z[P], b[P];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int e = i * L + a.sub;
        z[i] = b[i] = 0.0f;
        if (have && e < p.E) {
            z[i] = as_float(((const T*)p.logits)[(size_t)tok * p.E + e]);
            if (p.bias) b[i] = p.bias[e];
            a.exists |= 1u << i;
            if (!(z[i] > -INFINITY) || !(b[i] > -INFINITY)) a.out |= 1u << i;
            if (p.softmax && z[i] > -INFINITY) sum += exp((double)z[i] - (double)top_z);
        }
    }
    sum = lanes_sum<L>(sum);
    choose<double, T, L, P>(p, a, tok, have, z, b, 0.0f, top_z, 1.0 / sum, c, chosen);
}

// L lanes per token (P experts each), 32 / L tokens per warp.  ORDERED: there is a bias or a choice of groups, else z alone decides.
template <typename T, int L, int P, bool ORDERED>
__global__ void __launch_bounds__(32 * WARPS) route_kernel(const RouteP p)
{
    constexpr int TOKENS = 32 / L, SLOTS = TOKENS * (8 * L < ROUTE_MAX_K ? 8 * L : ROUTE_MAX_K);
    constexpr int SCORES = 32 * (TOKENS < P ? TOKENS : P);           // [tokens][groups]
    __shared__ double shc[ORDERED ? WARPS : 1][ORDERED ? 32 * P + SCORES : 1];
    __shared__ int32_t shi[WARPS][SLOTS];
    __shared__ float shw[WARPS][SLOTS];
    __shared__ float4 sht[WARPS][TOKENS];
    __shared__ int32_t hist[ROUTE_MAX_E];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Lane<L, P> a{lane % L, lane / L, 0, 0};
    pdl_wait();
    if (p.counts) {
        for (int e = threadIdx.x; e < p.E; e += 32 * WARPS) hist[e] = 0;
        __syncthreads();
    }
    float b[P], bmax = 0.0f;
    uint32_t no_bias = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int e = i * L + a.sub;
        b[i] = ORDERED && p.bias && e < p.E ? p.bias[e] : 0.0f;
        if (!(b[i] > -INFINITY)) no_bias |= 1u << i;
        else bmax = fmaxf(bmax, fabsf(b[i]));
    }
    if (ORDERED) bmax = lanes_max<L>(bmax);
    int32_t* const chosen = shi[warp];
    for (int tok0 = (blockIdx.x * WARPS + warp) * TOKENS; tok0 < p.n; tok0 += gridDim.x * WARPS * TOKENS) {
        const int tok = tok0 + a.t;
        const bool have = tok < p.n;
        float z[P], top = -INFINITY;
        a.exists = 0;
        a.out = no_bias;
        bool bad = false;                       // a NaN (softmax: or infinity) among the logits
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int e = i * L + a.sub;
            z[i] = 0.0f;
            if (have && e < p.E) {
                z[i] = as_float(((const T*)p.logits)[(size_t)tok * p.E + e]);
                a.exists |= 1u << i;
            }
        }
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (a.exists >> i & 1) {
                if (!(z[i] > -INFINITY)) a.out |= 1u << i;
                bad |= !(z[i] < INFINITY) && (p.softmax || z[i] != z[i]);
                top = fmaxf(top, z[i]);
            }
        const uint32_t bads = __ballot_sync(FULL, bad);
        float inv = 0.0f;
        if (p.softmax) {
            top = lanes_max<L>(top);
            if (ORDERED || !p.renorm) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (a.exists >> i & 1) sum += z[i] > -INFINITY ? expf(z[i] - top) : 0.0f;
                sum = lanes_sum<L>(sum);
                inv = sum > 0.0f ? 1.0f / sum : 0.0f;
            } else {
                inv = 1.0f;                     // the weights are divided by their sum, which has exp(0) in it
            }
        }
        if constexpr (ORDERED) {
            const bool unsure = choose<float, T, L, P>(p, a, tok, have, z, b, bmax, top, inv, (float*)shc[warp], chosen);
            if (__any_sync(FULL, unsure)) {
                __syncwarp();
                choose_again<T, L, P>(p, tok, have, top, shc[warp], chosen);
            }
        } else {
            uint32_t key[P];
#pragma unroll
            for (int i = 0; i < P; ++i) key[i] = !(a.exists >> i & 1) ? 0 : a.out >> i & 1 ? Ordered<float>::NONE : Ordered<float>::key(z[i]);
            const uint32_t mine = (L == 32 ? FULL : ((1u << (L & 31)) - 1) << (a.t * L));
            for (int j = 0; j < p.k; ++j) {
                uint32_t best = key[0];
#pragma unroll
                for (int i = 1; i < P; ++i) best = key[i] > best ? key[i] : best;
                const uint32_t m = lanes_max<L>(best);
                int e = 0x7fffffff;
#pragma unroll
                for (int i = P - 1; i >= 0; --i) e = key[i] == m ? i * L + a.sub : e;
                const uint32_t equal = __ballot_sync(FULL, best == m) & mine;
                if (__any_sync(FULL, equal & (equal - 1))) e = lanes_min<L>(e);
                else e = __shfl_sync(FULL, e, __ffs(equal) - 1);
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (e == i * L + a.sub) key[i] = 0;
                if (a.sub == 0) chosen[a.t * p.k + j] = e;
            }
        }
        // weights: a lane per chosen expert
        if (a.sub == 0) {
            float4 of = make_float4(top, inv, 0.0f, 0.0f);
            sht[warp][a.t] = of;
        }
        __syncwarp();
        const int slots = min(TOKENS, p.n - tok0) * p.k;
        for (int q = lane; q < slots; q += 32) {
            const int t = q * p.kdiv >> 16, e = chosen[q];
            const float v = as_float(((const T*)p.logits)[(size_t)(tok0 + t) * p.E + e]);
            const float4 of = sht[warp][t];
            float s = p.softmax ? (v > -INFINITY ? expf(v - of.x) * of.y : 0.0f) : sigmoid(v);
            if (ORDERED && p.bias && !(p.bias[e] > -INFINITY)) s = 0.0f;
            shw[warp][q] = s;
            p.idx[(size_t)tok0 * p.k + q] = e;
            if (p.counts) atomicAdd(&hist[e], 1);
        }
        __syncwarp();
        float factor = p.scale;
        if (p.renorm) {
            float sum = 0.0f;
            if (have)
                for (int j = 0; j < p.k; ++j) sum += shw[warp][a.t * p.k + j];
            factor = p.scale / (sum + TINY);
        }
        if (bads >> (a.t * L) & (L == 32 ? FULL : (1u << (L & 31)) - 1)) factor = NAN;
        if (a.sub == 0) sht[warp][a.t].z = factor;
        __syncwarp();
        for (int q = lane; q < slots; q += 32) p.w[(size_t)tok0 * p.k + q] = shw[warp][q] * sht[warp][q * p.kdiv >> 16].z;
        __syncwarp();
    }
    if (p.counts) {
        __syncthreads();
        for (int e = threadIdx.x; e < p.E; e += 32 * WARPS)
            if (hist[e]) atomicAdd(&p.counts[e], hist[e]);
    }
}

// The gradient of the logits: the chosen experts' dg scattered into the tokens' rows in shared memory, then whole rows written.
template <typename T, int L, int P>
__global__ void __launch_bounds__(32 * WARPS) route_bwd_kernel(const RouteP p)
{
    constexpr int TOKENS = 32 / L, SLOTS = TOKENS * (8 * L < ROUTE_MAX_K ? 8 * L : ROUTE_MAX_K);
    __shared__ float shr[WARPS][32 * P];        // [tokens][E]
    __shared__ float shg[WARPS][SLOTS], shd[WARPS][SLOTS];
    __shared__ float4 sht[WARPS][TOKENS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, mt = lane / L;
    float* const row = shr[warp];
    pdl_wait();
    for (int i = lane; i < 32 * P; i += 32) row[i] = 0.0f;
    for (int tok0 = (blockIdx.x * WARPS + warp) * TOKENS; tok0 < p.n; tok0 += gridDim.x * WARPS * TOKENS) {
        const int tok = tok0 + mt, tokens = min(TOKENS, p.n - tok0), slots = tokens * p.k;
        const bool have = tok < p.n;
        float pr[P], top = -INFINITY, inv = 0.0f;
        if (p.softmax) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int e = i * L + sub;
                pr[i] = have && e < p.E ? as_float(((const T*)p.logits)[(size_t)tok * p.E + e]) : -INFINITY;
                top = fmaxf(top, pr[i]);
            }
            top = lanes_max<L>(top);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                pr[i] = pr[i] == -INFINITY ? 0.0f : expf(pr[i] - top);
                sum += pr[i];
            }
            sum = lanes_sum<L>(sum);
            inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int i = 0; i < P; ++i) pr[i] *= inv;
            if (sub == 0) sht[warp][mt] = make_float4(top, inv, 0.0f, 0.0f);
        }
        __syncwarp();
        for (int q = lane; q < slots; q += 32) {
            const int t = q * p.kdiv >> 16, e = p.top[(size_t)tok0 * p.k + q];
            float s = 0.0f;
            if (e >= 0 && e < p.E && !(p.bias && !(p.bias[e] > -INFINITY))) {
                const float v = as_float(((const T*)p.logits)[(size_t)(tok0 + t) * p.E + e]);
                s = !p.softmax ? sigmoid(v) : v == -INFINITY ? 0.0f : expf(v - sht[warp][t].x) * sht[warp][t].y;
            }
            shg[warp][q] = s;
            shd[warp][q] = p.dw[(size_t)tok0 * p.k + q];
        }
        __syncwarp();
        // per token: 1 / S, A / S, and the softmax's sum of dg p
        float over = 1.0f, mean = 0.0f, D = 0.0f;
        if (have) {
            float S = 0.0f, A = 0.0f;
            for (int j = 0; j < p.k; ++j) {
                const float g = shg[warp][mt * p.k + j];
                S += g;
                if (g != 0.0f) A = fmaf(shd[warp][mt * p.k + j], g, A);
            }
            if (p.renorm) {
                over = 1.0f / (S + TINY);
                mean = A * over;
                D = p.scale * mean * (TINY * over);             // scale / S * (A - A * (S - 1e-20) / S)
            } else {
                D = p.scale * A;
            }
        }
        if (sub == 0) {
            sht[warp][mt].z = p.scale * over;
            sht[warp][mt].w = mean;
        }
        __syncwarp();
        for (int q = lane; q < slots; q += 32) {
            const int t = q * p.kdiv >> 16, e = p.top[(size_t)tok0 * p.k + q];
            if (e < 0 || e >= p.E || (p.bias && !(p.bias[e] > -INFINITY))) continue;
            const float4 of = sht[warp][t];
            float d = of.z * (shd[warp][q] - of.w);
            if (!p.softmax) {
                const float v = as_float(((const T*)p.logits)[(size_t)(tok0 + t) * p.E + e]);
                const float s = shg[warp][q];
                d = s == 0.0f ? 0.0f : d * s * sigmoid(-v);
            }
            atomicAdd(&row[t * p.E + e], d);                    // (one writer each, unless the caller repeats an index)
        }
        __syncwarp();
        if (p.softmax) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int e = i * L + sub;
                if (have && e < p.E) row[mt * p.E + e] = pr[i] == 0.0f ? 0.0f : pr[i] * (row[mt * p.E + e] - D);
            }
            __syncwarp();
        }
        T* const out = (T*)p.dz + (size_t)tok0 * p.E;
        for (int i = lane; i < tokens * p.E; i += 32) {
            if constexpr (sizeof(T) == 4) out[i] = row[i];
            else out[i] = __float2bfloat16(row[i]);
        }
        if (p.dz16) {
            for (int t = 0; t < tokens; ++t)
                for (int e = lane; e < p.E8; e += 32)
                    p.dz16[(size_t)(tok0 + t) * p.E8 + e] = __float2bfloat16(e < p.E ? row[t * p.E + e] : 0.0f);
        }
        __syncwarp();
        for (int i = lane; i < tokens * p.E; i += 32) row[i] = 0.0f;
        __syncwarp();
    }
}

template <typename T, int L, int P> int run_fwd(const RouteP& p, cudaStream_t st)
{
    const int per = WARPS * (32 / L), want = (p.n + per - 1) / per, most = 148 * 8;
    const bool ordered = p.bias || p.top_groups < p.groups;
    MGPT_CUDA(launch_pdl(ordered ? route_kernel<T, L, P, true> : route_kernel<T, L, P, false>, want < most ? want : most, 32 * WARPS, 0, st, p));
    MGPT_LAUNCHED("route_kernel");
    return 0;
}
template <typename T, int L, int P> int run_bwd(const RouteP& p, cudaStream_t st)
{
    const int per = WARPS * (32 / L), want = (p.n + per - 1) / per, most = 148 * 8;
    MGPT_CUDA(launch_pdl(route_bwd_kernel<T, L, P>, want < most ? want : most, 32 * WARPS, 0, st, p));
    MGPT_LAUNCHED("route_bwd_kernel");
    return 0;
}
// eight experts per lane, and as many lanes as that takes
#define MGPT_BY_EXPERTS(run, T)                       \
    (p.E <= 8 ? run<T, 1, 8>(p, st)                   \
     : p.E <= 16 ? run<T, 2, 8>(p, st)                \
     : p.E <= 32 ? run<T, 4, 8>(p, st)                \
     : p.E <= 64 ? run<T, 8, 8>(p, st)                \
     : p.E <= 128 ? run<T, 16, 8>(p, st)              \
     : p.E <= 256 ? run<T, 32, 8>(p, st) : run<T, 32, 16>(p, st))

int fill(RouteP& p, const mgpt_moe_routing* r, int n, int E, int k)
{
    if (!r) return fail(MGPT_MOE_EINVAL, "null argument");
    if (n < 0 || E <= 0 || E > ROUTE_MAX_E || k <= 0 || k > ROUTE_MAX_K || k > E)
        return fail(MGPT_MOE_EINVAL, "routing: 1 to 512 experts, top_k at most 32 and at most the experts");
    if ((long long)n * k > (1ll << 30)) return fail(MGPT_MOE_EINVAL, "routing: too many tokens");
    if (r->score != MGPT_MOE_SCORE_SOFTMAX && r->score != MGPT_MOE_SCORE_SIGMOID) return fail(MGPT_MOE_EINVAL, "routing: unknown score");
    if (r->groups < 1 || r->groups > ROUTE_MAX_GROUPS || E % r->groups) return fail(MGPT_MOE_EINVAL, "routing: 1 to 32 groups, of equal size");
    if (r->top_groups < 1 || r->top_groups > r->groups) return fail(MGPT_MOE_EINVAL, "routing: top_groups must be 1 to groups");
    if (r->group_top != 1 && r->group_top != 2) return fail(MGPT_MOE_EINVAL, "routing: group_top must be 1 or 2");
    if (k > r->top_groups * (E / r->groups)) return fail(MGPT_MOE_EINVAL, "routing: top_k is more than the experts of top_groups groups");
    if (!(r->scale > -INFINITY && r->scale < INFINITY)) return fail(MGPT_MOE_EINVAL, "routing: scale must be finite");
    MGPT_TRY(check_aligned(r->bias, "bias", 4));
    p.bias = r->bias;
    p.n = n; p.E = E; p.k = k;
    p.softmax = r->score == MGPT_MOE_SCORE_SOFTMAX;
    p.groups = r->groups; p.top_groups = r->top_groups; p.group_top = r->group_top;
    p.renorm = r->renormalise != 0;
    p.scale = r->scale;
    p.gsize = E / r->groups;
    p.gdiv = ((1u << 20) + p.gsize - 1) / p.gsize;
    p.kdiv = ((1u << 16) + k - 1) / k;
    return 0;
}

// Column sums of dz, in a fixed order: blocks of rows, then the blocks.  (The layer's router bias; d_bias is added to.)
__global__ void __launch_bounds__(256) route_bias_kernel(const float* dz, int n, int E, int rows, float* part)
{
    pdl_wait();
    const int r0 = blockIdx.x * rows, r1 = min(r0 + rows, n);
    for (int e = threadIdx.x; e < E; e += 256) {
        float s = 0.0f;
        for (int r = r0; r < r1; ++r) s += dz[(size_t)r * E + e];
        part[(size_t)blockIdx.x * E + e] = s;
    }
}
__global__ void __launch_bounds__(256) route_bias_join_kernel(const float* part, int parts, int E, float* d_bias)
{
    pdl_wait();
    for (int e = threadIdx.x; e < E; e += 256) {
        float s = 0.0f;
        for (int i = 0; i < parts; ++i) s += part[(size_t)i * E + e];
        d_bias[e] += s;
    }
}

}  // namespace

// ---- the layer's routing ------------------------------------------------------------------------------------------------
int check_routing(const mgpt_moe_routing* r, int E, int k)
{
    RouteP p = {};
    return fill(p, r, 0, E, k);
}

// The router's product, then this routing over its own.  (The logits lie where the probabilities do without one: what
// a saved routing holds has to be enough for backward.)
int launch_routed(mgpt_moe_layer* L, const Workspace& w, char* ws, const void* x, int io, cudaStream_t st)
{
    const Dims& d = L->d;
    Workspace r = w;
    r.logits = w.probs;
    r.probs = w.logits;
    int32_t* const idx = (int32_t*)(ws + w.top_idx);
    float* const weights = (float*)(ws + w.top_p);
    if (tc_router_usable(L, x, io, w.n_tokens))
        MGPT_TRY(tc_router_fwd(L, r, ws, x, st));
    else
        MGPT_TRY(launch_router_fwd(x, io, L->p_data[0], L->p_data[1], w.n_tokens, d.C, d.E, d.k, (float*)(ws + r.logits), (float*)(ws + r.probs),
                                   idx, weights, st, nullptr, nullptr, L->d_status));
    RouteP p = {};
    MGPT_TRY(fill(p, &L->routing, w.n_tokens, d.E, d.k));
    p.logits = ws + r.logits; p.idx = idx; p.w = weights;
    return MGPT_BY_EXPERTS(run_fwd, float);
}

// dlogits (and their BF16 copy, where there is one) from d_top_p; d_bias, where it is given, is added to.
int launch_routed_bwd(mgpt_moe_layer* L, const Workspace& w, char* ws, bf16* dl16, int E8, float* d_bias, cudaStream_t st)
{
    const Dims& d = L->d;
    RouteP p = {};
    MGPT_TRY(fill(p, &L->routing, w.n_tokens, d.E, d.k));
    p.logits = ws + w.probs;
    p.top = (const int32_t*)(ws + w.top_idx);
    p.dw = (const float*)(ws + w.d_top_p);
    p.dz = ws + w.dlogits;
    p.dz16 = dl16;
    p.E8 = E8;
    MGPT_TRY(MGPT_BY_EXPERTS(run_bwd, float));
    if (!d_bias) return 0;
    // (rw_part has at least C + 1 rows of E floats)
    int rows = 64;
    while ((p.n + rows - 1) / rows > 256 || (p.n + rows - 1) / rows > d.C) rows *= 2;
    const int parts = (p.n + rows - 1) / rows;
    float* const part = (float*)(ws + w.rw_part);
    MGPT_CUDA(launch_pdl(route_bias_kernel, parts, 256, 0, st, (const float*)p.dz, p.n, d.E, rows, part));
    MGPT_LAUNCHED("route_bias_kernel");
    MGPT_CUDA(launch_pdl(route_bias_join_kernel, 1, 256, 0, st, part, parts, d.E, d_bias));
    MGPT_LAUNCHED("route_bias_join_kernel");
    return 0;
}

}  // namespace mgpt

using namespace mgpt;

extern "C" {

int mgpt_moe_set_routing(mgpt_moe_layer* L, const mgpt_moe_routing* r)
{
    if (!L) return fail(MGPT_MOE_EINVAL, "null layer");
    if (r) MGPT_TRY(check_routing(r, L->d.E, L->d.k));
    L->routed = r != nullptr;
    if (r) L->routing = *r;
    L->fwd_done = false;        // a backward would take the other routing's gradient
    return 0;
}

int mgpt_moe_op_route(const void* logits, int io, int n, int E, int k, const mgpt_moe_routing* r, int32_t* top_idx, float* weights,
                      int32_t* counts, mgpt_stream_t stream)
{
    RouteP p = {};
    MGPT_TRY(fill(p, r, n, E, k));
    if (io != MGPT_MOE_IO_F32 && io != MGPT_MOE_IO_BF16) return fail(MGPT_MOE_EINVAL, "unknown io dtype");
    if (n == 0) return 0;
    if (!logits || !top_idx || !weights) return fail(MGPT_MOE_EINVAL, "null argument");
    MGPT_TRY(check_aligned(logits, "logits", io == MGPT_MOE_IO_F32 ? 4 : 2));
    MGPT_TRY(check_aligned(top_idx, "top_idx", 4));
    MGPT_TRY(check_aligned(weights, "weights", 4));
    MGPT_TRY(check_aligned(counts, "counts", 4));
    p.logits = logits; p.idx = top_idx; p.w = weights; p.counts = counts;
    cudaStream_t st = (cudaStream_t)stream;
    return io == MGPT_MOE_IO_F32 ? MGPT_BY_EXPERTS(run_fwd, float) : MGPT_BY_EXPERTS(run_fwd, bf16);
}

int mgpt_moe_op_route_backward(const void* logits, int io, const int32_t* top_idx, const float* d_weights, int n, int E, int k,
                               const mgpt_moe_routing* r, void* d_logits, mgpt_stream_t stream)
{
    RouteP p = {};
    MGPT_TRY(fill(p, r, n, E, k));
    if (io != MGPT_MOE_IO_F32 && io != MGPT_MOE_IO_BF16) return fail(MGPT_MOE_EINVAL, "unknown io dtype");
    if (n == 0) return 0;
    if (!logits || !top_idx || !d_weights || !d_logits) return fail(MGPT_MOE_EINVAL, "null argument");
    MGPT_TRY(check_aligned(logits, "logits", io == MGPT_MOE_IO_F32 ? 4 : 2));
    MGPT_TRY(check_aligned(d_logits, "d_logits", io == MGPT_MOE_IO_F32 ? 4 : 2));
    MGPT_TRY(check_aligned(top_idx, "top_idx", 4));
    MGPT_TRY(check_aligned(d_weights, "d_weights", 4));
    p.logits = logits; p.top = top_idx; p.dw = d_weights; p.dz = d_logits;
    cudaStream_t st = (cudaStream_t)stream;
    return io == MGPT_MOE_IO_F32 ? MGPT_BY_EXPERTS(run_bwd, float) : MGPT_BY_EXPERTS(run_bwd, bf16);
}

}  // extern "C"
