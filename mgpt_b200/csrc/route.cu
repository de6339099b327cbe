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
    bool vec;           // E is a multiple of 4, and every row starts where four values may be moved at once
    int gsize;          // experts per group
    int group_lanes;    // lanes that hold a group, where that is a power of two of whole lanes (route_kernel), else 0
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
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
        const V other = __shfl_xor_sync(FULL, v, o);
        v = other > v ? other : v;
    }
    return v;
}
template <int L, typename V> __device__ __forceinline__ V lanes_min(V v)
{
    if constexpr (L == 32 && sizeof(V) == 4 && (V)(-1) > (V)0) return __reduce_min_sync(FULL, v);
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
__device__ __forceinline__ float max_nan(float a, float b)
{
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
// the largest, or a NaN where there is one
template <int L> __device__ __forceinline__ float lanes_max_nan(float v)
{
    if constexpr (L == 32) return Ordered<float>::value(__reduce_max_sync(FULL, Ordered<float>::key(v)));      // (max.NaN's NaN is above infinity)
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(FULL, v, o));
    return v;
}
template <int L> __device__ __forceinline__ uint32_t lanes_of(int t) { return L == 32 ? FULL : ((1u << (L & 31)) - 1) << (t * L); }

// Four neighbouring values of a row, `none` beyond its end.
__device__ __forceinline__ void load4(const float* p, float (&v)[4])
{
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void load4(const bf16* p, float (&v)[4])
{
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
    v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ void load_four(const T* row, int e, int E, bool vec, float none, float (&v)[4])
{
    if (vec) {
        if (e < E) load4(row + e, v);
        else v[0] = v[1] = v[2] = v[3] = none;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = e + c < E ? as_float(row[e + c]) : none;
    }
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(bf16* p, const float (&v)[4])
{
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(bf16* p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ float sigmoid(float z) { return 1.0f / (1.0f + expf(-z)); }

// The groups that stay, a bit each, of a token's scores c (minus infinity: out): its lanes call it.  *close: the last that stays and the first
// that does not differ by `margin` or less.  The warp's shared memory: c [tokens][E], then room for [tokens][groups].
template <typename V, int L> __device__ __forceinline__ uint32_t choose_groups(const RouteP& p, V* c, int sub, int mt, float margin, bool* close)
{
    const V NOTHING = -(V)INFINITY;
    // S lanes to a group, L / S groups at a time
    int S = L;
    while (S > 1 && L / S < p.groups) S >>= 1;
    const int first = sub / S, part = sub % S;
    V* const scores = c + (32 / L) * p.E + mt * p.groups;
    for (int g0 = 0; g0 < p.groups; g0 += L / S) {
        const int g = g0 + first;
        V m1 = NOTHING, m2 = NOTHING;
        if (g < p.groups) {
            // every S-th expert, each group from another one on (the banks of shared memory)
            const V* from = c + mt * p.E + g * p.gsize + part;
            const int count = (p.gsize - part + S - 1) / S;
            int j = count ? g % count : 0;
            for (int i = 0; i < count; ++i, j = j + 1 == count ? 0 : j + 1) {
                const V v = from[j * S];
                m2 = v > m1 ? m1 : v > m2 ? v : m2;
                m1 = v > m1 ? v : m1;
            }
        }
        for (int o = S / 2; o > 0; o >>= 1) {
            const V n1 = __shfl_xor_sync(FULL, m1, o), n2 = __shfl_xor_sync(FULL, m2, o);
            const V low = n1 > m1 ? m1 : n1;
            m1 = n1 > m1 ? n1 : m1;
            m2 = n2 > m2 ? n2 : m2;
            m2 = low > m2 ? low : m2;
        }
        if (p.group_top == 2 && m2 > NOTHING) m1 += m2;
        if (g < p.groups && part == 0) scores[g] = m1;
    }
    __syncwarp();
    uint32_t kept = 0;
    V least = INFINITY, most = NOTHING;             // of the kept, of the others
    for (int g = sub; g < p.groups; g += L) {
        const V score = scores[g];
        int before = 0;
        for (int h = 0; h < p.groups; ++h) {
            const V v = scores[h];
            before += v > score || (v == score && h < g);
        }
        if (before < p.top_groups) {
            kept |= 1u << g;
            least = score < least ? score : least;
        } else {
            most = score > most ? score : most;
        }
    }
    if (sizeof(V) == 4) *close = !((float)(lanes_min<L>(least) - lanes_max<L>(most)) > margin);
    return lanes_or<L>(kept);
}

// The chosen experts of the warp's tokens into `chosen` [tokens][k], all in FP64.  top: the token's largest logit.
template <typename T, int L, int P>
__device__ __noinline__ void choose_again(const RouteP& p, int tok, bool have, float top, double* c, int32_t* chosen)
{
    using O = Ordered<double>;
    const int lane = threadIdx.x & 31, sub = lane % L, mt = lane / L;
    O::U key[P];
    double v[P], sum = 0.0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int e = i * L + sub;
        const float z = have && e < p.E ? as_float(((const T*)p.logits)[(size_t)tok * p.E + e]) : -INFINITY;
        v[i] = z;
        if (p.softmax && z > -INFINITY) sum += exp((double)z - (double)top);
    }
    const double inv = 1.0 / lanes_sum<L>(sum);
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int e = i * L + sub;
        const float b = p.bias && e < p.E ? p.bias[e] : 0.0f;
        const bool out = !(v[i] > -INFINITY) || !(b > -INFINITY);
        double s = -INFINITY;
        if (!out) s = (p.softmax ? exp(v[i] - (double)top) * inv : 1.0 / (1.0 + exp(-v[i]))) + (double)b;
        if (e < p.E) c[mt * p.E + e] = s;
        key[i] = e >= p.E ? 0 : out ? O::NONE : O::key(p.bias ? s : v[i]);
    }
    if (p.top_groups < p.groups) {
        __syncwarp();
        bool close;
        const uint32_t kept = choose_groups<double, L>(p, c, sub, mt, 0.0f, &close);
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (!(kept >> ((uint32_t)(i * L + sub) * p.gdiv >> 20) & 1)) key[i] = 0;
    }
    for (int j = 0; j < p.k; ++j) {
        O::U best = key[0];
#pragma unroll
        for (int i = 1; i < P; ++i) best = key[i] > best ? key[i] : best;
        const O::U m = lanes_max<L>(best);
        int e = 0x7fffffff;
#pragma unroll
        for (int i = P - 1; i >= 0; --i) e = key[i] == m ? i * L + sub : e;
        e = lanes_min<L>(e);
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (e == i * L + sub) key[i] = 0;
        if (sub == 0) chosen[mt * p.k + j] = e;
    }
    __syncwarp();
}

// L lanes per token, P neighbouring experts each; 32 / L tokens per warp.  ORDERED: there is a bias or a choice of groups, else z alone decides.
//
// The rounds of the choice: a score becomes the number of steps of R / 2^23 that it is below a bound on all of them (23 bits; further
// than R: the last step), and with 511 - e in the bits below, keys are unlike each other, equal scores go by index, and a round is the
// largest key below the last round's: a subtraction and a minimum per expert, one reduction, nothing to cross out.  Two
// keys in a row that are further apart than the scores may be wrong are in the right order.  Closer ones are looked at
// when the rounds are over: those of equal inputs are, any others send the token to choose_again.
template <typename T, int L, int P, bool ORDERED>
__global__ void __launch_bounds__(32 * WARPS, P > 8 ? 4 : 8) route_kernel(const RouteP p)
{
    constexpr int TOKENS = 32 / L, SLOTS = TOKENS * (8 * L < ROUTE_MAX_K ? 8 * L : ROUTE_MAX_K);
    constexpr int SCORES = 32 * (TOKENS < P ? TOKENS : P);              // [tokens][groups]
    constexpr uint32_t LAST = (1u << 23) - 3, OUT = 1u << 9;            // the last step; the keys of experts that are out (0: there is none)
    __shared__ double shc[WARPS][32 * P + SCORES];
    __shared__ int32_t shi[WARPS][SLOTS];
    __shared__ float shw[WARPS][SLOTS];
    __shared__ float4 sht[WARPS][TOKENS];
    __shared__ int32_t hist[ROUTE_MAX_E];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, mt = lane / L, e0 = sub * P;
    pdl_wait();
    if (p.counts) {
        for (int e = threadIdx.x; e < p.E; e += 32 * WARPS) hist[e] = 0;
        __syncthreads();
    }
    const bool by_score = ORDERED && p.bias;
    float b[P], bhi = -INFINITY, blo = INFINITY;                        // (out by the bias: minus infinity)
    if constexpr (ORDERED) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            b[i] = p.bias && e0 + i < p.E ? p.bias[e0 + i] : 0.0f;
            if (b[i] > -INFINITY) {
                bhi = fmaxf(bhi, b[i]);
                blo = fminf(blo, b[i]);
            } else {
                b[i] = -INFINITY;
            }
        }
        bhi = lanes_max<L>(bhi);
        blo = lanes_min<L>(blo);
        if (!(bhi >= blo)) bhi = blo = 0.0f;
    }
    const float bmax = fmaxf(fabsf(bhi), fabsf(blo)), rounding = 6e-8f * (1.0f + bmax);       // (of a score with its bias)
    int32_t* const chosen = shi[warp];
    for (int tok0 = (blockIdx.x * WARPS + warp) * TOKENS; tok0 < p.n; tok0 += gridDim.x * WARPS * TOKENS) {
        const int tok = tok0 + mt;
        const bool have = tok < p.n;
        const T* const row = (const T*)p.logits + (size_t)tok * p.E;
        float z[P], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            float v[4];
            load_four(row, have ? e0 + i : p.E, p.E, p.vec, -INFINITY, v);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                z[i + c] = v[c];
                top = max_nan(top, v[c]);
            }
        }
        // a NaN (softmax: or infinity) among the logits
        const bool bad = __ballot_sync(FULL, top != top || (p.softmax && top == INFINITY)) & lanes_of<L>(mt);
        if (!by_score || p.softmax) top = lanes_max_nan<L>(top);
        float inv = 1.0f;                       // (what the weights are divided by has exp(0) in it, where they are all there is)
        uint32_t key[P], apart = 1;
        bool unsure = false;
        if constexpr (ORDERED) {
            float c[P];
            if (p.softmax) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    c[i] = z[i] > -INFINITY ? __expf(z[i] - top) : 0.0f;
                    sum += c[i];
                }
                sum = lanes_sum<L>(sum);
                inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
                for (int i = 0; i < P; ++i) c[i] = z[i] > -INFINITY ? fmaf(c[i], inv, b[i]) : -INFINITY;
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i) c[i] = z[i] > -INFINITY ? __fdividef(1.0f, 1.0f + __expf(-z[i])) + b[i] : -INFINITY;
            }
            // How far a score may be off.  exp: (|argument| + 2) 2^-23 of itself.  A softmax's term: that, 0.37 * 2^-23 at most, and its
            // share of the sum's error: as much in the mean (6.3 + 2) and 21 roundings; a sigmoid: (0.23 + 0.5) 2^-23, and
            // 2^-24 and 2^-22 for the sum and the quotient.
            const float most = p.softmax ? inv : 1.0f, base = p.softmax ? fmaf(2.6e-6f, inv, 8e-8f) : 4e-7f;
            uint32_t outside = 0;               // bit i: not in a group that stays
            if (p.top_groups < p.groups) {
                // (a group's score: twice that, and three roundings of twice the size)
                const float margin = 4.0f * base + 9.0f * rounding;
                if (p.group_lanes) {
                    float m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        m2 = fmaxf(m2, fminf(m1, c[i]));
                        m1 = fmaxf(m1, c[i]);
                    }
                    for (int o = p.group_lanes / 2; o > 0; o >>= 1) {
                        const float n1 = __shfl_xor_sync(FULL, m1, o), n2 = __shfl_xor_sync(FULL, m2, o);
                        m2 = fmaxf(fmaxf(m2, n2), fminf(m1, n1));
                        m1 = fmaxf(m1, n1);
                    }
                    if (p.group_top == 2 && m2 > -INFINITY) m1 += m2;
                    // the groups that may be ahead of this one (it is among them), and those that are
                    int may = -1, are = 0;
                    for (int g = 0; g < p.groups; ++g) {
                        const float d = __shfl_sync(FULL, m1, mt * L + g * p.group_lanes) - m1;
                        may += !(d <= -margin);
                        are += d > margin;
                    }
                    if (may >= p.top_groups) {
                        outside = FULL;
                        unsure = e0 < p.E && are < p.top_groups;
                    }
                } else {
                    float* const cs = (float*)shc[warp];
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        if (e0 + i < p.E) cs[mt * p.E + e0 + i] = c[i];
                    __syncwarp();
                    const uint32_t kept = choose_groups<float, L>(p, cs, sub, mt, margin, &unsure);
#pragma unroll
                    for (int i = 0; i < P; ++i) outside |= (~kept >> ((uint32_t)(e0 + i) * p.gdiv >> 20) & 1) << i;
                }
            }
            if (by_score) {
                const float bound = most + bhi + 4.0f * (base + rounding), R = fminf(bound - blo, 4.0f), S = 8388600.0f / R;
                apart = (uint32_t)fminf(2.0f * S * (base + rounding) + 4.0f, 4e6f);      // (and two roundings to steps)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const uint32_t q = min(__float_as_uint(fmaf(bound - c[i], S, 8388608.0f)) - 0x4b000000u, LAST);
                    key[i] = c[i] > -INFINITY ? (0xffffffffu - e0 - i) - (q << 9) : OUT + 511 - e0 - i;
                }
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const uint32_t q = min(__float_as_uint(fmaf(top - z[i], 524288.0f, 8388608.0f)) - 0x4b000000u, LAST);
                    key[i] = z[i] > -INFINITY ? (0xffffffffu - e0 - i) - (q << 9) : OUT + 511 - e0 - i;
                }
            }
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (e0 + i >= p.E || outside >> i & 1) key[i] = 0;
        } else {
            // (the steps order logits: R = 16, and what is in another step is further up or down)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const uint32_t q = min(__float_as_uint(fmaf(top - z[i], 524288.0f, 8388608.0f)) - 0x4b000000u, LAST);
                key[i] = e0 + i >= p.E ? 0 : z[i] > -INFINITY ? (0xffffffffu - e0 - i) - (q << 9) : OUT + 511 - e0 - i;
            }
            if (p.softmax && !p.renorm) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < P; ++i) sum += z[i] > -INFINITY ? expf(z[i] - top) : 0.0f;
                sum = lanes_sum<L>(sum);
                inv = sum > 0.0f ? 1.0f / sum : 0.0f;
            }
        }
        apart <<= 9;
        uint32_t last = 0, close = 0;
        for (int j = 0; j <= p.k; ++j) {
            // (a key that was taken is last or more: its distance is last or more, all others' is less)
            uint32_t below = last - 1 - key[0];
#pragma unroll
            for (int i = 1; i < P; ++i) below = min(below, last - 1 - key[i]);
            const uint32_t m = last - 1 - lanes_min<L>(below);
            if (j > 0 && last - m < apart && m >= 2 * OUT) close |= 1u << (j - 1);
            if (sub == 0 && j < p.k) chosen[mt * p.k + j] = 511 - (m & 511);
            last = m;
        }
        __syncwarp();
        if (__any_sync(FULL, close && !bad)) {
            if (!unsure && have && !bad)
                for (uint32_t left = close; left; left &= left - 1) {
                    const int j = __ffs(left) - 1, e = chosen[mt * p.k + j], f = j + 1 < p.k ? chosen[mt * p.k + j + 1] : 511 - (last & 511);
                    unsure |= !(as_float(row[e]) == as_float(row[f]) && (!by_score || p.bias[e] == p.bias[f]));
                }
        }
        if (__any_sync(FULL, unsure && have)) {
            // (`top` is every token's largest logit, but for a sigmoid under a bias, which does not need it)
            __syncwarp();
            choose_again<T, L, P>(p, tok, have, top, shc[warp], chosen);
        }
        // weights: a lane per chosen expert
        if (sub == 0) sht[warp][mt] = make_float4(top, inv, 0.0f, 0.0f);
        __syncwarp();
        const int slots = min(TOKENS, p.n - tok0) * p.k;
        for (int q = lane; q < slots; q += 32) {
            const int t = q * p.kdiv >> 16, e = chosen[q];
            const float v = as_float(((const T*)p.logits)[(size_t)(tok0 + t) * p.E + e]);
            const float4 of = sht[warp][t];
            float s = p.softmax ? (v > -INFINITY ? expf(v - of.x) * of.y : 0.0f) : sigmoid(v);
            if (by_score && !(p.bias[e] > -INFINITY)) s = 0.0f;
            shw[warp][q] = s;
            p.idx[(size_t)tok0 * p.k + q] = e;
            if (p.counts) atomicAdd(&hist[e], 1);
        }
        __syncwarp();
        float factor = p.scale;
        if (p.renorm) {
            float sum = 0.0f;
#pragma unroll 4
            for (int j = 0; j < p.k; ++j) sum += shw[warp][mt * p.k + j];
            factor = p.scale / (sum + TINY);
        }
        if (sub == 0) sht[warp][mt].z = bad ? NAN : factor;
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

// dg of a chosen expert: the sums of its token's weights, scale / S and A / S
struct Token {
    float of, mean;
};
__device__ __forceinline__ Token token_of(const RouteP& p, float S, float A)
{
    const float over = 1.0f / (S + TINY);
    return p.renorm ? Token{p.scale * over, A * over} : Token{p.scale, 0.0f};
}
__device__ __forceinline__ bool has_gradient(const RouteP& p, int e) { return e >= 0 && e < p.E && !(p.bias && !(p.bias[e] > -INFINITY)); }

// The gradient of a sigmoid's logits: zeros but for the chosen.  A lane per chosen expert, as many tokens per warp as that gives (at most
// ROWS / E); their values go into rows of zeros in shared memory, which are then written whole.  Bound by what is written.
constexpr int ROWS = 1024;
template <typename T> __global__ void __launch_bounds__(32 * WARPS) route_sigmoid_bwd_kernel(const RouteP p, int per_warp)
{
    __shared__ __align__(16) float shr[WARPS][ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mt = lane * p.kdiv >> 16, first = mt * p.k;
    float* const rows = shr[warp];
    for (int i = lane; i < per_warp * p.E; i += 32) rows[i] = 0.0f;
    pdl_wait();
    __syncwarp();
    for (int64_t tok0 = (int64_t)(blockIdx.x * WARPS + warp) * per_warp; tok0 < p.n; tok0 += (int64_t)gridDim.x * WARPS * per_warp) {
        const int tokens = (int)min((int64_t)per_warp, p.n - tok0);
        const bool mine = mt < tokens;
        int e = -1;
        float dw = 0.0f, g = 0.0f, rest = 0.0f;
        if (mine) {
            e = p.top[tok0 * p.k + lane];
            dw = p.dw[tok0 * p.k + lane];
            if (has_gradient(p, e)) {
                const float v = as_float(((const T*)p.logits)[(tok0 + mt) * p.E + e]);
                g = v > -INFINITY || v != v ? sigmoid(v) : 0.0f;
                rest = sigmoid(-v);
            } else {
                e = -1;
            }
        }
        float S = 0.0f, A = 0.0f;
        if (p.renorm) {
            const float product = g != 0.0f ? dw * g : 0.0f;
            for (int j = 0; j < p.k; ++j) {
                S += __shfl_sync(FULL, g, (first + j) & 31);
                A += __shfl_sync(FULL, product, (first + j) & 31);
            }
        }
        const Token of = token_of(p, S, A);
        if (e >= 0 && g != 0.0f) atomicAdd(&rows[mt * p.E + e], of.of * (dw - of.mean) * g * rest);       // (one writer each, unless the caller repeats an index)
        __syncwarp();
        T* const out = (T*)p.dz + tok0 * p.E;
        const int count = tokens * p.E;
        if (p.vec) {
            for (int i = lane * 4; i < count; i += 128) {
                float v[4];
                load4(rows + i, v);
                store4(rows + i, {0.0f, 0.0f, 0.0f, 0.0f});
                store4(out + i, v);
                if (p.dz16) store4(p.dz16 + tok0 * p.E + i, v);         // (E is E8 then, or the other way is taken)
            }
        } else {
            for (int i = lane; i < count; i += 32) store1(out + i, rows[i]);
            if (p.dz16)
                for (int t = 0; t < tokens; ++t)
                    for (int i = lane; i < p.E8; i += 32) p.dz16[(tok0 + t) * p.E8 + i] = __float2bfloat16(i < p.E ? rows[t * p.E + i] : 0.0f);
            __syncwarp();
            for (int i = lane; i < count; i += 32) rows[i] = 0.0f;
        }
        __syncwarp();
    }
}

// That of a softmax's: L lanes per token, P experts each, four neighbouring ones at a time (a warp's accesses are runs of memory).
template <typename T, int L, int P>
__global__ void __launch_bounds__(32 * WARPS) route_softmax_bwd_kernel(const RouteP p)
{
    constexpr int TOKENS = 32 / L, SLOTS = TOKENS * (8 * L < ROUTE_MAX_K ? 8 * L : ROUTE_MAX_K);
    __shared__ __align__(16) float shr[WARPS][32 * P];          // [tokens][4 L i + ..]: dg, zeros but for the chosen
    __shared__ float shg[WARPS][SLOTS], shd[WARPS][SLOTS];
    __shared__ float4 sht[WARPS][TOKENS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, mt = lane / L;
    float* const rows = shr[warp];
    for (int i = lane; i < 32 * P; i += 32) rows[i] = 0.0f;
    pdl_wait();
    for (int tok0 = (blockIdx.x * WARPS + warp) * TOKENS; tok0 < p.n; tok0 += gridDim.x * WARPS * TOKENS) {
        const int tok = tok0 + mt, slots = min(TOKENS, p.n - tok0) * p.k;
        const bool have = tok < p.n;
        const T* const row = (const T*)p.logits + (size_t)tok * p.E;
        // (asked for before the rows' arithmetic)
        int e1 = lane < slots ? p.top[(size_t)tok0 * p.k + lane] : -1;
        const float d1 = lane < slots ? p.dw[(size_t)tok0 * p.k + lane] : 0.0f;
        float pr[P], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            float v[4];
            load_four(row, have ? (i / 4 * L + sub) * 4 : p.E, p.E, p.vec, -INFINITY, v);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                pr[i + c] = v[c];
                top = max_nan(top, v[c]);
            }
        }
        top = lanes_max_nan<L>(top);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            pr[i] = pr[i] == -INFINITY ? 0.0f : expf(pr[i] - top);
            sum += pr[i];
        }
        sum = lanes_sum<L>(sum);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (sub == 0) sht[warp][mt] = make_float4(top, inv, 0.0f, 0.0f);
        __syncwarp();
        for (int q = lane; q < slots; q += 32) {
            const int t = q * p.kdiv >> 16, e = q == lane ? e1 : p.top[(size_t)tok0 * p.k + q];
            float g = 0.0f;
            if (has_gradient(p, e)) {
                const float v = as_float(((const T*)p.logits)[(size_t)(tok0 + t) * p.E + e]);
                g = v == -INFINITY ? 0.0f : expf(v - sht[warp][t].x) * sht[warp][t].y;
            }
            shg[warp][q] = g;
            shd[warp][q] = q == lane ? d1 : p.dw[(size_t)tok0 * p.k + q];
        }
        __syncwarp();
        float S = 0.0f, A = 0.0f;
        if (have)
#pragma unroll 4
            for (int j = 0; j < p.k; ++j) {
                const float g = shg[warp][mt * p.k + j], d = shd[warp][mt * p.k + j];
                S += g;
                A += g != 0.0f ? d * g : 0.0f;
            }
        const Token of = token_of(p, S, A);
        // sum of dg p: renormalised, scale / S * (A - A * (S - 1e-20) / S)
        const float D = p.renorm ? of.mean * (of.of * TINY) : p.scale * A;
        if (sub == 0) *reinterpret_cast<float2*>(&sht[warp][mt].z) = make_float2(of.of, of.mean);
        __syncwarp();
        for (int q = lane; q < slots; q += 32) {
            const int t = q * p.kdiv >> 16, e = q == lane ? e1 : p.top[(size_t)tok0 * p.k + q];
            if (has_gradient(p, e)) atomicAdd(&rows[t * L * P + e], sht[warp][t].z * (shd[warp][q] - sht[warp][t].w));
        }
        __syncwarp();
        T* const out = (T*)p.dz + (size_t)tok * p.E;
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            const int e = (i / 4 * L + sub) * 4;
            float v[4];
            load4(rows + mt * L * P + e, v);
            store4(rows + mt * L * P + e, {0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float pc = pr[i + c] * inv;
                v[c] = pc == 0.0f ? 0.0f : pc * (v[c] - D);
            }
            if (!have || e >= p.E) continue;
            if (p.vec) {
                store4(out + e, v);
                if (p.dz16) store4(p.dz16 + (size_t)tok * p.E + e, v);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (e + c < p.E) store1(out + e + c, v[c]);
                    if (p.dz16 && e + c < p.E8) p.dz16[(size_t)tok * p.E8 + e + c] = __float2bfloat16(e + c < p.E ? v[c] : 0.0f);
                }
            }
        }
        if (p.dz16 && !p.vec && have)           // (what of the padding lies beyond the last four)
            for (int e = (p.E + 3) / 4 * 4 + sub; e < p.E8; e += L) p.dz16[(size_t)tok * p.E8 + e] = __float2bfloat16(0.0f);
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
template <typename T, int L, int P> int run_softmax_bwd(const RouteP& p, cudaStream_t st)
{
    const int per = WARPS * (32 / L), want = (p.n + per - 1) / per, most = 148 * 8;
    MGPT_CUDA(launch_pdl(route_softmax_bwd_kernel<T, L, P>, want < most ? want : most, 32 * WARPS, 0, st, p));
    MGPT_LAUNCHED("route_softmax_bwd_kernel");
    return 0;
}
template <typename T> int run_sigmoid_bwd(const RouteP& p, cudaStream_t st)
{
    int per_warp = 32 / p.k;
    if (per_warp > ROWS / p.E) per_warp = ROWS / p.E;
    const int per = WARPS * per_warp, want = (p.n + per - 1) / per, most = 148 * 8;
    MGPT_CUDA(launch_pdl(route_sigmoid_bwd_kernel<T>, want < most ? want : most, 32 * WARPS, 0, st, p, per_warp));
    MGPT_LAUNCHED("route_sigmoid_bwd_kernel");
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

template <typename T> int run_fwd(RouteP& p, cudaStream_t st)
{
    p.vec = p.E % 4 == 0 && ((uintptr_t)p.logits & (4 * sizeof(T) - 1)) == 0;
    const int per_lane = p.E <= 256 ? 8 : 16, lanes = p.gsize / per_lane;
    p.group_lanes = p.gsize % per_lane == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    return MGPT_BY_EXPERTS(run_fwd, T);
}
template <typename T> int run_bwd(RouteP& p, cudaStream_t st)
{
    p.vec = p.E % 4 == 0 && (((uintptr_t)p.logits | (uintptr_t)p.dz) & (4 * sizeof(T) - 1)) == 0 && (!p.dz16 || p.E8 == p.E);
    return p.softmax ? MGPT_BY_EXPERTS(run_softmax_bwd, T) : run_sigmoid_bwd<T>(p, st);
}

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
    return run_fwd<float>(p, st);
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
    MGPT_TRY(run_bwd<float>(p, st));
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
    return io == MGPT_MOE_IO_F32 ? run_fwd<float>(p, st) : run_fwd<bf16>(p, st);
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
    return io == MGPT_MOE_IO_F32 ? run_bwd<float>(p, st) : run_bwd<bf16>(p, st);
}

}  // extern "C"
