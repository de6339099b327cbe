// Routing to experts from their logits, and its gradient.  Token with logits z, bias b (order only), k chosen:
//
//   s_e = 1 / (1 + exp(-z_e))   or   exp(z_e) / sum exp(z),      c_e = s_e + b_e
//   the top_groups groups of consecutive experts with the largest sums of their group_top largest c stay;
//   chosen are their k largest c in falling order, equal ones by index; without a bias the order is that of z itself
//   w_j = scale * s_j / (sum of the chosen s + 1e-20)   or   scale * s_j
//
// Gradient, with S the sum of the chosen s plus 1e-20, A = sum dw_j s_j and T_j = sum_i s_i (dw_j - dw_i):
//   dg_j = scale / S * (dw_j - A / S) = scale / S * (T_j + 1e-20 dw_j) / S   or   scale * dw_j
//   sigmoid: dz_e = dg_j s_j (1 - s_j) for the chosen, 0 elsewhere;   softmax: dz_e = p_e ([chosen] dg_j - sum_j dg_j p_j),
//   of weights as they are scale p_e (T_j + dw_j * the sum of the p that were not chosen) for the chosen, -scale p_e A elsewhere
// (dw_j - A / S and dw_j - A as they stand have no digits left where one expert has nearly all of S; of a single chosen expert they are rounding.)
// The reference has clamped softmax and top-k only (utils/Tensor.cpp:850-909).
//
// What is chosen is what exact arithmetic chooses (up to FP64's rounding): scores are formed in FP32 with a known bound on their
// error, and what is closer than that is settled by exact values: of the few experts concerned, of a group's largest, or (a logit of
// infinity or a NaN, biases of very different size, long runs of equals) of all.  What is chosen does not depend on which way that goes.
//
// Bytes: the logits once, the weights and indices; backward the gradients' bytes, for a softmax the logits too.  Forward reaches no limit of the
// chip: about 180 instructions per token of 128 experts and 8 chosen, 690 per token of 256 in groups, at 52 to 58 % of the issue slots and 49 to 54 %
// of the integer pipe (minima and comparisons, at half the rate of additions), with 28 to 30 % of the warps: the rounds' reductions wait for one
// another.  us in a graph on a B200, FP32 logits: 8 x 256 in groups 4.4, 32768 x 64, 4 chosen 8.6, 32768 x 256 in groups, 8 chosen 35 (floor
// 5.3), 131072 x 128, 8 chosen 37 (floor 12).  Of equal logits, which BF16 has among the first k + 1 in 10 % of the tokens at 64 experts and a third at
// 128 and 256, the order is settled like that of close ones: 32768 x 64 10.5 us in BF16 against 7.3 in FP32 (without counts), 131072 x 128 64 against
// 37.  Backward: 32768 x 256 (sigmoid) 7.9 (4.3 TB/s), 131072 x 128 (softmax) 27.5 (4.9 TB/s; with six blocks per SM 29), of weights as they are
// 30.  Of the forward call 2 us are the counts' atomics, where counts are asked for.
// Not kept: the eight least by sorting and merging lists (38 against 36 us, 39 against 35: more minima), two warps per block (44 against 38),
// six to eight blocks per SM (37 to 41 against 36).
#include "common.cuh"

#include <cstring>

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
    uint32_t kdiv;      // 2^16 / k, rounded up: q * kdiv >> 16 is q / k for q < 512, as many as a warp's tokens have (q * (k - 1) < 2^16)
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

// Numbers as unsigned integers of the same order, and back.
__device__ __forceinline__ uint32_t ordered(float v)
{
    const uint32_t u = __float_as_uint(v);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
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
    if constexpr (L == 32 && sizeof(V) == 4 && (V)(-1) > (V)0) {
        return __reduce_min_sync(FULL, v);
    } else {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
            const V other = __shfl_xor_sync(FULL, v, o);
            v = other < v ? other : v;
        }
        return v;
    }
}
template <int L, typename V> __device__ __forceinline__ V lanes_sum(V v)
{
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
template <int L> __device__ __forceinline__ uint32_t lanes_or(uint32_t v)
{
    if constexpr (L == 32) {
        return __reduce_or_sync(FULL, v);
    } else {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) v |= __shfl_xor_sync(FULL, v, o);
        return v;
    }
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
    if constexpr (L == 32) {
        return from_ordered(__reduce_max_sync(FULL, ordered(v)));          // (max.NaN's NaN is above infinity)
    } else {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(FULL, v, o));
        return v;
    }
}
template <int L> __device__ __forceinline__ uint32_t lanes_of(int t) { return L == 32 ? FULL : ((1u << (L & 31)) - 1) << (t * L); }

// Four neighbouring values of a row, `none` beyond its end.
__device__ __forceinline__ void load4(const float* p, float (&v)[4])
{
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
// from global memory, here and not where the values are needed first
__device__ __forceinline__ void fetch4(const float* p, float (&v)[4])
{
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "l"(p));
}
__device__ __forceinline__ void fetch4(const bf16* p, float (&v)[4])
{
    uint2 a;
    asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(a.x), "=r"(a.y) : "l"(p));
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
    v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ void load_four(const T* row, int e, int E, bool vec, float none, float (&v)[4])
{
    if (vec) {
        if (e < E) fetch4(row + e, v);
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

// (of numbers far below zero too: neither exponential is infinite)
__device__ __forceinline__ float sigmoid(float z)
{
    const float e = expf(-fabsf(z));
    return (z < 0.0f ? e : 1.0f) / (1.0f + e);
}

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

// A token's weights from its chosen experts: a lane per chosen expert of the warp's tokens.  sht: top and 1 / sum of exp(z - top), then the factor.
template <typename T, int L>
__device__ __forceinline__ void weigh(const RouteP& p, int tok0, const int32_t* chosen, float* weights, float4* sht, int32_t* hist, float top, float inv, bool bad)
{
    const int lane = threadIdx.x & 31, sub = lane % L, mt = lane / L;
    if (sub == 0) sht[mt] = make_float4(top, inv, 0.0f, 0.0f);
    __syncwarp();
    const int slots = min(32 / L, p.n - tok0) * p.k;
    for (int q = lane; q < slots; q += 32) {
        const int t = q * p.kdiv >> 16, e = chosen[q];
        const float v = as_float(((const T*)p.logits)[(size_t)(tok0 + t) * p.E + e]);
        const float4 of = sht[t];
        float s = p.softmax ? (v > -INFINITY ? expf(v - of.x) * of.y : 0.0f) : sigmoid(v);
        if (p.bias && !(p.bias[e] > -INFINITY)) s = 0.0f;
        weights[q] = s;
        p.idx[(size_t)tok0 * p.k + q] = e;
        if (p.counts) atomicAdd(&hist[e], 1);
    }
    __syncwarp();
    float factor = p.scale;
    if (p.renorm) {
        float sum = 0.0f;
#pragma unroll 4
        for (int j = 0; j < p.k; ++j) sum += weights[mt * p.k + j];
        factor = p.scale / (sum + TINY);
    }
    if (sub == 0) sht[mt].z = bad ? NAN : factor;
    __syncwarp();
    for (int q = lane; q < slots; q += 32) p.w[(size_t)tok0 * p.k + q] = weights[q] * sht[q * p.kdiv >> 16].z;
    __syncwarp();
}

// The tokens of a warp from their logits, all scores in FP64.  (Loops rather than unrolled code: this is rare, and what is not in the
// instruction cache costs more than it computes.)  c: [tokens][E] scores, then [tokens][groups].
template <typename T, int L>
__device__ __noinline__ void route_again(const RouteP& p, int tok0, double* c, int32_t* chosen, float4* sht, int32_t* hist)
{
    const int lane = threadIdx.x & 31, sub = lane % L, mt = lane / L, tok = tok0 + mt;
    const bool have = tok < p.n;
    const T* const row = (const T*)p.logits + (size_t)tok * p.E;
    double* const mine = c + mt * p.E;
    float top = -INFINITY;                      // of the numbers
    bool bad = false;
    uint32_t taken = 0;                         // bits of the lane's experts i * L + sub
#pragma unroll 4
    for (int e = sub; e < p.E; e += L) {
        const float z = have ? as_float(row[e]) : -INFINITY;
        bad |= z != z;
        top = fmaxf(top, z);
    }
    top = lanes_max<L>(top);
    bad = (__ballot_sync(FULL, bad) & lanes_of<L>(mt)) || (p.softmax && top == INFINITY);
    double inv = 1.0;
    if (p.softmax) {
        double sum = 0.0;
#pragma unroll 2
        for (int e = sub; e < p.E; e += L) {
            const float z = have ? as_float(row[e]) : -INFINITY;
            const double s = z == top && z > -INFINITY ? 1.0 : z > -INFINITY ? exp((double)z - (double)top) : 0.0;      // (+inf less itself is no number)
            mine[e] = s;
            sum += s;
        }
        sum = lanes_sum<L>(sum);
        inv = sum > 0.0 ? 1.0 / sum : 0.0;
    }
    // (minus infinity: out)
#pragma unroll 2
    for (int e = sub; e < p.E; e += L) {
        const float z = have ? as_float(row[e]) : -INFINITY;
        double s = p.softmax ? mine[e] * inv : 1.0 / (1.0 + exp(-(double)z));
        if (p.bias) s = p.bias[e] > -INFINITY ? s + (double)p.bias[e] : -INFINITY;
        mine[e] = z > -INFINITY && s > -INFINITY ? s : -INFINITY;
    }
    if (p.top_groups < p.groups) {
        __syncwarp();
        bool close;
        const uint32_t kept = choose_groups<double, L>(p, c, sub, mt, 0.0f, &close);
        for (int i = 0, e = sub; e < p.E; ++i, e += L)
            if (!(kept >> ((uint32_t)e * p.gdiv >> 20) & 1)) taken |= 1u << i;
    }
    if (!p.bias && have)                        // the logits' own order
        for (int e = sub; e < p.E; e += L) mine[e] = as_float(row[e]) > -INFINITY ? (double)as_float(row[e]) : -INFINITY;
    for (int j = 0; j < p.k; ++j) {
        constexpr int NOBODY = 0x7fffffff;
        double best = -INFINITY;
        int at = NOBODY;
#pragma unroll 4
        for (int i = 0, e = sub; e < p.E; ++i, e += L) {
            const double v = mine[e];
            if (!(taken >> i & 1) && (at == NOBODY || v > best)) {
                best = v;
                at = e;
            }
        }
        const double m = lanes_max<L>(best);
        const int e = lanes_min<L>(best == m ? at : NOBODY);
        if (e % L == sub) taken |= 1u << (e / L);
        if (sub == 0) chosen[mt * p.k + j] = e;
    }
    __syncwarp();
    weigh<T, L>(p, tok0, chosen, (float*)c, sht, hist, top, (float)inv, bad);
}

// exp(-z) and 1 / x to 2^-22 of themselves and the argument's rounding (of scores that only have to be near enough)
__device__ __forceinline__ float near_exp(float v)
{
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * 1.4426950409f));
    return e;
}
__device__ __forceinline__ float near_over(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Whether a lane's group stays: known (`stays`), or `open`, and then by exact values of its experts that may be among its largest, those whose
// score is near `least` or above.  Lanes of groups (route_kernel).
template <typename T, int L, int P>
__device__ __noinline__ bool settle_group(const RouteP& p, int tok, bool have, float top, float least, bool open, bool stays)
{
    const int lane = threadIdx.x & 31, sub = lane % L, mt = lane / L, e0 = sub * P;
    const T* const row = (const T*)p.logits + (size_t)tok * p.E;
    double over = 1.0, d1 = -INFINITY, d2 = -INFINITY;
    open &= have;
    if (p.softmax) {
        double sum = 0.0;
#pragma unroll 2
        for (int e = sub; e < p.E; e += L)
            if (have && as_float(row[e]) > -INFINITY) sum += exp((double)as_float(row[e]) - (double)top);
        over = 1.0 / lanes_sum<L>(sum);
    }
    if (open)
        for (int i = 0; i < P; ++i) {
            const float z = as_float(row[e0 + i]), b = p.bias ? p.bias[e0 + i] : 0.0f;
            const float c = (p.softmax ? near_exp(z - top) * (float)over : near_over(1.0f + near_exp(-z))) + b;
            if (!(z > -INFINITY) || !(c >= least)) continue;
            const double v = (p.softmax ? exp((double)z - (double)top) * over : 1.0 / (1.0 + exp(-(double)z))) + (double)b;
            d2 = v > d1 ? d1 : v > d2 ? v : d2;
            d1 = v > d1 ? v : d1;
        }
    for (int o = p.group_lanes / 2; o > 0; o >>= 1) {
        const double n1 = __shfl_xor_sync(FULL, d1, o), n2 = __shfl_xor_sync(FULL, d2, o);
        const double low = n1 > d1 ? d1 : n1;
        d1 = n1 > d1 ? n1 : d1;
        d2 = n2 > d2 ? n2 : d2;
        d2 = low > d2 ? low : d2;
    }
    if (p.group_top == 2 && d2 > -INFINITY) d1 += d2;
    int before = 0;
    for (int g = 0; g < p.groups; ++g) {
        const int from = mt * L + g * p.group_lanes, state = __shfl_sync(FULL, stays ? 2 : open ? 1 : 0, from);
        const double d = __shfl_sync(FULL, d1, from);
        before += state == 2 || (state == 1 && (d > d1 || (d == d1 && g * p.group_lanes < sub - sub % p.group_lanes)));
    }
    return open ? before < p.top_groups : stays;
}

// L lanes per token, P experts each; 32 / L tokens per warp.
//
// The rounds of the choice: a score becomes the number of steps of R / 2^23 that it is below a bound on all of them (23 bits; further
// than R: the last step, and so is what is out), with e + 1 added below: keys are unlike each other, equal scores go by index, and a round
// is the least key above the last round's: an addition and a minimum per expert, one reduction, nothing to cross out.  Two
// keys in a row that are further apart than the scores may be wrong are in the right order.  Where some are not, what was chosen and
// what is not far enough behind it are put in order by their exact values (FP64; the logits themselves where they decide).  Of groups
// whose scores are too close settle_group decides; a token that is none of this (see `unsure`) is left to route_again.
enum { BY_LOGIT, BY_SCORE, BY_GROUP };          // no bias and no choice of groups; a bias; groups
template <typename T, int L, int P, int HOW>
__global__ void __launch_bounds__(32 * WARPS, P > 8 ? 5 : 8) route_kernel(const RouteP p)
{
    constexpr int TOKENS = 32 / L, KM = P * L < ROUTE_MAX_K ? P * L : ROUTE_MAX_K, EXTRA = 4;
    constexpr int FOR_GROUPS = 32 * P + 32 * (TOKENS < P ? TOKENS : P), FOR_ORDER = TOKENS * (KM + EXTRA + EXTRA / 2 + KM / 2);
    constexpr uint32_t LAST = 0x4b000000u + (1u << 23) - 3, NONE = 0xffffffffu;     // the last step, as a number of 2^23 and more; no expert
    __shared__ double shc[WARPS][FOR_GROUPS > FOR_ORDER ? FOR_GROUPS : FOR_ORDER];
    __shared__ int32_t shi[WARPS][TOKENS * KM];
    __shared__ float4 sht[WARPS][TOKENS];
    __shared__ int32_t hist[ROUTE_MAX_E];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, mt = lane / L;
    // The lane's experts: neighbours, so that a group is a run of lanes; else four and four (a warp's loads are runs of memory).
    const int e0 = HOW == BY_GROUP ? sub * P : sub * 4;
    auto expert = [&](int i) { return e0 + (HOW == BY_GROUP ? i : i / 4 * (4 * L) + i % 4); };
    double* const scratch = shc[warp];
    pdl_wait();
    if (p.counts) {
        for (int e = threadIdx.x; e < p.E; e += 32 * WARPS) hist[e] = 0;
        __syncthreads();
    }
    const bool by_score = HOW == BY_SCORE || (HOW == BY_GROUP && p.bias);
    float b[P], bhi = -INFINITY, blo = INFINITY;                        // (out by the bias: minus infinity)
    if constexpr (HOW != BY_LOGIT) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            b[i] = p.bias && expert(i) < p.E ? p.bias[expert(i)] : 0.0f;
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
    // Steps of scores.  How far a score may be off (base).  exp: (|argument| + 2) 2^-23 of itself.  A softmax's term: that, 0.37 * 2^-23 at
    // most, and its share of the sum's error: as much in the mean (6.3 + 2) and 21 roundings; a sigmoid: (0.23 + 0.5) 2^-23, and
    // 2^-24 and 2^-22 for the sum and the quotient.  A softmax's largest term, and so all of this, is its token's.
    float base, bound, S;
    uint32_t apart = 1u << 9;
    auto steps = [&](float most) {
        base = p.softmax ? fmaf(2.6e-6f, most, 8e-8f) : 4e-7f;
        bound = most + bhi + 4.0f * (base + rounding);
        S = __fdividef(8388600.0f, fminf(bound - blo, 4.0f));
        if (by_score) apart = (uint32_t)fminf(2.0f * S * (base + rounding) + 4.0f, 4e6f) << 9;      // (and two roundings to steps)
    };
    steps(1.0f);
    int32_t* const chosen = shi[warp];
    const int stride = gridDim.x * WARPS * TOKENS;
    float z[P];
    auto load = [&](int tok) {
        const T* const row = (const T*)p.logits + (size_t)tok * p.E;
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            float v[4];
            load_four(row, tok < p.n ? expert(i) : p.E, p.E, p.vec, -INFINITY, v);
#pragma unroll
            for (int c = 0; c < 4; ++c) z[i + c] = v[c];
        }
    };
    int begin = (blockIdx.x * WARPS + warp) * TOKENS;
    load(begin + mt);
    for (; begin < p.n; begin += 32 * stride) {
        uint32_t again = 0;                     // of 32 rounds of the loop, those with tokens that need route_again
        for (int round = 0, tok0 = begin; round < 32 && tok0 < p.n; ++round, tok0 += stride) {
            const int tok = tok0 + mt;
            const bool have = tok < p.n;
            float top = z[0];
#pragma unroll
            for (int i = 1; i < P; ++i) top = max_nan(top, z[i]);
            // a NaN (softmax: or infinity) among the logits
            const unsigned none = __ballot_sync(FULL, top != top || (p.softmax && top == INFINITY));
            if (HOW == BY_LOGIT && __builtin_expect(none, 0)) {      // (32768 x 256 in groups: 38 us in place of 34.7)
                again |= 1u << round;
                load(tok + stride);
                continue;
            }
            const bool bad = HOW != BY_LOGIT && none & lanes_of<L>(mt);
            bool unsure = bad || (HOW != BY_LOGIT && top == INFINITY);
            if (!by_score || p.softmax) top = lanes_max_nan<L>(top);
            float inv = 1.0f;                   // (what the weights are divided by has exp(0) in it, where they are all there is)
            uint32_t key[P];
            bool aside = false;                 // the lane's experts are not in a group that stays
            if constexpr (HOW != BY_LOGIT) {
                float c[P];                     // (NaN: out.  A logit of infinity has been seen to above)
                if (p.softmax) {
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        c[i] = z[i] > -INFINITY ? near_exp(z[i] - top) : 0.0f;
                        sum += c[i];
                    }
                    sum = lanes_sum<L>(sum);
                    inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
                    for (int i = 0; i < P; ++i) c[i] = fmaf(c[i], inv, fmaf(z[i], 0.0f, b[i]));
                } else {
#pragma unroll
                    for (int i = 0; i < P; ++i) c[i] = near_over(1.0f + near_exp(-z[i])) + fmaf(z[i], 0.0f, b[i]);
                }
                if (p.softmax) steps(inv);
                uint32_t outside = 0;           // bit i: not in a group that stays, where groups are not runs of lanes
                if constexpr (HOW == BY_GROUP) {
                    // (a group's score: twice that, and three roundings of twice the size)
                    const float margin = 4.0f * base + 9.0f * rounding;
                    if (p.group_lanes) {
                        float m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < P; ++i) {
                            const float v = fmaxf(c[i], -INFINITY);     // (of a NaN: the other)
                            m2 = fmaxf(m2, fminf(m1, v));
                            m1 = fmaxf(m1, v);
                        }
                        for (int o = p.group_lanes / 2; o > 0; o >>= 1) {
                            const float n1 = __shfl_xor_sync(FULL, m1, o), n2 = __shfl_xor_sync(FULL, m2, o);
                            m2 = fmaxf(fmaxf(m2, n2), fminf(m1, n1));
                            m1 = fmaxf(m1, n1);
                        }
                        const float least = p.group_top == 2 ? m2 : m1;
                        if (p.group_top == 2 && m2 > -INFINITY) m1 += m2;
                        // the groups that may be ahead of this one (it is among them), and those that are
                        int may = -1, are = 0;
                        for (int g = 0; g < p.groups; ++g) {
                            const float d = __shfl_sync(FULL, m1, mt * L + g * p.group_lanes) - m1;
                            may += !(d <= -margin);
                            are += d > margin;
                        }
                        bool stays = may < p.top_groups;
                        const bool open = e0 < p.E && !stays && are < p.top_groups;
                        if (__builtin_expect(__any_sync(FULL, open && have && !bad && margin < 1e-3f), 0)) stays = settle_group<T, L, P>(p, tok, have, top, least - margin, open && !bad, stays);
                        else unsure |= open;
                        aside = !stays;
                    } else {
                        float* const cs = (float*)scratch;
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < P; ++i)
                            if (expert(i) < p.E) cs[mt * p.E + expert(i)] = c[i];
                        __syncwarp();
                        bool near;
                        const uint32_t kept = choose_groups<float, L>(p, cs, sub, mt, margin, &near);
                        unsure |= near;
#pragma unroll
                        for (int i = 0; i < P; ++i) outside |= (~kept >> ((uint32_t)expert(i) * p.gdiv >> 20) & 1) << i;
                    }
                }
                if (by_score) {
#pragma unroll
                    for (int i = 0; i < P; ++i) key[i] = (min(__float_as_uint(fmaf(bound - c[i], S, 8388608.0f)), LAST) << 9) + (expert(i) + 1);
                } else {
#pragma unroll
                    for (int i = 0; i < P; ++i) key[i] = (min(__float_as_uint(fmaf(top - z[i], 524288.0f, 8388608.0f)), LAST) << 9) + (expert(i) + 1);
                }
                if (HOW == BY_GROUP && !p.group_lanes) {
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        if (outside >> i & 1) key[i] = NONE;
                }
                unsure = __ballot_sync(FULL, unsure) & lanes_of<L>(mt);         // (of all the token's lanes: there may be fewer than k keys then)
            } else {
                // (the steps order logits: R = 16, and what is in another step is further up or down)
#pragma unroll
                for (int i = 0; i < P; ++i) key[i] = (min(__float_as_uint(fmaf(top - z[i], 524288.0f, 8388608.0f)), LAST) << 9) + (expert(i) + 1);
                if (p.softmax && !p.renorm) {
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < P; ++i) sum += z[i] > -INFINITY ? expf(z[i] - top) : 0.0f;
                    sum = lanes_sum<L>(sum);
                    inv = sum > 0.0f ? 1.0f / sum : 0.0f;
                }
            }
            if (p.E != L * P) {
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (expert(i) >= p.E) key[i] = NONE;
            }
            load(tok + stride);                 // (what the next round needs, on its way meanwhile)
            // the least key above `last` (a key that was taken is further, modulo 2^32, than any other), and one less than how far it is
            auto beyond = [&](uint32_t last, uint32_t* m) {
                const uint32_t from = ~last;
                uint32_t part[4];               // (chains side by side)
#pragma unroll
                for (int i = 0; i < P; ++i) part[i % 4] = i < 4 ? key[i] + from : min(key[i] + from, part[i % 4]);
                uint32_t next = min(min(part[0], part[1]), min(part[2], part[3]));
                if (HOW == BY_GROUP && aside) next = NONE + from;
                next = lanes_min<L>(next);
                *m = next - from;
                return next;
            };
            uint32_t last = NONE, close = 0, bit = 0;
            int32_t* const to = chosen + mt * p.k;
            for (int j = 0; j < p.k; ++j) {
                if (beyond(last, &last) < apart) close |= bit;
                bit = bit ? bit << 1 : 1;
                if (sub == 0) to[j] = (last - 1) & 511;
            }
            uint32_t next;                      // the first that was not chosen
            if (beyond(last, &next) < apart && next != NONE && next > last) close |= bit;
            __syncwarp();
            if (__builtin_expect(__any_sync(FULL, close && !unsure), 0)) {
                double* const value = scratch + mt * (KM + EXTRA);
                int32_t* const behind = (int32_t*)(scratch + TOKENS * (KM + EXTRA)) + mt * EXTRA;
                int32_t* const sorted = (int32_t*)(scratch + TOKENS * (KM + EXTRA + EXTRA / 2)) + mt * KM;
                const T* const row = (const T*)p.logits + (size_t)tok * p.E;
                int count = close && have && !unsure ? p.k : 0;
                bool more = count && close & bit;
                while (__any_sync(FULL, more)) {
                    if (more) {
                        if (count < p.k + EXTRA) {
                            if (sub == 0) behind[count - p.k] = (next - 1) & 511;
                            ++count;
                        } else {
                            unsure = true;
                            more = false;
                            count = 0;
                        }
                    }
                    uint32_t m;
                    const uint32_t step = beyond(next, &m);
                    if (step >= apart || m == NONE || m < next) more = false;
                    if (more) next = m;
                }
                double over = 1.0;
                if (by_score && p.softmax) {
                    double sum = 0.0;
#pragma unroll 2
                    for (int e = sub; e < p.E; e += L)
                        if (count && as_float(row[e]) > -INFINITY) sum += exp((double)as_float(row[e]) - (double)top);
                    over = 1.0 / lanes_sum<L>(sum);
                }
                __syncwarp();
                for (int j = sub; j < count; j += L) {
                    const int e = j < p.k ? to[j] : behind[j - p.k];
                    const float x = as_float(row[e]), y = by_score ? p.bias[e] : 0.0f;
                    double v = x;
                    if (by_score) v = (p.softmax ? exp(v - (double)top) * over : 1.0 / (1.0 + exp(-v))) + (double)y;
                    value[j] = x > -INFINITY && y > -INFINITY ? v : -INFINITY;
                }
                __syncwarp();
                for (int j = sub; j < count; j += L) {
                    const int e = j < p.k ? to[j] : behind[j - p.k];
                    const double v = value[j];
                    int before = 0;
                    for (int i = 0; i < count; ++i) before += value[i] > v || (value[i] == v && (i < p.k ? to[i] : behind[i - p.k]) < e);
                    if (before < p.k) sorted[before] = e;
                }
                __syncwarp();
                if (count)
                    for (int j = sub; j < p.k; j += L) to[j] = sorted[j];
                __syncwarp();
            }
            if (__any_sync(FULL, unsure && have)) again |= 1u << round;
            else weigh<T, L>(p, tok0, chosen, (float*)scratch, sht[warp], hist, top, inv, false);
        }
        for (; again; again &= again - 1) route_again<T, L>(p, begin + (__ffs(again) - 1) * stride, scratch, chosen, sht[warp], hist);
    }
    if (p.counts) {
        __syncthreads();
        for (int e = threadIdx.x; e < p.E; e += 32 * WARPS)
            if (hist[e]) atomicAdd(&p.counts[e], hist[e]);
    }
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
        float share = g;                        // with its factor, dg of the weight
        if (p.renorm) {
            const float known = g != 0.0f ? dw : 0.0f;
            float S = 0.0f, diff = 0.0f;
            for (int j = 0; j < p.k; ++j) {
                const float gj = __shfl_sync(FULL, g, (first + j) & 31);
                S += gj;
                diff = fmaf(gj, dw - __shfl_sync(FULL, known, (first + j) & 31), diff);
            }
            const float over = 1.0f / (S + TINY);
            share *= over;
            dw = fmaf(TINY, dw, diff) * over;
        }
        if (e >= 0 && g != 0.0f) atomicAdd(&rows[mt * p.E + e], p.scale * dw * share * rest);       // (one writer each, unless the caller repeats an index)
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

// That of a softmax's: L lanes per token, at least as many as there are chosen experts, P experts each, four neighbouring ones at a time (a
// warp's accesses are runs of memory).  The next tokens' logits are on their way while these are worked on.
template <typename T, int L, int P, bool RENORM>
__global__ void __launch_bounds__(32 * WARPS, 8) route_softmax_bwd_kernel(const RouteP p)
{
    constexpr int TOKENS = 32 / L;
    __shared__ __align__(16) float shr[WARPS][32 * P];          // [tokens][L * P]: dg, zeros but for the chosen
    __shared__ uint32_t shb[RENORM ? 1 : WARPS][32];            // bits of a lane's experts that were chosen, for weights as they are
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, mt = lane / L;
    const int ct = min((int)(lane * p.kdiv >> 16), TOKENS - 1), cj = lane - ct * p.k;      // the token and place of the lane's chosen expert (cj < k)
    float* const rows = shr[warp];
    uint32_t* const bits = shb[RENORM ? 0 : warp];
    for (int i = lane; i < 32 * P; i += 32) rows[i] = 0.0f;
    if (!RENORM) bits[lane] = 0;
    pdl_wait();
    const int stride = gridDim.x * WARPS * TOKENS;
    int tok0 = (blockIdx.x * WARPS + warp) * TOKENS;
    float z[P], dw = 0.0f, v = 0.0f;
    int e = -1;
    auto load = [&](int tok0) {
        const int tok = tok0 + mt;
        const T* const row = (const T*)p.logits + (size_t)tok * p.E;
        e = -1;
        if (cj < p.k && tok0 + ct < p.n) {
            e = p.top[(size_t)(tok0 + ct) * p.k + cj];
            dw = p.dw[(size_t)(tok0 + ct) * p.k + cj];
        }
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            float four[4];
            load_four(row, tok < p.n ? (i / 4 * L + sub) * 4 : p.E, p.E, p.vec, -INFINITY, four);
#pragma unroll
            for (int c = 0; c < 4; ++c) z[i + c] = four[c];
        }
    };
    load(tok0);
    __syncwarp();
    for (; tok0 < p.n; tok0 += stride) {
        const int tok = tok0 + mt, e1 = e;
        const bool have = tok < p.n;
        bool mine = has_gradient(p, e1);
        float dw1 = dw, rest = 0.0f;
        if (mine) v = as_float(((const T*)p.logits)[(size_t)(tok0 + ct) * p.E + e1]);
        float pr[P], top = z[0], sum = 0.0f;
#pragma unroll
        for (int i = 1; i < P; ++i) top = max_nan(top, z[i]);
        top = lanes_max_nan<L>(top);
        if (top == -INFINITY) top = 0.0f;       // (all out: zeros)
#pragma unroll
        for (int i = 0; i < P; ++i) {
            pr[i] = expf(z[i] - top);
            sum += pr[i];
        }
        load(tok0 + stride);
        sum = lanes_sum<L>(sum);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        if constexpr (!RENORM) {
            // what was not chosen, and the entries that repeat an expert together, in the place of one of them
            bool one = false;
            if (mine) {
                const uint32_t bit = 1u << (e1 / (4 * L) * 4 + e1 % 4);
                atomicAdd(&rows[ct * L * P + e1], dw1);
                one = !(atomicOr(&bits[ct * L + e1 / 4 % L], bit) & bit);
            }
            __syncwarp();
            const uint32_t chosen = bits[lane];
            bits[lane] = 0;
#pragma unroll
            for (int i = 0; i < P; ++i) rest += chosen >> i & 1 ? 0.0f : pr[i];
            rest = lanes_sum<L>(rest) * inv;
            if (mine) dw1 = rows[ct * L * P + e1];
            mine = one;
        }
        // a lane per chosen expert
        const float ctop = __shfl_sync(FULL, top, ct * L), cinv = __shfl_sync(FULL, inv, ct * L);
        const float g = !mine || v == -INFINITY ? 0.0f : expf(v - ctop) * cinv, known = g != 0.0f ? dw1 : 0.0f;
        float S = 0.0f, A = 0.0f, diff = 0.0f;
#pragma unroll 1            // (unrolled: spills, 31 us against 27.6 at 131072 x 128)
        for (int j = 0; j < p.k; ++j) {
            const float gj = __shfl_sync(FULL, g, ct * p.k + j), dj = __shfl_sync(FULL, known, ct * p.k + j);
            S += gj;
            A = fmaf(gj, dj, A);
            diff = fmaf(gj, dw1 - dj, diff);
        }
        const float over = 1.0f / (S + TINY);
        // sum of dg p: renormalised, scale / S * (A - A * (S - 1e-20) / S)
        float D = __shfl_sync(FULL, RENORM ? A * over * (p.scale * over * TINY) : p.scale * A, mt * p.k);
        if constexpr (RENORM) {
            if (mine) atomicAdd(&rows[ct * L * P + e1], p.scale * over * (fmaf(TINY, dw1, diff) * over));       // (one writer each, unless the caller repeats an index)
        } else {
            const float crest = __shfl_sync(FULL, rest, ct * L);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < P; i += 4) store4(rows + mt * L * P + (i / 4 * L + sub) * 4, {-D, -D, -D, -D});
            D = 0.0f;
            __syncwarp();
            if (mine) rows[ct * L * P + e1] = p.scale * fmaf(dw1, crest, diff);
        }
        __syncwarp();
        T* const out = (T*)p.dz + (size_t)tok * p.E;
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            const int at = (i / 4 * L + sub) * 4;
            float d[4];
            load4(rows + mt * L * P + at, d);
            store4(rows + mt * L * P + at, {0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int c = 0; c < 4; ++c) d[c] = pr[i + c] * inv * (d[c] - D);
            if (!have || at >= p.E) continue;
            if (p.vec) {
                store4(out + at, d);
                if (p.dz16) store4(p.dz16 + (size_t)tok * p.E + at, d);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (at + c < p.E) store1(out + at + c, d[c]);
                    if (p.dz16 && at + c < p.E8) p.dz16[(size_t)tok * p.E8 + at + c] = __float2bfloat16(at + c < p.E ? d[c] : 0.0f);
                }
            }
        }
        if (p.dz16 && !p.vec && have)           // (what of the padding lies beyond the last four)
            for (int i = (p.E + 3) / 4 * 4 + sub; i < p.E8; i += L) p.dz16[(size_t)tok * p.E8 + i] = __float2bfloat16(0.0f);
        __syncwarp();
    }
}

bool many(const RouteP& p) { return (int64_t)p.n * p.E > 148 * 2048; }
template <typename T, int L, int P> int run_fwd(RouteP& p, cudaStream_t st)
{
    const int per = WARPS * (32 / L), want = (p.n + per - 1) / per, most = 148 * (P > 8 ? 5 : 8), lanes = p.gsize / P;
    p.group_lanes = p.gsize % P == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    void (*const kernel)(RouteP) = p.top_groups < p.groups ? route_kernel<T, L, P, BY_GROUP> : p.bias ? route_kernel<T, L, P, BY_SCORE> : route_kernel<T, L, P, BY_LOGIT>;
    MGPT_CUDA(launch_pdl(kernel, want < most ? want : most, 32 * WARPS, 0, st, p));
    MGPT_LAUNCHED("route_kernel");
    return 0;
}
template <typename T, int L, int P> int run_softmax_bwd(const RouteP& p, cudaStream_t st)
{
    const int per = WARPS * (32 / L), want = (p.n + per - 1) / per, most = 148 * 8;
    MGPT_CUDA(launch_pdl(p.renorm ? route_softmax_bwd_kernel<T, L, P, true> : route_softmax_bwd_kernel<T, L, P, false>, want < most ? want : most, 32 * WARPS, 0, st, p));
    MGPT_LAUNCHED("route_softmax_bwd_kernel");
    return 0;
}
template <typename T, int L> int run_softmax_bwd(const RouteP& p, cudaStream_t st)
{
    return p.E <= 4 * L ? run_softmax_bwd<T, L, 4>(p, st) : p.E <= 8 * L ? run_softmax_bwd<T, L, 8>(p, st) : run_softmax_bwd<T, L, 16>(p, st);
}
// at least as many lanes as chosen experts (one each), and 16 experts per lane at most (few tokens: 8, as above; 1021 x 155: 2.8 us against 3.5)
template <typename T> int run_softmax_bwd(const RouteP& p, cudaStream_t st)
{
    int lanes = 1;
    while (lanes < p.k || 16 * lanes < p.E || (lanes < 32 && 8 * lanes < p.E && !many(p))) lanes *= 2;
    switch (lanes) {
        case 1: return run_softmax_bwd<T, 1>(p, st);
        case 2: return run_softmax_bwd<T, 2>(p, st);
        case 4: return run_softmax_bwd<T, 4>(p, st);
        case 8: return run_softmax_bwd<T, 8>(p, st);
        case 16: return run_softmax_bwd<T, 16>(p, st);
        default: return run_softmax_bwd<T, 32>(p, st);
    }
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
template <typename T> int run_fwd(RouteP& p, cudaStream_t st)
{
    p.vec = p.E % 4 == 0 && ((uintptr_t)p.logits & (4 * sizeof(T) - 1)) == 0;
    // Sixteen experts per lane where that leaves an SM two thousand logits and more: what a round costs beside its minima is shared by more tokens
    // (131072 x 128: 39 us against 55 with eight, 4096 x 128: 3.5 against 5.1).  Fewer: eight, whose chains are shorter (64 x 256 in groups: 4.1
    // against 5.0).
    if (p.E > 256) return run_fwd<T, 32, 16>(p, st);
    if (many(p))
        return p.E <= 16 ? run_fwd<T, 1, 16>(p, st) : p.E <= 32 ? run_fwd<T, 2, 16>(p, st) : p.E <= 64 ? run_fwd<T, 4, 16>(p, st)
               : p.E <= 128 ? run_fwd<T, 8, 16>(p, st) : run_fwd<T, 16, 16>(p, st);
    return p.E <= 8 ? run_fwd<T, 1, 8>(p, st) : p.E <= 16 ? run_fwd<T, 2, 8>(p, st) : p.E <= 32 ? run_fwd<T, 4, 8>(p, st)
           : p.E <= 64 ? run_fwd<T, 8, 8>(p, st) : p.E <= 128 ? run_fwd<T, 16, 8>(p, st) : run_fwd<T, 32, 8>(p, st);
}
template <typename T> int run_bwd(RouteP& p, cudaStream_t st)
{
    p.vec = p.E % 4 == 0 && (((uintptr_t)p.logits | (uintptr_t)p.dz) & (4 * sizeof(T) - 1)) == 0 && (!p.dz16 || p.E8 == p.E);
    return p.softmax ? run_softmax_bwd<T>(p, st) : run_sigmoid_bwd<T>(p, st);
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

// Column sums of blocks of rows of [n, E], in a fixed order: 256 / E' threads to a column, E' the power of two that E fits.  (The layer's router
// bias: first its blocks of rows, then those sums; the last are added to what is there.)
__global__ void __launch_bounds__(256) route_columns_kernel(const float* from, int n, int E, int rows, float* to, bool add)
{
    pdl_wait();
    __shared__ float sums[256];
    int cols = 1;
    while (cols < E) cols *= 2;
    const int e = threadIdx.x % cols, group = threadIdx.x / cols, groups = 256 / cols;
    const int r0 = blockIdx.x * rows, r1 = min(r0 + rows, n);
    float s = 0.0f;
    if (e < E)
#pragma unroll 8
        for (int r = r0 + group; r < r1; r += groups) s += from[(size_t)r * E + e];
    sums[threadIdx.x] = s;
    __syncthreads();
    if (group == 0 && e < E) {
        for (int g = 1; g < groups; ++g) s += sums[g * cols + e];
        float* const out = to + (size_t)blockIdx.x * E + e;
        *out = add ? *out + s : s;
    }
}

}  // namespace

// ---- the layer's routing ------------------------------------------------------------------------------------------------
int check_routing(const mgpt_moe_routing* r, int E, int k)
{
    RouteP p = {};
    return fill(p, r, 0, E, k);
}

// What tells settings apart: 0 for the reference's, else a hash of all but the bias's address.
uint32_t routing_tag(const mgpt_moe_layer* L)
{
    if (!L->routed) return 0;
    const mgpt_moe_routing& r = L->routing;
    uint32_t bits, h = 2166136261u;             // FNV-1a
    memcpy(&bits, &r.scale, 4);
    for (uint32_t v : {(uint32_t)r.score, (uint32_t)r.groups, (uint32_t)r.top_groups, (uint32_t)r.group_top, (uint32_t)(r.renormalise != 0), bits, (uint32_t)(r.bias != nullptr)})
        for (int i = 0; i < 32; i += 8) h = (h ^ (v >> i & 255)) * 16777619u;
    return h ? h : 1;
}

// The router's product, then this routing over its own.
int launch_routed(mgpt_moe_layer* L, const Workspace& w, char* ws, const void* x, int io, cudaStream_t st)
{
    const Dims& d = L->d;
    int32_t* const idx = (int32_t*)(ws + w.top_idx);
    float* const weights = (float*)(ws + w.top_p);
    if (tc_router_usable(L, x, io, w.n_tokens))
        MGPT_TRY(tc_router_fwd(L, w, ws, x, st));
    else
        MGPT_TRY(launch_router_fwd(x, io, L->p_data[0], L->p_data[1], w.n_tokens, d.C, d.E, d.k, (float*)(ws + w.logits), (float*)(ws + w.probs),
                                   idx, weights, st, nullptr, nullptr, L->d_status));
    RouteP p = {};
    MGPT_TRY(fill(p, &L->routing, w.n_tokens, d.E, d.k));
    p.logits = ws + w.logits; p.idx = idx; p.w = weights;
    return run_fwd<float>(p, st);
}

// dlogits (and their BF16 copy, where there is one) from d_top_p; d_bias, where it is given, is added to.
int launch_routed_bwd(mgpt_moe_layer* L, const Workspace& w, char* ws, bf16* dl16, int E8, float* d_bias, cudaStream_t st)
{
    const Dims& d = L->d;
    RouteP p = {};
    MGPT_TRY(fill(p, &L->routing, w.n_tokens, d.E, d.k));
    p.logits = ws + w.logits;
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
    MGPT_CUDA(launch_pdl(route_columns_kernel, parts, 256, 0, st, (const float*)p.dz, p.n, d.E, rows, part, false));
    MGPT_LAUNCHED("route_columns_kernel");
    MGPT_CUDA(launch_pdl(route_columns_kernel, 1, 256, 0, st, (const float*)part, parts, d.E, parts, d_bias, true));
    MGPT_LAUNCHED("route_columns_kernel");
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
    L->counts_left |= L->fwd_done;
    L->fwd_done = false;        // a backward would take the other routing's gradient
    L->plan_outdated = true;
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
