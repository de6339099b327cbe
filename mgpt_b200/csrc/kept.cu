// Activations into 8 bits and back (the format: kept.cuh).  Bound by HBM: a thread moves 16 bytes of x at a time, a warp's accesses are
// runs of memory, and four pieces are on their way at once.  32768 x 2048 BF16 on a B200: kept in 32 us (6.4 TB/s), restored in 35 (5.9).
#include "kept.cuh"

namespace mgpt {

namespace {

constexpr int THREADS = 256, UNROLL = 4;

template <typename T> constexpr int piece() { return 16 / sizeof(T); }
__device__ __forceinline__ void widen_piece(const uint4 u, F2 (&v)[4], bf16)
{
    v[0] = widen(u.x); v[1] = widen(u.y); v[2] = widen(u.z); v[3] = widen(u.w);
}
__device__ __forceinline__ void widen_piece(const uint4 u, F2 (&v)[2], float)
{
    v[0] = F2(__uint_as_float(u.x), __uint_as_float(u.y));
    v[1] = F2(__uint_as_float(u.z), __uint_as_float(u.w));
}
__device__ __forceinline__ uint4 narrow_piece(const F2 (&v)[4], bf16) { return make_uint4(narrow(v[0]), narrow(v[1]), narrow(v[2]), narrow(v[3])); }
__device__ __forceinline__ uint4 narrow_piece(const F2 (&v)[2], float)
{
    return make_uint4(__float_as_uint(v[0].lo()), __float_as_uint(v[0].hi()), __float_as_uint(v[1].lo()), __float_as_uint(v[1].hi()));
}
// N bytes: 8 or 4
template <int N> __device__ __forceinline__ void store_words(int8_t* p, const uint32_t (&w)[N / 4])
{
    if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}
template <int N> __device__ __forceinline__ void load_words(const int8_t* p, uint32_t (&w)[N / 4])
{
    if constexpr (N == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x;
        w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// The pieces of a thread: where a row's last group is whole, of one run of pieces (flat: a row of everything); else `lanes` threads to a row.
struct KeptP {
    const void* x;
    void* out;
    int8_t* v;
    uint8_t* e;
    int64_t rows, C;
    bool flat;
    int lanes;          // a power of two, 32 at most
};

// f(piece's place in x and v in elements, group's place in e, whether there is such a piece); every lane of a warp makes the same calls
template <typename T, typename F> __device__ __forceinline__ void for_pieces(const KeptP& p, F f)
{
    constexpr int E = piece<T>(), G = KEPT_GROUP / E;
    if (p.flat) {
        for (int64_t i = (int64_t)blockIdx.x * THREADS * UNROLL + threadIdx.x; i - (int)threadIdx.x < p.C / E; i += (int64_t)gridDim.x * THREADS * UNROLL)
            f(i * E, i / G, THREADS * E, THREADS / G, p.C);
    } else {
        const int sub = threadIdx.x % p.lanes, per = THREADS / p.lanes, groups = kept_groups((int)p.C);
        const int row_pieces = groups * G;
        for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += (int64_t)gridDim.x * per) {
            const int64_t r = r0 + threadIdx.x / p.lanes;
            for (int q = sub; q - sub < row_pieces; q += p.lanes * UNROLL)
                f(r * p.C + q * E, r * groups + q / G, p.lanes * E, p.lanes / G, r < p.rows ? (r + 1) * p.C : 0);
        }
    }
}

template <typename T> __global__ void __launch_bounds__(THREADS) keep8_kernel(const KeptP p)
{
    constexpr int E = piece<T>(), G = KEPT_GROUP / E;
    pdl_wait();
    for_pieces<T>(p, [&](int64_t at, int64_t group, int step, int group_step, int64_t end) {
        uint4 u[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
            u[k] = at + k * step < end ? *reinterpret_cast<const uint4*>((const T*)p.x + at + k * step) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
            F2 v[E / 2];
            uint32_t w[E / 4];
            widen_piece(u[k], v, T());
            const uint32_t byte = kept_pack<T>(u[k], v, w);
            if (at + k * step < end) {
                store_words<E>(p.v + at + k * step, w);
                if (threadIdx.x % G == 0) p.e[group + k * group_step] = (uint8_t)byte;
            }
        }
    });
}

template <typename T> __global__ void __launch_bounds__(THREADS) restore8_kernel(const KeptP p)
{
    constexpr int E = piece<T>();
    pdl_wait();
    for_pieces<T>(p, [&](int64_t at, int64_t group, int step, int group_step, int64_t end) {
        uint32_t w[UNROLL][E / 4], byte[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
            if (at + k * step < end) {
                load_words<E>(p.v + at + k * step, w[k]);
                byte[k] = p.e[group + k * group_step];
            }
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
            if (at + k * step < end) {
                F2 v[E / 2];
                const F2 unit(kept_unit(byte[k]));
#pragma unroll
                for (int j = 0; j < E / 4; ++j) {
                    kept_unpack(w[k][j], v[2 * j], v[2 * j + 1]);
                    v[2 * j] = v[2 * j] * unit;
                    v[2 * j + 1] = v[2 * j + 1] * unit;
                }
                *reinterpret_cast<uint4*>((T*)p.out + at + k * step) = narrow_piece(v, T());
            }
    });
}

int check_kept(int64_t n, int C, int io)
{
    if (n < 0 || n > (1 << 30) || C <= 0) return fail(MGPT_MOE_EINVAL, "kept activations: sizes out of range");
    if (C % 8) return fail(MGPT_MOE_EINVAL, "kept activations: channels must be a multiple of 8");
    if (io != MGPT_MOE_IO_F32 && io != MGPT_MOE_IO_BF16) return fail(MGPT_MOE_EINVAL, "unknown io dtype");
    return 0;
}
// how the pieces are dealt out, and the number of blocks
int deal(KeptP& p, int n, int C, int io)
{
    const int E = io == MGPT_MOE_IO_BF16 ? 8 : 4;
    int64_t blocks;
    if (C % KEPT_GROUP == 0) {
        p.flat = true;
        p.rows = 1;
        p.C = (int64_t)n * C;
        blocks = (p.C / E + THREADS * UNROLL - 1) / (THREADS * UNROLL);
    } else {
        p.rows = n;
        p.C = C;
        const int pieces = kept_groups(C) * (KEPT_GROUP / E);
        p.lanes = KEPT_GROUP / E;
        while (p.lanes < 32 && p.lanes * UNROLL < pieces) p.lanes *= 2;
        blocks = ((int64_t)n * p.lanes + THREADS - 1) / THREADS;
    }
    const int64_t most = 148 * 8;
    return (int)(blocks < most ? blocks : most);
}

}  // namespace

}  // namespace mgpt

using namespace mgpt;

extern "C" {

int mgpt_moe_op_keep8(const void* x, int io, int n, int C, int8_t* values, uint8_t* exponents, mgpt_stream_t stream)
{
    MGPT_TRY(check_kept(n, C, io));
    if (n == 0) return 0;
    if (!x || !values || !exponents) return fail(MGPT_MOE_EINVAL, "null argument");
    MGPT_TRY(check_aligned(x, "x"));
    MGPT_TRY(check_aligned(values, "values", 8));
    KeptP p = {};
    p.x = x; p.v = values; p.e = exponents;
    const int blocks = deal(p, n, C, io);
    MGPT_CUDA(launch_pdl(io == MGPT_MOE_IO_BF16 ? keep8_kernel<bf16> : keep8_kernel<float>, blocks, THREADS, 0, (cudaStream_t)stream, p));
    MGPT_LAUNCHED("keep8_kernel");
    return 0;
}

int mgpt_moe_op_restore8(const int8_t* values, const uint8_t* exponents, int n, int C, void* x, int io, mgpt_stream_t stream)
{
    MGPT_TRY(check_kept(n, C, io));
    if (n == 0) return 0;
    if (!x || !values || !exponents) return fail(MGPT_MOE_EINVAL, "null argument");
    MGPT_TRY(check_aligned(x, "x"));
    MGPT_TRY(check_aligned(values, "values", 8));
    KeptP p = {};
    p.out = x; p.v = const_cast<int8_t*>(values); p.e = const_cast<uint8_t*>(exponents);
    const int blocks = deal(p, n, C, io);
    MGPT_CUDA(launch_pdl(io == MGPT_MOE_IO_BF16 ? restore8_kernel<bf16> : restore8_kernel<float>, blocks, THREADS, 0, (cudaStream_t)stream, p));
    MGPT_LAUNCHED("restore8_kernel");
    return 0;
}

}  // extern "C"
