// Softmax cross entropy of a vocabulary product, and its gradients, without keeping the logits.
//
//   z[i,v] = <x[i,:], w[v,:]>,  lse[i] = log sum_v exp z[i,v],  loss[i] = lse[i] - z[i, target[i]]
//   dz[i,v] = d_loss[i] * (exp(z[i,v] - lse[i]) - [v == target[i]]),  dx = dz w,  dw = dz^T x
//
// The reference forms all logits in FP32 and passes over them for the loss and again for the gradient
// (layers/CrossEntropyLossLayer.cpp; utils/cuda_ops.cu:748-876).  Here the loss is an epilogue of the product: each 256 x 256
// tile of logits leaves a row maximum and a row sum of exponentials.  The gradients take the vocabulary piece by piece: the
// piece's logits are computed again, the epilogue turns them into dz (BF16, the operand type of the two products that
// follow; FP32 until then), and one launch forms the piece's rows of dw and adds its share of dx.
//
// dz is kept over the largest |d_loss|, which the results are multiplied by in FP32: with the usual d_loss, one number for
// all tokens, a target's entry is then -(1 - p) and rounds by less than p.  (Rounded with its factor it is off by the factor's own
// rounding, up to 2^-8, in every token alike: gradients of 1800 tokens were 2.9e-3 off the exact ones, of which 1.7e-3 are the
// results' own rounding.)
//
// Tokens whose target is not in [0, vocabulary) take no part: the others are packed first, so that an ignored token costs
// nothing and its x, whatever it holds, is not read.  The loss of at most TILE tokens of the operand type reads them as they lie:
// leaving some out would not make their one tile of products shorter.  A row of it is one token, so that what an ignored one holds
// stays there, and is dropped when the columns are joined.
#include "pairs.cuh"
#include "tc_common.cuh"

namespace mgpt {

namespace {

using namespace tcx;

constexpr int TILE = 256;                            // tokens and vocabulary rows of a pair's tile
constexpr int BK = 64;
constexpr uint32_t OPER_BYTES = 128 * BK * 2;        // one operand's share of a stage in one CTA: 16 KiB
constexpr uint32_t STAGE_BYTES = 2 * OPER_BYTES;
constexpr uint32_t BOX_BYTES = 64 * BK * 2;
constexpr int EPI_WARPS = 16;                        // four per TMEM lane quarter, 64 columns each
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr uint32_t TMEM_COLS = 2 * TILE;
constexpr uint32_t STAGING = 4096;                   // per epilogue warp: 32 rows x 128 B
constexpr int QUEUE = 4;
constexpr int NARROW = 512;                          // LOSS_NARROW, DLOGITS_NARROW up to this C
constexpr int PART = 512 / BK;                       // LOSS, DLOGITS: k-blocks summed in one accumulator
constexpr int CLAIM = 6;                             // GRADS: the next item is claimed this many k-blocks before the last one's loads end
constexpr int MAX_PIECES = 1024;
constexpr int COUNTERS = 2 * MAX_PIECES + 2;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int ST_BAD_TARGET = ST_BAD_EXPERT;         // the status bit of an index outside its range

enum { LOSS = 0, DLOGITS = 1, GRADS = 2, LOSS_NARROW = 3, DLOGITS_NARROW = 4 };
constexpr bool is_loss(int kind) { return kind == LOSS || kind == LOSS_NARROW; }
constexpr bool in_parts(int kind) { return kind == LOSS || kind == DLOGITS; }       // logits: several accumulators, joined in registers

struct HeadP {
    const int32_t* n_valid;     // null: n tokens, as they lie
    int n;                      // of the call
    int few[2];                 // without n_valid: rows of x that each CTA of a pair loads, at most 128; the other rows are never looked at
    int direct;                 // x has the operand type: where no token is left out, it is read as it lies
    int32_t* sched;             // next item; zero before the launch (null: items by stride)
    int32_t* status;
    int C, V;
    int v0;                     // first vocabulary row of the piece
    int v_tiles;                // 256-row tiles of the vocabulary in this launch
    int group;                  // token tiles that share a pass over the vocabulary (LOSS, DLOGITS)
    int c_tiles;                // GRADS: 256-column tiles of C
    int k_slices, slice_tiles;  // GRADS, dx: the piece's vocabulary in k_slices of slice_tiles tiles
    int n_pad;                  // row pitch of part; rows of a slice of acc
    const int32_t* target;      // packed
    const float *lse, *d_loss;  // packed; d_loss over *scale
    const float* scale;
    float2* part;               // LOSS: [v_tiles][n_pad] maximum and sum
    float* z_target;
    bf16* dz;                   // DLOGITS: [token tile of 128][64-column block] of swizzled 128 x 64 tiles
    float* acc;                 // GRADS: [k_slices][n_pad][C], dx so far
    int first;                  // acc is written, not added to
    int last;                   // the sums for dx are complete: they are written there
    const int32_t* rows;        // packed -> token
    void* dx;
    int dx_f32;
    void* dw;
    int dw_f32;                 // dw is FP32 and added to
};

// exp(from - to), 1 where both are the same infinity
__device__ __forceinline__ float shift(float from, float to) { return from == to ? 1.0f : exp2f((from - to) * LOG2E); }

// (exponents below -126 give 0: terms that a sum with a 1 in it, or a rounding to 8 bits beside the target's, does not see)
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// four channels of dx
__device__ __forceinline__ void put_dx(void* dx, int f32, size_t at, float4 x, float scale)
{
    x.x *= scale; x.y *= scale; x.z *= scale; x.w *= scale;
    if (f32) {
        *reinterpret_cast<float4*>((float*)dx + at) = x;
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
        *reinterpret_cast<uint2*>((bf16*)dx + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

// An arrival that hands over nothing that was written: the accumulator's columns, or a queue entry, have been read.  (With release at
// cluster scope each one waited for the warp's stores to global memory before it, about 2000 cycles of an item.)
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }

// What an item is.  LOSS, DLOGITS: m (256 tokens), n (256 vocabulary rows), reduction over C.
// GRADS: dx (m: 256 tokens, n: 256 channels, reduction over a slice of the vocabulary) or dw (m: 256 vocabulary rows, n: 256
// channels, reduction over the tokens).  The leader's producer works an item out and passes it to everyone.
struct __align__(16) Item {
    int m, n;               // m < 0: no more
    int slice;              // GRADS: the vocabulary's slice, -1: dw
    int nkb;                // 64-element blocks of the reduction
    __device__ __forceinline__ bool dw() const { return slice < 0; }
    __device__ __forceinline__ int half(int C) const { return C - n * TILE <= TILE / 2 ? 64 : 128; }     // GRADS: columns per CTA
};
struct Shared {
    Item item[QUEUE];
    uint64_t full[6], empty[6], acc_full[2], acc_empty[2], item_full[QUEUE], item_empty[QUEUE], joined[8][4];
    uint32_t tmem;
};
template <int KIND> constexpr int stages() { return is_loss(KIND) ? 6 : 5; }
template <int KIND> constexpr uint32_t extra_bytes() { return is_loss(KIND) ? 4 * 4 * 128 * sizeof(float2) : EPI_WARPS * STAGING; }
template <int KIND> constexpr uint32_t smem_bytes() { return 1024 + stages<KIND>() * STAGE_BYTES + extra_bytes<KIND>() + sizeof(Shared); }
static_assert(smem_bytes<LOSS>() <= 232448 && smem_bytes<GRADS>() <= 232448, "shared memory of one CTA");

template <int KIND> __device__ __forceinline__ int item_count(const HeadP& p, int n_valid)
{
    const int mt = (n_valid + TILE - 1) / TILE;
    return KIND == GRADS ? (mt * p.k_slices + p.v_tiles) * p.c_tiles : mt * p.v_tiles;
}
template <int KIND> __device__ __forceinline__ Item decode(const HeadP& p, int n_valid, int i)
{
    Item w;
    const int mt = (n_valid + TILE - 1) / TILE;
    w.slice = 0;
    if (KIND != GRADS) {
        // group token tiles at a time run through the whole vocabulary, so that x stays in L2
        const int g = i / (p.group * p.v_tiles), r = i - g * p.group * p.v_tiles, in = min(p.group, mt - g * p.group);
        w.n = r / in;
        w.m = g * p.group + r - w.n * in;
        w.nkb = (p.C + BK - 1) / BK;
        return w;
    }
    const int dx = mt * p.k_slices * p.c_tiles;
    if (i < dx) {
        w.slice = i / (mt * p.c_tiles);
        const int r = i - w.slice * mt * p.c_tiles;
        w.m = r / p.c_tiles;
        w.n = r - w.m * p.c_tiles;
        w.nkb = min(p.slice_tiles, p.v_tiles - w.slice * p.slice_tiles) * (TILE / BK);
    } else {
        w.slice = -1;
        w.m = (i - dx) / p.c_tiles;
        w.n = (i - dx) - w.m * p.c_tiles;
        w.nkb = (n_valid + BK - 1) / BK;
    }
    return w;
}

// tmA: LOSS, DLOGITS x (box 64 x 128 rows); GRADS the dz tiles as {64, 128 rows, tiles} in boxes of {64, 128, 1}
// tmA2: GRADS the dz tiles in boxes of {64, 64, 2}
// tmB: LOSS, DLOGITS w (box 64 x 128 rows); GRADS w (box 64 x 64 rows); tmB2: x (box 64 x 64 rows)
// tmX: x as it lies in the caller's memory, in boxes like those of x above, which is the packed copy
// The epilogue's 16 warps: all of them on an item, 64 columns each; or two groups of eight that take items in turn, 128 columns
// each.  What a warp of DLOGITS_NARROW does for an item is a chain of some 6000 cycles (tcgen05.ld, exponentials, shared memory, the copy
// that has to have left it), of which an item of C = 512 with 4100 cycles of products hides one only half: 1.3 % of the gradients' time where
// the power limit sets the clock, 6 % where it does not.  LOSS and DLOGITS, all sixteen on an item, add its accumulators in registers and
// give each back at once.  One accumulator over all channels for the gradients' logits, beside the loss's several, was 1 % faster
// (1501 of 3001 tokens, 1024 x 50021 458 us, now 464; 8192, 2048 x 131072 12.70 ms, now 12.83) and left exp(z - lse) with what the
// tensor core cuts off such a sum: 2e-3 of d_loss for a token that is certain (logit 400, 2048 channels), now 3e-5.
template <int KIND> constexpr int item_warps() { return KIND == DLOGITS_NARROW || KIND == LOSS_NARROW ? EPI_WARPS / 2 : EPI_WARPS; }

template <int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
head_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmA2,
            const __grid_constant__ CUtensorMap tmB2, const __grid_constant__ CUtensorMap tmX, const HeadP p)
{
    constexpr int NS = stages<KIND>(), ITEM_WARPS = item_warps<KIND>(), GROUPS = EPI_WARPS / ITEM_WARPS, UNITS = 16 / ITEM_WARPS;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    uint8_t* const tiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* const extra = tiles + NS * STAGE_BYTES;
    Shared& sh = *reinterpret_cast<Shared*>(extra + extra_bytes<KIND>());
    const uint32_t full = smem_u32(sh.full), empty = smem_u32(sh.empty), acc_full = smem_u32(sh.acc_full), acc_empty = smem_u32(sh.acc_empty);
    const uint32_t item_full = smem_u32(sh.item_full), item_empty = smem_u32(sh.item_empty);
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(full + 8 * s, 1);                     // (the leader's; the peer's loads count on it too)
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + 8 * b, 1);
            mbar_init(acc_empty + 8 * b, 2 * ITEM_WARPS);
        }
        for (int i = 0; i < QUEUE; ++i) {
            mbar_init(item_full + 8 * i, 1);
            mbar_init(item_empty + 8 * i, 2 * ITEM_WARPS + 2);      // the leader's: the epilogue, its MMA thread, the peer's producer
        }
        for (int q = 0; q < 32; ++q) mbar_init(smem_u32(&sh.joined[q >> 2][q & 3]), ITEM_WARPS / 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(&sh.tmem), TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                         // the peer's barriers exist before anything is sent to them
    tc_fence_after();
    const uint32_t tmem_base = sh.tmem;
    pdl_wait();
    const int n_valid = p.n_valid ? *p.n_valid : p.n;
    const bool as_it_lies = p.direct && n_valid == p.n;
    const int x_rows0 = p.n_valid ? 128 : p.few[0], x_rows1 = p.n_valid ? 128 : p.few[1];
    const float scale = KIND == GRADS ? *p.scale : 1.0f;

    const uint32_t lead_item_empty = mapa(item_empty, 0);
    // the pair's n-th item; false: no more
    auto consume = [&](uint32_t n, Item& w) -> bool {
        const int slot = n % QUEUE;
        if (!mbar_wait_cluster(item_full + 8 * slot, (n / QUEUE) & 1, p.status, ERR_SCHED_WAIT)) return false;
        const int4 v = taken<int4>(smem_u32(&sh.item[slot]));
        w.m = v.x; w.n = v.y; w.slice = v.z; w.nkb = v.w;
        return w.m >= 0;
    };
    auto release = [&](uint32_t n) { arrive_remote(lead_item_empty + 8 * (n % QUEUE)); };

    if (warp == 0) {
        if (elect_one()) {
            const int total = item_count<KIND>(p, n_valid), grid = gridDim.x >> 1;
            const uint32_t lead_full = mapa(full, 0), tile0 = smem_u32(tiles);
            const uint32_t peer_item = mapa(smem_u32(sh.item), 1), peer_item_full = mapa(item_full, 1);
            // The logits' items, all alike, are passed on one ahead, so that the peer's loads, which share the leader's barriers, do not wait to
            // hear of one: a pair's first two are its own by number, those that follow are claimed two ahead (8192 x 512 x 32000: 202 -> 190
            // us).  The gradients' items are of two lengths and claimed as late as hides the counter (7570 x 312 x 7261: 114 us ahead, 93 so).
            // Behind the last item come two entries that say so: either group of the epilogue may be the one to read on.
            constexpr bool AHEAD = KIND != GRADS;
            int s = 0, after = (blockIdx.x >> 1) + grid, claimed = 0;
            uint32_t free_phase = 1;                        // (the first round finds every stage free)
            bool ok = true;
            auto item_of = [&](int i) {
                Item w = {-1, 0, 0, 0};
                if (i < total) w = decode<KIND>(p, n_valid, i);
                return w;
            };
            auto publish = [&](uint32_t n, const Item& w) {
                const int slot = n % QUEUE;
                if (!mbar_wait(item_empty + 8 * slot, ((n / QUEUE) & 1) ^ 1, p.status, ERR_SCHED_WAIT)) return false;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(&sh.item[slot])), "r"(w.m), "r"(w.n), "r"(w.slice), "r"(w.nkb) : "memory");
                asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(peer_item + (uint32_t)sizeof(Item) * slot), "r"(w.m), "r"(w.n), "r"(w.slice), "r"(w.nkb) : "memory");
                mbar_arrive(item_full + 8 * slot);
                mbar_arrive_cluster(peer_item_full + 8 * slot);             // (release at cluster scope: the item is visible)
                return true;
            };
            Item w, following;
            if (rank == 0) {
                w = item_of(blockIdx.x >> 1);
                ok = publish(0, w);
            }
            for (uint32_t n = 0; ok; ++n) {
                if (rank == 0) {
                    if (AHEAD || w.m < 0) {
                        following = item_of(w.m < 0 ? total : after);
                        if (!publish(n + 1, following) || w.m < 0) break;
                    }
                    if (AHEAD || w.nkb <= CLAIM) claimed = p.sched ? atomicAdd(p.sched, 1) : 0;      // (looked at when this item's loads are under way)
                } else {
                    const bool more = consume(n, w);
                    release(n);
                    if (!more) break;
                }
                for (int kb = 0; kb < w.nkb; ++kb) {
                    if (!AHEAD && rank == 0 && w.nkb - kb == CLAIM + 1) claimed = atomicAdd(p.sched, 1);
                    if (!mbar_wait(empty + 8 * s, free_phase, p.status, ERR_EMPTY_WAIT)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a_dst = tile0 + s * STAGE_BYTES, b_dst = a_dst + OPER_BYTES, bar = lead_full + 8 * s;
                    if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * OPER_BYTES + (x_rows0 + x_rows1) * (BK * 2));       // both CTAs' bytes
                    if (KIND != GRADS) {
                        // (one tile of tokens: tmX has the leader's rows, tmA the peer's)
                        if ((rank == 0 ? x_rows0 : x_rows1) > 0)
                            tma_load_2d_pair(a_dst, as_it_lies && (p.n_valid || rank == 0) ? &tmX : &tmA, kb * BK, w.m * TILE + rank * 128, bar);
                        tma_load_2d_pair(b_dst, &tmB, kb * BK, p.v0 + w.n * TILE + rank * 128, bar);
                    } else {
                        const int blocks = p.v_tiles * (TILE / 64), col = w.n * TILE + rank * w.half(p.C), k0 = w.slice * p.slice_tiles * (TILE / BK);
                        const CUtensorMap* mB;
                        int row;
                        if (!w.dw()) {
                            tma_load_3d_pair(a_dst, &tmA, 0, 0, (w.m * 2 + rank) * blocks + k0 + kb, bar);
                            mB = &tmB;
                            row = p.v0 + (k0 + kb) * BK;
                        } else {
                            tma_load_3d_pair(a_dst, &tmA2, 0, (kb & 1) * 64, (kb >> 1) * blocks + w.m * (TILE / 64) + rank * 2, bar);
                            mB = as_it_lies ? &tmX : &tmB2;
                            row = kb * BK;
                        }
                        tma_load_2d_pair(b_dst, mB, col, row, bar);
                        tma_load_2d_pair(b_dst + BOX_BYTES, mB, col + 64, row, bar);
                    }
                    if (++s == NS) {
                        s = 0;
                        free_phase ^= 1;
                    }
                }
                if (rank == 0) {
                    if (AHEAD) {
                        after = p.sched ? 2 * grid + claimed : after + grid;
                    } else {
                        following = item_of(grid + claimed);
                        ok = ok && publish(n + 1, following);
                    }
                    w = following;
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            uint32_t t = 0, phase = 0;
            int s = 0;
            bool ok = true;
            Item w;
            const uint32_t peer_empty = mapa(empty, 1), peer_acc_full = mapa(acc_full, 1);
            const uint32_t tile0 = smem_u32(tiles);
            const uint64_t k_major = make_desc(tile0, 16, 1024), mn_major = make_desc(tile0, BOX_BYTES, 1024);
            for (uint32_t n = 0; ok && consume(n, w); ++n) {
                release(n);
                if (w.nkb == 0) continue;
                const bool a_mn = KIND == GRADS && w.dw(), b_mn = KIND == GRADS;
                const uint32_t idesc = make_idesc(TILE, KIND == GRADS ? 2 * w.half(p.C) : TILE, a_mn, b_mn);
                const uint64_t a0 = a_mn ? mn_major : k_major, b0 = (b_mn ? mn_major : k_major) + (OPER_BYTES >> 4);
                const uint32_t a_step = a_mn ? 2048 >> 4 : 32 >> 4, b_step = b_mn ? 2048 >> 4 : 32 >> 4;     // (the address field: 16-byte units)
                for (int k0 = 0; ok && k0 < w.nkb; ++t) {
                    const uint32_t buf = t & 1u, d_tmem = tmem_base + buf * TILE;
                    const int k1 = in_parts(KIND) ? min(k0 + PART, w.nkb) : w.nkb;
                    if (!mbar_wait(acc_empty + 8 * buf, ((t >> 1) & 1) ^ 1, p.status, ERR_ACC_WAIT)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    for (int kb = k0; kb < k1; ++kb) {
                        if (!mbar_wait(full + 8 * s, phase, p.status, ERR_FULL_WAIT)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t ad = a0 + s * (STAGE_BYTES >> 4), bd = b0 + s * (STAGE_BYTES >> 4);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            umma_bf16_pair(d_tmem, ad + k * a_step, bd + k * b_step, idesc, (kb > k0 || k > 0) ? 1u : 0u);
                        umma_commit_pair(empty + 8 * s);
                        umma_commit_pair(peer_empty + 8 * s);
                        if (++s == NS) {
                            s = 0;
                            phase ^= 1;
                        }
                    }
                    if (ok) {
                        umma_commit_pair(acc_full + 8 * buf);
                        umma_commit_pair(peer_acc_full + 8 * buf);
                    }
                    k0 = k1;
                }
            }
        }
    } else {
        // TMEM lane quarter q, the h-th of the warps that share its columns
        const int q = warp & 3, group = (warp - 2) / ITEM_WARPS, h = (warp - 2) % ITEM_WARPS >> 2;
        uint8_t* const stage = extra + (warp - 2) * STAGING;
        const uint32_t acc_free = mapa(acc_empty, 0), joined = smem_u32(sh.joined[group * 4 + q]);
        uint32_t t = 0;
        Item w, before = {};
        uint32_t k = 0;                                     // items of the group so far
        constexpr int SHARERS = ITEM_WARPS / 4;             // warps of a lane quarter
        float2* const sums = reinterpret_cast<float2*>(extra) + group * 4 * SHARERS * 128 + q * 32 + lane;      // [4 items][SHARERS][128 rows]
        auto join = [&](uint32_t k, const Item& of) {
            if (!mbar_wait(joined + 8 * (k & 3), k >> 2 & 1, p.status, ERR_ACC_WAIT)) return false;
            float2 o[SHARERS];
            float m = -INFINITY, all = 0.0f;
#pragma unroll
            for (int i = 0; i < SHARERS; ++i) {
                o[i] = sums[((k & 3) * SHARERS + i) * 128];
                m = fmaxf(m, o[i].x);
            }
#pragma unroll
            for (int i = 0; i < SHARERS; ++i) all = fmaf(o[i].y, shift(o[i].x, m), all);
            const int row = of.m * TILE + rank * 128 + q * 32 + lane;
            if (row < n_valid) p.part[(size_t)of.n * p.n_pad + row] = make_float2(m, all);
            return true;
        };
        for (uint32_t n = group; __any_sync(0xffffffffu, consume(n, w)); n += GROUPS, ++k) {
            __syncwarp();
            if (lane == 0) release(n);
            const bool empty_sum = w.nkb == 0;              // no token takes part: dw is zero
            uint32_t buf = 0, t_lane = 0;
            auto next_acc = [&]() {                         // the next accumulator is complete; false: the wait ran out
                buf = GROUPS == 2 ? group : t & 1u;         // (two groups: an item is one accumulator, theirs)
                t_lane = tmem_base + buf * TILE + ((uint32_t)(q * 32) << 16) + h * (UNITS * 64);
                if (!mbar_wait(acc_full + 8 * buf, (GROUPS == 2 ? t : t >> 1) & 1, p.status, ERR_ACC_WAIT)) return false;
                tc_fence_after();
                ++t;
                return true;
            };
            auto give_back = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_remote(acc_free + 8 * buf);
            };
            // this thread's token, and where its target lies behind the warp's first column
            const int row = w.m * TILE + rank * 128 + q * 32 + lane, v = p.v0 + w.n * TILE + h * (UNITS * 64);
            const bool real = KIND != GRADS && row < n_valid;
            const int at = real ? p.target[row] - v : -1;
            constexpr bool dlogits = KIND != GRADS && !is_loss(KIND);
            const float up = dlogits && real ? p.d_loss[row] : 0.0f, lse = dlogits && real ? p.lse[row] : 0.0f;
            if (!empty_sum && !next_acc()) break;
            // the item's other accumulators, added to what the first one left in z; false: a wait ran out
            auto add_parts = [&](float (&z)[64]) {
                for (int kb = PART; kb < w.nkb; kb += PART) {
                    if (!next_acc()) return false;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float o[16];
                        tmem_ld16(t_lane + 16 * c, o);
                        tmem_ld_wait();
                        if (c == 3) give_back();
#pragma unroll
                        for (int j = 0; j < 16; ++j) z[16 * c + j] += o[j];
                    }
                }
                return true;
            };
            if (is_loss(KIND)) {
                float top = -INFINITY, sum = 0.0f;
                bool ok = true;
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    const int valid = p.V - v - u * 64, a = at - u * 64;
                    float z[64];
                    {
                        float (&z0)[32] = *reinterpret_cast<float (*)[32]>(z), (&z1)[32] = *reinterpret_cast<float (*)[32]>(z + 32);
                        tmem_ld32(t_lane + u * 64, z0);
                        tmem_ld32(t_lane + u * 64 + 32, z1);
                    }
                    tmem_ld_wait();
                    if (u + 1 == UNITS) give_back();
                    if (KIND == LOSS && !(ok = add_parts(z))) break;
                    if (valid < 64) {
#pragma unroll
                        for (int j = 0; j < 64; ++j)
                            if (j >= valid) z[j] = -INFINITY;
                    }
                    if (__any_sync(0xffffffffu, (a >> 6) == 0)) {           // a target in these columns: rare
                        float zt = 0.0f;
#pragma unroll
                        for (int j = 0; j < 64; ++j)
                            if (a == j) zt = z[j];
                        if ((a >> 6) == 0) p.z_target[row] = zt;
                    }
                    float t4[4] = {fmaxf(z[0], top), z[1], z[2], z[3]};
#pragma unroll
                    for (int j = 4; j < 64; ++j) t4[j & 3] = fmaxf(t4[j & 3], z[j]);
                    const float m = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                    const F2 ref(m == -INFINITY ? 0.0f : -m * LOG2E);               // (columns beyond the vocabulary alone)
                    F2 s2[2] = {F2(u ? sum * shift(top, m) : 0.0f, 0.0f), F2(0.0f)};
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const F2 e = fma2(F2(z[2 * j], z[2 * j + 1]), F2(LOG2E), ref);
                        s2[j & 1] = s2[j & 1] + F2(ex2(e.lo()), ex2(e.hi()));
                    }
                    const F2 both = s2[0] + s2[1];
                    sum = both.lo() + both.hi();
                    top = m;
                }
                if (!ok) break;
                // The warps of a lane quarter join their columns, in turn, an item later, so that none waits for another.  Four barriers and
                // buffers, for items k, k + 1 ..: a warp that arrives for item k + 4 has met an accumulator that every other warp gave back
                // at item k + 2 (k + 3 in groups) or later, after it had arrived for k + 1 and, if it was the one to join k, had read
                // it.  (With one barrier a warp that is an item ahead arrives twice where another has not yet.)
                if (k > 0 && h == (int)((k - 1) & (SHARERS - 1)) && !join(k - 1, before)) break;
                before = w;
                sums[((k & 3) * SHARERS + h) * 128] = make_float2(top, sum);
                __syncwarp();
                if (lane == 0) mbar_arrive(joined + 8 * (k & 3));
            } else if (dlogits) {
                const F2 ref(-lse * LOG2E), up2(up);        // (rows behind the last token: logits 0, up 0)
                const uint32_t line = smem_u32(stage) + lane * 128;
                float all[KIND == DLOGITS ? 64 : 1];
                if constexpr (KIND == DLOGITS) {
                    tmem_ld32(t_lane, *reinterpret_cast<float (*)[32]>(all));
                    tmem_ld32(t_lane + 32, *reinterpret_cast<float (*)[32]>(all + 32));
                    tmem_ld_wait();
                    give_back();
                    if (!add_parts(all)) break;
                }
#pragma unroll 1
                for (int u = 0; u < UNITS; ++u) {
                    const int valid = p.V - v - u * 64, a = at - u * 64;
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the staging tile is free again
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float z[32];
                        if constexpr (KIND == DLOGITS) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) z[j] = all[c * 32 + j];
                        } else {
                            tmem_ld32(t_lane + u * 64 + c * 32, z);
                            tmem_ld_wait();
                            if (c == 1 && u + 1 == UNITS) give_back();
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const F2 e = fma2(F2(z[j], z[j + 1]), F2(LOG2E), ref);
                            (F2(ex2(e.lo()), ex2(e.hi())) * up2).get(z[j], z[j + 1]);
                        }
                        if (valid < (c + 1) * 32) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (c * 32 + j >= valid) z[j] = 0.0f;
                        }
                        if (__any_sync(0xffffffffu, (a >> 5) == c)) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (a == c * 32 + j) z[j] -= up;
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {       // 16-byte pieces in the 128-byte swizzle
                            uint32_t b[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) b[i] = narrow(F2(z[8 * j + 2 * i], z[8 * j + 2 * i + 1]));
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(line + (((uint32_t)(c * 4 + j) ^ (lane & 7u)) << 4)),
                                         "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3]) : "memory");
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        const size_t block = (size_t)(w.m * 2 + rank) * (p.v_tiles * (TILE / 64)) + w.n * (TILE / 64) + h * UNITS + u;
                        bf16* dst = p.dz + (block * 128 + q * 32) * 64;
                        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(stage)), "r"(STAGING) : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            } else {
                // rows r0.. of the result (tokens, or vocabulary rows), columns c0..; 8 lanes share a 128-byte line of a row
                const int r0 = w.m * TILE + rank * 128 + q * 32, c0 = w.n * TILE + h * 64;
                const int rows = w.dw() ? p.V - p.v0 - r0 : n_valid - r0;
                const int sub = lane >> 3, piece = lane & 7;
                const uint32_t base = smem_u32(stage), line = base + lane * 128;
                float a[2][32];
                if (empty_sum) {
#pragma unroll
                    for (int j = 0; j < 64; ++j) a[j >> 5][j & 31] = 0.0f;
                } else {
                    tmem_ld32(t_lane, a[0]);
                    tmem_ld32(t_lane + 32, a[1]);
                    tmem_ld_wait();
                    give_back();
                    if (w.dw()) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) a[j >> 5][j & 31] *= scale;
                    }
                }
                if (c0 >= p.C || (w.half(p.C) == 64 && h >= 2)) continue;
                auto put = [&](int j, const uint32_t (&b)[4]) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(line + (((uint32_t)j ^ (lane & 7u)) << 4)),
                                 "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3]) : "memory");
                };
                auto get = [&](int r) {                     // this lane's piece of row r
                    uint4 u;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                                 : "r"(base + r * 128 + (((uint32_t)piece ^ (r & 7u)) << 4)) : "memory");
                    return u;
                };
                if (w.dw() && !p.dw_f32) {
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t b[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const __nv_bfloat162 two = __floats2bfloat162_rn(a[j >> 2][(8 * j + 2 * i) & 31], a[j >> 2][(8 * j + 2 * i + 1) & 31]);
                            b[i] = *reinterpret_cast<const uint32_t*>(&two);
                        }
                        put(j, b);
                    }
                    __syncwarp();
                    bf16* dst = (bf16*)p.dw + (size_t)(p.v0 + r0) * p.C + c0 + piece * 8;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = 4 * i + sub;
                        if (r < rows && c0 + piece * 8 < p.C) *reinterpret_cast<uint4*>(dst + (size_t)r * p.C) = get(r);
                    }
                } else {
                    float* const out = w.dw() ? (float*)p.dw + (size_t)(p.v0 + r0) * p.C : p.acc + ((size_t)w.slice * p.n_pad + r0) * p.C;
                    const bool add = w.dw() || !p.first, done = !w.dw() && p.last;
                    const int to = done && lane < rows ? p.rows[r0 + lane] : 0;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t b[4] = {__float_as_uint(a[c][4 * j]), __float_as_uint(a[c][4 * j + 1]), __float_as_uint(a[c][4 * j + 2]),
                                                   __float_as_uint(a[c][4 * j + 3])};
                            put(j, b);
                        }
                        __syncwarp();
                        const int col = c0 + c * 32 + piece * 4;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int r = 4 * i + sub;
                            const int token = __shfl_sync(0xffffffffu, to, r);
                            if (r < rows && col < p.C) {
                                float4* d = reinterpret_cast<float4*>(out + (size_t)r * p.C + col);
                                const uint4 u = get(r);
                                float4 x = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
                                if (add) {
                                    const float4 o = *d;
                                    x.x += o.x; x.y += o.y; x.z += o.z; x.w += o.w;
                                }
                                if (done) put_dx(p.dx, p.dx_f32, (size_t)token * p.C + col, x, scale);
                                else *d = x;
                            }
                        }
                    }
                }
            }
        }
        if (is_loss(KIND) && k > 0 && h == (int)((k - 1) & (SHARERS - 1))) join(k - 1, before);
        if (KIND != GRADS && !is_loss(KIND) && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    // neither CTA may leave (or give its TMEM back) while the other can still read its shared memory or signal it
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// ---- packing ----------------------------------------------------------------------------------------------------------
struct PackP {
    const void* x;
    const int32_t* targets;
    int n, C, Cp, V, n_pad, per_block;
    int direct;                 // no copy where no token is left out
    int32_t* n_valid;           // [0], followed by the counters of the products
    int32_t *rows, *target;     // packed -> token; its target
    bf16* xp;                   // [n_pad][Cp]
    int32_t* status;
    // the loss
    float *loss, *lse;          // zero for tokens that take no part
    // the gradients
    const float *lse_in, *d_loss_in;
    float *lse_p, *d_loss_p, *scale;
    void* dx;                   // zero for tokens that take no part
};

// The tokens that take part, packed in their order, and zeros up to whole tiles.  Every block counts the targets before its
// own tokens (and all of them, for the zeros): N * 4 bytes out of L2 for each of at most 296 blocks.
template <typename TIo, bool GRAD>
__global__ void __launch_bounds__(256) head_pack_kernel(const PackP p)
{
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int t0 = blockIdx.x * p.per_block, t1 = min(p.n, t0 + p.per_block);
    __shared__ int sums[2][8];
    __shared__ float tops[8];
    int before = 0, all = 0;
    float top = 0.0f;
    bool bad = false;
    for (int i = tid; i < p.n; i += 256) {
        const int t = p.targets[i], in = t >= 0 && t < p.V;
        bad |= t >= p.V;
        all += in;
        before += i < t0 ? in : 0;
        if (GRAD && in) top = fmaxf(top, fabsf(p.d_loss_in[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
        if (GRAD) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (lane == 0) sums[0][warp] = before, sums[1][warp] = all, tops[warp] = top;
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) before += sums[0][i], all += sums[1][i], top = fmaxf(top, tops[i]);
    if (!(top > 0.0f && top < INFINITY)) top = 1.0f;        // (a d_loss that is not finite spoils its own token only)
    if (blockIdx.x == 0) {
        for (int i = tid; i < COUNTERS; i += 256) p.n_valid[i] = i == 0 ? all : 0;
        if (GRAD && tid == 0) *p.scale = top;
        if (bad && p.status) atomicOr(p.status, ST_BAD_TARGET);
    }
    const bool copy = !(p.direct && all == p.n);
    constexpr int PER = 8;
    auto copy_row = [&](const TIo* from, bf16* to) {        // one warp; columns beyond C (and all without `from`) are zero
        for (int c = lane * PER; c < p.Cp; c += 32 * PER) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (from && c < p.C) {
                if constexpr (sizeof(TIo) == 2) {
                    u = *reinterpret_cast<const uint4*>(from + c);
                } else {
                    const float4 a = *reinterpret_cast<const float4*>(from + c), b = *reinterpret_cast<const float4*>(from + c + 4);
                    const __nv_bfloat162 h[4] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w),
                                                 __floats2bfloat162_rn(b.x, b.y), __floats2bfloat162_rn(b.z, b.w)};
                    u = *reinterpret_cast<const uint4*>(h);
                }
            }
            *reinterpret_cast<uint4*>(to + c) = u;
        }
    };
    // 32 tokens at a time: every warp finds their places, and takes every eighth of them
    for (int i0 = t0; i0 < t1; i0 += 32) {
        const int i = i0 + lane, t = i < t1 ? p.targets[i] : -1;
        const bool in = t >= 0 && t < p.V;
        const uint32_t mask = __ballot_sync(0xffffffffu, in);
        const int j = before + __popc(mask & ((1u << lane) - 1u));
        if (warp == 0 && i < t1) {
            if (in) {
                p.rows[j] = i;
                p.target[j] = t;
                if (GRAD) {
                    p.lse_p[j] = p.lse_in[i];
                    p.d_loss_p[j] = p.d_loss_in[i] / top;
                }
            } else if (!GRAD) {
                p.loss[i] = 0.0f;
                p.lse[i] = 0.0f;
            }
        }
        for (int r = warp; r < min(32, t1 - i0); r += 8) {
            const size_t o = (size_t)(i0 + r) * p.C;
            const int at = __shfl_sync(0xffffffffu, j, r);
            if (mask >> r & 1) {
                if (copy) copy_row((const TIo*)p.x + o, p.xp + (size_t)at * p.Cp);
            } else if (GRAD) {
                for (int c = lane * PER; c < p.C; c += 32 * PER)
#pragma unroll
                    for (int k = 0; k < (int)sizeof(TIo) / 2; ++k) reinterpret_cast<uint4*>((TIo*)p.dx + o + c)[k] = make_uint4(0, 0, 0, 0);
            }
        }
        before += __popc(mask);
    }
    const int end = (all + TILE - 1) / TILE * TILE;
    if (copy)
        for (int j = all + blockIdx.x * 8 + warp; j < end; j += gridDim.x * 8) copy_row(nullptr, p.xp + (size_t)j * p.Cp);
}

// ---- joining ----------------------------------------------------------------------------------------------------------
// lse and loss from the tiles' maxima and sums: 32 tokens per block, WARPS warps that take runs of eight tiles in turn, joined in order.
// targets: of tokens that were not packed (null: packed ones)
template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
head_join_kernel(const int32_t* n_valid, const float2* part, const float* z_target, const int32_t* rows, const int32_t* targets, int n, int V, int n_pad, float* loss,
                 float* lse, int32_t* status)
{
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * 32 + lane, all_rows = targets ? n : *n_valid, v_tiles = (V + TILE - 1) / TILE;
    if (blockIdx.x * 32 >= all_rows) return;
    const bool real = row < all_rows;
    __shared__ float2 sh[WARPS][32];
    float top = -INFINITY, sum = 0.0f;
    if (real)
        for (int v0 = warp * 8; v0 < v_tiles; v0 += WARPS * 8) {
            float2 o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = v0 + i < v_tiles ? part[(size_t)(v0 + i) * n_pad + row] : make_float2(-INFINITY, 0.0f);
            float m = top;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, o[i].x);
            sum *= shift(top, m);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(o[i].y, shift(o[i].x, m), sum);
            top = m;
        }
    sh[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp > 0 || !real) return;
    float m = -INFINITY, all = 0.0f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) m = fmaxf(m, sh[i][lane].x);
#pragma unroll
    for (int i = 0; i < WARPS; ++i)
        if (i * 8 < v_tiles) all = fmaf(sh[i][lane].y, shift(sh[i][lane].x, m), all);
    const float l = m + logf(all);
    const int i = targets ? row : rows[row], t = targets ? targets[row] : 0;
    const bool in = t >= 0 && t < V;
    if (t >= V) atomicOr(status, ST_BAD_TARGET);
    lse[i] = in ? l : 0.0f;
    loss[i] = in ? l - z_target[row] : 0.0f;
}

// dx from several slices of the vocabulary: a token per block of x, four channels per thread.
__global__ void __launch_bounds__(128)
head_dx_kernel(const int32_t* n_valid, const float* scale, const float* acc, const int32_t* rows, int slices, int n_pad, int C, void* dx, int f32)
{
    pdl_wait();
    const int row = blockIdx.x, c = (blockIdx.y * 128 + threadIdx.x) * 4;
    if (row >= *n_valid || c >= C) return;
    const float* from = acc + (size_t)row * C + c;
    const size_t pitch = (size_t)n_pad * C;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int i = 0; i < slices; ++i) {
        const float4 o = *reinterpret_cast<const float4*>(from + i * pitch);
        s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
    }
    put_dx(dx, f32, (size_t)rows[row] * C + c, s, *scale);
}

// ---- host side --------------------------------------------------------------------------------------------------------
size_t up(size_t v, size_t a) { return (v + a - 1) / a * a; }

struct HeadWs {
    size_t counters, scale, rows, target, lse, d_loss, z_target, xp, part, acc, dz;
    size_t fixed;               // all of it but dz
    int n_pad, Cp, v_tiles, c_tiles;
};
HeadWs head_ws(int n, int C, int V, bool grad, int slices)
{
    HeadWs w = {};
    w.n_pad = (int)up(n, TILE);
    w.Cp = (int)up(C, 64);
    w.v_tiles = (int)(up(V, TILE) / TILE);
    w.c_tiles = (int)(up(C, TILE) / TILE);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t o = off;
        off = up(off + bytes, 1024);
        return o;
    };
    const size_t N = w.n_pad;
    w.counters = take(COUNTERS * 4);
    w.scale = take(4);
    w.rows = take(N * 4);
    w.target = take(N * 4);
    w.xp = take(N * w.Cp * 2);
    if (grad) {
        w.lse = take(N * 4);
        w.d_loss = take(N * 4);
        w.acc = take(N * C * 4 * slices);
        w.dz = off;
    } else {
        w.z_target = take(N * 4);
        w.part = take(N * w.v_tiles * 8);
    }
    w.fixed = off;
    return w;
}
size_t dz_tile_bytes(int n_pad) { return (size_t)n_pad * TILE * 2; }     // of 256 vocabulary rows

int check_shape(int n, int C, int V, int io)
{
    if (n < 0 || C <= 0 || V <= 0) return fail(MGPT_MOE_EINVAL, "head loss: sizes must be positive");
    if (C % 8) return fail(MGPT_MOE_EINVAL, "head loss: embed_dim must be a multiple of 8");
    if (io != MGPT_MOE_IO_F32 && io != MGPT_MOE_IO_BF16) return fail(MGPT_MOE_EINVAL, "unknown io dtype");
    if (up(n, TILE) > (1u << 30) || up(V, TILE) > (1u << 30) || (double)(up(n, TILE) / TILE) * (up(V, TILE) / TILE) > 1e9 || C > (1 << 20))
        return fail(MGPT_MOE_EINVAL, "head loss: sizes out of range");
    return 0;
}
// Whether x is read where it lies rather than from a packed copy, if no token is left out.  Rows off 32-byte boundaries cost two sectors
// for one (4740 x 296 x 65753: 227 us, 168 at C = 288), boxes that reach beyond the last token as much as full ones and more (3 tokens of
// 1376 channels, gradient of the logits: 45 us, 37 from the copy); a copy of few tokens costs nothing.
bool as_it_lies(int n, int C, int io) { return io == MGPT_MOE_IO_BF16 && C % 16 == 0 && (n % TILE == 0 || n >= 8 * TILE); }
// token tiles whose x (and dz) share the L2 with a vocabulary tile
int group_of(int n_pad, int Cp)
{
    const size_t tile = (size_t)TILE * Cp * 2, most = (size_t)32 << 20;
    const int mt = n_pad / TILE, g = (int)(most / tile);
    return g < 1 ? 1 : g > mt ? mt : g;
}
// Slices of the vocabulary that dx is summed in.  dx and dw are the same work, so of the 74 pairs' shares half is dx: 60 items are
// enough for none to be more than two thirds of a share, and more only cost sums.  us, both products and the sum of the slices, at
// 148 / 74 / 37 items: 1 of 3 tokens, 1376 x 52191 83 / 79 / 76; 300 tokens, 488 x 37571 45 / 40 / 40; 8192 tokens, 512 x 32000
// 390 / 388 / 366 (one slice); 1501 of 3001 tokens, 1024 x 50021, half of whose items turn out not to exist 234 / 224 / 275 (one).
int slices_of(int n_pad, int c_tiles, int v_tiles)
{
    const int items = n_pad / TILE * c_tiles;
    int s = (60 + items - 1) / items;
    if (s > v_tiles / 4) s = v_tiles / 4;
    return s < 1 ? 1 : s;
}

template <int KIND>
int launch_head(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& a2, const CUtensorMap& b2, const CUtensorMap& x, const HeadP& p, int pairs, cudaStream_t st)
{
    static bool done[64] = {};
    int dev = 0;
    MGPT_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !done[dev]) {
        MGPT_CUDA(cudaFuncSetAttribute(head_kernel<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<KIND>()));
        if (dev < 64) done[dev] = true;
    }
    MGPT_CUDA(launch_pdl(head_kernel<KIND>, 2 * pairs, THREADS, smem_bytes<KIND>(), st, a, b, a2, b2, x, p));
    MGPT_LAUNCHED("head_kernel");
    return 0;
}
int sm_count(int* sms)
{
    static int known[64];
    int dev = 0;
    MGPT_CUDA(cudaGetDevice(&dev));
    *sms = dev < 64 ? known[dev] : 0;
    if (!*sms) MGPT_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 64) known[dev] = *sms;
    if (*sms < 2) return fail(MGPT_MOE_ECUDA, "head loss: needs two SMs");
    return 0;
}

template <bool GRAD> int launch_pack(PackP& p, int io, cudaStream_t st)
{
    p.per_block = (p.n + 295) / 296;
    int blocks = (p.n + p.per_block - 1) / p.per_block;
    if (blocks < 32) blocks = 32;                       // (the zeros behind the last token)
    if (io == MGPT_MOE_IO_BF16) MGPT_CUDA(launch_pdl(head_pack_kernel<bf16, GRAD>, blocks, 256, 0, st, p));
    else MGPT_CUDA(launch_pdl(head_pack_kernel<float, GRAD>, blocks, 256, 0, st, p));
    MGPT_LAUNCHED("head_pack_kernel");
    return 0;
}

}  // namespace

}  // namespace mgpt

using namespace mgpt;

extern "C" {

size_t mgpt_moe_op_head_loss_workspace_bytes(int n, int C, int V)
{
    if (check_shape(n, C, V, MGPT_MOE_IO_BF16) || n == 0) return 0;
    return head_ws(n, C, V, false, 1).fixed;
}

size_t mgpt_moe_op_head_loss_backward_workspace_bytes(int n, int C, int V, size_t piece_bytes)
{
    if (check_shape(n, C, V, MGPT_MOE_IO_BF16) || n == 0) return 0;
    HeadWs w = head_ws(n, C, V, true, 1);
    w = head_ws(n, C, V, true, slices_of(w.n_pad, w.c_tiles, w.v_tiles));
    const size_t tile = dz_tile_bytes(w.n_pad);
    size_t tiles = piece_bytes / tile;
    const size_t least = ((size_t)w.v_tiles + MAX_PIECES - 1) / MAX_PIECES;
    tiles = tiles < least ? least : tiles > (size_t)w.v_tiles ? w.v_tiles : tiles;
    return w.fixed + tiles * tile;
}

int mgpt_moe_op_head_loss(const void* x, int io, const void* w, const int32_t* targets, int n, int C, int V, float* loss, float* lse,
                          int32_t* status, void* workspace, size_t ws_bytes, mgpt_stream_t stream)
{
    MGPT_TRY(check_shape(n, C, V, io));
    if (n == 0) return 0;
    if (!x || !w || !targets || !loss || !lse || !status) return fail(MGPT_MOE_EINVAL, "null argument");
    MGPT_TRY(check_aligned(x, "x"));
    MGPT_TRY(check_aligned(w, "w"));
    if (!workspace || ((uintptr_t)workspace & 255)) return fail(MGPT_MOE_EINVAL, "workspace must be 256-byte aligned");
    const HeadWs h = head_ws(n, C, V, false, 1);
    if (ws_bytes < h.fixed) return fail(MGPT_MOE_ENOMEM, "workspace smaller than mgpt_moe_op_head_loss_workspace_bytes()");
    cudaStream_t st = (cudaStream_t)stream;
    char* ws = (char*)workspace;
    int sms;
    MGPT_TRY(sm_count(&sms));
    CUtensorMap mx, mw, mx0;
    const bool packed = io != MGPT_MOE_IO_BF16 || n > TILE, direct = !packed || as_it_lies(n, C, io);
    MGPT_TRY(make_map_kind(&mx, ws + h.xp, h.n_pad, h.Cp, 128, false));
    MGPT_TRY(make_map_kind(&mw, w, V, C, 128, false));
    // One tile of tokens: only the rows that there are (a box that reaches beyond them is slower than one that is full: 3 tokens of
    // 1376 channels against 208764 vocabulary rows 153 us, 200 tokens 113).
    const int few[2] = {n < 128 ? (int)up(n, 8) : 128, n <= 128 ? 0 : (int)up(n - 128, 8)};
    if (direct) MGPT_TRY(make_map_kind(&mx0, x, n, C, packed ? 128 : few[0], false));
    if (!packed && few[1]) MGPT_TRY(make_map_kind(&mx, x, n, C, few[1], false));
    PackP k = {};
    k.x = x; k.targets = targets; k.n = n; k.C = C; k.Cp = h.Cp; k.V = V; k.n_pad = h.n_pad; k.direct = direct;
    k.n_valid = (int32_t*)(ws + h.counters);
    k.rows = (int32_t*)(ws + h.rows); k.target = (int32_t*)(ws + h.target); k.xp = (bf16*)(ws + h.xp);
    k.status = status; k.loss = loss; k.lse = lse;
    // one tile of tokens costs the same with or without those that take no part: no need to sort them out
    if (packed) MGPT_TRY(launch_pack<false>(k, io, st));
    HeadP p = {};
    p.n_valid = packed ? k.n_valid : nullptr; p.n = n; p.few[0] = few[0]; p.few[1] = few[1]; p.direct = direct; p.sched = packed ? k.n_valid + 1 : nullptr;
    p.status = status; p.C = C; p.V = V; p.v_tiles = h.v_tiles;
    p.group = group_of(h.n_pad, h.Cp); p.n_pad = h.n_pad; p.target = packed ? k.target : targets;
    p.part = (float2*)(ws + h.part); p.z_target = (float*)(ws + h.z_target);
    const long items = (long)(h.n_pad / TILE) * h.v_tiles;
    const int pairs = (int)(items < sms / 2 ? items : sms / 2);
    if (C <= NARROW) MGPT_TRY(launch_head<LOSS_NARROW>(mx, mw, mx, mw, direct ? mx0 : mx, p, pairs, st));
    else MGPT_TRY(launch_head<LOSS>(mx, mw, mx, mw, direct ? mx0 : mx, p, pairs, st));
    const int32_t* as_given = packed ? nullptr : targets;
    if (n < 32 * sms) MGPT_CUDA(launch_pdl(head_join_kernel<16>, (n + 31) / 32, 512, 0, st, p.n_valid, p.part, p.z_target, k.rows, as_given, n, V, h.n_pad, loss, lse, status));
    else MGPT_CUDA(launch_pdl(head_join_kernel<4>, (n + 31) / 32, 128, 0, st, p.n_valid, p.part, p.z_target, k.rows, as_given, n, V, h.n_pad, loss, lse, status));
    MGPT_LAUNCHED("head_join_kernel");
    return 0;
}

int mgpt_moe_op_head_loss_backward(const void* x, int io, const void* w, const int32_t* targets, const float* lse, const float* d_loss,
                                   int n, int C, int V, void* dx, void* dw, int dw_dtype, int32_t* status,
                                   void* workspace, size_t ws_bytes, mgpt_stream_t stream)
{
    MGPT_TRY(check_shape(n, C, V, io));
    if (dw_dtype != MGPT_MOE_IO_F32 && dw_dtype != MGPT_MOE_IO_BF16) return fail(MGPT_MOE_EINVAL, "unknown dtype of dw");
    cudaStream_t st = (cudaStream_t)stream;
    if (!dw) return fail(MGPT_MOE_EINVAL, "null argument");
    MGPT_TRY(check_aligned(dw, "dw"));
    if (n == 0) {
        if (dw_dtype == MGPT_MOE_IO_BF16) MGPT_CUDA(cudaMemsetAsync(dw, 0, (size_t)V * C * 2, st));
        return 0;
    }
    if (!x || !w || !targets || !lse || !d_loss || !dx || !status) return fail(MGPT_MOE_EINVAL, "null argument");
    MGPT_TRY(check_aligned(x, "x"));
    MGPT_TRY(check_aligned(w, "w"));
    MGPT_TRY(check_aligned(dx, "dx"));
    if (!workspace || ((uintptr_t)workspace & 255)) return fail(MGPT_MOE_EINVAL, "workspace must be 256-byte aligned");
    HeadWs h = head_ws(n, C, V, true, 1);
    const int slices = slices_of(h.n_pad, h.c_tiles, h.v_tiles);
    h = head_ws(n, C, V, true, slices);
    const size_t tile = dz_tile_bytes(h.n_pad);
    const size_t room = ws_bytes > h.fixed ? (ws_bytes - h.fixed) / tile : 0;
    if (room < ((size_t)h.v_tiles + MAX_PIECES - 1) / MAX_PIECES)
        return fail(MGPT_MOE_ENOMEM, "workspace smaller than mgpt_moe_op_head_loss_backward_workspace_bytes()");
    const int most = room > (size_t)h.v_tiles ? h.v_tiles : (int)room;
    const int pieces = (h.v_tiles + most - 1) / most, per = (h.v_tiles + pieces - 1) / pieces;
    char* ws = (char*)workspace;
    int sms;
    MGPT_TRY(sm_count(&sms));
    CUtensorMap mx, mw, mx_t, mw_t, mz, mz_t, mx0, mx0_t;
    const bool direct = as_it_lies(n, C, io);
    MGPT_TRY(make_map_kind(&mx, ws + h.xp, h.n_pad, h.Cp, 128, false));
    MGPT_TRY(make_map_kind(&mw, w, V, C, 128, false));
    MGPT_TRY(make_map_kind(&mx_t, ws + h.xp, h.n_pad, h.Cp, 64, false));
    MGPT_TRY(make_map_kind(&mw_t, w, V, C, 64, false));
    mx0 = mx; mx0_t = mx_t;
    if (direct) {
        MGPT_TRY(make_map_kind(&mx0, x, n, C, 128, false));
        MGPT_TRY(make_map_kind(&mx0_t, x, n, C, 64, false));
    }
    const uint64_t tiles = (uint64_t)(h.n_pad / 128) * per * (TILE / 64);
    MGPT_TRY(make_map_tiles(&mz, ws + h.dz, tiles, 128, 1));
    MGPT_TRY(make_map_tiles(&mz_t, ws + h.dz, tiles, 64, 2));
    PackP k = {};
    k.x = x; k.targets = targets; k.n = n; k.C = C; k.Cp = h.Cp; k.V = V; k.n_pad = h.n_pad;
    k.n_valid = (int32_t*)(ws + h.counters);
    k.rows = (int32_t*)(ws + h.rows); k.target = (int32_t*)(ws + h.target); k.xp = (bf16*)(ws + h.xp);
    k.direct = direct; k.status = status; k.lse_in = lse; k.d_loss_in = d_loss; k.lse_p = (float*)(ws + h.lse); k.d_loss_p = (float*)(ws + h.d_loss); k.scale = (float*)(ws + h.scale); k.dx = dx;
    MGPT_TRY(launch_pack<true>(k, io, st));
    HeadP p = {};
    p.n_valid = k.n_valid; p.n = n; p.direct = direct; p.rows = k.rows; p.dx = dx; p.dx_f32 = io == MGPT_MOE_IO_F32; p.status = status; p.C = C; p.V = V; p.group = group_of(h.n_pad, h.Cp); p.n_pad = h.n_pad;
    p.target = k.target; p.lse = k.lse_p; p.d_loss = k.d_loss_p; p.scale = k.scale; p.dz = (bf16*)(ws + h.dz); p.acc = (float*)(ws + h.acc);
    p.c_tiles = h.c_tiles; p.dw = dw; p.dw_f32 = dw_dtype == MGPT_MOE_IO_F32;
    for (int i = 0; i < pieces; ++i) {
        p.v0 = i * per * TILE;
        p.v_tiles = h.v_tiles - i * per < per ? h.v_tiles - i * per : per;
        p.slice_tiles = (per + slices - 1) / slices;            // (of a full piece, whose slices the others keep within)
        p.k_slices = (p.v_tiles + p.slice_tiles - 1) / p.slice_tiles;
        p.first = i == 0;
        p.last = slices == 1 && i == pieces - 1;
        const long items = (long)(h.n_pad / TILE) * p.v_tiles;
        p.sched = k.n_valid + 1 + 2 * i;
        const int pairs = (int)(items < sms / 2 ? items : sms / 2);
        if (C <= NARROW) MGPT_TRY(launch_head<DLOGITS_NARROW>(mx, mw, mx, mw, mx0, p, pairs, st));
        else MGPT_TRY(launch_head<DLOGITS>(mx, mw, mx, mw, mx0, p, pairs, st));
        p.sched = k.n_valid + 2 + 2 * i;
        const long grads = ((long)(h.n_pad / TILE) * p.k_slices + p.v_tiles) * p.c_tiles;
        MGPT_TRY(launch_head<GRADS>(mz, mw_t, mz_t, mx_t, mx0_t, p, (int)(grads < sms / 2 ? grads : sms / 2), st));
    }
    if (slices == 1) return 0;
    const int used = (per + p.slice_tiles - 1) / p.slice_tiles;
    MGPT_CUDA(launch_pdl(head_dx_kernel, dim3(n, (C + 511) / 512), 128, 0, st, k.n_valid, p.scale, p.acc, k.rows, used, h.n_pad, C, dx, p.dx_f32));
    MGPT_LAUNCHED("head_dx_kernel");
    return 0;
}

}  // extern "C"
