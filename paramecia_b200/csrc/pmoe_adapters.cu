// Low-rank adapters of many requests beside one projection: out_t = base_t + s_i B_i (A_i x_t) with i = ids[t], for a
// batch whose rows belong to different adapters.  base is the shared projection's output (pmoe_qmatmul's, say); a row whose
// id is outside [0, L) keeps it.  The reference's QMatMul holds one low-rank update and merges it
// (paramecia-model/src/models/with_tracing.rs:103-337).
//
// What bounds it: 2 r (K + N) flops over K x + 2 N out elements a row, at most r flops a byte, below the ridge of the card
// (258) for every rank served (r <= 128): the rows' stream from memory for prompts, latency for single tokens.
//
// One kernel does both products.  A tile of rows of one adapter belongs to a cluster of one to eight CTAs: each takes a part of
// K for its share of h = A x, the shares are added through distributed shared memory, and each CTA then takes a part of the N
// output columns.  h never goes to memory, and a single token still uses eight SMs.  Two kernels of that form: tiles of
// sixteen rows on the warp-level matrix instructions (k_adapters), and of 128 rows on tcgen05 (k_adapters_tc).
#include <cooperative_groups.h>

#include "pmoe_internal.h"
#include "pmoe_status.h"
#include "pmoe_tcgen05.cuh"
#include "pmoe_vec.cuh"

namespace pmoe {

namespace cg = cooperative_groups;

constexpr int ADAPTER_MAX_RANK = 128, ADAPTER_MAX = 4096;
constexpr int ADAPTER_ROWS_UNSORTED = 1024;   // rows that are grouped by id without pmoe_sort_pairs
constexpr int ADAPTER_ROWS_LEADER = 128;       // ... where every row looks for the rows of its own id alone
constexpr int AD_MAX_CTAS = 8;                // CTAs of a cluster

// c += a b, 16 x 8 x 16, bf16 operands, f32 sums.  Lane l, g = l / 4, q = l % 4: a0 / a1 = rows g / g + 8 at the inner pair
// (2q, 2q + 1), a2 / a3 the same at inner pair 2q + 8; b0, b1 the same inner pairs of column g; c0, c1 = row g, columns
// 2q, 2q + 1; c2, c3 = row g + 8.  The inner index is summed over, so any renaming of it that a and b share is allowed:
// a lane's pairs are taken from consecutive elements (one wide load) instead of the two places the layout names.
__device__ inline void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A pair of f32 values as three pairs of bf16 whose sum is the value: they hold all 24 bits of it (8 + 8 + 8, each remainder
// is exact: the upper half of the bits left is cut off, which makes no infinity of a large number).  An infinity has no remainder; a
// NaN's is one, also where its upper half is an infinity's.  So do f32 rows and h, whatever the result's type: two pieces of h were off by 2^-17 of what the adapter adds, which
// is more than a bf16 result's own rounding where its terms or base cancel.
constexpr int PIECES = 3;

__device__ inline void split_pair(float lo, float hi, uint32_t (&w)[PIECES])
{
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        const uint32_t l = __float_as_uint(lo), h = __float_as_uint(hi);
        w[p] = __byte_perm(l, h, 0x7632);
        const float rest_l = lo - __uint_as_float(l & 0xffff0000u), rest_h = hi - __uint_as_float(h & 0xffff0000u);
        lo = p == 0 && fabsf(lo) == INFINITY ? 0.f : rest_l;
        hi = p == 0 && fabsf(hi) == INFINITY ? 0.f : rest_h;
    }
}

// Eight consecutive inner elements of a row as matrix operands, four pairs: in one piece for bf16, in three for f32 (whose
// second sixteen bytes lie one unit of the warp further).
template <typename XT> struct XFrag;
template <> struct XFrag<__nv_bfloat16> {
    static constexpr int WORDS = 1;
    static __device__ void words(const uint4 *p, uint32_t (&w)[4][1])
    {
        const uint4 v = p[0];
        w[0][0] = v.x; w[1][0] = v.y; w[2][0] = v.z; w[3][0] = v.w;
    }
};
template <> struct XFrag<float> {
    static constexpr int WORDS = PIECES;
    static __device__ void words(const uint4 *p, uint32_t (&w)[4][PIECES])
    {
        const float4 v0 = reinterpret_cast<const float4 *>(p)[0], v1 = reinterpret_cast<const float4 *>(p)[32];
        split_pair(v0.x, v0.y, w[0]);
        split_pair(v0.z, v0.w, w[1]);
        split_pair(v1.x, v1.y, w[2]);
        split_pair(v1.z, v1.w, w[3]);
    }
};

// Asynchronous copies of 16 (8) bytes to shared memory at byte offsets that the instruction carries; size 0 writes zeros
// and reads nothing.
template <int D, int S> __device__ inline void copy16(uint32_t dst, const void *src, int size)
{
    asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, %2;" ::"r"(dst), "l"(src), "r"(size), "n"(D), "n"(S) : "memory");
}
__device__ inline void copy8(uint32_t dst, const void *src, int size)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
}
__device__ inline void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ inline void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// f(Const<0>), ..., f(Const<N - 1>): offsets that depend on the index stay constants
template <int I> struct Const {
    __host__ __device__ constexpr operator int() const { return I; }
};
template <int N, typename F> __device__ __forceinline__ void each(F &&f)
{
    if constexpr (N > 0) {
        each<N - 1>(f);
        f(Const<N - 1>{});
    }
}

struct AdapterArgs {
    int n, K, N, r, L;
    const __nv_bfloat16 *a, *b;
    const float *scales;
    const int *ids, *order, *offsets;
};

// out = base in the rows that have no adapter.  They are in no tile, and may be any number of them side by side, so every CTA
// of the grid takes the rows blockIdx.x, blockIdx.x + gridDim.x, ... when its tile is done (copied by the tiles' slots,
// 64 rows each before their tile, they doubled the time of 8192 rows with a thirteenth of them bare).
// The lanes of a warp look at 32 of them at a time; the first ids are loaded when the kernel begins.
__device__ inline int id_of_share(const AdapterArgs &P, int first)
{
    const int64_t t = blockIdx.x + (int64_t)gridDim.x * (first + (threadIdx.x & 31));
    return t < P.n ? P.ids[t] : 0;
}

template <int THREADS, typename OT> __device__ inline void copy_bare_rows(const AdapterArgs &P, int my_id, const OT *base, OT *out)
{
    if (out == base) return;
    const int units = P.N / 8;
    for (int first = 0;;) {
        unsigned bare = __ballot_sync(0xffffffffu, (unsigned)my_id >= (unsigned)P.L);
        int u = threadIdx.x;   // this thread's next unit, of the lowest row left in `bare`
        while (true) {
            float v[4][8];
            size_t at[4];
            int got = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                while (bare && u >= units) { u -= units; bare &= bare - 1; }
                if (!bare) break;
                at[k] = (size_t)(blockIdx.x + (int64_t)gridDim.x * (first + __ffs(bare) - 1)) * P.N + u * 8;
                load_units<8>(base + at[k], v[k]);
                u += THREADS;
                got++;
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (k < got) store_units<8>(out + at[k], v[k]);
            if (got < 4) break;
        }
        first += 32;
        if (blockIdx.x + (int64_t)gridDim.x * first >= P.n) return;
        __syncwarp();
        my_id = id_of_share(P, first);
    }
}

// The sum of four floats at the same place in CTAS CTAs of the cluster, in CTA order; the loads are independent
template <int CTAS> __device__ inline float4 sum_of_cluster(cg::cluster_group &cluster, const float *p)
{
    float4 v[CTAS], s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int o = 0; o < CTAS; o++) v[o] = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(const_cast<float *>(p), o));
#pragma unroll
    for (int o = 0; o < CTAS; o++) { s.x += v[o].x; s.y += v[o].y; s.z += v[o].z; s.w += v[o].w; }
    return s;
}

// f(Const<ctas>): clusters are of 1, 2, 4 or 8 CTAs
template <typename F> __device__ __forceinline__ void with_cluster_size(int ctas, F &&f)
{
    if (ctas == 1) f(Const<1>{});
    else if (ctas == 2) f(Const<2>{});
    else if (ctas == 4) f(Const<4>{});
    else f(Const<8>{});
}

// The tile of a slot: its adapter and rows (-1: none), the same for every CTA that asks for it.  With the adapters' rows one
// after another (the first of adapter e at offsets[e]), its tile slots begin at offsets[e] / T + e: with one slot more than whole
// multiples of T inside its range that is never fewer than it has tiles, and each adapter finds its own without a scan.
template <int T, int THREADS>
__device__ inline void tile_of_slot(const AdapterArgs &P, const int *offsets, int slot, int &tile_id, int &tile_rows, int &tile_first)
{
    for (int e = threadIdx.x; e < P.L; e += THREADS) {
        const int from = offsets[e], to = min(offsets[e + 1], P.n), nth = slot - (from / T + e);
        if (from >= 0 && nth >= 0 && nth < (to - from + T - 1) / T) {   // one adapter at most
            tile_id = e;
            tile_first = from + nth * T;
            tile_rows = min(T, to - from - nth * T);
        }
    }
}

// From pmoe_sort_pairs's arrays
template <int T, int THREADS>
__device__ inline void find_tile(const AdapterArgs &P, int slot, int *rows, int &tile_id, int &tile_rows, int &tile_first)
{
    const int tid = threadIdx.x;
    if (tid == 0) tile_rows = 0;
    __syncthreads();
    tile_of_slot<T, THREADS>(P, P.offsets, slot, tile_id, tile_rows, tile_first);
    __syncthreads();
    if (tid < T) rows[tid] = tid < tile_rows ? P.order[tile_first + tid] : -1;
    __syncthreads();
}

// From the ids alone: every CTA counts them, then looks for the rows of its own tile.  A sort in front is a launch of its own,
// 4 us for few rows (1000 rows, 4 adapters of rank 64: 16.7 us without it, 20.9 us with it; 1024 rows, 16 adapters: 18.6 and 17.6), but it
// reads the ids once where here every CTA does: 8192 rows took 56 us without and 47 us with it.
// offsets: L + 1 words of shared memory
template <int T, int THREADS>
__device__ inline void find_tile_by_ids(const AdapterArgs &P, int slot, int *rows, int &tile_id, int &tile_rows, int &tile_first, int *offsets)
{
    constexpr int WARPS = THREADS / 32;
    __shared__ int found_by[WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int e = tid; e <= P.L; e += THREADS) offsets[e] = 0;
    if (tid == 0) tile_rows = 0;
    __syncthreads();
#pragma unroll 4
    for (int t = tid; t - lane < P.n; t += THREADS) {
        const int id = t < P.n ? P.ids[t] : -1;
        const int same = __all_sync(0xffffffffu, id == __shfl_sync(0xffffffffu, id, 0));   // a prompt's rows
        if ((unsigned)id < (unsigned)P.L && (!same || lane == 0)) atomicAdd(offsets + id, same ? 32 : 1);
    }
    __syncthreads();
    if (warp == 0) {   // the counts become their exclusive sums
        int before = 0;
        for (int e = lane; e - lane <= P.L; e += 32) {
            const int count = e < P.L ? offsets[e] : 0;
            int incl = count;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += y;
            }
            if (e <= P.L) offsets[e] = before + incl - count;
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    __syncthreads();
    tile_of_slot<T, THREADS>(P, offsets, slot, tile_id, tile_rows, tile_first);
    if (tid < T) rows[tid] = -1;
    __syncthreads();
    if (tile_rows == 0) return;
    // a warp's part of the ids; its rows of this adapter are counted, then those of the tile's range written down
    const int id = tile_id, first = tile_first - offsets[id], part = (P.n + THREADS - 1) / THREADS * 32;
    const int t0 = warp * part, t1 = min(P.n, t0 + part);
    int count = 0;
#pragma unroll 4
    for (int t = t0 + lane; t - lane < t1; t += 32) count += __popc(__ballot_sync(0xffffffffu, t < t1 && P.ids[t] == id));
    if (lane == 0) found_by[warp] = count;
    __syncthreads();
    int nth = -first;
#pragma unroll
    for (int w = 0; w < WARPS; w++)
        if (w < warp) nth += found_by[w];
    if (nth < T && nth + count > 0)
        for (int t = t0 + lane; t - lane < t1 && nth < T; t += 32) {
            const bool mine = t < t1 && P.ids[t] == id;
            const unsigned m = __ballot_sync(0xffffffffu, mine);
            const int at = nth + __popc(m & ((1u << lane) - 1));
            if (mine && at >= 0 && at < T) rows[at] = t;
            nth += __popc(m);
        }
    __syncthreads();
}

// ---------------------------------------------------------------- few rows of an adapter, or f32 rows: sixteen rows a tile
// A CTA of four warps walks its share of K and then its share of N in stages of four chunks of 32, a chunk a warp: a stage
// holds what the matrix instructions of a chunk need, as the lanes need it (sixteen bytes per lane, lanes side by side, so no
// access meets a bank twice), and a warp reads what its own lanes fetched.  The copies are asynchronous and STAGES stages are on
// their way, the first ones of N while the shares of h are still being added: one decoding row of 2048 x 2048 takes 5 us, 64
// rows with 36 adapters of rank 32 (2048 to 4096) 10.1 us, which is the chain id -> rows -> h -> exchange -> columns.
// RT: groups of eight ranks that the accumulators are sized for.
constexpr int FEW_M = 16, FEW_THREADS = 128;

template <typename XT, typename OT, int RT> struct AdapterStage {
    static constexpr int SIZE = sizeof(XT) > sizeof(OT) ? sizeof(XT) : sizeof(OT);
    static constexpr int WEIGHTS = 4 * RT * 32 * 16;                     // A: 4 chunks x RT rank groups; B: 4 chunks x 4 products x RT / 4 rank steps
    static constexpr int ROW_CHUNK = 2 * 32 * 8 * SIZE;                 // two rows of eight elements a lane
    static constexpr int BYTES = WEIGHTS + 4 * ROW_CHUNK;
    static constexpr int HS = RT == 2 ? 16 : RT * 8 + 16;               // floats between two rows of h: no two rows of a quarter warp start in one bank
    static constexpr int H_BYTES = 3 * FEW_M * HS * 4;
    static constexpr int ROOM = (RT == 16 ? 222 : 110) * 1024 - H_BYTES;   // of the 227 KB of an SM: one or two CTAs at least
    static constexpr int STAGES = ROOM / BYTES < 2 ? 2 : ROOM / BYTES > 4 ? 4 : ROOM / BYTES;
    static constexpr int SMEM = STAGES * BYTES + H_BYTES;
    static_assert(SMEM <= 222 * 1024, "fits an SM beside the static arrays");
};

template <typename XT, typename OT, int RT>
__global__ void __launch_bounds__(FEW_THREADS, RT == 16 ? 1 : 4) k_adapters(AdapterArgs P, const XT *__restrict__ x, const OT *base, OT *out)
{
    using S = AdapterStage<XT, OT, RT>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int rows[FEW_M];
    __shared__ int tile_id, tile_rows, tile_first;
    __shared__ int all_ids[ADAPTER_ROWS_LEADER];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), c = (int)cluster.block_rank(), slot = blockIdx.x / ctas;
    constexpr int HS = S::HS;
    float *part = reinterpret_cast<float *>(smem + S::STAGES * S::BYTES);   // [2][16][HS] this CTA's share of h
    float *h = part + 2 * FEW_M * HS;                                       // [16][HS]
    pdl_wait();
    pdl_launch_dependents();

    const int share_id = id_of_share(P, 0);

    // ---- the tile: its adapter and rows.  Every CTA of the cluster finds the same.
    if (P.order) {
        find_tile<FEW_M, FEW_THREADS>(P, slot, rows, tile_id, tile_rows, tile_first);
    } else if (P.n > ADAPTER_ROWS_LEADER) {
        find_tile_by_ids<FEW_M, FEW_THREADS>(P, slot, rows, tile_id, tile_rows, tile_first, reinterpret_cast<int *>(smem));
    } else {
        // slot t leads a tile when the number of earlier rows with its id is a multiple of sixteen
        const int id = P.ids[slot];
        if (tid < FEW_M) rows[tid] = -1;
        for (int t = tid; t < P.n; t += FEW_THREADS) all_ids[t] = P.ids[t];
        __syncthreads();
        if (warp == 0) {
            int before = 0, found = 0;
            for (int t = 0; t < P.n && found < FEW_M; t += 32) {
                const bool same = t + lane < P.n && all_ids[t + lane] == id;
                const unsigned m = __ballot_sync(0xffffffffu, same);
                const unsigned early = t + 32 <= slot ? m : t > slot ? 0u : m & ((1u << (slot - t)) - 1);
                before += __popc(early);
                const int at = found + __popc(m & ~early & ((1u << lane) - 1));
                if (same && !(early >> lane & 1) && at < FEW_M) rows[at] = t + lane;
                found += __popc(m & ~early);
            }
            if (lane == 0) {
                tile_id = id;
                tile_rows = (unsigned)id >= (unsigned)P.L || before % FEW_M ? 0 : min(found, FEW_M);
            }
        }
        __syncthreads();
    }
    if (tile_rows == 0) {
        copy_bare_rows<FEW_THREADS>(P, share_id, base, out);
        return;
    }
    const int id = tile_id, t0 = rows[g], t1 = rows[g + 8];
    const bool has0 = (unsigned)t0 < (unsigned)P.n, has1 = (unsigned)t1 < (unsigned)P.n;

    // ---- the stages of this CTA
    const int kc = (P.K + 31) / 32, nc = (P.N + 31) / 32;
    const int k0 = (int)((int64_t)kc * c / ctas), k1 = (int)((int64_t)kc * (c + 1) / ctas);
    const int n0 = (int)((int64_t)nc * c / ctas), n1 = (int)((int64_t)nc * (c + 1) / ctas);
    const int kstages = (k1 - k0 + 3) / 4, stages = kstages + (n1 - n0 + 3) / 4;
    const int size0 = has0 ? 16 : 0, size1 = has1 ? 16 : 0;
    // Where this lane fetches from, a stage further after each: its two rows in x, later in base; the weights of this warp's
    // chunk in A, later in B.  EX, EO: elements of x and base in sixteen bytes.
    constexpr int EX = 16 / sizeof(XT), EO = 16 / sizeof(OT);
    const XT *x0 = x + (has0 ? (size_t)t0 * P.K : 0) + (k0 + warp) * 32 + q * EX, *x1 = x + (has1 ? (size_t)t1 * P.K : 0) + (k0 + warp) * 32 + q * EX;
    const OT *b0 = base + (has0 ? (size_t)t0 * P.N : 0) + (n0 + warp) * 32 + q * EO, *b1 = base + (has1 ? (size_t)t1 * P.N : 0) + (n0 + warp) * 32 + q * EO;
    const __nv_bfloat16 *aw = P.a + ((size_t)id * P.r + g) * P.K + (k0 + warp) * 32 + q * 8;
    const size_t aw_step = (size_t)8 * P.K;
    const __nv_bfloat16 *bw = P.b + ((size_t)id * P.N + (n0 + warp) * 32 + (g >> 1) * EO + (g & 1)) * P.r + q * (RT == 2 ? 4 : 8);
    const uint32_t to_weights = smem_u32(smem) + warp * (S::WEIGHTS / 4), to_rows = smem_u32(smem) + S::WEIGHTS + warp * S::ROW_CHUNK;
    const bool all_ranks = P.r == RT * 8;

    // Rows: a copy instruction takes 64 consecutive bytes of each of eight rows.  For f32 that is half a chunk (v = 0, 1);
    // x's pieces go to the lane that multiplies them (eight consecutive elements, like the weights' sixteen bytes), base's
    // stay with the lane that adds them: its columns are four and four, sixteen apart.
    const uint32_t x_lane = sizeof(XT) == 2 ? lane * 16 : (q & 1) * 512 + (g * 4 + (q >> 1)) * 16;
    constexpr int X_STEP = 32, B_STEP = 512;   // from v = 0 to v = 1
    auto fetch_rows = [&](uint32_t dst, auto step, auto *p0, auto *p1, bool whole, int first, int limit) {
        using VT = std::remove_cv_t<std::remove_pointer_t<decltype(p0)>>;
        constexpr int V = sizeof(VT) / 2, STEP = decltype(step)();   // V units of sixteen bytes in eight elements
        each<V>([&](auto v) {
            if (whole) {
                copy16<v * STEP, v * 64>(dst, p0, size0);
                copy16<v * STEP + V * 512, v * 64>(dst, p1, size1);
            } else {   // a copy of nothing still gets an address inside a tensor
                const bool in = first + v * 16 < limit;
                copy16<v * STEP, 0>(dst, in ? (const char *)p0 + v * 64 : (const char *)P.a, in ? size0 : 0);
                copy16<v * STEP + V * 512, 0>(dst, in ? (const char *)p1 + v * 64 : (const char *)P.a, in ? size1 : 0);
            }
        });
    };
    int fetch_at = 0;   // the buffer of the next stage to fetch
    auto fetch = [&](int st) {
        const int buffer = fetch_at;
        fetch_at = fetch_at == (S::STAGES - 1) * S::BYTES ? 0 : fetch_at + S::BYTES;
        if (st < kstages) {
            const int ch = k0 + st * 4 + warp;
            const bool whole = ch < k1 && ch * 32 + 32 <= P.K && all_ranks;   // nothing of the chunk is missing
            const int limit = ch < k1 ? P.K : 0;
            const uint32_t dw = to_weights + buffer + lane * 16;
            if (whole) {
                const __nv_bfloat16 *src = aw;
                each<RT>([&](auto i) {
                    copy16<i * 512, 0>(dw, src, 16);
                    src += aw_step;
                });
            } else {
                each<RT>([&](auto i) {
                    const bool there = ch * 32 + q * 8 < limit && i * 8 < P.r;
                    copy16<i * 512, 0>(dw, there ? aw + i * aw_step : P.a, there ? 16 : 0);
                });
            }
            fetch_rows(to_rows + buffer + x_lane, Const<X_STEP>{}, x0, x1, whole, ch * 32 + q * EX, limit);
            x0 += 128; x1 += 128; aw += 128;
        } else if (st < stages) {
            const int ch = n0 + (st - kstages) * 4 + warp;
            const bool whole = ch < n1 && ch * 32 + 32 <= P.N && all_ranks;
            const int limit = ch < n1 ? P.N : 0, col = ch * 32 + (g >> 1) * EO + (g & 1);
            each<4>([&](auto j) {
                constexpr int skip = sizeof(OT) == 2 ? j * 2 : j / 2 * 16 + j % 2 * 2;
                const __nv_bfloat16 *src = bw + skip * P.r;
                const bool in = col + skip < limit;
                if constexpr (RT == 2) {
                    const bool there = in && q * 4 < P.r;
                    copy8(to_weights + buffer + j * 256 + lane * 8, there ? src : P.b, there ? 8 : 0);
                } else {
                    const uint32_t dw = to_weights + buffer + lane * 16;
                    if (whole)
                        each<RT / 4>([&](auto s) { copy16<(j * (RT / 4) + s) * 512, s * 64>(dw, src, 16); });
                    else
                        each<RT / 4>([&](auto s) {
                            const bool there = in && s * 32 + q * 8 < P.r;
                            copy16<(j * (RT / 4) + s) * 512, 0>(dw, there ? src + s * 32 : P.b, there ? 16 : 0);
                        });
                }
            });
            fetch_rows(to_rows + buffer + lane * 16, Const<B_STEP>{}, b0, b1, whole, ch * 32 + q * EO, limit);
            b0 += 128; b1 += 128; bw += (size_t)128 * P.r;
        }
        copies_commit();
    };
    int buffer = 0;          // of the stage that is being used
    auto landed = [&] {
        copies_wait<S::STAGES - 1>();
        __syncwarp();
    };
    auto done_with = [&](int st) {
        __syncwarp();
        buffer = buffer == (S::STAGES - 1) * S::BYTES ? 0 : buffer + S::BYTES;
        fetch(st + S::STAGES);
    };
#pragma unroll
    for (int st = 0; st < S::STAGES; st++) fetch(st);
    const uint8_t *my_rows = smem + S::WEIGHTS + warp * S::ROW_CHUNK + lane * 16, *my_weights = smem + warp * (S::WEIGHTS / 4);

    // ---- this warp's share of h = A x; chunks behind the CTA's share are zeros
    float acc[RT][4] = {};
    for (int st = 0; st < kstages; st++) {
        landed();
        constexpr int V = sizeof(XT) / 2, PC = XFrag<XT>::WORDS;
        const uint4 *rv = reinterpret_cast<const uint4 *>(my_rows + buffer);
        const uint4 *av = reinterpret_cast<const uint4 *>(my_weights + buffer) + lane;
        uint32_t w0[4][PC], w1[4][PC];
        XFrag<XT>::words(rv, w0);
        XFrag<XT>::words(rv + V * 32, w1);
#pragma unroll
        for (int t = 0; t < RT; t += 2) {
            const uint4 a = av[t * 32], b = av[(t + 1) * 32];
#pragma unroll
            for (int p = 0; p < PC; p++) {
                mma_bf16(acc[t], w0[0][p], w1[0][p], w0[1][p], w1[1][p], a.x, a.y);
                mma_bf16(acc[t + 1], w0[0][p], w1[0][p], w0[1][p], w1[1][p], b.x, b.y);
                mma_bf16(acc[t], w0[2][p], w1[2][p], w0[3][p], w1[3][p], a.z, a.w);
                mma_bf16(acc[t + 1], w0[2][p], w1[2][p], w0[3][p], w1[3][p], b.z, b.w);
            }
        }
        done_with(st);
    }

    // the four warps have the same rows: the upper half hands its sums to the lower half, lane to lane, until one has them all
    auto at_part = [&](int buffer, int i, int half) {
        return reinterpret_cast<float2 *>(part + (buffer * FEW_M + g + half * 8) * HS + i * 8 + 2 * q);
    };
    auto put = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < RT; i++) {
            *at_part(buffer, i, 0) = make_float2(acc[i][0], acc[i][1]);
            *at_part(buffer, i, 1) = make_float2(acc[i][2], acc[i][3]);
        }
    };
    auto add = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const float2 u = *at_part(buffer, i, 0), v = *at_part(buffer, i, 1);
            acc[i][0] += u.x; acc[i][1] += u.y; acc[i][2] += v.x; acc[i][3] += v.y;
        }
    };
    if (warp >= 2) put(warp - 2);
    __syncthreads();
    if (warp < 2) add(warp);
    if (warp == 1) put(1);
    __syncthreads();
    if (warp == 0) {
        add(1);
        put(0);
    }

    // ---- the shares of the cluster added, in CTA order, times the adapter's scale
    const float scale = P.scales ? P.scales[id] : 1.f;
    constexpr int per_row = RT * 2;
    cluster.sync();
    with_cluster_size(ctas, [&](auto n) {   // every CTA adds all of it: one barrier less on the way
        constexpr int CTAS = decltype(n)();
        for (int i = tid; i < FEW_M * per_row; i += FEW_THREADS) {
            const int at = i / per_row * HS + i % per_row * 4;
            const float4 s = sum_of_cluster<CTAS>(cluster, part + at);
            const bool rank = i % per_row * 4 < P.r;   // ranks behind r are zeros, also where x is infinite
            *reinterpret_cast<float4 *>(h + at) = rank ? make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    });
    __syncthreads();

    // ---- out = base + B h over this CTA's chunks of 32 columns.  Column i of a chunk's j-th product is the chunk's column
    // (i / 2) * 8 + j * 2 + i % 2, so that a lane ends with eight consecutive columns of its two rows (f32: with columns
    // 4 (i / 2) + 2 j + i % 2 of the first or second half, four consecutive ones of each).  Ranks: a lane takes four
    // (RT = 2) or eight consecutive ones, which are one or two steps of the matrix instruction.
    constexpr int KS = RT / 2;
    uint32_t hf[KS][PIECES][4];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int k = RT == 2 ? q * 4 : s / 2 * 32 + q * 8 + s % 2 * 4;
        const float4 v0 = *reinterpret_cast<const float4 *>(h + g * HS + k);
        const float4 v1 = *reinterpret_cast<const float4 *>(h + (g + 8) * HS + k);
        uint32_t w[4][PIECES];
        split_pair(v0.x, v0.y, w[0]);
        split_pair(v1.x, v1.y, w[1]);
        split_pair(v0.z, v0.w, w[2]);
        split_pair(v1.z, v1.w, w[3]);
#pragma unroll
        for (int p = 0; p < PIECES; p++)
#pragma unroll
            for (int i = 0; i < 4; i++) hf[s][p][i] = w[i][p];
    }
    OT *o0 = out + (has0 ? (size_t)t0 * P.N : 0) + (n0 + warp) * 32 + q * EO, *o1 = out + (has1 ? (size_t)t1 * P.N : 0) + (n0 + warp) * 32 + q * EO;
    for (int st = kstages; st < stages; st++) {
        landed();
        const int ch = n0 + (st - kstages) * 4 + warp;
        float o[4][4] = {};
        const uint8_t *wv = my_weights + buffer;
        // the four products of a step are independent: in turn, so that none waits for its own sum
        if constexpr (RT == 2) {
            uint2 v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = reinterpret_cast<const uint2 *>(wv)[j * 32 + lane];
#pragma unroll
            for (int p = 0; p < PIECES; p++)
#pragma unroll
                for (int j = 0; j < 4; j++) mma_bf16(o[j], hf[0][p][0], hf[0][p][1], hf[0][p][2], hf[0][p][3], v[j].x, v[j].y);
        } else {
#pragma unroll
            for (int s = 0; s < RT / 4; s++) {
                uint4 v[4];
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = reinterpret_cast<const uint4 *>(wv)[(j * (RT / 4) + s) * 32 + lane];
#pragma unroll
                for (int p = 0; p < PIECES; p++) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        mma_bf16(o[j], hf[2 * s][p][0], hf[2 * s][p][1], hf[2 * s][p][2], hf[2 * s][p][3], v[j].x, v[j].y);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        mma_bf16(o[j], hf[2 * s + 1][p][0], hf[2 * s + 1][p][1], hf[2 * s + 1][p][2], hf[2 * s + 1][p][3], v[j].z, v[j].w);
                }
            }
        }
        constexpr int V = sizeof(OT) / 2, E = 8 / V;   // V groups of E consecutive columns
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (!(half ? has1 : has0) || ch >= n1 || ch * 32 + v * 16 + q * E >= P.N) continue;
                float y[E];
                load_units<E>(reinterpret_cast<const OT *>(my_rows + buffer + (half * V + v) * 512), y);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    y[e] += o[v * (E / 2) + e / 2][2 * half];
                    y[e + 1] += o[v * (E / 2) + e / 2][2 * half + 1];
                }
                store_units<E>((half ? o1 : o0) + v * 16, y);
            }
        o0 += 128; o1 += 128;
        done_with(st);
    }
    copy_bare_rows<FEW_THREADS>(P, share_id, base, out);
    cluster.sync();   // no CTA leaves while another reads its shares
}

// ---------------------------------------------------------------- many rows of an adapter: tcgen05
// For prompts the warp-level instructions become the limit: their operands pass through registers, once for every sixteen
// rows, and at rank 64 the second product alone keeps them busy for longer than the rows' bytes take (8192 rows of 2048 bf16:
// 42 us for this part).  Here a tile of 128 rows of one adapter is the M of tcgen05.mma, read from shared memory and summed in
// tensor memory:
//   h[128, r]     = X[128, K] A^T   stages of 64 of K: the rows' and A's pieces of 128 bytes, 128-byte swizzle
//   out[128, 128] = H B^T + base    chunks of 128 columns, each of h's three bf16 pieces its own product
// with the cluster's exchange of h between them as above.  All threads copy (asynchronously, LEAD stages ahead), one
// issues the products, and a chunk's sums are read, added to base and stored while the next chunk's product runs.  The
// columns of B lie permuted in shared memory so that a lane reads eight consecutive ones of a row.
constexpr int TC_M = 128, TC_THREADS = 256;
// Rows an adapter has on average from which these tiles are taken.  K = N = 2048, bf16, us of 16-row and 128-row tiles, 16 adapters in sorted order:
//   rows an adapter    64          96          128         192         512
//   rank 16         8.5 / 29    15 / 29     10 / 18     19 / 20     31 / 31
//   rank 64         13 / 28     24 / 29     19 / 20     37 / 21     58 / 34
//   rank 128        21 / 36     38 / 38     31 / 26     60 / 27    118 / 42
// The crossing lies between 96 and 192 for ranks of 64 and more and at 512 for rank 16; with four adapters or one, whose tiles of 128 do not
// fill the card, 16-row tiles stay ahead to 512 rows (four of rank 64: 19 / 29).  96 is the lower end of that range.
constexpr int TC_MIN_ROWS = 96;

// Waits that ran out, of all streams since the library was loaded (pmoe_rows_status), and where the last one was
struct Failures {
    unsigned count;
    int detail;
};
__device__ Failures g_failures;

template <typename OT, int RT> struct TcTile {
    static constexpr int R = RT * 8, KB = (R + 63) / 64;              // ranks, blocks of 64 of them
    static constexpr int X_BYTES = TC_M * 128, A_BYTES = R * 128, B_BYTES = KB * 128 * 128;
    static constexpr int STAGE = X_BYTES + A_BYTES > B_BYTES ? X_BYTES + A_BYTES : B_BYTES;
    static constexpr int PS = R + 4;                                  // floats between two rows of this CTA's share of h
    static constexpr int PART = TC_M * PS * 4, H_BYTES = PIECES * KB * TC_M * 128;
    static constexpr bool OVERLAY = RT == 16;                         // the share lies over the stages, which wait for the exchange
    static constexpr int ROOM = 218 * 1024 - H_BYTES - (OVERLAY ? 0 : PART);
    static constexpr int STAGES = ROOM / STAGE > 6 ? 6 : ROOM / STAGE;
    static constexpr int SMEM = 1024 + STAGES * STAGE + H_BYTES + (OVERLAY ? 0 : PART);
    // A stage is fetched into the buffer of the stage LAG before the last: with a lag of two its product has had a whole step
    // to end; where the buffers are few they are worth more as stages on their way.
    static constexpr int LAG = STAGES >= 5 ? 2 : 1, LEAD = STAGES - LAG;
    static_assert(STAGES >= 3 && (!OVERLAY || PART <= STAGES * STAGE), "room for the pipeline");
};

// The row of B's tile that holds a column of a chunk: in groups of 32, row 8 j + i is the column that k_adapters gives to column
// i of its j-th product.
template <typename OT> __device__ inline int row_of(int col)
{
    const int c = col % 32;
    return col / 32 * 32 + (sizeof(OT) == 2 ? c / 2 % 4 * 8 + c / 8 * 2 + c % 2 : (c / 16 * 2 + c / 2 % 2) * 8 + c / 4 % 4 * 2 + c % 2);
}

template <typename OT, int RT>
__global__ void __launch_bounds__(TC_THREADS, 1) k_adapters_tc(AdapterArgs P, const __nv_bfloat16 *__restrict__ x, const OT *base, OT *out)
{
    using S = TcTile<OT, RT>;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ int rows[TC_M];
    __shared__ int tile_id, tile_rows, tile_first;
    __shared__ uint64_t bars[S::STAGES];
    __shared__ uint32_t tmem_at;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), c = (int)cluster.block_rank(), slot = blockIdx.x / ctas;
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the swizzle counts from 1024-byte boundaries
    uint8_t *hs = smem + S::STAGES * S::STAGE;                                      // [PIECES][KB][128 rows of 128 bytes]
    float *part = reinterpret_cast<float *>(S::OVERLAY ? smem : hs + S::H_BYTES);   // [128][PS]
    pdl_wait();
    pdl_launch_dependents();
    const int share_id = id_of_share(P, 0);
    if (P.order) find_tile<TC_M, TC_THREADS>(P, slot, rows, tile_id, tile_rows, tile_first);
    else find_tile_by_ids<TC_M, TC_THREADS>(P, slot, rows, tile_id, tile_rows, tile_first, reinterpret_cast<int *>(smem));
    if (tile_rows == 0) {
        copy_bare_rows<TC_THREADS>(P, share_id, base, out);
        return;
    }
    const int id = tile_id;
    if (tid == 0) {
        for (int i = 0; i < S::STAGES; i++) mbar_init(&bars[i], 1);
        fence_mbar_init();
    }
    if (warp == 0) tmem_alloc(&tmem_at, 256);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    bool ok = true;
    // the product of stage `use` (counted over both parts) is complete, and its buffer free
    auto product_done = [&](int use) {
        if (ok && !mbar_wait_spin(&bars[use % S::STAGES], (use / S::STAGES) & 1)) {
            ok = false;
            atomicExch(&g_failures.detail, use);
            atomicAdd(&g_failures.count, 1u);
        }
    };

    // ---- what this CTA takes of K and of N
    const int kc = (P.K + 63) / 64, nc = (P.N + 127) / 128;
    const int k0 = (int)((int64_t)kc * c / ctas), kst = (int)((int64_t)kc * (c + 1) / ctas) - k0;
    const int n0 = (int)((int64_t)nc * c / ctas), nst = (int)((int64_t)nc * (c + 1) / ctas) - n0;

    // copies: eight lanes take the 128 bytes of a row; this thread's rows are tid / 8 + 32 i
    const int chunk = tid & 7, row8 = tid >> 3;
    const uint32_t to = smem_u32(smem) + row8 * 128 + ((chunk ^ (row8 & 7)) << 4);
    const __nv_bfloat16 *xr[4];
    int x_size[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int t = rows[row8 + 32 * i];
        x_size[i] = (unsigned)t < (unsigned)P.n ? 16 : 0;
        xr[i] = x + (x_size[i] ? (size_t)t * P.K : 0);
    }
    const __nv_bfloat16 *aw = P.a + ((size_t)id * P.r + row8) * P.K;
    const __nv_bfloat16 *bw = P.b + (size_t)id * P.N * P.r;
    auto fetch_k = [&](int st) {
        if (st < kst) {
            const uint32_t dst = to + (st % S::STAGES) * S::STAGE;
            const int k = (k0 + st) * 64 + chunk * 8;
            const bool in = k < P.K;
            each<4>([&](auto i) { copy16<i * 32 * 128, 0>(dst, in ? xr[i] + k : x, in ? x_size[i] : 0); });
            each<(S::R + 31) / 32>([&](auto i) {
                const bool there = in && row8 + i * 32 < P.r;
                if (S::R >= 32 || row8 < S::R) copy16<S::X_BYTES + i * 32 * 128, 0>(dst, there ? aw + (size_t)i * 32 * P.K + k : P.a, there ? 16 : 0);
            });
        }
        copies_commit();
    };
    auto fetch_n = [&](int st) {
        if (st < nst) {
            const uint32_t dst = smem_u32(smem) + ((kst + st) % S::STAGES) * S::STAGE;
            const int col0 = (n0 + st) * 128;
#pragma unroll
            for (int i = 0; i < RT / 2; i++) {
                const int m = tid + i * TC_THREADS, col = m / RT, k8 = m % RT, n = row_of<OT>(col);
                const bool there = col0 + col < P.N && k8 * 8 < P.r;
                copy16<0, 0>(dst + k8 / 8 * 16384 + n * 128 + ((k8 % 8 ^ n % 8) << 4), there ? bw + (size_t)(col0 + col) * P.r + k8 * 8 : P.b, there ? 16 : 0);
            }
        }
        copies_commit();
    };

    // ---- this CTA's share of h
    constexpr uint32_t IDESC_H = make_idesc(1, 1, 1, S::R, TC_M), IDESC_OUT = make_idesc(1, 1, 1, 128, TC_M);   // bf16 x bf16 -> f32
    for (int st = 0; st < S::LEAD; st++) fetch_k(st);
    for (int st = 0; st < kst; st++) {
        copies_wait<S::LEAD - 1>();
        fence_proxy_async();
        __syncthreads();
        if (tid == 0) {
            tc_fence_after();
            const uint8_t *buffer = smem + (st % S::STAGES) * S::STAGE;
            const uint64_t da = smem_desc_sw128(buffer), db = smem_desc_sw128(buffer + S::X_BYTES);
#pragma unroll
            for (int ks = 0; ks < 4; ks++) mma_f16(tmem, da + ks * 2, db + ks * 2, IDESC_H, st > 0 || ks > 0);
            tc_commit(&bars[st % S::STAGES]);
        }
        if (st >= S::LAG) product_done(st - S::LAG);
        fetch_k(st + S::LEAD);
    }
    if (kst > 0) product_done(kst - 1);
    tc_fence_after();
    if (!S::OVERLAY)
        for (int st = 0; st < S::LEAD; st++) fetch_n(st);
    else
        __syncthreads();

    // ---- the shares of the cluster added, in CTA order, times the adapter's scale, and given to all as bf16 pieces
    for (int i = warp / 4; i < S::R / 16; i += 2) {
        uint32_t v[16];
        if (kst > 0) {
            tmem_ld16(tmem + ((uint32_t)(warp % 4 * 32) << 16) + i * 16, v);
            tmem_ld_wait();
        }
        float4 *p = reinterpret_cast<float4 *>(part + (warp % 4 * 32 + lane) * S::PS + i * 16);
#pragma unroll
        for (int e = 0; e < 4; e++)
            p[e] = kst > 0 ? make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]), __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]))
                           : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    tc_fence_before();
    cluster.sync();
    const float scale = P.scales ? P.scales[id] : 1.f;
    with_cluster_size(ctas, [&](auto n) {
        constexpr int CTAS = decltype(n)();
        for (int i = c * TC_THREADS + tid; i < TC_M * RT; i += CTAS * TC_THREADS) {   // eight ranks of a row
            const int row = i / RT, k8 = i % RT;
            const float4 u = sum_of_cluster<CTAS>(cluster, part + row * S::PS + k8 * 8), v = sum_of_cluster<CTAS>(cluster, part + row * S::PS + k8 * 8 + 4);
            uint32_t w[4][PIECES];
            const uint32_t rank = k8 * 8 < P.r ? ~0u : 0u;   // ranks behind r are zeros, also where x is infinite
            split_pair(u.x * scale, u.y * scale, w[0]);
            split_pair(u.z * scale, u.w * scale, w[1]);
            split_pair(v.x * scale, v.y * scale, w[2]);
            split_pair(v.z * scale, v.w * scale, w[3]);
            uint8_t *at = hs + k8 / 8 * (TC_M * 128) + row * 128 + ((k8 % 8 ^ row % 8) << 4);
#pragma unroll
            for (int o = 0; o < CTAS; o++) {
                uint8_t *there = cluster.map_shared_rank(at, o);
#pragma unroll
                for (int p = 0; p < PIECES; p++)
                    *reinterpret_cast<uint4 *>(there + p * S::KB * TC_M * 128) = make_uint4(w[0][p] & rank, w[1][p] & rank, w[2][p] & rank, w[3][p] & rank);
            }
        }
    });
    asm volatile("fence.proxy.async;" ::: "memory");   // h is read by the tensor cores, here and in the other CTAs
    cluster.sync();
    asm volatile("fence.proxy.async;" ::: "memory");
    if (S::OVERLAY)
        for (int st = 0; st < S::LEAD; st++) fetch_n(st);

    // ---- out = base + h B.  Warp w reads the rows of quarter w % 4 and the columns of half w / 4: two groups of 32 columns
    // times two of sixteen rows, a lane eight columns of rows g and g + 8 of each.
    constexpr int V = sizeof(OT) / 2, E = 8 / V;    // V groups of E consecutive columns
    const OT *bp[4];
    OT *op[4];
    bool has[4];
    const int first_col = warp / 4 * 64 + q * E;
#pragma unroll
    for (int i = 0; i < 4; i++) {                    // rows g, g + 8, g + 16, g + 24 of the quarter
        const int t = rows[warp % 4 * 32 + g + i * 8];
        has[i] = (unsigned)t < (unsigned)P.n;
        bp[i] = base + (has[i] ? (size_t)t * P.N : 0);
        op[i] = out + (has[i] ? (size_t)t * P.N : 0);
    }
    auto ahead_base = [&](int st) {                  // towards L2, one lane for the bytes of four
        const int col = (n0 + st) * 128 + first_col;
        if (q == 0 && st < nst)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (has[i] && col + u * 32 < P.N) asm volatile("prefetch.global.L2 [%0];" ::"l"(bp[i] + col + u * 32));
    };
    float4 held[2][2][4][V];                         // base of two chunks, as loaded: [32 columns][row][16 bytes]
    auto load_base = [&](int st, auto which) {
        const int col = (n0 + st) * 128 + first_col;
        if (st < nst)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int v = 0; v < V; v++)
                        if (has[i] && col + u * 32 + v * 16 < P.N) held[which][u][i][v] = *reinterpret_cast<const float4 *>(bp[i] + col + u * 32 + v * 16);
    };
    auto finish = [&](int st, auto which) {          // `which` is st % 2
        const int col = (n0 + st) * 128 + first_col;
        uint32_t o[2][16];                           // the sums of sixteen rows, read while those before are stored
        auto read = [&](auto k) { tmem_ld_16x32(tmem + which * 128 + warp / 4 * 64 + k / 2 * 32 + ((uint32_t)(warp % 4 * 32 + k % 2 * 16) << 16), o[k % 2]); };
        read(Const<0>{});
        each<4>([&](auto k) {
            constexpr int u = k / 2, half = k % 2;
            tmem_ld_wait();
            if constexpr (k < 3) read(Const<k + 1>{});
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int v = 0; v < V; v++) {
                    constexpr int i0 = half * 2;
                    if (!has[i0 + r] || col + u * 32 + v * 16 >= P.N) continue;
                    float y[E];
                    load_units<E>(reinterpret_cast<const OT *>(&held[which][u][i0 + r][v]), y);
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        const int j = v * (E / 2) + e / 2;
                        y[e] += __uint_as_float(o[half][4 * j + 2 * r]);
                        y[e + 1] += __uint_as_float(o[half][4 * j + 2 * r + 1]);
                    }
                    store_units<E>(op[i0 + r] + col + u * 32 + v * 16, y);
                }
        });
        tc_fence_before();
    };
    auto step = [&](int st, auto which) {            // `which` is st % 2
        copies_wait<S::LEAD - 1>();
        fence_proxy_async();
        __syncthreads();   // the copies of all threads, and their reads of this half of tensor memory
        if (tid == 0) {
            tc_fence_after();
            const uint8_t *buffer = smem + ((kst + st) % S::STAGES) * S::STAGE;
#pragma unroll
            for (int p = 0; p < PIECES; p++)
#pragma unroll
                for (int kb = 0; kb < S::KB; kb++) {
                    const uint64_t da = smem_desc_sw128(hs + (p * S::KB + kb) * TC_M * 128), db = smem_desc_sw128(buffer + kb * 16384);
#pragma unroll
                    for (int ks = 0; ks < (S::R < 64 ? S::R / 16 : 4); ks++)
                        mma_f16(tmem + which * 128, da + ks * 2, db + ks * 2, IDESC_OUT, p > 0 || kb > 0 || ks > 0);
                }
            tc_commit(&bars[(kst + st) % S::STAGES]);
        }
        if (st > 0) product_done(kst + st - 1);
        fetch_n(st + S::LEAD);
        if (st > 0) {
            tc_fence_after();
            finish(st - 1, Const<1 - which>{});
        }
        load_base(st + 1, Const<1 - which>{});
        ahead_base(st + 3);
    };
    for (int st = 1; st < 3; st++) ahead_base(st);
    load_base(0, Const<0>{});
    for (int st = 0; st < nst; st += 2) {
        step(st, Const<0>{});
        if (st + 1 < nst) step(st + 1, Const<1>{});
    }
    if (nst > 0) {
        product_done(kst + nst - 1);
        tc_fence_after();
        if (nst % 2) finish(nst - 1, Const<0>{});
        else finish(nst - 1, Const<1>{});
    }
    copies_wait<0>();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 256);
    copy_bare_rows<TC_THREADS>(P, share_id, base, out);
}

// slots clusters of `ctas` CTAs
template <typename Kern, typename XT, typename OT>
static cudaError_t launch_clusters(Kern kern, std::atomic<uint64_t> &asked, int slots, int ctas, int threads, size_t smem, const AdapterArgs &P, const XT *x, const OT *base, OT *out,
                                   cudaStream_t s)
{
    if (smem > 40 * 1024) {   // with the static arrays, more than a launch may have without asking
        cudaError_t e = allow_smem((const void *)kern, smem, asked);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)slots * ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kern, P, x, base, out);
}

// The cluster's size: more CTAs share a tile's K and N (`shared` of work), each with the same work around it (finding the
// tile, the exchange of h: `around`).  Taken is the size with the shortest sum over the waves that the grid makes: eight where
// the rows are few, one or two where the tiles alone fill the card's `room`.  Measured, us with clusters of 1, 2, 4, 8 CTAs (* is taken):
//   16-row tiles: 1 row 12.2 8.2 6.1 5.1*; 64 rows of 48 ids 18.6 11.7 11.9 11.6*; 128 rows of as many ids, rank 64 19.7 19.2 25.1* 41.7;
//     1024 f32 rows of 4 ids 29.9 20.5 18.5* 32.1; 4096 f32 rows of 12 ids 28.0* 29.1 32.1 41.7; 8192 rows of 100 ids 80.6* 86.3 108 189
//   128-row tiles: 1024 rows of 4 ids 46.9 28.4 19.2 16.8*; 2048 rows of 4 ids 46.8 27.5 18.4 28.5*; 8192 rows of 12 ids 50.2 33.1* 59.1 84.1;
//     16384 rows of 12 ids, rank 16 49.8* 58.1 78.4 155
// The sum takes `room` for as many SMs as the card has.  Clusters of eight with a CTA an SM fill it less than that, and slots without a tile are not
// counted, which costs 10 us in the case of 2048 rows and 6 in that of 128.
static int cluster_size(int64_t tiles, int64_t room, double around, double shared)
{
    int ctas = AD_MAX_CTAS;
    double best = 1e30;
    for (int c = AD_MAX_CTAS; c >= 1; c /= 2) {
        const double cost = max(1.0, (double)(tiles * c) / room) * (around + shared / c);
        if (cost < best) { best = cost; ctas = c; }
    }
    return ctas;
}
// tiles of T rows, about: an adapter's last one is half full
static int64_t tiles_of(const AdapterArgs &P, int T) { return min((int64_t)P.n, (int64_t)(P.n + T - 1) / T + min(P.L, P.n) / 2); }

template <typename XT, typename OT, int RT>
static cudaError_t launch_adapters_as(const AdapterArgs &P, const XT *x, const OT *base, OT *out, cudaStream_t s)
{
    using S = AdapterStage<XT, OT, RT>;
    static_assert(S::STAGES * S::BYTES >= (ADAPTER_MAX + 1) * 4, "room for the offsets");
    const bool slots_by_id = P.order || P.n > ADAPTER_ROWS_LEADER;   // else every row is a slot
    const int64_t room = 148 * (int64_t)max(1, min(8, (int)(227 * 1024 / (S::SMEM + 6144))));
    const int ctas = cluster_size(slots_by_id ? tiles_of(P, FEW_M) : min(P.n, P.L), room, 8.0, (P.K + P.N) / 128.0);   // in stages
    static std::atomic<uint64_t> asked{0};
    return launch_clusters(k_adapters<XT, OT, RT>, asked, slots_by_id ? P.n / FEW_M + P.L : P.n, ctas, FEW_THREADS, S::SMEM, P, x, base, out, s);
}

template <typename OT, int RT>
static cudaError_t launch_adapters_tc(const AdapterArgs &P, const __nv_bfloat16 *x, const OT *base, OT *out, cudaStream_t s)
{
    const int ctas = cluster_size(tiles_of(P, TC_M), 148, 8.0, P.K / 64 * 0.35 + P.N / 128 * 0.9);   // in microseconds
    static std::atomic<uint64_t> asked{0};
    return launch_clusters(k_adapters_tc<OT, RT>, asked, P.n / TC_M + P.L, ctas, TC_THREADS, TcTile<OT, RT>::SMEM, P, x, base, out, s);
}

cudaError_t launch_adapters(const void *base, int out_dtype, const void *x, int x_dtype, const AdapterArgs &P, void *out, cudaStream_t s)
{
    // tiles of 128 rows where an adapter has enough of them and the rows are the tensor cores' own type; else of 16
    const bool wide = P.n > ADAPTER_ROWS_LEADER && P.n / P.L >= TC_MIN_ROWS && x_dtype == PMOE_BF16;
    return with_type(out_dtype, [&](auto *op) {
        using OT = std::remove_pointer_t<decltype(op)>;
        const OT *bb = (const OT *)base;
        OT *oo = (OT *)out;
        if (wide) {
            const __nv_bfloat16 *xx = (const __nv_bfloat16 *)x;
            return P.r <= 16   ? launch_adapters_tc<OT, 2>(P, xx, bb, oo, s)
                   : P.r <= 32 ? launch_adapters_tc<OT, 4>(P, xx, bb, oo, s)
                   : P.r <= 64 ? launch_adapters_tc<OT, 8>(P, xx, bb, oo, s)
                               : launch_adapters_tc<OT, 16>(P, xx, bb, oo, s);
        }
        return with_type(x_dtype, [&](auto *xp) {
            using XT = std::remove_pointer_t<decltype(xp)>;
            const XT *xx = (const XT *)x;
            return P.r <= 16   ? launch_adapters_as<XT, OT, 2>(P, xx, bb, oo, s)
                   : P.r <= 32 ? launch_adapters_as<XT, OT, 4>(P, xx, bb, oo, s)
                   : P.r <= 64 ? launch_adapters_as<XT, OT, 8>(P, xx, bb, oo, s)
                               : launch_adapters_as<XT, OT, 16>(P, xx, bb, oo, s);
        });
    });
}

}  // namespace pmoe

using namespace pmoe;

extern "C" int pmoe_adapters_add(int device, const void *base, const void *x, int x_dtype, int n, int K, int N, int rank, int n_adapters,
                                 const void *a, const void *b, const float *scales, const int *ids, const int *order, const int *offsets,
                                 void *out, int out_dtype, void *stream)
{
    if (n < 0 || n > (1 << 30) || n_adapters <= 0 || n_adapters > ADAPTER_MAX)
        return fail(PMOE_ERR_INVALID_ARG, "bad n / n_adapters (1 to %d)", ADAPTER_MAX);
    if (K <= 0 || K % 8 || N <= 0 || N % 8 || K > (1 << 20) || N > (1 << 20))
        return fail(PMOE_ERR_UNSUPPORTED_SHAPE, "K and N must be multiples of 8 up to 2^20 (got %d, %d)", K, N);
    if (rank <= 0 || rank % 8 || rank > ADAPTER_MAX_RANK)
        return fail(PMOE_ERR_UNSUPPORTED_SHAPE, "rank must be a multiple of 8 up to %d (got %d); pad with zero rows", ADAPTER_MAX_RANK, rank);
    if (!f32_or_bf16(x_dtype) || !f32_or_bf16(out_dtype)) return fail(PMOE_ERR_UNSUPPORTED_DTYPE, "x / out must be F32 or BF16");
    if (!n) return PMOE_OK;
    if (!base || !x || !a || !b || !ids || !out) return fail(PMOE_ERR_INVALID_ARG, "base / x / a / b / ids / out is NULL");
    if ((order == nullptr) != (offsets == nullptr)) return fail(PMOE_ERR_INVALID_ARG, "order and offsets come together");
    if (!order && n > ADAPTER_ROWS_UNSORTED)
        return fail(PMOE_ERR_TOO_MANY_TOKENS, "%d rows need the order of their ids (pmoe_sort_pairs); without it at most %d are served", n,
                    ADAPTER_ROWS_UNSORTED);
    if (!aligned16(base) || !aligned16(x) || !aligned16(a) || !aligned16(b) || !aligned16(out))
        return fail(PMOE_ERR_INVALID_ARG, "base, x, a, b and out must be 16-byte aligned");
    const size_t ids_bytes = (size_t)n * sizeof(int), out_bytes = (size_t)n * N * block_bytes(out_dtype), L = n_adapters;
    if (overlap({{out, out_bytes}}, {{base == out ? nullptr : base, out_bytes}, {x, (size_t)n * K * block_bytes(x_dtype)}, {a, L * rank * K * 2}, {b, L * N * rank * 2},
                                     {scales, L * sizeof(float)}, {ids, ids_bytes}, {order, ids_bytes}, {offsets, (L + 1) * sizeof(int)}}))
        return fail(PMOE_ERR_INVALID_ARG, "out must not overlap an input (it may be base)");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    const AdapterArgs args{n, K, N, rank, n_adapters, (const __nv_bfloat16 *)a, (const __nv_bfloat16 *)b, scales, ids, order, offsets};
    CU(launch_adapters(base, out_dtype, x, x_dtype, args, out, (cudaStream_t)stream));
    return PMOE_OK;
}

extern "C" int pmoe_rows_status(int device, void *stream)
{
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    cudaStream_t s = (cudaStream_t)stream;
    Failures f{};
    CU(cudaMemcpyFromSymbolAsync(&f, g_failures, sizeof f, 0, cudaMemcpyDeviceToHost, s));
    CU(cudaStreamSynchronize(s));
    static FailureCounts counts;
    bool news = f.count != 0;
    try {
        news = counts.news(device, stream, f.count);
    } catch (...) {   // no memory for a stream's entry: an old failure is reported once more
    }
    return news ? fail(PMOE_ERR_TIMEOUT, "a wait inside pmoe_adapters_add ran out (%u so far, the last at stage %d)", f.count, f.detail) : PMOE_OK;
}
