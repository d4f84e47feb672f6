// Low-rank adapters of many requests beside one projection: out_t = base_t + s_i B_i (A_i x_t) with i = ids[t], for a
// batch whose rows belong to different adapters.  base is the shared projection's output (pmoe_qmatmul's, say); a row whose
// id is outside [0, L) keeps it.  The reference's QMatMul holds one low-rank update and merges it
// (paramecia-model/src/models/with_tracing.rs:103-337).
//
// What bounds it: 2 r (K + N) flops over K x + 2 N out elements a row, at most r flops a byte, below the ridge of the card
// for every rank served (r <= 128), so the rows' stream from memory is the limit for prompts, and latency for single
// tokens.  The warp-level matrix instructions are fast enough for that rate and take their operands from registers, where
// the loads put them: no shared-memory staging of x, A or B at all.
//
// One kernel does both products.  A tile of up to T rows of one adapter belongs to a cluster of eight CTAs: each takes an
// eighth of K for its share of h = A x, the shares are added through distributed shared memory, and each CTA
// then takes an eighth of the N output columns.  h never goes to memory, and a single token still uses eight SMs.
#include <cooperative_groups.h>

#include "pmoe_internal.h"
#include "pmoe_vec.cuh"

namespace pmoe {

namespace cg = cooperative_groups;

constexpr int ADAPTER_MAX_RANK = 128;
constexpr int ADAPTER_ROWS_UNSORTED = 1024;   // rows that are grouped by id without pmoe_sort_pairs
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

// A pair of f32 values as PIECES pairs of bf16 whose sum is the value: three hold all 24 bits of it (8 + 8 + 8, each
// remainder is exact), two hold 16.
template <int PIECES> __device__ inline void split_pair(float lo, float hi, uint32_t (&w)[PIECES])
{
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        w[p] = pack_bf16(lo, hi);
        lo -= __uint_as_float(w[p] << 16);
        hi -= __uint_as_float(w[p] & 0xffff0000u);
    }
}

// eight consecutive inner elements of a row as matrix operands: four pairs, in one piece for bf16 and in three for f32
template <typename XT> struct XFrag;
template <> struct XFrag<__nv_bfloat16> {
    static constexpr int PIECES = 1;
    static __device__ void words(const uint4 *p, uint32_t (&w)[4][1])
    {
        const uint4 v = p[0];
        w[0][0] = v.x; w[1][0] = v.y; w[2][0] = v.z; w[3][0] = v.w;
    }
};
template <> struct XFrag<float> {
    static constexpr int PIECES = 3;
    static __device__ void words(const uint4 *p, uint32_t (&w)[4][3])
    {
        const float4 v0 = reinterpret_cast<const float4 *>(p)[0], v1 = reinterpret_cast<const float4 *>(p)[32];
        split_pair<3>(v0.x, v0.y, w[0]);
        split_pair<3>(v0.z, v0.w, w[1]);
        split_pair<3>(v1.x, v1.y, w[2]);
        split_pair<3>(v1.z, v1.w, w[3]);
    }
};

// Asynchronous copies of 16 (8) bytes to shared memory; size 0 writes zeros and reads nothing.
__device__ inline void copy16(void *dst, const void *src, int size)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(size) : "memory");
}
__device__ inline void copy8(void *dst, const void *src, int size)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(size) : "memory");
}
__device__ inline void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ inline void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

struct AdapterArgs {
    int n, K, N, r, L;
    const __nv_bfloat16 *a, *b;
    const float *scales;
    const int *ids, *order, *offsets;
};

// floats between two rows of h in shared memory: sixteen more where rows would start in the same bank
__host__ __device__ inline int h_stride(int r16) { return r16 % 32 ? r16 : r16 + 16; }

// out = base in the listed rows, eight elements at a time; four loads are on their way before the first is stored
template <typename OT>
__device__ inline void copy_rows_of(const OT *base, OT *out, int N, const int *list, int count, int first, int step)
{
    const int units = N / 8, total = count * units;
    for (int u = first; u < total; u += 4 * step) {
        float v[4][8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = u + i * step;
            if (k < total) load_units<8>(base + (size_t)list[k / units] * N + k % units * 8, v[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = u + i * step;
            if (k < total) store_units<8>(out + (size_t)list[k / units] * N + k % units * 8, v[i]);
        }
    }
}

// A CTA walks its share of K and then its share of N in stages of four chunks of 32: a stage holds what the matrix
// instructions of those chunks need, as the lanes need it (sixteen bytes per lane, lanes side by side, so no
// access meets a bank twice).  The copies are asynchronous and STAGES stages are on their way, the first ones of N
// while the shares of h are still being added.
//
// A warp has sixteen rows and KH of them share a stage's four chunks: what a warp does per chunk is a chain of dependent
// steps (read, multiply, add the base, write), so it takes about sixteen warps an SM to fill each other's gaps.  With one warp
// per sixteen rows (four to eight an SM) 8192 rows of 2048 bf16, rank 64, took 82 us.
// RT: groups of eight ranks that the accumulators are sized for.
template <typename XT, typename OT, int T, int RT> struct AdapterStage {
    static constexpr int SIZE = sizeof(XT) > sizeof(OT) ? sizeof(XT) : sizeof(OT);
    static constexpr int KH = T == 16 ? 4 : SIZE == 4 && RT < 16 ? 4 : 2;
    static constexpr int WARPS = T / 16 * KH, THREADS = WARPS * 32, CPW = 4 / KH;
    static constexpr int MIN_CTAS = T == 16 ? 4 : WARPS == 8 && RT < 16 ? 2 : 1;
    static constexpr int STAGES = T == 16 ? 4 : 2;
    static constexpr int WEIGHTS = 4 * RT * 32 * 16;                     // A: 4 chunks x RT rank groups; B: 4 chunks x 4 products x RT / 4 rank steps
    static constexpr int ROW_CHUNK = 2 * 32 * 8 * SIZE;                 // two rows of eight elements a lane
    static constexpr int ROWS = T / 16 * 4 * ROW_CHUNK;
    static constexpr int BYTES = WEIGHTS + ROWS;
    static size_t smem(int r16) { return STAGES * BYTES + (size_t)(KH / 2 + 1) * T * h_stride(r16) * sizeof(float); }
};

template <typename XT, typename OT, int T, int RT>
__global__ void __launch_bounds__(AdapterStage<XT, OT, T, RT>::THREADS, AdapterStage<XT, OT, T, RT>::MIN_CTAS) k_adapters(AdapterArgs P, const XT *__restrict__ x, const OT *base, OT *out)
{
    using S = AdapterStage<XT, OT, T, RT>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int rows[T];
    __shared__ int tile_id, tile_rows, tile_first, bare_list[T];
    __shared__ unsigned bare_mask[2];
    __shared__ int all_ids[T == 16 ? ADAPTER_ROWS_UNSORTED : 1];   // without an order T is 16
    constexpr int THREADS = S::THREADS, CPW = S::CPW;
    constexpr int HP = std::is_same<OT, float>::value ? 3 : 2;   // pieces of h: an f32 result keeps all of it, a bf16 result 16 bits
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int rg = warp % (T / 16), kh = warp / (T / 16);   // this warp's sixteen rows and its chunks of a stage
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), c = (int)cluster.block_rank(), slot = blockIdx.x / ctas;
    const int r16 = (P.r + 15) / 16 * 16, hs = h_stride(r16);
    float *part = reinterpret_cast<float *>(smem + S::STAGES * S::BYTES);   // [KH / 2][T][hs] this CTA's share of h
    float *h = part + S::KH / 2 * T * hs;                                   // [T][hs]
    pdl_wait();
    pdl_launch_dependents();

    // ---- the tile: its adapter and rows.  Every CTA of the cluster finds the same.
    if (P.order) {
        // Tile slots of adapter e begin at offsets[e] / T + e: with one slot more than whole multiples of T inside its
        // range that is never fewer than it has tiles, and needs no scan over the adapters.
        if (tid == 0) tile_rows = 0;
        __syncthreads();
        for (int e = tid; e < P.L; e += THREADS) {
            const int from = P.offsets[e], to = min(P.offsets[e + 1], P.n), nth = slot - (from / T + e);
            if (from >= 0 && nth >= 0 && nth < (to - from + T - 1) / T) {   // one adapter at most
                tile_id = e;
                tile_first = from + nth * T;
                tile_rows = min(T, to - from - nth * T);
            }
        }
        // rows without an adapter are nowhere in the order: the slots pass over the batch once more for them
        const int t = slot * T + tid;
        const bool bare = tid < T && t < P.n && (unsigned)P.ids[min(t, P.n - 1)] >= (unsigned)P.L;
        const unsigned bare_here = __ballot_sync(0xffffffffu, bare);
        if (lane == 0 && warp < (T + 31) / 32) bare_mask[warp] = bare_here;
        const int any = __syncthreads_count(bare);
        if (tid < T) rows[tid] = tid < tile_rows ? P.order[tile_first + tid] : -1;
        if (any && out != base) {
            // listed in ascending order: the CTAs of the cluster share the list out among them
            if (bare) bare_list[__popc(bare_here & ((1u << lane) - 1)) + (warp > 0 ? __popc(bare_mask[0]) : 0)] = t;
            __syncthreads();
            copy_rows_of(base, out, P.N, bare_list, any, c * THREADS + tid, ctas * THREADS);
        }
        __syncthreads();
        if (tile_rows == 0) return;
    } else if constexpr (T == 16) {
        // slot t leads a tile when the number of earlier rows with its id is a multiple of T
        const int id = P.ids[slot];
        if ((unsigned)id >= (unsigned)P.L) {
            if (out != base) {
                if (tid == 0) bare_list[0] = slot;
                __syncthreads();
                copy_rows_of(base, out, P.N, bare_list, 1, c * THREADS + tid, ctas * THREADS);
            }
            return;
        }
        if (tid < T) rows[tid] = -1;
        for (int t = tid; t < P.n; t += THREADS) all_ids[t] = P.ids[t];
        __syncthreads();
        if (warp == 0) {
            int before = 0, found = 0;
            for (int t = 0; t < P.n && found < T; t += 32) {
                const bool same = t + lane < P.n && all_ids[t + lane] == id;
                const unsigned m = __ballot_sync(0xffffffffu, same);
                const unsigned early = t + 32 <= slot ? m : t > slot ? 0u : m & ((1u << (slot - t)) - 1);
                before += __popc(early);
                const int at = found + __popc(m & ~early & ((1u << lane) - 1));
                if (same && !(early >> lane & 1) && at < T) rows[at] = t + lane;
                found += __popc(m & ~early);
            }
            if (lane == 0) {
                tile_id = id;
                tile_rows = before % T ? 0 : min(found, T);
            }
        }
        __syncthreads();
        if (tile_rows == 0) return;
    }
    const int id = tile_id, nrows = tile_rows;
    const int row_base = rg * 16;
    const int t0 = rows[row_base + g], t1 = rows[row_base + g + 8];
    const bool has0 = (unsigned)t0 < (unsigned)P.n, has1 = (unsigned)t1 < (unsigned)P.n;
    const bool busy = row_base < nrows;       // a warp of a T = 64 tile may have no rows

    // ---- the stages of this CTA
    const int kc = (P.K + 31) / 32, nc = (P.N + 31) / 32;
    const int k0 = (int)((int64_t)kc * c / ctas), k1 = (int)((int64_t)kc * (c + 1) / ctas);
    const int n0 = (int)((int64_t)nc * c / ctas), n1 = (int)((int64_t)nc * (c + 1) / ctas);
    const int kstages = (k1 - k0 + 3) / 4, stages = kstages + (n1 - n0 + 3) / 4;
    const int tiles = P.r / 8;
    const XT *x0 = x + (has0 ? (size_t)t0 * P.K : 0), *x1 = x + (has1 ? (size_t)t1 * P.K : 0);
    const OT *b0 = base + (has0 ? (size_t)t0 * P.N : 0), *b1 = base + (has1 ? (size_t)t1 * P.N : 0);
    const __nv_bfloat16 *aw = P.a + ((size_t)id * P.r + g) * P.K;
    const __nv_bfloat16 *bw = P.b + (size_t)id * P.N * P.r;
    // chunk i of a stage: its weights are fetched by the warps i, i + 4, ...; its rows by the warp that uses them
    auto weights_of = [&](int st, int i) { return reinterpret_cast<uint4 *>(smem + (st % S::STAGES) * S::BYTES + i * (S::WEIGHTS / 4)) + lane; };
    auto rows_of = [&](int st, int i) {
        return reinterpret_cast<uint4 *>(smem + (st % S::STAGES) * S::BYTES + S::WEIGHTS + (rg * 4 + i) * S::ROW_CHUNK) + lane;
    };
    const int size0 = has0 ? 16 : 0, size1 = has1 ? 16 : 0;
    auto copy_rows = [&](uint4 *dst, const auto *p0, const auto *p1, int n0, int n1) {
        constexpr int V = sizeof(*p0) / 2;   // 16-byte units of eight elements
#pragma unroll
        for (int v = 0; v < V; v++) {
            copy16(dst + v * 32, reinterpret_cast<const uint4 *>(p0) + v, n0);
            copy16(dst + (V + v) * 32, reinterpret_cast<const uint4 *>(p1) + v, n1);
        }
    };
    // WHOLE: every chunk of the stage lies inside the share and inside K or N
    auto fetch_k = [&](int st, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int ch0 = k0 + st * 4;
        {
            const int wc = warp % 4, k = (ch0 + wc) * 32 + q * 8;
            const bool in = WHOLE || (ch0 + wc < k1 && k < P.K);
            uint4 *dst = weights_of(st, wc) + warp / 4 * 32;
            const __nv_bfloat16 *src = in ? aw + (size_t)(warp / 4) * 8 * P.K + k : P.a;
            const size_t step = in ? (size_t)(S::WARPS / 4) * 8 * P.K : 0;
#pragma unroll
            for (int i = 0; i < RT; i += S::WARPS / 4) {
                if (i + warp / 4 >= tiles) break;
                copy16(dst + i * 32, src, in ? 16 : 0);
                src += step;
            }
        }
        const XT *p0 = x0 + ch0 * 32 + q * 8, *p1 = x1 + ch0 * 32 + q * 8;
#pragma unroll
        for (int u = 0; u < CPW; u++) {
            const int i = kh * CPW + u;
            const bool in = WHOLE || (ch0 + i < k1 && (ch0 + i) * 32 + q * 8 < P.K);
            copy_rows(rows_of(st, i), in ? p0 + i * 32 : x, in ? p1 + i * 32 : x, in ? size0 : 0, in ? size1 : 0);
        }
    };
    auto fetch_n = [&](int st, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int ch0 = n0 + (st - kstages) * 4;
        constexpr int JW = 16 / S::WARPS;    // of the four products of a chunk, those that this warp fetches the weights of
        const int wc = warp % 4, j0 = warp / 4 * JW;
        uint4 *dst = weights_of(st, wc);
        const int col0 = (ch0 + wc) * 32 + (g >> 1) * 8 + j0 * 2 + (g & 1);
        const __nv_bfloat16 *br = bw + (size_t)col0 * P.r + q * (RT == 2 ? 4 : 8);
#pragma unroll
        for (int jj = 0; jj < JW; jj++) {
            const int j = j0 + jj;
            const bool in = WHOLE || (ch0 + wc < n1 && col0 + jj * 2 < P.N);
            if constexpr (RT == 2) {
                const bool there = in && q * 4 < P.r;
                copy8(reinterpret_cast<uint2 *>(dst - lane) + j * 32 + lane, there ? br : P.b, there ? 8 : 0);
            } else {
#pragma unroll
                for (int s = 0; s < RT / 4; s++) {
                    const bool there = in && s * 32 + q * 8 < P.r;
                    copy16(dst + (j * (RT / 4) + s) * 32, there ? br + s * 32 : P.b, there ? 16 : 0);
                }
            }
            br += 2 * P.r;
        }
        const OT *p0 = b0 + ch0 * 32 + q * 8, *p1 = b1 + ch0 * 32 + q * 8;
#pragma unroll
        for (int u = 0; u < CPW; u++) {
            const int i = kh * CPW + u;
            const bool in = WHOLE || (ch0 + i < n1 && (ch0 + i) * 32 + q * 8 < P.N);
            copy_rows(rows_of(st, i), in ? p0 + i * 32 : base, in ? p1 + i * 32 : base, in ? size0 : 0, in ? size1 : 0);
        }
    };
    auto fetch = [&](int st) {
        if (st < kstages) {
            const int last = k0 + st * 4 + 4;
            if (last <= k1 && last * 32 <= P.K) fetch_k(st, std::true_type{});
            else fetch_k(st, std::false_type{});
        } else if (st < stages) {
            const int last = n0 + (st - kstages) * 4 + 4;
            if (last <= n1 && last * 32 <= P.N) fetch_n(st, std::true_type{});
            else fetch_n(st, std::false_type{});
        }
        copies_commit();
    };
    // T = 16: a warp reads what its own lanes fetched; T = 64: the weights come from all warps
    auto landed = [&] {
        copies_wait<S::STAGES - 1>();
        if (T == 16) __syncwarp();
        else __syncthreads();
    };
    auto done_with = [&](int st) {
        if (T == 16) __syncwarp();
        else __syncthreads();
        fetch(st + S::STAGES);
    };
#pragma unroll
    for (int st = 0; st < S::STAGES; st++) fetch(st);

    // ---- this warp's share of h = A x
    float acc[RT][4] = {};
    for (int st = 0; st < kstages; st++) {
        landed();
        const int here = min(4, k1 - k0 - st * 4);
        if (busy)
#pragma unroll
            for (int u = 0; u < CPW; u++) {
                const int i = kh * CPW + u;
                if (i >= here) continue;
                constexpr int V = sizeof(XT) / 2, PC = XFrag<XT>::PIECES;
                uint32_t w0[4][PC], w1[4][PC];
                XFrag<XT>::words(rows_of(st, i), w0);
                XFrag<XT>::words(rows_of(st, i) + V * 32, w1);
                const uint4 *av = weights_of(st, i);
#pragma unroll
                for (int t = 0; t < RT; t += 2) {
                    if (t >= tiles) break;
                    const uint4 u = av[t * 32], v = t + 1 < tiles ? av[(t + 1) * 32] : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int p = 0; p < PC; p++) {
                        mma_bf16(acc[t], w0[0][p], w1[0][p], w0[1][p], w1[1][p], u.x, u.y);
                        mma_bf16(acc[t + 1], w0[0][p], w1[0][p], w0[1][p], w1[1][p], v.x, v.y);
                        mma_bf16(acc[t], w0[2][p], w1[2][p], w0[3][p], w1[3][p], u.z, u.w);
                        mma_bf16(acc[t + 1], w0[2][p], w1[2][p], w0[3][p], w1[3][p], v.z, v.w);
                    }
                }
            }
        done_with(st);
    }
    // the warps of the same rows: the upper half hands its sums to the lower half, lane to lane, until one has them all
    auto at_part = [&](int buffer, int i, int half) {
        return reinterpret_cast<float2 *>(part + (buffer * T + row_base + g + half * 8) * hs + i * 8 + 2 * q);
    };
    auto put = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < RT; i++)
            if (i * 8 < r16) {
                *at_part(buffer, i, 0) = make_float2(acc[i][0], acc[i][1]);
                *at_part(buffer, i, 1) = make_float2(acc[i][2], acc[i][3]);
            }
    };
    auto add = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < RT; i++)
            if (i * 8 < r16) {
                const float2 u = *at_part(buffer, i, 0), v = *at_part(buffer, i, 1);
                acc[i][0] += u.x; acc[i][1] += u.y; acc[i][2] += v.x; acc[i][3] += v.y;
            }
    };
    if constexpr (S::KH == 4) {
        if (kh >= 2) put(kh - 2);
        __syncthreads();
        if (kh < 2) add(kh);
        if (kh == 1) put(1);
        __syncthreads();
        if (kh == 0) add(1);
    } else {
        if (kh == 1) put(0);
        __syncthreads();
        if (kh == 0) add(0);
    }
    if (kh == 0) put(0);

    // ---- the shares of the cluster added, in CTA order, times the adapter's scale
    const float scale = P.scales ? P.scales[id] : 1.f;
    const int per_row = r16 / 4;
    if (T == 16) {
        cluster.sync();
        for (int i = tid; i < 16 * per_row; i += THREADS) {   // every CTA adds all of it: one barrier less on the way
            float *p = part + i / per_row * hs + i % per_row * 4;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int o = 0; o < AD_MAX_CTAS; o++) {
                if (o >= ctas) break;
                const float4 v = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(p, o));
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            *reinterpret_cast<float4 *>(h + i / per_row * hs + i % per_row * 4) = make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale);
        }
        __syncthreads();
    } else {
        cluster.sync();
        for (int i = c * THREADS + tid; i < T * per_row; i += ctas * THREADS) {   // each CTA its part, given to all
            const int at = i / per_row * hs + i % per_row * 4;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int o = 0; o < AD_MAX_CTAS; o++) {
                if (o >= ctas) break;
                const float4 v = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(part + at, o));
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            s = make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale);
#pragma unroll
            for (int o = 0; o < AD_MAX_CTAS; o++)
                if (o < ctas) *reinterpret_cast<float4 *>(cluster.map_shared_rank(h + at, o)) = s;
        }
        cluster.sync();
    }

    // ---- out = base + B h over this CTA's chunks of 32 columns.  Column (i / 2) * 8 + j * 2 + i % 2 of a chunk is column i
    // of its j-th product, so that a lane ends with eight consecutive columns of its two rows.  Ranks: a lane takes four
    // (RT = 2) or eight consecutive ones, which are one or two steps of the matrix instruction.
    constexpr int KS = RT / 2;
    uint32_t hf[KS][HP][4];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int k = RT == 2 ? q * 4 : s / 2 * 32 + q * 8 + s % 2 * 4;
        float4 v0 = make_float4(0.f, 0.f, 0.f, 0.f), v1 = v0;
        if (k < r16) {
            v0 = *reinterpret_cast<const float4 *>(h + (row_base + g) * hs + k);
            v1 = *reinterpret_cast<const float4 *>(h + (row_base + g + 8) * hs + k);
        }
        uint32_t w[4][HP];
        split_pair<HP>(v0.x, v0.y, w[0]);
        split_pair<HP>(v1.x, v1.y, w[1]);
        split_pair<HP>(v0.z, v0.w, w[2]);
        split_pair<HP>(v1.z, v1.w, w[3]);
#pragma unroll
        for (int p = 0; p < HP; p++)
#pragma unroll
            for (int i = 0; i < 4; i++) hf[s][p][i] = w[i][p];
    }
    for (int st = kstages; st < stages; st++) {
        landed();
        const int ch0 = n0 + (st - kstages) * 4;
        if (busy)
#pragma unroll
            for (int u = 0; u < CPW; u++) {
                const int i = kh * CPW + u;
                if (ch0 + i >= n1) continue;
                float o[4][4] = {};
                const uint4 *bv = weights_of(st, i);
                // the four products of a step are independent: in turn, so that none waits for its own sum
                if constexpr (RT == 2) {
#pragma unroll
                    for (int p = 0; p < HP; p++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint2 v = (reinterpret_cast<const uint2 *>(bv - lane) + j * 32)[lane];
                            mma_bf16(o[j], hf[0][p][0], hf[0][p][1], hf[0][p][2], hf[0][p][3], v.x, v.y);
                        }
                } else {
#pragma unroll
                    for (int s = 0; s < RT / 4; s++) {
                        if (s * 32 >= P.r) break;
                        uint4 v[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) v[j] = bv[(j * (RT / 4) + s) * 32];
#pragma unroll
                        for (int p = 0; p < HP; p++) {
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                mma_bf16(o[j], hf[2 * s][p][0], hf[2 * s][p][1], hf[2 * s][p][2], hf[2 * s][p][3], v[j].x, v[j].y);
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                mma_bf16(o[j], hf[2 * s + 1][p][0], hf[2 * s + 1][p][1], hf[2 * s + 1][p][2], hf[2 * s + 1][p][3], v[j].z, v[j].w);
                        }
                    }
                }
                const int col = (ch0 + i) * 32 + q * 8;
                if (col < P.N) {
                    constexpr int V = sizeof(OT) / 2;
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        if (!(half ? has1 : has0)) continue;
                        float v[8];
                        const uint4 *bp = rows_of(st, i) + half * V * 32;
                        if constexpr (V == 1) {
                            load_units<8>(reinterpret_cast<const OT *>(bp), v);
                        } else {
                            float u[4];
                            load_units<4>(reinterpret_cast<const OT *>(bp), u);
#pragma unroll
                            for (int e = 0; e < 4; e++) v[e] = u[e];
                            load_units<4>(reinterpret_cast<const OT *>(bp + 32), u);
#pragma unroll
                            for (int e = 0; e < 4; e++) v[4 + e] = u[e];
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            v[2 * j] += o[j][2 * half];
                            v[2 * j + 1] += o[j][2 * half + 1];
                        }
                        store_units<8>(out + (size_t)(half ? t1 : t0) * P.N + col, v);
                    }
                }
            }
        done_with(st);
    }
    if (T == 16) cluster.sync();   // no CTA leaves while another reads its shares
}

template <typename XT, typename OT, int T, int RT>
static cudaError_t launch_adapters_as(const AdapterArgs &P, const XT *x, const OT *base, OT *out, cudaStream_t s)
{
    using S = AdapterStage<XT, OT, T, RT>;
    const size_t smem = S::smem((P.r + 15) / 16 * 16);
    auto *kern = k_adapters<XT, OT, T, RT>;
    if (smem > 40 * 1024) {   // with the static arrays, more than a launch may have without asking
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    // The cluster's size: more CTAs share a tile's K and N, each with the same work around it (finding the tile, the
    // exchange of h: about as long as eight stages).  Taken is the size with the shortest sum over the waves
    // that the grid makes: eight where the rows are few, one or two where the tiles alone fill the card.
    const int slots = P.order ? P.n / T + P.L : P.n;
    const int64_t room = 148 * (int64_t)max(1, min(2 * S::MIN_CTAS, (int)(227 * 1024 / (smem + 6144))));
    int ctas = AD_MAX_CTAS;
    double best = 1e30;
    for (int c = AD_MAX_CTAS; c >= 1; c /= 2) {
        const int64_t tiles = P.order ? (P.n + T - 1) / T + min(P.L, (P.n + T - 1) / T) / 2 : min(P.n, P.L);
        const double cost = (double)((tiles * c + room - 1) / room) * (8.0 + (P.K + P.N) / 128.0 / c);
        if (cost < best) { best = cost; ctas = c; }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)slots * ctas);
    cfg.blockDim = dim3(S::THREADS);
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

cudaError_t launch_adapters(const void *base, int out_dtype, const void *x, int x_dtype, const AdapterArgs &P, void *out, cudaStream_t s)
{
    // tiles of 64 rows where an adapter has that many on average; else of 16
    const bool wide = P.order && P.n / P.L >= 48;
    return with_type(x_dtype, [&](auto *xp) {
        return with_type(out_dtype, [&](auto *op) {
            using XT = std::remove_pointer_t<decltype(xp)>;
            using OT = std::remove_pointer_t<decltype(op)>;
            const XT *xx = (const XT *)x;
            const OT *bb = (const OT *)base;
            OT *oo = (OT *)out;
            if (wide)
                return P.r <= 16   ? launch_adapters_as<XT, OT, 64, 2>(P, xx, bb, oo, s)
                       : P.r <= 32 ? launch_adapters_as<XT, OT, 64, 4>(P, xx, bb, oo, s)
                       : P.r <= 64 ? launch_adapters_as<XT, OT, 64, 8>(P, xx, bb, oo, s)
                                   : launch_adapters_as<XT, OT, 64, 16>(P, xx, bb, oo, s);
            return P.r <= 16   ? launch_adapters_as<XT, OT, 16, 2>(P, xx, bb, oo, s)
                   : P.r <= 32 ? launch_adapters_as<XT, OT, 16, 4>(P, xx, bb, oo, s)
                   : P.r <= 64 ? launch_adapters_as<XT, OT, 16, 8>(P, xx, bb, oo, s)
                               : launch_adapters_as<XT, OT, 16, 16>(P, xx, bb, oo, s);
        });
    });
}

}  // namespace pmoe

using namespace pmoe;

extern "C" int pmoe_adapters_add(int device, const void *base, const void *x, int x_dtype, int n, int K, int N, int rank, int n_adapters,
                                 const void *a, const void *b, const float *scales, const int *ids, const int *order, const int *offsets,
                                 void *out, int out_dtype, void *stream)
{
    if (n < 0 || n > (1 << 30) || n_adapters <= 0 || n_adapters > 4096) return fail(PMOE_ERR_INVALID_ARG, "bad n / n_adapters (1 to 4096)");
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
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    const AdapterArgs args{n, K, N, rank, n_adapters, (const __nv_bfloat16 *)a, (const __nv_bfloat16 *)b, scales, ids, order, offsets};
    CU(launch_adapters(base, out_dtype, x, x_dtype, args, out, (cudaStream_t)stream));
    return PMOE_OK;
}
