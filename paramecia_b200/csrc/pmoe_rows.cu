// Rows to the experts and back as operators of their own: the stable sort of the (token, slot) pairs by expert, the
// dispatch of a token's row to its places in expert order, the weighted sum back, and the gradients of both.
//
// The block's own kernels do the same inside (launch_group, launch_combine) without ever writing the sorted rows; these
// entry points are for hosts that run something else between the two: their own experts, per-expert adapters, a
// training step.  With key_p = idx_p - base kept where 0 <= key_p < E:
//   offsets[e] = #{p kept : key_p < e},  place_p = offsets[key_p] + #{q < p : key_q = key_p}  (-1: not kept),
//   order[place_p] = p  (-1 from offsets[E] on).
// The order is stable, so all of it is a function of idx alone (the block's grouping leaves the order inside an expert
// to its atomics).
#include <climits>
#include <cooperative_groups.h>
#include <initializer_list>
#include <utility>

#include "pmoe_internal.h"
#include "pmoe_vec.cuh"

namespace pmoe {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------- sort
// A counting sort in one launch, by one CTA or by a cluster of eight.  Every warp owns a run of consecutive pairs, takes it
// 32 pairs at a time, and ranks the pairs of such a step among those of the same expert: ranks inside the step, steps,
// warps and CTAs are four levels of the same order, so the result is stable without atomics that decide anything.
//   1. cnt[w][e]  pairs of expert e in warp w's run
//   2. the CTAs' totals are exchanged through distributed shared memory; scans over (e, CTA, w): cnt[w][e] becomes the
//      place of that warp's first pair of e among this CTA's pairs, shift[e] what leads from there to the place among all
//   3. the runs once more: place = cnt[w][e] + rank inside the step + shift[e]
// The pairs are few bytes (4 to read, 8 to write): what counts is latency up to some 40960 pairs, and beyond the work of the eight SMs,
// about 4 us for each further 40960; from 131073 pairs on a run has more steps than a lane keeps, and its keys are read twice.
// - A lane loads its keys of sixteen steps at once and keeps them, with their ranks, from 1. to 3. where the run is no longer.
// - The lanes of a step with the same expert meet in a mask in shared memory, one word per warp and expert (__match_any_sync
//   and ballots over the bits of the expert's number took 2000 and 1300 cycles a step with 32 warps an SM).
// - The pairs are written to `order` from shared memory, where 3. leaves them in this CTA's order: neighbours of an
//   expert then leave in one sector instead of one each.
// 40960 pairs of 512 experts: 17 us with __match_any_sync, 12.6 us with ballots and direct writes, now 10.6 us (81920: 30, 19, 14.5 us).
// 163840: 29 us; 40960 of 128 experts: 9.9 us.  1024 threads leave 64 registers each: the cluster's form spills 64 bytes a thread, the other 20.
constexpr int SORT_MAX_E = 4096;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_CTAS = 8;
constexpr int SORT_BATCH = 16;
constexpr int SORT_ONE_CTA = 4096;   // pairs up to which one CTA sorts
constexpr int SORT_SMEM = 200 * 1024;

struct SortKeys {
    uint32_t v[SORT_BATCH];
    // the keys of the steps from pair p on; pairs behind p1 get one that no expert has
    __device__ void load(const uint32_t *idx, int64_t p, int64_t p1, uint32_t base, int lane)
    {
#pragma unroll
        for (int i = 0; i < SORT_BATCH; i++) v[i] = p + i * 32 + lane < p1 ? __ldg(idx + p + i * 32 + lane) - base : 0xffffffffu;
    }
};

// the lanes whose key equals this lane's (none for a key that no expert has); mask: this warp's words, zero before and after
__device__ inline unsigned lanes_of_key(uint32_t key, uint32_t E, unsigned *mask, int lane)
{
    const bool kept = key < E;
    if (kept) atomicOr(mask + key, 1u << lane);
    __syncwarp();
    const unsigned same = kept ? mask[key] : 0u;
    __syncwarp();
    if (kept && (same & ((1u << lane) - 1)) == 0) mask[key] = 0;
    return same;
}

template <int CTAS>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_pairs(const uint32_t *__restrict__ idx, int P, uint32_t base, int E, int warps,
                                                             int run, int *__restrict__ order, int *__restrict__ place,
                                                             int *__restrict__ offsets)
{
    extern __shared__ __align__(16) int cnt[];                           // [warps][E]
    unsigned *masks = reinterpret_cast<unsigned *>(cnt + warps * E);     // [warps][E]; later the pairs in this CTA's order
    int *mine = cnt + 2 * warps * E, *shift = mine + E;                  // [E] this CTA's totals, [E]
    __shared__ int warp_tot[32], warp_own[32];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = CTAS > 1 ? (int)cluster.block_rank() : 0;
    for (int i = tid; i < warps * E / 2; i += SORT_THREADS) reinterpret_cast<int4 *>(cnt)[i] = make_int4(0, 0, 0, 0);
    if (tid == 0 && (warps * E & 1)) reinterpret_cast<int2 *>(cnt)[warps * E - 1] = make_int2(0, 0);
    pdl_wait();
    pdl_launch_dependents();

    const int64_t cta0 = min((int64_t)P, (int64_t)rank * warps * run);
    const int64_t p0 = min((int64_t)P, cta0 + (int64_t)w * run), p1 = w < warps ? min((int64_t)P, p0 + run) : p0;
    const bool once = run <= SORT_BATCH * 32;
    SortKeys keys;
    uint16_t rank_of[SORT_BATCH];   // of the run's only batch: earlier lanes of the step with this key, and all of them << 8
    keys.load(idx, p0, p1, base, lane);
    __syncthreads();
    int *my_cnt = cnt + w * E;
    unsigned *my_mask = masks + w * E;
    for (int64_t p = p0; p < p1; p += SORT_BATCH * 32) {
        if (p != p0) keys.load(idx, p, p1, base, lane);
#pragma unroll
        for (int i = 0; i < SORT_BATCH; i++) {
            if (p + i * 32 >= p1) break;
            const uint32_t key = keys.v[i];
            const unsigned same = lanes_of_key(key, E, my_mask, lane);
            const int nth = __popc(same & ((1u << lane) - 1)), all = __popc(same);
            rank_of[i] = (uint16_t)(nth | all << 8);
            if (same && nth == 0) my_cnt[key] += all;
            __syncwarp();
        }
    }
    __syncthreads();

    // thread t scans experts [t*q, t*q + q)
    const int q = (E + SORT_THREADS - 1) / SORT_THREADS, e0 = min(E, tid * q), e1 = min(E, e0 + q);
    int own = 0;      // over this thread's experts, of this CTA
    for (int e = e0; e < e1; e++) {
        int t = 0;
#pragma unroll 8
        for (int v = 0; v < warps; v++) t += cnt[v * E + e];
        mine[e] = t;
        own += t;
    }
    int sum = own;    // of all CTAs
    if (CTAS > 1) {
        cluster.sync();
        sum = 0;
        for (int e = e0; e < e1; e++)
#pragma unroll
            for (int o = 0; o < CTAS; o++) sum += *cluster.map_shared_rank(mine + e, o);
    }
    int incl = sum, incl_own = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, off), z = __shfl_up_sync(0xffffffffu, incl_own, off);
        if (lane >= off) { incl += y; incl_own += z; }
    }
    if (lane == 31) { warp_tot[w] = incl; warp_own[w] = incl_own; }
    __syncthreads();
    int upto = warp_tot[lane], upto_own = warp_own[lane];      // every warp scans the 32 warp totals for itself
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, off), z = __shfl_up_sync(0xffffffffu, upto_own, off);
        if (lane >= off) { upto += y; upto_own += z; }
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31), total_own = __shfl_sync(0xffffffffu, upto_own, 31);
    const int earlier = __shfl_sync(0xffffffffu, upto, max(0, w - 1)), earlier_own = __shfl_sync(0xffffffffu, upto_own, max(0, w - 1));
    int before = incl - sum + (w > 0 ? earlier : 0), at_own = incl_own - own + (w > 0 ? earlier_own : 0);
    for (int e = e0; e < e1; e++) {
        if (rank == 0) offsets[e] = before;
        int first = before;     // where this CTA's pairs of e begin among all
        if (CTAS > 1) {
#pragma unroll
            for (int o = 0; o < CTAS; o++) {
                const int t = *cluster.map_shared_rank(mine + e, o);
                if (o < rank) first += t;
                before += t;
            }
        } else {
            before += mine[e];
        }
        shift[e] = first - at_own;
#pragma unroll 8
        for (int v = 0; v < warps; v++) {
            const int t = cnt[v * E + e];
            cnt[v * E + e] = at_own;
            at_own += t;
        }
    }
    if (rank == 0 && tid == 0) offsets[E] = total;
    __syncthreads();

    // the pairs' number inside this CTA and their expert in one word (14 and 12 bits), where the masks were
    const bool staged = once && run <= E && order;
    unsigned *sorted = masks;
    for (int64_t p = p0; p < p1; p += SORT_BATCH * 32) {
        if (!once) keys.load(idx, p, p1, base, lane);
#pragma unroll
        for (int i = 0; i < SORT_BATCH; i++) {
            const int64_t pair = p + i * 32 + lane;
            if (p + i * 32 >= p1) break;
            const uint32_t key = keys.v[i];
            int nth = rank_of[i] & 255, all = rank_of[i] >> 8;
            if (!once) {
                const unsigned same = lanes_of_key(key, E, my_mask, lane);
                nth = __popc(same & ((1u << lane) - 1));
                all = __popc(same);
            }
            const bool kept = key < (uint32_t)E;
            int at = -1;
            if (kept) at = my_cnt[key] + nth;
            __syncwarp();
            if (kept && nth == 0) my_cnt[key] = at + all;
            __syncwarp();
            const int to = kept ? at + shift[key] : -1;
            if (pair < p1 && place) place[pair] = to;
            if (kept) {
                if (staged) sorted[at] = (unsigned)(pair - cta0) << 12 | key;
                else if (order) order[to] = (int)pair;
            }
        }
    }
    if (staged) {
        __syncthreads();
        for (int i = tid; i < total_own; i += SORT_THREADS) order[i + shift[sorted[i] & 4095]] = (int)cta0 + (int)(sorted[i] >> 12);
    }
    if (order)
        for (int64_t p = total + rank * SORT_THREADS + tid; p < P; p += CTAS * SORT_THREADS) order[p] = -1;
    if (CTAS > 1) cluster.sync();   // no CTA leaves while another reads its totals
}

cudaError_t launch_sort_pairs(const uint32_t *idx, int P, int base, int E, int *order, int *place, int *offsets, cudaStream_t s)
{
    // counts and masks of all warps within SORT_SMEM; no more warps than there are steps of 32 pairs
    const int most = min(32, (int)((SORT_SMEM - 8 * E) / (8 * E)));
    const bool one = P <= SORT_ONE_CTA;
    const int ctas = one ? 1 : SORT_CTAS;
    const int warps = min(most, max(1, (P + 31) / 32 / ctas));
    const int run = (int)((((int64_t)P + ctas * warps - 1) / (ctas * warps) + 31) / 32 * 32);
    const size_t smem = ((size_t)2 * warps + 2) * E * sizeof(int);
    auto *kern = one ? k_sort_pairs<1> : k_sort_pairs<SORT_CTAS>;
    static std::atomic<uint64_t> asked[2] = {};
    if (smem > 40 * 1024) {
        cudaError_t e = allow_smem((const void *)kern, SORT_SMEM, asked[one]);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = ctas;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = one ? 1 : 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kern, idx, P, (uint32_t)base, E, warps, run, order, place, offsets);
}

// ---------------------------------------------------------------- rows
// Dispatch, combine and their gradients move every row once, so memory bounds them; what the kernels have to do is to keep
// enough loads on their way for any row length and any number of rows.  A row is cut into units (16 bytes of a row where
// its length and address allow), and a token gets as many threads as its row has units: 32 to 256 of them share a CTA with
// other tokens' threads, a longer row takes several CTAs.
struct RowThreads {
    int log2_threads;   // threads of a token inside a CTA of 256
    int ctas;           // CTAs of a token (1 unless its threads are all 256)
    unsigned grid;
    static RowThreads of(int64_t units, int n)
    {
        RowThreads r{5, 1, 0};
        while ((1 << r.log2_threads) < units && r.log2_threads < 8) r.log2_threads++;
        if (units > 256) r.ctas = (int)min((units + 255) / 256, (int64_t)max(1, (1 << 30) / n));
        const int tokens = 256 >> r.log2_threads;
        r.grid = (unsigned)((int64_t)((n + tokens - 1) / tokens) * r.ctas);
        return r;
    }
    // the token of this thread, its first unit and the step to its next ones
    __device__ void mine(int &t, int &first, int &step) const
    {
        t = (int)(blockIdx.x / ctas) * (256 >> log2_threads) + (threadIdx.x >> log2_threads);
        first = (int)(blockIdx.x % ctas) * 256 + (threadIdx.x & ((1 << log2_threads) - 1));
        step = ctas << log2_threads;
    }
};

// Rows are moved as bytes, so any element type goes: a unit is read once and written to the token's places.  The rows behind
// the last kept pair are zeroed by the same CTAs.
// M: units a thread takes at once, `step` apart; four where a unit is small, so that a place is read once for all of them.
template <typename V, int M>
__global__ void __launch_bounds__(256) k_dispatch_rows(const V *__restrict__ x, int units, int n, int top_k, const int *__restrict__ place,
                                                       const int *__restrict__ offsets, int E, V *__restrict__ out, RowThreads rt)
{
    pdl_wait();
    pdl_launch_dependents();
    const int P = n * top_k;
    int t, first, step;
    rt.mine(t, first, step);
    if (t < n)
        for (int u = first; u < units; u += step * M) {
            V v[M];
#pragma unroll
            for (int m = 0; m < M; m++) v[m] = u + m * step < units ? x[(size_t)t * units + u + m * step] : V{};
#pragma unroll 4
            for (int j = 0; j < top_k; j++) {
                const int to = place[(size_t)t * top_k + j];
                if ((unsigned)to >= (unsigned)P) continue;
                V *row = out + (size_t)to * units + u;
#pragma unroll
                for (int m = 0; m < M; m++)
                    if (u + m * step < units) row[m * step] = v[m];
            }
        }
    for (int64_t r = (int64_t)max(0, offsets[E]) + blockIdx.x; r < P; r += gridDim.x)
        for (int u = threadIdx.x; u < units; u += 256) out[(size_t)r * units + u] = V{};
}

cudaError_t launch_dispatch_rows(const void *x, size_t row_bytes, int n, int top_k, const int *place, const int *offsets, int E,
                                 void *out, cudaStream_t s)
{
    const uintptr_t a = (uintptr_t)x | (uintptr_t)out | row_bytes;
    auto go = [&](auto v) {
        using V = decltype(v);
        constexpr int M = sizeof(V) <= 4 ? 4 : 1;
        const int units = (int)(row_bytes / sizeof(V));
        const RowThreads rt = RowThreads::of((units + M - 1) / M, n);
        return launch_pdl(k_dispatch_rows<V, M>, dim3(rt.grid), dim3(256), 0, s, (const V *)x, units, n, top_k, place, offsets, E, (V *)out, rt);
    };
    count_launch();
    return a % 16 == 0 ? go(uint4{}) : a % 8 == 0 ? go(uint2{}) : a % 4 == 0 ? go(0u) : a % 2 == 0 ? go((uint16_t)0) : go((uint8_t)0);
}

// out_t = extra_t + sum_j w_tj rows[place_tj], f32 in slot order.  Without weights it is the gradient of the dispatch.
// (extra may be out: a thread reads the elements it later writes.)
template <int U, typename RT, typename ET, typename OT>
__global__ void __launch_bounds__(256) k_combine_rows(const RT *__restrict__ rows, int H, int n, int top_k, int n_rows,
                                                      const int *__restrict__ place, const float *__restrict__ w, const ET *extra,
                                                      OT *out, RowThreads rt)
{
    pdl_wait();
    pdl_launch_dependents();
    const int units = H / U;
    int t, first, step;
    rt.mine(t, first, step);
    if (t >= n) return;
    place += (size_t)t * top_k;
    if (w) w += (size_t)t * top_k;
    // M units at once, `step` apart (four where a unit is one or two elements: a place and a weight are read once for all), of
    // BATCH rows, without a branch between the loads: the first row and the last unit stand in for what does not count.
    constexpr int M = U <= 2 ? 4 : 1, BATCH = U <= 2 ? 2 : 4;
    for (int u = first; u < units; u += step * M) {
        float acc[M][U] = {};
        int at[M];
#pragma unroll
        for (int m = 0; m < M; m++) at[m] = M == 1 ? u * U : min(u + m * step, units - 1) * U;
        for (int j = 0; j < top_k && n_rows > 0; j += BATCH) {
            float v[BATCH][M][U], f[BATCH];
            bool there[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int r = j + i < top_k ? place[j + i] : -1;
                there[i] = (unsigned)r < (unsigned)n_rows;
                f[i] = w && j + i < top_k ? w[j + i] : 1.f;
#pragma unroll
                for (int m = 0; m < M; m++) load_units<U>(rows + (size_t)(there[i] ? r : 0) * H + at[m], v[i][m]);
            }
#pragma unroll
            for (int i = 0; i < BATCH; i++)
                if (there[i])
#pragma unroll
                    for (int m = 0; m < M; m++)
#pragma unroll
                        for (int e = 0; e < U; e++) acc[m][e] = fmaf(f[i], v[i][m][e], acc[m][e]);
        }
#pragma unroll
        for (int m = 0; m < M; m++) {
            if (M > 1 && u + m * step >= units) break;
            if (extra) {
                float v[U];
                load_units<U>(extra + (size_t)t * H + at[m], v);
#pragma unroll
                for (int e = 0; e < U; e++) acc[m][e] += v[e];
            }
            store_units<U>(out + (size_t)t * H + at[m], acc[m]);
        }
    }
}

// Elements of a unit: 16 bytes of the widest type among those given, fewer where H or an address does not allow it.
static int unit_elements(int H, bool any_f32, std::initializer_list<std::pair<const void *, int>> tensors)
{
    for (int u = any_f32 ? 4 : 8; u > 1; u /= 2) {
        bool fits = H % u == 0;
        for (auto &t : tensors) fits = fits && (uintptr_t)t.first % min(16, u * (t.second == PMOE_F32 ? 4 : 2)) == 0;
        if (fits) return u;
    }
    return 1;
}

// f(Units<u>) for a unit of u elements; eight only where all types are bf16
template <int U_> struct Units { static constexpr int U = U_; };
template <bool EIGHT, typename F> static auto with_units(int u, F &&f)
{
    if constexpr (EIGHT)
        if (u == 8) return f(Units<8>{});
    return u == 4 ? f(Units<4>{}) : u == 2 ? f(Units<2>{}) : f(Units<1>{});
}

cudaError_t launch_combine_rows(const void *rows, int rows_dtype, int n_rows, int n, int top_k, int H, const int *place, const float *w,
                                const void *extra, int extra_dtype, void *out, int out_dtype, cudaStream_t s)
{
    count_launch();
    const int u = unit_elements(H, rows_dtype == PMOE_F32 || extra_dtype == PMOE_F32 || out_dtype == PMOE_F32,
                                {{rows, rows_dtype}, {extra, extra_dtype}, {out, out_dtype}});
    const RowThreads rt = RowThreads::of(u <= 2 ? (H / u + 3) / 4 : H / u, n);
    return with_type(rows_dtype, [&](auto *rp) {
        return with_type(extra_dtype, [&](auto *ep) {
            return with_type(out_dtype, [&](auto *op) {
                using RT = std::remove_pointer_t<decltype(rp)>;
                using ET = std::remove_pointer_t<decltype(ep)>;
                using OT = std::remove_pointer_t<decltype(op)>;
                return with_units<sizeof(RT) + sizeof(ET) + sizeof(OT) == 6>(u, [&](auto units) {
                    return launch_pdl(k_combine_rows<decltype(units)::U, RT, ET, OT>, dim3(rt.grid), dim3(256), 0, s, (const RT *)rows, H, n,
                                      top_k, n_rows, place, w, (const ET *)extra, (OT *)out, rt);
                });
            });
        });
    });
}

// Gradient of combine: grad_rows[place_p] = w_p grad_out[t],  grad_w_p = <grad_out[t], rows[place_p]> for pair p = (t, j): one
// warp per pair, whose token's row comes from the cache for all slots but one.
template <int U, typename GT, typename RT>
__global__ void __launch_bounds__(256) k_combine_grad(const GT *__restrict__ grad_out, const RT *__restrict__ rows, int H, int top_k, int P,
                                                      const int *__restrict__ place, const int *__restrict__ offsets, int E,
                                                      const float *__restrict__ w, RT *__restrict__ grad_rows, float *__restrict__ grad_w)
{
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t p = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (p >= P) return;
    const int at = place[p];
    const bool kept = (unsigned)at < (unsigned)P;
    float dot = 0.f;
    if (kept) {
        const float wt = w ? w[p] : 1.f;
        const GT *g = grad_out + (size_t)(p / top_k) * H;
        const RT *r = rows + (size_t)at * H;
        RT *gr = grad_rows + (size_t)at * H;
#pragma unroll 4
        for (int h = lane * U; h < H; h += 32 * U) {
            float a[U], b[U];
            load_units<U>(g + h, a);
            if (grad_w) {
                load_units<U>(r + h, b);
#pragma unroll
                for (int i = 0; i < U; i++) dot = fmaf(a[i], b[i], dot);
            }
            if (grad_rows) {
#pragma unroll
                for (int i = 0; i < U; i++) a[i] *= wt;
                store_units<U>(gr + h, a);
            }
        }
    }
    if (grad_w) {
#pragma unroll
        for (int s = 16; s >= 1; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
        if (lane == 0) grad_w[p] = dot;
    }
    const int64_t r = (int64_t)max(0, offsets[E]) + p;   // one row behind the last kept pair each
    if (grad_rows && r < P) {
        const float zero[U] = {};
        for (int h = lane * U; h < H; h += 32 * U) store_units<U>(grad_rows + (size_t)r * H + h, zero);
    }
}

cudaError_t launch_combine_grad(const void *grad_out, int grad_dtype, const void *rows, int rows_dtype, int n, int top_k, int H,
                                const int *place, const int *offsets, int E, const float *w, void *grad_rows, float *grad_w,
                                cudaStream_t s)
{
    count_launch();
    const int P = n * top_k;
    const int u = unit_elements(H, grad_dtype == PMOE_F32 || rows_dtype == PMOE_F32, {{grad_out, grad_dtype}, {rows, rows_dtype}, {grad_rows, rows_dtype}});
    return with_type(grad_dtype, [&](auto *gp) {
        return with_type(rows_dtype, [&](auto *rp) {
            using GT = std::remove_pointer_t<decltype(gp)>;
            using RT = std::remove_pointer_t<decltype(rp)>;
            return with_units<sizeof(GT) + sizeof(RT) == 4>(u, [&](auto units) {
                return launch_pdl(k_combine_grad<decltype(units)::U, GT, RT>, dim3((P + 7) / 8), dim3(256), 0, s, (const GT *)grad_out,
                                  (const RT *)rows, H, top_k, P, place, offsets, E, w, (RT *)grad_rows, grad_w);
            });
        });
    });
}

constexpr int MAX_ROW = 1 << 30;   // a thread's place in a row and its step to the next one add up in 32 bits

static int check_pairs(int n, int top_k, int E)
{
    if (n < 0 || top_k <= 0 || (int64_t)n * top_k > (1 << 30)) return fail(PMOE_ERR_INVALID_ARG, "n >= 0, top_k >= 1 and n * top_k <= 2^30 are served");
    if (E <= 0 || E > SORT_MAX_E) return fail(PMOE_ERR_UNSUPPORTED_SHAPE, "1 to %d experts are served (got %d)", SORT_MAX_E, E);
    return PMOE_OK;
}

}  // namespace pmoe

using namespace pmoe;

extern "C" {

int pmoe_sort_pairs(int device, const uint32_t *idx, int n, int top_k, int expert_base, int E, int *order, int *place, int *offsets,
                    void *stream)
{
    int rc = check_pairs(n, top_k, E);
    if (rc) return rc;
    if (expert_base < 0 || expert_base > INT_MAX - E) return fail(PMOE_ERR_INVALID_ARG, "expert_base must be 0 to 2^31 - 1 - E");
    if (!offsets || (n && !idx)) return fail(PMOE_ERR_INVALID_ARG, "idx / offsets is NULL");
    const size_t pairs = (size_t)n * top_k * sizeof(int);
    if (overlap({{order, pairs}, {place, pairs}, {offsets, ((size_t)E + 1) * sizeof(int)}}, {{idx, pairs}}))
        return fail(PMOE_ERR_INVALID_ARG, "order, place and offsets must not overlap idx or one another");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    CU(launch_sort_pairs(idx, n * top_k, expert_base, E, order, place, offsets, (cudaStream_t)stream));
    return PMOE_OK;
}

int pmoe_dispatch_rows(int device, const void *x, size_t row_bytes, int n, int top_k, const int *place, const int *offsets, int E,
                       void *out, void *stream)
{
    int rc = check_pairs(n, top_k, E);
    if (rc) return rc;
    if (!row_bytes || row_bytes > MAX_ROW) return fail(PMOE_ERR_INVALID_ARG, "row_bytes must be 1 to 2^30");
    if (!n) return PMOE_OK;
    if (!x || !place || !offsets || !out) return fail(PMOE_ERR_INVALID_ARG, "x / place / offsets / out is NULL");
    const size_t pairs = (size_t)n * top_k;
    if (overlap({{out, pairs * row_bytes}}, {{x, (size_t)n * row_bytes}, {place, pairs * sizeof(int)}, {offsets, ((size_t)E + 1) * sizeof(int)}}))
        return fail(PMOE_ERR_INVALID_ARG, "out must not overlap x, place or offsets");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    CU(launch_dispatch_rows(x, row_bytes, n, top_k, place, offsets, E, out, (cudaStream_t)stream));
    return PMOE_OK;
}

int pmoe_combine_rows(int device, const void *rows, int rows_dtype, int n_rows, int n, int top_k, int H, const int *place,
                      const float *w, const void *extra, int extra_dtype, void *out, int out_dtype, void *stream)
{
    int rc = check_pairs(n, top_k, 1);
    if (rc) return rc;
    if (H <= 0 || H > MAX_ROW || n_rows < 0) return fail(PMOE_ERR_INVALID_ARG, "H must be 1 to 2^30 and n_rows not negative");
    if (!f32_or_bf16(rows_dtype) || !f32_or_bf16(out_dtype) || (extra && !f32_or_bf16(extra_dtype)))
        return fail(PMOE_ERR_UNSUPPORTED_DTYPE, "rows / extra / out must be F32 or BF16");
    if (!n) return PMOE_OK;
    if ((n_rows && !rows) || !place || !out) return fail(PMOE_ERR_INVALID_ARG, "rows / place / out is NULL");
    const size_t pairs = (size_t)n * top_k, out_bytes = (size_t)n * H * block_bytes(out_dtype);
    const bool in_place = extra == out && extra_dtype == out_dtype;
    if (overlap({{out, out_bytes}}, {{rows, (size_t)n_rows * H * block_bytes(rows_dtype)}, {place, pairs * sizeof(int)}, {w, pairs * sizeof(float)},
                                     {in_place ? nullptr : extra, (size_t)n * H * block_bytes(extra_dtype)}}))
        return fail(PMOE_ERR_INVALID_ARG, "out must not overlap rows, place or w, and extra only as a whole and in the same type");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    CU(launch_combine_rows(rows, rows_dtype, n_rows, n, top_k, H, place, w, extra, extra ? extra_dtype : out_dtype, out, out_dtype,
                           (cudaStream_t)stream));
    return PMOE_OK;
}

int pmoe_combine_rows_grad(int device, const void *grad_out, int grad_dtype, const void *rows, int rows_dtype, int n, int top_k, int H,
                           const int *place, const int *offsets, int E, const float *w, void *grad_rows, float *grad_w, void *stream)
{
    int rc = check_pairs(n, top_k, E);
    if (rc) return rc;
    if (H <= 0 || H > MAX_ROW) return fail(PMOE_ERR_INVALID_ARG, "H must be 1 to 2^30");
    if (!f32_or_bf16(grad_dtype) || !f32_or_bf16(rows_dtype)) return fail(PMOE_ERR_UNSUPPORTED_DTYPE, "grad_out / rows must be F32 or BF16");
    if (!n) return PMOE_OK;
    if (!grad_rows && !grad_w) return fail(PMOE_ERR_INVALID_ARG, "neither grad_rows nor grad_w is asked for");
    if (!grad_out || !place || !offsets || (grad_w && !rows)) return fail(PMOE_ERR_INVALID_ARG, "grad_out / rows / place / offsets is NULL");
    const size_t pairs = (size_t)n * top_k, rows_bytes = pairs * H * block_bytes(rows_dtype);
    if (overlap({{grad_rows, rows_bytes}, {grad_w, pairs * sizeof(float)}},
                {{grad_out, (size_t)n * H * block_bytes(grad_dtype)}, {rows, rows_bytes}, {place, pairs * sizeof(int)},
                 {offsets, ((size_t)E + 1) * sizeof(int)}, {w, pairs * sizeof(float)}}))
        return fail(PMOE_ERR_INVALID_ARG, "grad_rows and grad_w must not overlap an input or one another");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    CU(launch_combine_grad(grad_out, grad_dtype, rows, rows_dtype, n, top_k, H, place, offsets, E, w, grad_rows, grad_w,
                           (cudaStream_t)stream));
    return PMOE_OK;
}

}  // extern "C"
