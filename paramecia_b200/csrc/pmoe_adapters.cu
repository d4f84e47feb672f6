// Low-rank adapters of many requests beside one projection: out_t = base_t + s_i B_i (A_i x_t) with i = ids[t], for a
// batch whose rows belong to different adapters.  base is the shared projection's output (pmoe_qmatmul's, say); a row whose
// id is outside [0, L) keeps it.  The reference's QMatMul holds one low-rank update and merges it
// (paramecia-model/src/models/with_tracing.rs:103-337).
#include "pmoe_internal.h"
#include "pmoe_vec.cuh"

namespace pmoe {

constexpr int ADAPTER_MAX_RANK = 128;
constexpr int ADAPTER_ROWS_UNSORTED = 1024;   // rows that are grouped by id without pmoe_sort_pairs

// one CTA per row: h = A x by one warp per rank, then one output column per thread
template <typename XT, typename OT>
__global__ void __launch_bounds__(256) k_adapters(const OT *base, const XT *__restrict__ x, int K, int N, int r,
                                                  const __nv_bfloat16 *__restrict__ a, const __nv_bfloat16 *__restrict__ b,
                                                  const float *__restrict__ scales, int L, const int *__restrict__ ids, OT *out)
{
    __shared__ float h[ADAPTER_MAX_RANK];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t t = blockIdx.x;
    const int id = ids[t];
    const bool has = (unsigned)id < (unsigned)L;
    if (has) {
        const float s = scales ? scales[id] : 1.f;
        for (int c = warp; c < r; c += 8) {
            const __nv_bfloat16 *ar = a + ((size_t)id * r + c) * K;
            float acc = 0.f;
            for (int k = lane; k < K; k += 32) acc = fmaf(load_as_float(x, t * K + k), __bfloat162float(ar[k]), acc);
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
            if (lane == 0) h[c] = acc * s;
        }
    }
    __syncthreads();
    for (int o = threadIdx.x; o < N; o += 256) {
        float v = load_as_float(base, t * N + o);
        if (has) {
            const __nv_bfloat16 *br = b + ((size_t)id * N + o) * r;
            float acc = 0.f;
            for (int c = 0; c < r; c++) acc = fmaf(h[c], __bfloat162float(br[c]), acc);
            v += acc;
        }
        store_from_float(out, t * N + o, v);
    }
}

cudaError_t launch_adapters(const void *base, int out_dtype, const void *x, int x_dtype, int n, int K, int N, int r, const void *a,
                            const void *b, const float *scales, int L, const int *ids, void *out, cudaStream_t s)
{
    count_launch();
    return with_type(x_dtype, [&](auto *xp) {
        return with_type(out_dtype, [&](auto *op) {
            using XT = std::remove_pointer_t<decltype(xp)>;
            using OT = std::remove_pointer_t<decltype(op)>;
            return launch_pdl(k_adapters<XT, OT>, dim3(n), dim3(256), 0, s, (const OT *)base, (const XT *)x, K, N, r,
                              (const __nv_bfloat16 *)a, (const __nv_bfloat16 *)b, scales, L, ids, (OT *)out);
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
    CU(launch_adapters(base, out_dtype, x, x_dtype, n, K, N, rank, a, b, scales, n_adapters, ids, out, (cudaStream_t)stream));
    return PMOE_OK;
}
