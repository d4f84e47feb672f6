// The residual add and RMS norm of pmoe_add_rms_norm with the normalised row in 8 bits: LayerWeights::forward_with_stats
// (paramecia-model/src/qwen3_next.rs:4273-4286) and RmsNorm::forward (quantized_nn.rs:172-190), followed by the
// activation quantiser that a mat-mul over 8-bit rows would run as a pass of its own.
//   r = round(resid + delta) in the residual's type (what is stored is what is normalised),
//   v = r / sqrt(mean(r^2) + eps) * weight,
//   per group of g values: a = max |v|, scale = a / 127 (int8) or a / 448 (e4m3), q = round(v / scale),
//   values = q * scale (optional).
// A group that holds an infinity or a NaN gets a scale that is not finite and zeros: its values read NaN, as the row does.
#include <cuda_fp8.h>

#include "pmoe_internal.h"
#include "pmoe_vec.cuh"

namespace pmoe {

constexpr int NORM_Q8_MAX_H = 16384;

// |v| as ordered bits: unsigned integers compare like the magnitudes, infinity above all numbers and NaN above infinity,
// so an integer maximum carries a NaN through where fmaxf would drop it.
__device__ inline uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <bool E4M3> __device__ inline uint8_t to_8bit(float ratio)
{
    if constexpr (E4M3) return (uint8_t)__nv_cvt_float_to_fp8(ratio, __NV_SATFINITE, __NV_E4M3);
    else return (uint8_t)(int8_t)max(-127, min(127, __float2int_rn(ratio)));
}
template <bool E4M3> __device__ inline float from_8bit(uint8_t q)
{
    if constexpr (E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)q, __NV_E4M3)));
    else return (float)(int8_t)q;
}

// one CTA per row, the row in shared memory, one warp per group
template <typename RT, typename DT, typename VT, bool E4M3>
__global__ void __launch_bounds__(256) k_norm_q8(const RT *resid_in, const DT *__restrict__ delta, const float *__restrict__ weight, int H,
                                                 float eps, int group, RT *resid_out, uint8_t *__restrict__ q, float *__restrict__ scales,
                                                 VT *__restrict__ values)
{
    extern __shared__ float row[];
    __shared__ float red[8];
    pdl_wait();
    pdl_launch_dependents();
    const size_t base = (size_t)blockIdx.x * H;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float ss = 0.f;
    for (int h = threadIdx.x; h < H; h += 256) {
        float v = load_as_float(resid_in, base + h);
        if (delta) v += load_as_float(delta, base + h);
        RT r;
        store_from_float(&r, 0, v);
        v = load_as_float(&r, 0);
        if (resid_out) resid_out[base + h] = r;
        row[h] = v;
        ss = fmaf(v, v, ss);
    }
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, s);
    if (lane == 0) red[warp] = ss;
    __syncthreads();
    float tot = 0.f;
    for (int w = 0; w < 8; w++) tot += red[w];
    const float m = sqrtf(tot / (float)H + eps);
    const int G = (H + group - 1) / group;
    for (int g = warp; g < G; g += 8) {
        const int h0 = g * group, h1 = min(H, h0 + group);
        uint32_t top = 0;
        for (int h = h0 + lane; h < h1; h += 32) {
            const float v = __fdiv_rn(row[h], m) * (weight ? weight[h] : 1.f);
            row[h] = v;
            top = max(top, magnitude(v));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        const float scale = __fdiv_rn(__uint_as_float(top), E4M3 ? 448.f : 127.f);
        const bool usable = scale > 0.f && scale < INFINITY;
        if (lane == 0) scales[(size_t)blockIdx.x * G + g] = scale;
        for (int h = h0 + lane; h < h1; h += 32) {
            const uint8_t b = usable ? to_8bit<E4M3>(__fdiv_rn(row[h], scale)) : 0;
            q[base + h] = b;
            if (values) store_from_float(values, base + h, from_8bit<E4M3>(b) * scale);
        }
    }
}

cudaError_t launch_norm_q8(const void *resid_in, int resid_dtype, const void *delta, int delta_dtype, const float *weight, int n, int H,
                           float eps, int group, void *resid_out, int q_dtype, void *q, float *scales, void *values, int values_dtype,
                           cudaStream_t s)
{
    count_launch();
    return with_type(resid_dtype, [&](auto *rp) {
        return with_type(delta_dtype, [&](auto *dp) {
            return with_type(values_dtype, [&](auto *vp) {
                using RT = std::remove_pointer_t<decltype(rp)>;
                using DT = std::remove_pointer_t<decltype(dp)>;
                using VT = std::remove_pointer_t<decltype(vp)>;
                auto *kern = q_dtype == PMOE_F8_E4M3 ? k_norm_q8<RT, DT, VT, true> : k_norm_q8<RT, DT, VT, false>;
                if (H > 12000) {   // beyond what a launch may have without asking
                    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_Q8_MAX_H * (int)sizeof(float));
                    if (e != cudaSuccess) return e;
                }
                return launch_pdl(kern, dim3(n), dim3(256),
                                  (size_t)H * sizeof(float), s, (const RT *)resid_in, (const DT *)delta, weight, H, eps, group,
                                  (RT *)resid_out, (uint8_t *)q, scales, (VT *)values);
            });
        });
    });
}

}  // namespace pmoe

using namespace pmoe;

extern "C" int pmoe_add_rms_norm_q8(int device, const void *resid_in, int resid_dtype, const void *delta, int delta_dtype,
                                    const float *weight, int n, int H, float eps, int group, void *resid_out, int q_dtype, void *q,
                                    float *scales, void *values, int values_dtype, void *stream)
{
    if (n < 0 || H <= 0 || H > NORM_Q8_MAX_H) return fail(PMOE_ERR_INVALID_ARG, "bad n / H (H <= %d)", NORM_Q8_MAX_H);
    if (group != 0 && group != 32 && group != 64 && group != 128 && group != 256)
        return fail(PMOE_ERR_UNSUPPORTED_SHAPE, "group must be 32, 64, 128, 256 or 0 for the whole row (got %d)", group);
    if (!f32_or_bf16(resid_dtype) || (delta && !f32_or_bf16(delta_dtype)) || (values && !f32_or_bf16(values_dtype)))
        return fail(PMOE_ERR_UNSUPPORTED_DTYPE, "resid / delta / values must be F32 or BF16");
    if (q_dtype != PMOE_I8 && q_dtype != PMOE_F8_E4M3) return fail(PMOE_ERR_UNSUPPORTED_DTYPE, "q must be I8 or F8_E4M3 (got %d)", q_dtype);
    if (!(eps >= 0.f)) return fail(PMOE_ERR_INVALID_ARG, "eps must not be negative");
    if (!n) return PMOE_OK;
    if (!resid_in || !q || !scales) return fail(PMOE_ERR_INVALID_ARG, "resid_in / q / scales is NULL");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    CU(launch_norm_q8(resid_in, resid_dtype, delta, delta ? delta_dtype : resid_dtype, weight, n, H, eps, group ? group : H, resid_out,
                      q_dtype, q, scales, values, values ? values_dtype : resid_dtype, (cudaStream_t)stream));
    return PMOE_OK;
}
