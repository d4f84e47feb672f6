// Loads and stores of a few consecutive row elements as f32, shared by the row operators (sort / dispatch / combine,
// 8-bit norm, low-rank adapters).  Addresses are multiples of 16 bytes, or of the whole unit where that is shorter.
#pragma once
#include "pmoe_common.cuh"

namespace pmoe {

template <int U, typename T> __device__ inline void load_units(const T *p, float (&v)[U])
{
    if constexpr (U == 1) {
        v[0] = load_as_float(p, 0);
    } else if constexpr (U == 2 && sizeof(T) == 4) {
        const float2 a = *reinterpret_cast<const float2 *>(p);
        v[0] = a.x; v[1] = a.y;
    } else if constexpr (sizeof(T) == 4) {
        static_assert(U % 4 == 0, "whole 16-byte loads");
#pragma unroll
        for (int i = 0; i < U / 4; i++) {
            const float4 a = reinterpret_cast<const float4 *>(p)[i];
            v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
        }
    } else if constexpr (U < 8) {   // a bf16 is the upper half of its f32
        uint32_t w[U / 2];
        if constexpr (U == 2) {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
            const uint2 a = *reinterpret_cast<const uint2 *>(p);
            w[0] = a.x; w[1] = a.y;
        }
#pragma unroll
        for (int j = 0; j < U / 2; j++) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
        static_assert(U % 8 == 0, "whole 16-byte loads");
#pragma unroll
        for (int i = 0; i < U / 8; i++) {
            const uint4 a = reinterpret_cast<const uint4 *>(p)[i];
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
                v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    }
}

__device__ inline uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}

template <int U, typename T> __device__ inline void store_units(T *p, const float (&v)[U])
{
    if constexpr (U == 1) {
        store_from_float(p, 0, v[0]);
    } else if constexpr (U == 2 && sizeof(T) == 4) {
        *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    } else if constexpr (U == 2) {
        *reinterpret_cast<uint32_t *>(p) = pack_bf16(v[0], v[1]);
    } else if constexpr (U == 4 && sizeof(T) == 2) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < U / 4; i++)
            reinterpret_cast<float4 *>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < U / 8; i++)
            reinterpret_cast<uint4 *>(p)[i] = make_uint4(pack_bf16(v[8 * i], v[8 * i + 1]), pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                                                         pack_bf16(v[8 * i + 4], v[8 * i + 5]), pack_bf16(v[8 * i + 6], v[8 * i + 7]));
    }
}

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// f(float) or f(__nv_bfloat16) for a dtype id that the caller has checked
template <typename F> inline auto with_type(int dtype, F &&f)
{
    return dtype == PMOE_F32 ? f((float *)nullptr) : f((__nv_bfloat16 *)nullptr);
}
inline bool f32_or_bf16(int dtype) { return dtype == PMOE_F32 || dtype == PMOE_BF16; }

}  // namespace pmoe
