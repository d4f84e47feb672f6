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

// max(m, |v|) that keeps a NaN, which fmaxf would drop
__device__ inline float max_abs(float m, float v)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
    return r;
}

// the same in 64 bits
__device__ inline double max_nan(double m, double v) { return v > m || v != v ? v : m; }

// How a group becomes 8 bits.  With u = r * weight and top = max |u| over the group, v = u / m and
//   scale = max |v| / 127 = top * (1 / m) / 127,   v / scale = u * (127 / top):
// the quotient needs neither m nor the rounded scale, which saves two products an element and lets both statistics be
// reduced at once.  For int8 it is taken in f32 (u, top, 127 / top: three roundings, where dividing v by its scale takes five): a
// value within 2^-15 of the middle between two steps may become either (of 24 million values none was another than the exact
// quotient's).  An e4m3 q is the rounding of the exact quotient: every value is rounded twice, from a quotient that is certainly too small and one that is certainly too large, and where the
// two differ, as for one value in 10^5, the group is done again in 64 bits from the row as it was stored.
constexpr float BELOW = 1.f - 0x1.6p-22f, ABOVE = 1.f + 0x1.6p-22f;   // five roundings of 2^-24 and a little

struct GroupScale {
    float scale, top;
    bool plain;    // scale is a number above 0, and `most / top` does not overflow
    template <bool E4M3> __device__ static GroupScale of(float top, float inv_m)
    {
        GroupScale g;
        g.scale = __fdiv_rn(top * inv_m, E4M3 ? 448.f : 127.f);
        g.top = top;
        g.plain = top >= 0x1p-100f && g.scale > 0.f && g.scale < INFINITY;
        return g;
    }
    template <bool E4M3> __device__ float inverse() const { return __fdiv_rn(E4M3 ? 448.f : 127.f, top); }
    // u * (127 / top) for the other groups: 0 where the scale is 0, infinite or NaN
    template <bool E4M3> __device__ float ratio(float u) const
    {
        return scale > 0.f && scale < INFINITY ? __fdiv_rn(u, top) * (E4M3 ? 448.f : 127.f) : 0.f;
    }
};

// 1 / sqrt(mean + eps); of 0 it is infinite and of an infinity 0, so that u * inv_m is u / m there too
__device__ inline float inverse_rms(float ss, int H, float eps) { return __frcp_rn(sqrtf(ss / (float)H + eps)); }

// N numbers u[i] * f to 8 bits, the bytes of `packed` in order.  N is 1 or a multiple of 4.
template <bool E4M3, int N> __device__ inline void to_8bit(const float (&u)[N], float f, uint32_t *packed)
{
    if constexpr (E4M3) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const __nv_fp8x2_storage_t b = __nv_cvt_float2_to_fp8x2(make_float2(u[i] * f, i + 1 < N ? u[i + 1] * f : 0.f), __NV_SATFINITE, __NV_E4M3);
            if (i % 4 == 0) packed[i / 4] = N == 1 ? b & 0xff : b;
            else packed[i / 4] |= (uint32_t)b << 16;
        }
    } else {
        // 1.5 * 2^23 + x rounds x to the nearest integer, ties to even, and its low byte is that integer's
        uint32_t t[N];
#pragma unroll
        for (int i = 0; i < N; i++) t[i] = __float_as_uint(fmaf(u[i], f, 12582912.f));
        if constexpr (N == 1) packed[0] = t[0] & 0xff;
        else
#pragma unroll
            for (int i = 0; i < N; i += 4) packed[i / 4] = __byte_perm(__byte_perm(t[i], t[i + 1], 0x0040), __byte_perm(t[i + 2], t[i + 3], 0x0040), 0x5410);
    }
}

// The quotient of d by the group's largest magnitude, rounded once to an 8-bit float.  d and top are products of two f32 numbers:
// 448 d is exact, and a quotient that is not a tie of e4m3 (five significant bits) is further from it than half a step of 64 bits,
// so the 64-bit quotient lies on the same side of every tie as the exact one, or on it where that does.  On the way to f32 the last
// bit says whether anything was cut off: rounding to nearest there would put a quotient beside a tie onto it.
__device__ inline uint32_t to_e4m3_exact(double d, double top)
{
    const double quotient = d * 448.0 / top;
    const float cut = __double2float_rz(quotient);
    const float f = __uint_as_float(__float_as_uint(cut) | ((double)cut != quotient ? 1u : 0u));
    return (uint32_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
}

// What four bytes stand for in units of the scale
template <bool E4M3> __device__ inline void held4(uint32_t packed, float *y)
{
    if constexpr (E4M3) {
        const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)packed, __NV_E4M3)));
        const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(packed >> 16), __NV_E4M3)));
        y[0] = a.x; y[1] = a.y; y[2] = b.x; y[3] = b.y;
    } else {
        // byte + 128 as the low byte of 2^23
        const uint32_t t = packed ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = __uint_as_float(__byte_perm(t, 0x4b000000u, 0x7650 | i)) - 8388736.f;
    }
}

// v + d rounded to the type of the residual, eight elements, written where the residual goes (if it goes anywhere)
__device__ inline void add_and_store(float (&v)[8], const float (&d)[8], float *to)
{
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += d[i];
    if (to) store_units<8>(to, v);
}
__device__ inline void add_and_store(float (&v)[8], const float (&d)[8], __nv_bfloat16 *to)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i] = pack_bf16(v[2 * i] + d[2 * i], v[2 * i + 1] + d[2 * i + 1]);
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    if (to) *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}

// One CTA per row.  The operator reads and writes each element once (17 bytes for f32 + f32 -> f32, int8, f32 values, 13 without
// values; 7 for bf16 + bf16 -> bf16, e4m3), so memory bounds it and the row must stay on the chip between its two statistics: here in
// registers, eight consecutive elements a thread and pass, a row never longer than threads * PASSES * 8.  A group is 4, 8, 16
// or 32 neighbouring threads of a pass (its maximum by shuffles) or the whole row (shuffles and a shared array).  The second
// limit is the issue rate: with two quotients an element 16384 rows of 2048 bf16 took 126 us to e4m3.  Now 51 us, 0.72 of the
// measured copy rate, with 44 instructions an element in 85 % of the issue slots; to int8 45 us, 0.81 of it, and from f32 rows 67 to 71 us, 0.95 and more.
// Where many quotients are ties (bf16 rows without weights) the 64-bit part runs for most rows: 87 us by groups of 128, 97 us by rows.
// THREADS: the most a launch has.  With one pass the registers are held to what fills an SM (2048 threads): the part in 64 bits wants
// twice as many.  It is compiled in with 192 to 240 bytes of spills a thread for e4m3; with the registers 16384 rows took 60 us for 51.
template <typename RT, typename DT, typename VT, bool E4M3, int PASSES, int THREADS>
__global__ void __launch_bounds__(THREADS, PASSES == 1 ? 2048 / THREADS : 1) k_norm_q8(const RT *resid_in, const DT *__restrict__ delta, const float *__restrict__ weight, int H,
                                                  float eps, int group, RT *resid_out, uint8_t *__restrict__ q,
                                                  float *__restrict__ scales, VT *__restrict__ values)
{
    __shared__ float red[32], red_max[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const size_t base = (size_t)blockIdx.x * H;
    pdl_wait();
    pdl_launch_dependents();
    float v[PASSES][8];
    float ss = 0.f;
    if (delta) {
        float d[PASSES][8];
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            const int h = (p * blockDim.x + tid) * 8;
            if (h >= H) continue;
            load_units<8>(resid_in + base + h, v[p]);
            load_units<8>(delta + base + h, d[p]);
        }
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            const int h = (p * blockDim.x + tid) * 8;
            if (h < H) add_and_store(v[p], d[p], resid_out ? resid_out + base + h : (RT *)nullptr);
        }
    } else {
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            const int h = (p * blockDim.x + tid) * 8;
            if (h >= H) continue;
            load_units<8>(resid_in + base + h, v[p]);
            if (resid_out) store_units<8>(resid_out + base + h, v[p]);
        }
    }
    float top[PASSES], row_top = 0.f;
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        const int h = (p * blockDim.x + tid) * 8;
        top[p] = 0.f;
        if (h >= H) continue;
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(v[p][i], v[p][i], ss);
        if (weight) {
            float w[8];
            load_units<8>(weight + h, w);
#pragma unroll
            for (int i = 0; i < 8; i++) v[p][i] *= w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) top[p] = max_abs(top[p], v[p][i]);
        if (group >= H) row_top = max_abs(row_top, top[p]);
    }
    const int log2_group = 31 - __clz(group), G = group >= H ? 1 : (H + group - 1) >> log2_group;   // more than one group: a power of two
    float *row_scales = scales + (size_t)blockIdx.x * G;
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, s);
        if (G == 1) row_top = max_abs(row_top, __shfl_xor_sync(0xffffffffu, row_top, s));
    }
    if (lane == 0) { red[warp] = ss; red_max[warp] = row_top; }
    if (G > 1) {   // groups of 32 to 256 values: up to a warp's
#pragma unroll
        for (int p = 0; p < PASSES; p++)
#pragma unroll
            for (int s = 1; s < 32; s <<= 1)
                if (s * 8 < group) top[p] = max_abs(top[p], __shfl_xor_sync(0xffffffffu, top[p], s));
    }
    __syncthreads();
    ss = lane < warps ? red[lane] : 0.f;
    row_top = lane < warps ? red_max[lane] : 0.f;
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, s);
        if (G == 1) row_top = max_abs(row_top, __shfl_xor_sync(0xffffffffu, row_top, s));
    }
    const float inv_m = inverse_rms(ss, H, eps);
    bool border[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        const int h = (p * blockDim.x + tid) * 8;
        border[p] = false;
        if (h >= H) continue;
        const GroupScale gs = GroupScale::of<E4M3>(G == 1 ? row_top : top[p], inv_m);
        if (G == 1 ? h == 0 : (h & (group - 1)) == 0) row_scales[G == 1 ? 0 : h >> log2_group] = gs.scale;
        uint32_t packed[2];
        if (gs.plain) {
            const float inverse = gs.inverse<E4M3>();
            to_8bit<E4M3>(v[p], E4M3 ? inverse * BELOW : inverse, packed);
            if constexpr (E4M3) {
                uint32_t above[2];
                to_8bit<E4M3>(v[p], inverse * ABOVE, above);
                border[p] = packed[0] != above[0] || packed[1] != above[1];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[p][i] = gs.ratio<E4M3>(v[p][i]);
            to_8bit<E4M3>(v[p], 1.f, packed);
        }
        *reinterpret_cast<uint2 *>(q + base + h) = make_uint2(packed[0], packed[1]);
        if (values) {
            float y[8];
            held4<E4M3>(packed[0], y);
            held4<E4M3>(packed[1], y + 4);
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] *= gs.scale;   // NaN where the scale is not finite: 0 * inf
            store_units<8>(values + base + h, y);
        }
    }
    if constexpr (E4M3) {
        bool any = false;
#pragma unroll
        for (int p = 0; p < PASSES; p++) any |= border[p];
        if (G == 1 ? !__syncthreads_or(any) : !__any_sync(0xffffffffu, any)) return;
        __shared__ double red_exact[32];
        double d[8], t = 0;
        // the exact products of a pass; the stored residual is what was normalised
        auto products = [&](int p) {
            const int h = (p * blockDim.x + tid) * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) d[i] = 0;
            if (h < H) {
                float r[8], w[8], a[8];
                load_units<8>((resid_out ? resid_out : resid_in) + base + h, r);
                if (weight) load_units<8>(weight + h, w);
                if (delta && !resid_out) {
                    load_units<8>(delta + base + h, a);
                    add_and_store(r, a, (RT *)nullptr);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) d[i] = weight ? (double)r[i] * (double)w[i] : (double)r[i];
            }
            double most = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) most = max_nan(most, fabs(d[i]));
            return most;
        };
        auto store = [&](int p) {
            const int h = (p * blockDim.x + tid) * 8;
            const GroupScale gs = GroupScale::of<E4M3>((float)t, inv_m);   // rounding keeps the order: t's rounding is `top`
            if (h >= H || !gs.plain) return;
            uint32_t packed[2] = {0u, 0u};
#pragma unroll
            for (int i = 0; i < 8; i++) packed[i / 4] |= to_e4m3_exact(d[i], t) << (8 * (i & 3));
            *reinterpret_cast<uint2 *>(q + base + h) = make_uint2(packed[0], packed[1]);
            if (values) {
                float y[8];
                held4<E4M3>(packed[0], y);
                held4<E4M3>(packed[1], y + 4);
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] *= gs.scale;
                store_units<8>(values + base + h, y);
            }
        };
        if (G > 1) {
#pragma unroll 1
            for (int p = 0; p < PASSES; p++) {
                t = products(p);
#pragma unroll
                for (int s = 1; s < 32; s <<= 1)
                    if (s * 8 < group) t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, s));
                store(p);
            }
        } else {
#pragma unroll 1
            for (int p = 0; p < PASSES; p++) t = max_nan(t, products(p));
#pragma unroll
            for (int s = 16; s >= 1; s >>= 1) t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, s));
            if (lane == 0) red_exact[warp] = t;
            __syncthreads();
            t = lane < warps ? red_exact[lane] : 0.0;
#pragma unroll
            for (int s = 16; s >= 1; s >>= 1) t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, s));
#pragma unroll 1
            for (int p = 0; p < PASSES; p++) {
                if (PASSES > 1) products(p);
                store(p);
            }
        }
    }
}

// Rows that no vector load fits (H not a multiple of 8, or an address off its boundary).  A warp has 256 consecutive
// elements a pass, lane l those at l, l + 32, ...: its loads are whole lines whatever the address, and a group of 32 to
// 256 values is one to eight registers of a warp.  16384 rows of 2047, us: f32 to int8 95 by rows and 113 by groups of 128; bf16 to int8 121 and
// 141, to e4m3 158 and 178, and 266 and 356 where most rows hold ties: an element a load, a store and a conversion.
template <typename RT, typename DT, typename VT, bool E4M3>
__global__ void __launch_bounds__(1024) k_norm_q8_any(const RT *resid_in, const DT *__restrict__ delta, const float *__restrict__ weight,
                                                      int H, float eps, int group, RT *resid_out, uint8_t *__restrict__ q,
                                                      float *__restrict__ scales, VT *__restrict__ values)
{
    constexpr int PASSES = NORM_Q8_MAX_H / (1024 * 8);
    __shared__ float red[32], red_max[32];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const size_t base = (size_t)blockIdx.x * H;
    resid_in += base;
    if (delta) delta += base;
    if (resid_out) resid_out += base;
    q += base;
    if (values) values += base;
    float v[PASSES][8];
    float ss = 0.f, row_top = 0.f;
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        const int h0 = (p * warps + warp) * 256 + lane;
        if (h0 - lane >= H) break;
        float d[8] = {}, w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int h = h0 + i * 32;
            v[p][i] = h < H ? load_as_float(resid_in, h) : 0.f;
            if (delta && h < H) d[i] = load_as_float(delta, h);
            w[i] = weight && h < H ? weight[h] : 1.f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int h = h0 + i * 32;
            RT r;
            store_from_float(&r, 0, delta ? v[p][i] + d[i] : v[p][i]);
            v[p][i] = load_as_float(&r, 0);
            if (resid_out && h < H) resid_out[h] = r;
            ss = fmaf(v[p][i], v[p][i], ss);
            v[p][i] *= w[i];
            if (group >= H) row_top = max_abs(row_top, v[p][i]);
        }
    }
    const int log2_group = 31 - __clz(group), G = group >= H ? 1 : (H + group - 1) >> log2_group;   // more than one group: a power of two
    float *row_scales = scales + (size_t)blockIdx.x * G;
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, s);
        if (G == 1) row_top = max_abs(row_top, __shfl_xor_sync(0xffffffffu, row_top, s));
    }
    if (lane == 0) { red[warp] = ss; red_max[warp] = row_top; }
    __syncthreads();
    ss = lane < warps ? red[lane] : 0.f;
    row_top = lane < warps ? red_max[lane] : 0.f;
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, s);
        if (G == 1) row_top = max_abs(row_top, __shfl_xor_sync(0xffffffffu, row_top, s));
    }
    const float inv_m = inverse_rms(ss, H, eps);
    bool border = false;
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        const int h0 = (p * warps + warp) * 256 + lane;
        if (h0 - lane >= H) break;
        float top[8];
#pragma unroll
        for (int i = 0; i < 8; i++) top[i] = fabsf(v[p][i]);
        if (G > 1)
#pragma unroll
            for (int s = 1; s < 8; s <<= 1)
                if (s * 32 < group)
#pragma unroll
                    for (int i = 0; i < 8; i += 2 * s) top[i] = max_abs(top[i], top[i + s]);
        GroupScale gs = GroupScale::of<E4M3>(row_top, inv_m);
        float inverse = gs.inverse<E4M3>();
        if (G == 1 && h0 == 0) row_scales[0] = gs.scale;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int h = h0 + i * 32;
            if (G > 1 && (i * 32 & (group - 1)) == 0) {   // a group begins
#pragma unroll
                for (int s = 16; s >= 1; s >>= 1) top[i] = max_abs(top[i], __shfl_xor_sync(0xffffffffu, top[i], s));
                gs = GroupScale::of<E4M3>(top[i], inv_m);
                inverse = gs.inverse<E4M3>();
                if (lane == 0 && h < H) row_scales[h >> log2_group] = gs.scale;
            }
            if (h >= H) continue;
            const float x[1] = {gs.plain ? v[p][i] : gs.ratio<E4M3>(v[p][i])};
            uint32_t low;
            to_8bit<E4M3>(x, !gs.plain ? 1.f : E4M3 ? inverse * BELOW : inverse, &low);
            if constexpr (E4M3) {
                uint32_t high;
                to_8bit<E4M3>(x, gs.plain ? inverse * ABOVE : 1.f, &high);
                border |= low != high;
            }
            q[h] = (uint8_t)low;
            if (values) {
                float y[4];
                held4<E4M3>(low, y);
                store_from_float(values, h, y[0] * gs.scale);
            }
        }
    }
    if constexpr (E4M3) {
        if (G == 1 ? !__syncthreads_or(border) : !__any_sync(0xffffffffu, border)) return;
        __shared__ double red_exact[32];
        auto product = [&](int h) {   // exact; the stored residual is what was normalised
            if (h >= H) return 0.0;
            RT r;
            store_from_float(&r, 0, resid_out ? load_as_float(resid_out, h) : load_as_float(resid_in, h) + (delta ? load_as_float(delta, h) : 0.f));
            return (double)load_as_float(&r, 0) * (weight ? (double)weight[h] : 1.0);
        };
        auto store = [&](int h, double t) {
            const GroupScale gs = GroupScale::of<E4M3>((float)t, inv_m);
            if (h >= H || !gs.plain) return;
            const uint32_t b = to_e4m3_exact(product(h), t);
            q[h] = (uint8_t)b;
            if (values) {
                float y[4];
                held4<E4M3>(b, y);
                store_from_float(values, h, y[0] * gs.scale);
            }
        };
        if (G > 1) {
            for (int p = 0; p < PASSES; p++)
                for (int i0 = 0; i0 < 256; i0 += group) {
                    const int h0 = (p * warps + warp) * 256 + i0 + lane;
                    double t = 0;
                    for (int k = 0; k < group; k += 32) t = max_nan(t, fabs(product(h0 + k)));
#pragma unroll
                    for (int s = 16; s >= 1; s >>= 1) t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, s));
                    for (int k = 0; k < group; k += 32) store(h0 + k, t);
                }
        } else {
            // over the elements that this thread wrote: no other thread touches their bytes
            double t = 0;
            for (int p = 0; p < PASSES; p++)
                for (int i = 0; i < 256; i += 32) t = max_nan(t, fabs(product((p * warps + warp) * 256 + i + lane)));
#pragma unroll
            for (int s = 16; s >= 1; s >>= 1) t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, s));
            if (lane == 0) red_exact[warp] = t;
            __syncthreads();
            t = lane < warps ? red_exact[lane] : 0.0;
#pragma unroll
            for (int s = 16; s >= 1; s >>= 1) t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, s));
            for (int p = 0; p < PASSES; p++)
                for (int i = 0; i < 256; i += 32) store((p * warps + warp) * 256 + i + lane, t);
        }
    }
}

cudaError_t launch_norm_q8(const void *resid_in, int resid_dtype, const void *delta, int delta_dtype, const float *weight, int n, int H,
                           float eps, int group, void *resid_out, int q_dtype, void *q, float *scales, void *values, int values_dtype,
                           cudaStream_t s)
{
    count_launch();
    const bool wide = H % 8 == 0 && aligned16(resid_in) && aligned16(delta) && aligned16(weight) && aligned16(resid_out) &&
                      aligned16(values) && ((uintptr_t)q & 7) == 0;
    const int passes = H > 8192 ? 2 : 1;   // 1024 threads take 8192 elements at once
    const int threads = min(1024, ((H + 8 * passes - 1) / (8 * passes) + 31) / 32 * 32);
    return with_type(resid_dtype, [&](auto *rp) {
        return with_type(delta_dtype, [&](auto *dp) {
            return with_type(values_dtype, [&](auto *vp) {
                using RT = std::remove_pointer_t<decltype(rp)>;
                using DT = std::remove_pointer_t<decltype(dp)>;
                using VT = std::remove_pointer_t<decltype(vp)>;
                auto go = [&](auto *kern, int block) {
                    return launch_pdl(kern, dim3(n), dim3(block), 0, s, (const RT *)resid_in, (const DT *)delta, weight, H, eps, group,
                                      (RT *)resid_out, (uint8_t *)q, scales, (VT *)values);
                };
                const bool f8 = q_dtype == PMOE_F8_E4M3;
                if (wide)
                    return threads <= 256 ? go(f8 ? k_norm_q8<RT, DT, VT, true, 1, 256> : k_norm_q8<RT, DT, VT, false, 1, 256>, threads)
                           : passes == 1  ? go(f8 ? k_norm_q8<RT, DT, VT, true, 1, 1024> : k_norm_q8<RT, DT, VT, false, 1, 1024>, threads)
                                          : go(f8 ? k_norm_q8<RT, DT, VT, true, 2, 1024> : k_norm_q8<RT, DT, VT, false, 2, 1024>, threads);
                return go(f8 ? k_norm_q8_any<RT, DT, VT, true> : k_norm_q8_any<RT, DT, VT, false>, min(1024, (H + 255) / 256 * 32));
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
    const size_t values_n = (size_t)n * H, G = group ? ((size_t)H + group - 1) / group : 1;
    const Span in{resid_in, values_n * block_bytes(resid_dtype)}, more{delta, values_n * block_bytes(delta_dtype)}, stored{resid_out, in.bytes};
    if (overlap({{q, values_n}, {scales, n * G * sizeof(float)}, {values, values_n * block_bytes(values_dtype)}},
                {in, more, stored, {weight, (size_t)H * sizeof(float)}}) ||
        (resid_out != resid_in && stored.over(in)) || ((resid_out != delta || resid_dtype != delta_dtype) && stored.over(more)))
        return fail(PMOE_ERR_INVALID_ARG, "the outputs must not overlap the inputs (resid_out may be resid_in) or one another");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(PMOE_ERR_NO_DEVICE, "cannot select device %d", device);
    CU(launch_norm_q8(resid_in, resid_dtype, delta, delta ? delta_dtype : resid_dtype, weight, n, H, eps, group ? group : H, resid_out,
                      q_dtype, q, scales, values, values ? values_dtype : resid_dtype, (cudaStream_t)stream));
    return PMOE_OK;
}
