// train_common.cuh -- what the training kernels share: gates with both
// halves of a sigmoid, the 8-bit checkpoint format, a fixed-order column sum.
#pragma once

#include <cuda_fp8.h>

#include "scan_kernel.cuh"

namespace need {

// ------------------------------------------------------------------ gates
// s = sigmoid(x) and n = 1 - s = sigmoid(-x) of a pair, both with full relative
// precision: t = e^-x, s = 1 / (1 + t), n = t s.  16-bit streams use the
// hardware exp2 and reciprocal (about 1e-7 relative, against the 2^-9 and 2^-12
// of the rounding that follows); fp32 streams the library exp and IEEE division.
template <typename T>
__device__ __forceinline__ void sig_pair(float2 x, float2& s, float2& n) {
    if constexpr (Ops<T>::BYTES == 4) {
        const float t0 = expf(-fabsf(x.x)), t1 = expf(-fabsf(x.y));
        const float r0 = __fdiv_rn(1.0f, 1.0f + t0), r1 = __fdiv_rn(1.0f, 1.0f + t1);
        const float m0 = t0 * r0, m1 = t1 * r1;
        s = make_float2(x.x < 0.0f ? m0 : r0, x.y < 0.0f ? m1 : r1);
        n = make_float2(x.x < 0.0f ? r0 : m0, x.y < 0.0f ? r1 : m1);
    } else {
        // e^-x may overflow: s is then 0 -- not the least number, which times a value near
        // the type's largest is no zero -- and t s is not a number.  Below x = 0 the
        // difference is exact enough
        const float2 k = fmul2(x, splat2(-1.4426950408889634f));
        float t0, t1;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(k.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(k.y));
        const float2 d = fadd2(make_float2(t0, t1), splat2(1.0f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(d.x));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(d.y));
        const float2 m = fmul2(make_float2(t0, t1), s), c = fadd2(splat2(1.0f), make_float2(-s.x, -s.y));
        n = make_float2(k.x > 0.0f ? c.x : m.x, k.y > 0.0f ? c.y : m.y);
    }
}

// s and its slope s (1 - s) = t s^2 of a 16-bit pair.  Where e^-x overflows s is 0, and so
// is the slope: t is capped for it.  A NaN stays in s.
template <typename T>
__device__ __forceinline__ void sig_slope(float2 x, float2& s, float2& slope) {
    static_assert(Ops<T>::BYTES == 2, "fp32 streams keep their sigmoids");
    const float2 k = fmul2(x, splat2(-1.4426950408889634f));
    float t0, t1;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(k.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(k.y));
    const float2 d = fadd2(make_float2(t0, t1), splat2(1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(d.y));
    constexpr float top = 0x1p126f;
    slope = fmul2(fmul2(make_float2(fminf(t0, top), fminf(t1, top)), s), s);
}

// s alone (e^-x may overflow: s is then 0)
template <typename T>
__device__ __forceinline__ float2 sig_only(float2 x) {
    if constexpr (Ops<T>::BYTES == 4) {
        return make_float2(sigmoid_exact(x.x), sigmoid_exact(x.y));
    } else {
        return sig2<T>(x);
    }
}

// a = e^-r and n = 1 - a of a pair, 0 <= r <= 1/4: six terms of the series of
// 1 - e^-r (the seventh is r^6 / 5040 of it, 4.8e-8).
__device__ __forceinline__ void exp_neg_small(float2 r, float2& a, float2& n) {
    float2 q = ffma2(r, splat2(-1.0f / 720.0f), splat2(1.0f / 120.0f));
    q = ffma2(r, q, splat2(-1.0f / 24.0f));
    q = ffma2(r, q, splat2(1.0f / 6.0f));
    q = ffma2(r, q, splat2(-0.5f));
    q = ffma2(r, q, splat2(1.0f));
    n = fmul2(r, q);
    a = fadd2(splat2(1.0f), make_float2(-n.x, -n.y));
}

// The same for any r >= 0.  fp32: expm1.  16 bit: below 2^-4
// the first five terms of the series of 1 - e^-r (the next is r^5 / 720 of it,
// 1.3e-9), above it the difference (2^-24 / 2^-4 relative).
template <typename T>
__device__ __forceinline__ void exp_neg(float2 r, float2& a, float2& n) {
    if constexpr (Ops<T>::BYTES == 4) {
        a = make_float2(expf(-r.x), expf(-r.y));
        n = make_float2(-expm1f(-r.x), -expm1f(-r.y));
    } else {
        a = make_float2(exp_approx(-r.x), exp_approx(-r.y));
        float2 q = ffma2(r, splat2(1.0f / 120.0f), splat2(-1.0f / 24.0f));
        q = ffma2(r, q, splat2(1.0f / 6.0f));
        q = ffma2(r, q, splat2(-0.5f));
        q = ffma2(r, q, splat2(1.0f));
        q = fmul2(r, q);
        n = make_float2(r.x < 0.0625f ? q.x : 1.0f - a.x, r.y < 0.0625f ? q.y : 1.0f - a.y);
    }
}

// ------------------------------------------------------------------ 8 bits
// A group's scale is 2^e, e the least exponent >= -126 with every |value| <=
// 448 * 2^e (448: e4m3's largest), kept as the byte e + 127; 255 marks a group
// that holds an infinity or NaN and reads back as NaN.  `top` is the bit
// pattern of the group's largest magnitude.  A power of two scales without
// rounding, so a value is rounded once, by the conversion.
__device__ __forceinline__ uint32_t e4m3_scale_byte(uint32_t top) {
    const int b = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return top >= 0x7f800000u ? 255u : static_cast<uint32_t>(b < 1 ? 1 : b);
}
__device__ __forceinline__ float e4m3_scale(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}
__device__ __forceinline__ float e4m3_inverse(uint32_t byte) {  // 2^-e
    return __uint_as_float((254u - min(byte, 253u)) << 23);
}
__device__ __forceinline__ uint16_t e4m3_round(float2 x) {
    return __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint16_t e4m3_pair(float2 x, uint32_t byte) {
    return e4m3_round(fmul2(x, splat2(e4m3_inverse(byte))));
}

// ------------------------------------------------------------------ TMA
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* tm, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
        "l"(tm), "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(bar))
        : "memory");
}

// Its counterpart: shared -> global, rows and channels outside the tensor left
// out.  The shared bytes must have been fenced for the async proxy.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* tm, const void* src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(tm),
                 "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(src))
                 : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// This thread's committed stores have read their shared memory (which the CTA may then give up).
__device__ __forceinline__ void tma_store_drain() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// out[c] = sum over rows of part[row][c], in a fixed order (train_norm.cu).
int column_sums(const float* part, int64_t rows, int64_t C, float* out, cudaStream_t stream);

}  // namespace need
