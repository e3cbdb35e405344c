// Shared parts of the product in 8-bit integers: rows to 8 bits (int8_quantize.cu), few tokens (int8_rows.cu), many (int8_matmul.cu).
#pragma once

#include <math.h>

#include "common.cuh"
#include "launch.cuh"

static inline size_t katsu_int8_pitch(size_t k) { return (k + 15) / 16 * 16; }

// A row's scale, and what turns its values into whole numbers.
struct KatsuInt8Scale {
    float scale;         // largest magnitude / 127: what results are multiplied by
    float lift, s, inv;  // s = scale * lift, inv = 1 / s
    float half;          // s / 2; 0 where the quick way does not do: the scale is 0, no number, or lifted
};

__device__ __forceinline__ KatsuInt8Scale katsu_int8_scale(float largest) {
    KatsuInt8Scale q;
    q.scale = largest < INFINITY ? __fdiv_rn(largest, 127.f) : __int_as_float(0x7fffffff);  // (false for a NaN)
    // Scales near the end of the f32 range: everything times 2^64, exactly, so that 1 / s does not overflow.
    q.lift = q.scale < 0x1p-100f ? 0x1p64f : 1.f;
    q.s = q.scale * q.lift;
    q.inv = q.s > 0.f ? __fdiv_rn(1.f, q.s) : 0.f;
    q.half = q.s > 0.f && q.lift == 1.f ? 0.5f * q.s : 0.f;
    return q;
}

// v / scale to the nearest whole number, halves to the even one, of the exact quotient: a product with the rounded
// reciprocal is off by up to 2e-5 and would put values next to a border on its other side.  The remainder
// d = v - q scale decides instead, and is exact where that matters: for |v| >= scale it is a multiple of scale's last
// place, and 24 bits hold it up to |d| = scale; for smaller |v| q is 0 (d = v) or 1 (a difference within a factor of two).
__device__ __forceinline__ int katsu_int8_quotient(float v, const KatsuInt8Scale &q) {
    if (!(q.s > 0.f)) return 0;  // zeros only, or a scale that is no number
    const float t = v * q.lift;
    float n = rintf(t * q.inv);
    const float d = fmaf(-n, q.s, t), twice = fabsf(d) + fabsf(d);
    if (twice > q.s || (twice == q.s && (int(n) & 1))) n += copysignf(1.f, d);
    return int(fminf(fmaxf(n, -127.f), 127.f));
}

// Four values to four bytes by the definition.
__device__ __forceinline__ unsigned katsu_int8_pack_exactly(const float (&v)[4], const KatsuInt8Scale &q) {
    unsigned out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) out |= (unsigned(katsu_int8_quotient(v[i], q)) & 0xffu) << (8 * i);
    return out;
}

// The same almost always, the quick way: v / scale rounded by adding 1.5 * 2^23, whose last places are then the whole number.
// *sure turns false where a remainder is not below half a scale; the caller takes such pieces again, by the definition.  (With a
// rounding instruction and a comparison for each value the conversions, 16 a clock and SM, took twice the time of the loads.)
__device__ __forceinline__ unsigned katsu_int8_pack(const float (&v)[4], const KatsuInt8Scale &q, bool *sure) {
    constexpr float magic = 12582912.f;
    float n[4], most = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        n[i] = fmaf(v[i], q.inv, magic);
        most = fmaxf(most, fabsf(fmaf(magic - n[i], q.s, v[i])));
    }
    *sure = *sure && most < q.half;
    return __byte_perm(__byte_perm(__float_as_uint(n[0]), __float_as_uint(n[1]), 0x0040),
                       __byte_perm(__float_as_uint(n[2]), __float_as_uint(n[3]), 0x0040), 0x5410);
}

// The larger magnitude; a NaN wins.
__device__ __forceinline__ float katsu_larger(float a, float b) {
    float out;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(out) : "f"(a), "f"(fabsf(b)));
    return out;
}

__device__ __forceinline__ float katsu_larger4(float most, const float (&v)[4]) {
    return katsu_larger(katsu_larger(katsu_larger(katsu_larger(most, v[0]), v[1]), v[2]), v[3]);
}

// The same over a warp: no magnitude has the sign's bit, so they compare as integers, NaNs above an infinity.
__device__ __forceinline__ float katsu_larger_of_warp(float most) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
}

// A result from its sum: the roundings that the header counts.
__device__ __forceinline__ float katsu_int8_result(int sum, float xs, float ws, float bias) {
    return __fadd_rn(__fmul_rn(__fmul_rn(float(sum), xs), ws), bias);
}

// Rows of x -> 8 bits and scales.
int32_t katsu_int8_quantize(katsu_cuda_ctx *ctx, const float *x, int8_t *q, float *scale, size_t m, size_t k);

// Few tokens, on the CUDA cores: x (f32, quantised by the kernel) or xq and xs.  *handled = 0: not for these sizes.
int32_t katsu_int8_few(katsu_cuda_ctx *ctx, const float *x, const int8_t *xq, const float *xs, const int8_t *wq,
                       const float *ws, const float *bias, float *y, size_t m, size_t k, size_t n, int *handled);
