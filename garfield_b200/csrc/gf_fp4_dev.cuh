// Device code of the 4-bit block floating-point format (gf_fp4.h): codes and scales from elements and back.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <cmath>

#include "gf_device.cuh"
#include "gf_fp4.h"

namespace gf {
namespace fp4 {

constexpr uint32_t kOct = 8;  // elements that one thread quantises

// The format's kernels may start while the kernel before them on the stream still runs, and wait for its end
// before they touch memory: what overlaps is their launch and set-up.  The quantiser lets the next kernel
// start at once; the others leave that to their end.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// W bytes of elements.
template <typename T, uint32_t W>
struct alignas(W < 16 ? W : 16) Vec {
    T v[W / sizeof(T)];
};

// Eight codes from eight floats, element i in bits 4i .. 4i + 3 (nearest, ties to even, saturating).
__device__ __forceinline__ uint32_t e2m1x8(const float* x) {
    uint32_t r;
    asm("{\n .reg .b8 a, b, c, d;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n mov.b32 %0, {a, b, c, d};\n}\n"
        : "=r"(r)
        : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
    return r;
}
// Two floats from a byte of two codes.
__device__ __forceinline__ float2 e2m1x2_to_f32(uint32_t b) {
    uint32_t h;
    asm("{\n .reg .b8 b;\n cvt.u8.u32 b, %1;\n cvt.rn.f16x2.e2m1x2 %0, b;\n}\n" : "=r"(h) : "r"(b));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}
__device__ __forceinline__ float scale_to_f32(uint32_t b, bool block16) {
    if (block16) return e4m3_to_f32(b);
    // E8M0: 2^(b - 127); 0 stands for 2^-127 (half the smallest normal float), 255 for NaN
    return __uint_as_float(b == 255u ? 0x7FC00000u : (b == 0u ? 0x00400000u : b << 23));
}

// max(a, b) of magnitudes, NaN if either is.
__device__ __forceinline__ float amax2(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// max(|a|, |b|, |c|), NaN if one is.
__device__ __forceinline__ float amax3(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Largest magnitude of eight elements, NaN if one is.
__device__ __forceinline__ float amax8(const float* x) {
    return amax2(amax3(amax3(x[0], x[1], x[2]), x[6], x[7]), amax3(x[3], x[4], x[5]));
}
// A quotient by a number y is held as x hi + x lo, hi + lo being 1 / y within 2^-41 of it and lo >= 0 (so that -0
// stays -0).  Where x / y is a boundary between codes the sum rounds to it.  Where it is not, it is more than half
// a last place away from it, by 1/32 of one at least (y and a boundary have few bits), which is far more than
// this sum errs by before it is rounded.  (Results too small for that are far below the first boundary.)
__device__ __forceinline__ float times(float x, float hi, float lo) { return __fmaf_rn(x, hi, __fmul_rn(x, lo)); }
// hi and lo for the finite E4M3 values s > 0: the hardware's approximation, which errs by a last place, taken four
// down, and what is missing.
__device__ __forceinline__ float rcp_e4m3(float s, float& lo) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    r = __uint_as_float(__float_as_uint(r) - 4u);
    lo = __fmul_rn(r, __fmaf_rn(-s, r, 1.0f));
    return r;
}

// Whether multiplying by alpha can be left to the multiplication by the block's factor: scaling by a power
// of two commutes with rounding, and in blocks of 32 the factor is one; in blocks of 16 alpha has to be.
// (Far from the ends of fp32's range, where rounding does not commute; encode8 looks after small blocks.)
inline bool fold_alpha(float alpha, uint32_t block) {
    int e = 0;
    return alpha >= 0x1p-30f && alpha <= 0x1p30f && (block == 32 || std::frexp(alpha, &e) == 0.5f);
}

// Scale byte of a block and the codes of this thread's eight elements x, which are to be multiplied by alpha.
// amax: the block's largest magnitude after that multiplication (rounding keeps order: the largest product is
// the largest element's).  FOLD: fold_alpha.
template <uint32_t BLOCK, bool FOLD>
__device__ __forceinline__ uint32_t encode8(float* x, float amax, float alpha, uint32_t& codes) {
    const uint32_t ef = __float_as_uint(amax) >> 23;
    float f = 1.0f;  // what the elements still have to be multiplied by
    if (!FOLD) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], alpha);
    } else {
        f = alpha;
        if (ef < 64u) {  // products may be subnormal, and rounded as such
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], alpha);
            f = 1.0f;
        }
    }
    uint32_t s8;
    if (BLOCK == 32) {
        s8 = ef == 255u ? 255u : max(ef, 2u) - 2u;
        f = __fmul_rn(f, __uint_as_float((254u - min(s8, 253u)) << 23));  // f / s, s a power of two
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const dev::f2x y = dev::mul2(dev::pack2(x[e], x[e + 1]), dev::pack2(f, f));
            x[e] = dev::lo2(y);
            x[e + 1] = dev::hi2(y);
        }
    } else {
        constexpr float kHi = 0x1.555554p-3f, kLo = (float)(1.0 / 6.0 - (double)kHi);
        s8 = ef == 255u ? 0x7Fu : (uint32_t)__nv_cvt_float_to_fp8(times(amax, kHi, kLo), __NV_SATFINITE, __NV_E4M3);
        float lo;
        const float hi = __fmul_rn(rcp_e4m3(e4m3_to_f32(s8), lo), f);
        lo = __fmul_rn(lo, f);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {  // times, two at a time
            const dev::f2x v = dev::pack2(x[e], x[e + 1]);
            const dev::f2x y = dev::fma2(v, dev::pack2(hi, hi), dev::mul2(v, dev::pack2(lo, lo)));
            x[e] = dev::lo2(y);
            x[e + 1] = dev::hi2(y);
        }
    }
    codes = ef == 255u || (BLOCK == 16 && s8 == 0u) ? 0u : e2m1x8(x);
    return s8;
}

// Launch attribute of a kernel that begins with wait_for_previous.
inline cudaLaunchAttribute early_start() {
    cudaLaunchAttribute a = {};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    return a;
}

}  // namespace fp4
}  // namespace gf
