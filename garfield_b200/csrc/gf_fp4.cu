// 4-bit block floating point: a row codec beside the byte codecs of gf_codec.cu.
//
// A row is cut into blocks of 32 or 16 consecutive elements.  With x = data * alpha and
// amax = max |x| over the block, the block's scale s and the elements' codes c are
//   block 32:  s = 2^(floor(log2 amax) - 2), exponent at least -127, held as E8M0 (bias 127)
//   block 16:  s = amax / 6 rounded to E4M3 (nearest, ties to even, at most 448)
//   c = x / s rounded to E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives): nearest, ties to
//       the even code, at most 6 in size; 0 where s = 0
// and the element is held as c * s / alpha.  Block 32 scales with one subtraction on the
// float's exponent field and its division is exact; the largest elements of a block (above 6 s,
// when amax is in the upper quarter of its binade) saturate.  Block 16 spends twice the scale
// bytes and keeps every element within half a code step, as long as amax / 6 stays inside E4M3's
// range [2^-9, 448]: alpha moves the data there.  A block holding an infinity or a NaN (after
// the multiplication by alpha) gets a NaN scale (0xFF, 0x7F) and codes 0, so what is read back
// and every product with it is NaN.
//
// x / s is an IEEE division before the rounding to a code, and that double rounding is harmless:
// s has at most 4 significant bits and a code boundary at most 3, so x either equals
// boundary * s or differs from it by at least 2^-24 of its value, which the fp32 quotient keeps.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "gf_device.cuh"
#include "gf_fp4.h"

namespace gf {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kColPitch = kFp4ColBytes + 16;  // shared-memory columns, one bank quad apart

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// Four consecutive elements in one load or store.
template <typename T>
struct alignas(sizeof(T) * 4) Quad {
    T v[4];
};

// Two codes from two floats: lo in bits 0-3, hi in bits 4-7 (nearest, ties to even, saturating).
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n .reg .b8 b;\n cvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n cvt.u32.u8 %0, b;\n}\n" : "=r"(r) : "f"(hi), "f"(lo));
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

// Scale byte of a block from the bits of amax, and the codes of this lane's four elements.
template <uint32_t BLOCK>
__device__ __forceinline__ uint32_t encode4(const float* x, float amax, uint32_t& codes) {
    const uint32_t ef = __float_as_uint(amax) >> 23;
    if (BLOCK == 32) {
        const uint32_t s8 = ef == 255u ? 255u : (ef >= 2u ? ef - 2u : 0u);
        if (ef == 255u) {
            codes = 0;
            return s8;
        }
        const float inv = __uint_as_float((254u - s8) << 23);  // 1 / s, a power of two
        codes = e2m1x2(x[0] * inv, x[1] * inv) | e2m1x2(x[2] * inv, x[3] * inv) << 8;
        return s8;
    }
    const uint32_t s8 = ef == 255u ? 0x7Fu : (uint32_t)__nv_cvt_float_to_fp8(__fdiv_rn(amax, 6.0f), __NV_SATFINITE, __NV_E4M3);
    if (ef == 255u || s8 == 0u) {
        codes = 0;
        return s8;
    }
    const float s = e4m3_to_f32(s8);
    codes = e2m1x2(__fdiv_rn(x[0], s), __fdiv_rn(x[1], s)) | e2m1x2(__fdiv_rn(x[2], s), __fdiv_rn(x[3], s)) << 8;
    return s8;
}

// One group of one panel per block step.  A warp takes a row's 128 elements, four to a lane, so
// its load is one contiguous run of 512 (fp32) or 256 bytes; the block maximum is a butterfly over the
// 8 or 4 lanes of the block; codes and scales gather in shared memory in the panel's order and
// leave as 16-byte pieces.  VEC: rows start on a four-element boundary and dim % 4 == 0.
template <typename T, uint32_t BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(const T* __restrict__ data, uint64_t ld, uint32_t n,
                                                                uint32_t dim, float alpha, uint8_t* __restrict__ packed,
                                                                Fp4Layout Lo, uint64_t tiles) {
    constexpr uint32_t kSb = kFp4Group / BLOCK * kFp4Rows;  // scale bytes of a group
    constexpr int U = 8;                                    // rows in flight per warp
    __shared__ __align__(16) uint8_t codes_s[4 * kColPitch];
    __shared__ __align__(16) uint8_t scales_s[kSb];
    const uint32_t lane = dev::lane_id(), warp = threadIdx.x >> 5;
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t p = (uint32_t)(t / Lo.groups), g = (uint32_t)(t % Lo.groups);
        const uint32_t row0 = p * kFp4Rows, valid = min(kFp4Rows, n - row0);
        const uint32_t cols = min(4u, Lo.cols - 4 * g);
        const uint32_t k = g * kFp4Group + lane * 4;
        for (uint32_t r0 = warp; r0 < valid; r0 += kWarps * U) {
            float x[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t r = r0 + u * kWarps;
                const T* src = data + (uint64_t)(row0 + r) * ld + k;
                if (VEC) {
                    Quad<T> q = {};
                    if (r < valid && k < dim) q = *reinterpret_cast<const Quad<T>*>(src);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[u][e] = __fmul_rn(to_f32(q.v[e]), alpha);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[u][e] = r < valid && k + e < dim ? __fmul_rn(to_f32(src[e]), alpha) : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t r = r0 + u * kWarps;
                // the bits of |x| order like |x|, with NaN above infinity: an integer maximum
                // sees every non-finite element
                uint32_t mb = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) mb = max(mb, __float_as_uint(x[u][e]) & 0x7FFFFFFFu);
#pragma unroll
                for (int o = BLOCK / 8; o > 0; o >>= 1) mb = max(mb, __shfl_xor_sync(dev::kFull, mb, o));
                uint32_t c;
                const uint32_t s8 = encode4<BLOCK>(x[u], __uint_as_float(mb), c);
                if (r < valid) {
                    *reinterpret_cast<uint16_t*>(codes_s + (lane >> 3) * kColPitch + r * 16 + (lane & 7u) * 2) = (uint16_t)c;
                    if (lane % (BLOCK / 4) == 0) scales_s[fp4_scale_at(r, lane / (BLOCK / 4))] = (uint8_t)s8;
                }
            }
        }
        __syncthreads();
        uint32_t* dst_s = reinterpret_cast<uint32_t*>(packed + Lo.scales_at(p, g));
        uint8_t* dst = packed + Lo.col_at(p, 4 * g);
        for (uint32_t i = threadIdx.x; i < kSb / 4; i += kThreads) {
            const uint32_t r = (i & 3u) * 32 + ((i >> 2) & 31u);
            if (r < valid) dst_s[i] = reinterpret_cast<const uint32_t*>(scales_s)[i];
        }
        for (uint32_t i = threadIdx.x; i < cols * kFp4Rows; i += kThreads) {
            const uint32_t c = i / kFp4Rows, r = i % kFp4Rows;
            if (r < valid)
                *reinterpret_cast<uint4*>(dst + c * Lo.col_bytes + r * 16) =
                    *reinterpret_cast<const uint4*>(codes_s + c * kColPitch + r * 16);
        }
        __syncthreads();
    }
}

// The reverse: a group's bytes come in as 16-byte pieces, a warp writes a row's 128 elements.
// The scale is divided by alpha once per block (rounded), and the code times it rounded again: with
// a power of two as alpha both are exact in fp32, otherwise a value is within 2^-23 of
// c * s / alpha.
template <typename T, uint32_t BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ packed, uint32_t n,
                                                                  uint32_t dim, float alpha, T* __restrict__ out,
                                                                  uint64_t ld, Fp4Layout Lo, uint64_t tiles) {
    constexpr uint32_t kSb = kFp4Group / BLOCK * kFp4Rows;
    __shared__ __align__(16) uint8_t codes_s[4 * kColPitch];
    __shared__ __align__(16) uint8_t scales_s[kSb];
    const uint32_t lane = dev::lane_id(), warp = threadIdx.x >> 5;
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t p = (uint32_t)(t / Lo.groups), g = (uint32_t)(t % Lo.groups);
        const uint32_t row0 = p * kFp4Rows, valid = min(kFp4Rows, n - row0);
        const uint32_t cols = min(4u, Lo.cols - 4 * g);
        const uint32_t k = g * kFp4Group + lane * 4;
        const uint4* src_s = reinterpret_cast<const uint4*>(packed + Lo.scales_at(p, g));
        const uint8_t* src = packed + Lo.col_at(p, 4 * g);
        for (uint32_t i = threadIdx.x; i < kSb / 16; i += kThreads) reinterpret_cast<uint4*>(scales_s)[i] = src_s[i];
        for (uint32_t i = threadIdx.x; i < cols * kFp4Rows; i += kThreads) {
            const uint32_t c = i / kFp4Rows, r = i % kFp4Rows;
            if (r < valid)
                *reinterpret_cast<uint4*>(codes_s + c * kColPitch + r * 16) =
                    *reinterpret_cast<const uint4*>(src + c * Lo.col_bytes + r * 16);
        }
        __syncthreads();
        if (k < dim) {
#pragma unroll 4
            for (uint32_t r = warp; r < valid; r += kWarps) {
                const uint32_t c = *reinterpret_cast<const uint16_t*>(codes_s + (lane >> 3) * kColPitch + r * 16 + (lane & 7u) * 2);
                const float s = __fdiv_rn(scale_to_f32(scales_s[fp4_scale_at(r, lane / (BLOCK / 4))], BLOCK == 16), alpha);
                const float2 a = e2m1x2_to_f32(c & 255u), b = e2m1x2_to_f32(c >> 8);
                Quad<T> q;
                from_f32(__fmul_rn(a.x, s), q.v[0]);
                from_f32(__fmul_rn(a.y, s), q.v[1]);
                from_f32(__fmul_rn(b.x, s), q.v[2]);
                from_f32(__fmul_rn(b.y, s), q.v[3]);
                T* dst = out + (uint64_t)(row0 + r) * ld + k;
                if (VEC) {
                    *reinterpret_cast<Quad<T>*>(dst) = q;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k + e < dim) dst[e] = q.v[e];
                }
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ host form

constexpr float kMags[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};

uint32_t e2m1_host(float y) {
    const uint32_t sign = std::signbit(y) ? 8u : 0u;
    const float a = std::fabs(y);
    // boundaries between neighbouring codes; a tie goes to the even code
    const bool up[7] = {a > 0.25f, a >= 0.75f, a > 1.25f, a >= 1.75f, a > 2.5f, a >= 3.5f, a > 5.0f};
    uint32_t c = 0;
    for (bool u : up) c += u;
    return sign | c;
}
float e4m3_host(uint32_t b) {
    const uint32_t e = (b >> 3) & 15u, m = b & 7u;
    if (e == 15u && m == 7u) return std::nanf("");
    return e ? std::ldexp(1.0f + (float)m / 8.0f, (int)e - 7) : std::ldexp((float)m / 8.0f, -6);
}
uint32_t to_e4m3_host(float t) {  // t >= 0, finite
    if (t >= 448.0f) return 0x7Eu;
    int e = 0;
    std::frexp(std::max(t, 0x1p-6f), &e);       // t in [2^(e-1), 2^e), or below the normals
    const float step = std::ldexp(1.0f, e - 4);  // 8 steps to a binade
    const float q = std::nearbyint(t / step);    // exact division by a power of two; ties to even
    return (uint32_t)((e + 5) * 8 + (int)q);     // q = 8 .. 16 (16 carries into the exponent; below 8: subnormals)
}
float scale_host(uint32_t b, uint32_t block) {
    if (block == 16) return e4m3_host(b);
    return b == 255u ? std::nanf("") : std::ldexp(1.0f, (int)b - 127);
}

void quantize_host(const float* data, uint32_t n, uint32_t dim, float alpha, uint32_t block, uint8_t* packed) {
    const Fp4Layout Lo = fp4_layout(n, dim, block);
    std::memset(packed, 0, Lo.panel_bytes * fp4_panels(n));
    for (uint32_t i = 0; i < n; ++i)
        for (uint32_t k0 = 0; k0 < dim; k0 += block) {
            const uint32_t k1 = std::min(dim, k0 + block), r = i % kFp4Rows;
            const float* x = data + (uint64_t)i * dim;
            float amax = 0.0f;
            bool bad = false;
            for (uint32_t k = k0; k < k1; ++k) {
                const float v = std::fabs(x[k] * alpha);
                bad |= !std::isfinite(v);
                amax = std::fmax(amax, v);
            }
            uint32_t s8;
            if (bad) {
                s8 = block == 16 ? 0x7Fu : 0xFFu;
            } else if (block == 16) {
                s8 = to_e4m3_host(amax / 6.0f);
            } else {
                int e = 0;
                std::frexp(amax, &e);  // amax in [2^(e-1), 2^e)
                s8 = amax > 0.0f ? (uint32_t)std::max(e - 3 + 127, 0) : 0u;
            }
            packed[Lo.scales_at(i / kFp4Rows, k0 / kFp4Group) + fp4_scale_at(r, (k0 % kFp4Group) / block)] = (uint8_t)s8;
            if (bad || (block == 16 && s8 == 0)) continue;
            const float s = scale_host(s8, block);
            for (uint32_t k = k0; k < k1; ++k) {
                // block 32: multiplied by 1 / s, a power of two that fp32 holds for every s
                const float y = block == 16 ? x[k] * alpha / s : std::ldexp(x[k] * alpha, 127 - (int)s8);
                uint8_t* b = packed + Lo.col_at(i / kFp4Rows, k / kFp4Col) + r * 16 + (k % kFp4Col) / 2;
                *b = (uint8_t)(*b | e2m1_host(y) << (4 * (k & 1u)));
            }
        }
}

void dequantize_host(const uint8_t* packed, uint32_t n, uint32_t dim, uint32_t block, float alpha, float* out) {
    const Fp4Layout Lo = fp4_layout(n, dim, block);
    for (uint32_t i = 0; i < n; ++i)
        for (uint32_t k = 0; k < dim; ++k) {
            const uint32_t r = i % kFp4Rows, p = i / kFp4Rows;
            const uint32_t c = (packed[Lo.col_at(p, k / kFp4Col) + r * 16 + (k % kFp4Col) / 2] >> (4 * (k & 1u))) & 15u;
            const uint32_t s8 = packed[Lo.scales_at(p, k / kFp4Group) + fp4_scale_at(r, k % kFp4Group / block)];
            const float s = scale_host(s8, block) / alpha;
            out[(uint64_t)i * dim + k] = (c & 8u ? -kMags[c & 7u] : kMags[c & 7u]) * s;
        }
}

// ------------------------------------------------------------------ launches

bool good_alpha(float alpha) { return std::isfinite(alpha) && alpha > 0.0f; }

unsigned grid_of(uint64_t tiles) { return (unsigned)std::min<uint64_t>(tiles, 0x7FFFFFFFu); }

template <typename T, uint32_t BLOCK>
void launch_quantize(const void* data, uint64_t ld, uint32_t n, uint32_t dim, float alpha, uint8_t* packed, cudaStream_t s) {
    const Fp4Layout Lo = fp4_layout(n, dim, BLOCK);
    const uint64_t tiles = (uint64_t)fp4_panels(n) * Lo.groups;
    const T* x = static_cast<const T*>(data);
    if (aligned(data, 4 * sizeof(T)) && ld % 4 == 0 && dim % 4 == 0)
        fp4_quantize_kernel<T, BLOCK, true><<<grid_of(tiles), kThreads, 0, s>>>(x, ld, n, dim, alpha, packed, Lo, tiles);
    else
        fp4_quantize_kernel<T, BLOCK, false><<<grid_of(tiles), kThreads, 0, s>>>(x, ld, n, dim, alpha, packed, Lo, tiles);
}
template <typename T, uint32_t BLOCK>
void launch_dequantize(const uint8_t* packed, uint32_t n, uint32_t dim, float alpha, void* out, uint64_t ld, cudaStream_t s) {
    const Fp4Layout Lo = fp4_layout(n, dim, BLOCK);
    const uint64_t tiles = (uint64_t)fp4_panels(n) * Lo.groups;
    T* y = static_cast<T*>(out);
    if (aligned(out, 4 * sizeof(T)) && ld % 4 == 0 && dim % 4 == 0)
        fp4_dequantize_kernel<T, BLOCK, true><<<grid_of(tiles), kThreads, 0, s>>>(packed, n, dim, alpha, y, ld, Lo, tiles);
    else
        fp4_dequantize_kernel<T, BLOCK, false><<<grid_of(tiles), kThreads, 0, s>>>(packed, n, dim, alpha, y, ld, Lo, tiles);
}

}  // namespace

}  // namespace gf

using namespace gf;

extern "C" uint64_t gf_fp4_bytes(uint32_t n, uint32_t dim, uint32_t block) {
    if (!fp4_shape(dim, block)) return 0;
    return fp4_layout(n, dim, block).panel_bytes * fp4_panels(n);
}

extern "C" gf_status gf_quantize_fp4(const void* data, uint32_t dtype, uint64_t ld, uint32_t n, uint32_t dim, float alpha,
                                     uint32_t block, void* packed_out, void* stream) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!dtype_bytes(dtype)) return fail(GF_ERR_ARG, "unknown dtype");
    if (!good_alpha(alpha)) return fail(GF_ERR_ARG, "alpha must be positive and finite");
    if (ld < dim) return fail(GF_ERR_ARG, "row stride below dim");
    if (n == 0) return GF_OK;
    if (!data || !packed_out) return fail(GF_ERR_ARG, "null argument");
    if (!aligned(data, dtype_bytes(dtype)) || !aligned(packed_out, 16)) return fail(GF_ERR_ARG, "misaligned pointer");
    cudaStream_t s = (cudaStream_t)stream;
    uint8_t* out = static_cast<uint8_t*>(packed_out);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (block == 16)
            launch_quantize<T, 16>(data, ld, n, dim, alpha, out, s);
        else
            launch_quantize<T, 32>(data, ld, n, dim, alpha, out, s);
    };
    if (dtype == GF_F32)
        go(float{});
    else if (dtype == GF_F16)
        go(__half{});
    else
        go(__nv_bfloat16{});
    GF_CUDA(cudaGetLastError());
    return GF_OK;
}

extern "C" gf_status gf_dequantize_fp4(const void* packed, uint32_t n, uint32_t dim, uint32_t block, float alpha, void* out,
                                       uint32_t dtype, uint64_t ld, void* stream) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!dtype_bytes(dtype)) return fail(GF_ERR_ARG, "unknown dtype");
    if (!good_alpha(alpha)) return fail(GF_ERR_ARG, "alpha must be positive and finite");
    if (ld < dim) return fail(GF_ERR_ARG, "row stride below dim");
    if (n == 0) return GF_OK;
    if (!packed || !out) return fail(GF_ERR_ARG, "null argument");
    if (!aligned(out, dtype_bytes(dtype)) || !aligned(packed, 16)) return fail(GF_ERR_ARG, "misaligned pointer");
    cudaStream_t s = (cudaStream_t)stream;
    const uint8_t* in = static_cast<const uint8_t*>(packed);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (block == 16)
            launch_dequantize<T, 16>(in, n, dim, alpha, out, ld, s);
        else
            launch_dequantize<T, 32>(in, n, dim, alpha, out, ld, s);
    };
    if (dtype == GF_F32)
        go(float{});
    else if (dtype == GF_F16)
        go(__half{});
    else
        go(__nv_bfloat16{});
    GF_CUDA(cudaGetLastError());
    return GF_OK;
}

extern "C" gf_status gf_quantize_fp4_host(const float* data, uint32_t n, uint32_t dim, float alpha, uint32_t block,
                                          void* packed_out) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!good_alpha(alpha)) return fail(GF_ERR_ARG, "alpha must be positive and finite");
    if (n == 0) return GF_OK;
    if (!data || !packed_out) return fail(GF_ERR_ARG, "null argument");
    quantize_host(data, n, dim, alpha, block, static_cast<uint8_t*>(packed_out));
    return GF_OK;
}

extern "C" gf_status gf_dequantize_fp4_host(const void* packed, uint32_t n, uint32_t dim, uint32_t block, float alpha,
                                            float* out) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!good_alpha(alpha)) return fail(GF_ERR_ARG, "alpha must be positive and finite");
    if (n == 0) return GF_OK;
    if (!packed || !out) return fail(GF_ERR_ARG, "null argument");
    dequantize_host(static_cast<const uint8_t*>(packed), n, dim, block, alpha, out);
    return GF_OK;
}
