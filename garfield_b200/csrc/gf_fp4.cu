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
// x / s is rounded to fp32 before it is rounded to a code, and that double rounding is harmless: s
// has at most 4 significant bits and a code boundary at most 3, so x either equals boundary * s or
// differs from it by at least 2^-24 of its value, which the fp32 quotient keeps.
//
// Both directions move 2.5 to 4.5 bytes an element, which leaves some 15 to 27 instructions for one at the
// HBM rate.  The quantiser's threads take eight consecutive elements: one to four loads, one
// 4-byte word of codes, and the block maximum in two shuffles (one for blocks of 16).  Four
// neighbouring lanes hold a row's column of 32 elements and the next lanes the next row, so a warp's
// codes fill whole 32-byte sectors of the panel.  The reader's threads take what one store
// holds (16 bytes, or 8, as the rows are aligned; else four elements), so a warp's stores leave no sector
// half written.  A CTA is short (one group of a panel); four to six of them on an SM overlap their loads and arithmetic.
// Rows in flight per thread: 16-bit data 2, with 6 CTAs on an SM (4 rows and the 4 CTAs that their registers
// allow win and lose: bf16 1M x 128 57 us against 61, bf16 8192 x 8192 in blocks of 16 35 against 37, fp16 1M x 128
// in blocks of 16 62 against 57; 1 row and 8 CTAs: 64, 39 and 66), fp32 4 (1M x 128: 83 us against 86, in blocks of
// 16 84 against 92), but 2 where short rows leave a thread few (1M x 16: 18 us against 22, 1M x 33 36 against 37).
// fp32 1M x 128 moves 7.0 TB/s both ways (part of it in L2); 16-bit data are bound by instructions as much
// as by bytes: bf16 1M x 128 5.7 TB/s, 8192 x 8192 in blocks of 16 5.0.
#include <algorithm>
#include <type_traits>
#include <cmath>
#include <cstring>

#include "gf_fp4_dev.cuh"

namespace gf {
namespace {

using namespace fp4;

constexpr uint32_t kThreads = 256;
constexpr float kNormal = 0x1p-126f;  // the smallest normal fp32 number

// Lanes of a row, as a power of two: enough for `cols` columns at `per` lanes each (per a power of two).
__device__ __forceinline__ uint32_t row_shift(uint32_t cols, uint32_t per) {
    return 31u - __clz(per) + (cols > 2 ? 2u : cols - 1u);
}

// One group of one panel.  W: bytes of a load, which rows are aligned to; kRows: rows in flight per thread.
template <typename T, uint32_t BLOCK, uint32_t W, bool FOLD, uint32_t kRows>
__global__ void __launch_bounds__(kThreads, kRows == 4 ? 4 : 6)
    fp4_quantize_kernel(const T* __restrict__ data, uint64_t ld, uint32_t n, uint32_t dim, float alpha,
                        uint8_t* __restrict__ packed, Fp4Layout Lo) {
    constexpr uint32_t kSb = kFp4Group / BLOCK * kFp4Rows;  // scale bytes of a group
    constexpr uint32_t kV = W / sizeof(T);                  // elements of a load
    constexpr uint32_t kBo = BLOCK / kOct;                  // threads of a block
    constexpr uint32_t kB = kFp4Group / BLOCK;              // blocks of a row's group
    __shared__ __align__(16) uint8_t scales_s[kSb];         // [row][block]
    const uint32_t p = blockIdx.x;
    wait_for_previous();
    let_next_start();
    for (uint32_t g = blockIdx.y; g < Lo.groups; g += gridDim.y) {
        const uint32_t row0 = p * kFp4Rows, valid = min(kFp4Rows, n - row0);
        const uint32_t cols = min(4u, Lo.cols - 4 * g), lsh = row_shift(cols, 4);
        const uint32_t o = threadIdx.x & ((1u << lsh) - 1u), rstep = kThreads >> lsh;
        const uint32_t k = g * kFp4Group + o * kOct, first = threadIdx.x >> lsh;
        const uint32_t left = k < dim ? dim - k : 0u;  // elements of the row from k on
        const T* src = data + (uint64_t)(row0 + first) * ld + k;
        const uint64_t step = ld * rstep;
        uint8_t* dst = packed + Lo.col_at(p, 4 * g + (o >> 2)) + (o & 3u) * 4;
        // scales of blocks in columns that the group lacks are 0
        if (cols < 4)
            for (uint32_t i = threadIdx.x; i < kSb; i += kThreads)
                if (i % kB * BLOCK >= cols * kFp4Col) scales_s[i] = 0;
        typedef Vec<T, W> Oct[kOct / kV];
        auto encode = [&](const Oct& q, uint32_t r, bool in) {
            float x[kOct];
#pragma unroll
            for (uint32_t e = 0; e < kOct; ++e) x[e] = to_f32(q[e / kV].v[e % kV]);
            float mx = __fmul_rn(amax8(x), alpha);
            if (BLOCK == 32) mx = amax2(mx, __shfl_xor_sync(dev::kFull, mx, 2));
            mx = amax2(mx, __shfl_xor_sync(dev::kFull, mx, 1));
            uint32_t c;
            const uint32_t s8 = encode8<BLOCK, FOLD>(x, mx, alpha, c);
            if (in) {
                *reinterpret_cast<uint32_t*>(dst + r * 16) = c;
                if (o % kBo == 0) scales_s[r * kB + o / kBo] = (uint8_t)s8;  // (0 for a block past the row's end)
            }
        };
        if (valid == kFp4Rows && dim % kV == 0) {  // a load's elements all exist or none does, the same in every row
            for (uint32_t r0 = 0; r0 < kFp4Rows; r0 += rstep * kRows) {
                Oct q[kRows] = {};
                // (short rows step by up to half a panel, of which two fit)
                auto there = [&](uint32_t u) { return u < 2 || r0 + u * rstep < kFp4Rows; };
#pragma unroll
                for (uint32_t u = 0; u < kRows; ++u)
#pragma unroll
                    for (uint32_t w = 0; w < kOct / kV; ++w)
                        if (there(u) && left > w * kV) q[u][w] = *reinterpret_cast<const Vec<T, W>*>(src + u * step + w * kV);
                src += step * kRows;
#pragma unroll
                for (uint32_t u = 0; u < kRows; ++u)
                    if (there(u)) encode(q[u], r0 + first + u * rstep, o < 4 * cols);
            }
        } else {
            for (uint32_t r0 = 0; r0 < valid; r0 += rstep, src += step) {
                const uint32_t r = r0 + first;
                Oct q = {};
                if (r < valid && left >= kOct) {
#pragma unroll
                    for (uint32_t w = 0; w < kOct / kV; ++w) q[w] = *reinterpret_cast<const Vec<T, W>*>(src + w * kV);
                } else if (r < valid) {
#pragma unroll
                    for (uint32_t e = 0; e < kOct; ++e)
                        if (e < left) q[e / kV].v[e % kV] = src[e];
                }
                encode(q, r, r < valid && o < 4 * cols);
            }
        }
        __syncthreads();
        uint32_t* dst_s = reinterpret_cast<uint32_t*>(packed + Lo.scales_at(p, g));
        for (uint32_t i = threadIdx.x; i < kSb / 4; i += kThreads) {
            const uint32_t r = (i & 3u) * 32 + ((i >> 2) & 31u);  // the inverse of fp4_scale_at, four blocks at a time
            if (r < valid) dst_s[i] = reinterpret_cast<const uint32_t*>(scales_s)[r * (kB / 4) + (i >> 7)];
        }
        __syncthreads();
    }
}

// The reverse.  W: bytes of a store.  inv is 1 / alpha rounded; the scale is multiplied by it once
// per thread and the code times that rounded again: with a power of two as alpha all is exact in
// fp32, otherwise a value is within 3 * 2^-24 of c * s / alpha.  Where s * inv is below fp32's normal numbers it
// keeps fewer bits, or none while 6 s inv has some left: there c * s, which is exact, is multiplied by inv.  A
// value below the normal numbers is off by another half of the smallest number at most, unless fp32 holds it.
// SMALL: whether that can happen.  In blocks of 32 it can (1M x 96 to fp16 46.5 us without this, 44.4 with it, 1M x 33
// 36.7 and 37.7, 1M x 128 to fp32 93.0 both; a branch takes 47.7 and 42.4); blocks of 16 have scales of 2^-9
// and more, so only an alpha above 2^117 brings it about (1M x 128 to bf16 51.7 us without, 58.8 with it).
template <typename T, uint32_t BLOCK, uint32_t W, bool SMALL>
__global__ void __launch_bounds__(kThreads, 6) fp4_dequantize_kernel(const uint8_t* __restrict__ packed, uint32_t n,
                                                                  uint32_t dim, float inv, T* __restrict__ out,
                                                                  uint64_t ld, Fp4Layout Lo) {
    constexpr uint32_t kV = W > sizeof(T) ? W / sizeof(T) : 4;  // elements of a thread: 2, 4 or 8
    constexpr uint32_t kCb = kV / 2;                            // their bytes of codes
    constexpr uint32_t kRows = 4;                               // rows in flight per thread
    const uint32_t p = blockIdx.x;
    wait_for_previous();
    for (uint32_t g = blockIdx.y; g < Lo.groups; g += gridDim.y) {
        const uint32_t row0 = p * kFp4Rows, valid = min(kFp4Rows, n - row0);
        const uint32_t lsh = row_shift(min(4u, Lo.cols - 4 * g), kFp4Col / kV);
        const uint32_t k0 = (threadIdx.x & ((1u << lsh) - 1u)) * kV, rstep = kThreads >> lsh;  // element of the group
        const uint32_t k = g * kFp4Group + k0;
        if (k >= dim) continue;
        const uint32_t left = dim - k;
        const uint8_t* src = packed + Lo.col_at(p, 4 * g + k0 / kFp4Col) + k0 % kFp4Col / 2;
        const uint8_t* src_s = packed + Lo.scales_at(p, g);
        uint32_t r = threadIdx.x >> lsh;
        T* dst = out + (uint64_t)(row0 + r) * ld + k;
        const uint64_t step = ld * rstep;
        auto codes_of = [&](uint32_t i) -> uint32_t {
            return kCb == 4   ? *reinterpret_cast<const uint32_t*>(src + i * 16)
                   : kCb == 2 ? *reinterpret_cast<const uint16_t*>(src + i * 16)
                              : src[i * 16];
        };
        auto write = [&](uint32_t c, uint32_t s8, bool whole) {
            const float held = scale_to_f32(s8, BLOCK == 16), both = __fmul_rn(held, inv);
            const bool small = SMALL && both < kNormal;
            const float s = small ? held : both, f = small ? inv : 1.0f;
            Vec<T, kV * sizeof(T)> y;
#pragma unroll
            for (uint32_t e = 0; e < kV; e += 2) {
                const float2 v = e2m1x2_to_f32((c >> (4 * e)) & 255u);
                if (SMALL) {  // two products of pairs, in place of a branch
                    const dev::f2x x = dev::mul2(dev::mul2(dev::pack2(v.x, v.y), dev::pack2(s, s)), dev::pack2(f, f));
                    from_f32(dev::lo2(x), y.v[e]);
                    from_f32(dev::hi2(x), y.v[e + 1]);
                } else {
                    from_f32(__fmul_rn(v.x, s), y.v[e]);
                    from_f32(__fmul_rn(v.y, s), y.v[e + 1]);
                }
            }
            if (W > sizeof(T) && whole) {
                *reinterpret_cast<decltype(y)*>(dst) = y;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < kV; ++e)
                    if (whole || e < left) dst[e] = y.v[e];
            }
            dst += step;
        };
        if (valid == kFp4Rows && rstep * kRows <= kFp4Rows) {
            for (; r < kFp4Rows; r += rstep * kRows) {
                uint32_t c[kRows], s8[kRows];
#pragma unroll
                for (uint32_t u = 0; u < kRows; ++u) {
                    c[u] = codes_of(r + u * rstep);
                    s8[u] = src_s[fp4_scale_at(r + u * rstep, k0 / BLOCK)];
                }
#pragma unroll
                for (uint32_t u = 0; u < kRows; ++u) write(c[u], s8[u], left >= kV);
            }
        } else {
            for (; r < valid; r += rstep) write(codes_of(r), src_s[fp4_scale_at(r, k0 / BLOCK)], left >= kV);
        }
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
    const float inv = 1.0f / alpha;
    for (uint32_t i = 0; i < n; ++i)
        for (uint32_t k = 0; k < dim; ++k) {
            const uint32_t r = i % kFp4Rows, p = i / kFp4Rows;
            const uint32_t c = (packed[Lo.col_at(p, k / kFp4Col) + r * 16 + (k % kFp4Col) / 2] >> (4 * (k & 1u))) & 15u;
            const uint32_t s8 = packed[Lo.scales_at(p, k / kFp4Group) + fp4_scale_at(r, k % kFp4Group / block)];
            const float held = scale_host(s8, block), s = held * inv, v = c & 8u ? -kMags[c & 7u] : kMags[c & 7u];
            out[(uint64_t)i * dim + k] = s < kNormal ? v * held * inv : v * s;
        }
}

// ------------------------------------------------------------------ launches

// A CTA per panel and group (at most 2^25 panels).
dim3 grid_of(uint32_t n, const Fp4Layout& Lo) { return dim3(fp4_panels(n), std::min(Lo.groups, 65535u)); }

// Bytes that the rows of a matrix are all aligned to: 16, 8 or an element.
uint32_t row_alignment(const void* p, uint64_t ld, uint32_t esize) {
    const uint64_t a = reinterpret_cast<uintptr_t>(p) | ld * esize;
    return a % 16 == 0 ? 16 : a % 8 == 0 ? 8 : esize;
}

template <typename... P, typename... A>
gf_status launch(void (*k)(P...), dim3 grid, cudaStream_t s, A... args) {
    cudaLaunchAttribute at = early_start();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    GF_CUDA(cudaLaunchKernelEx(&cfg, k, args...));
    return GF_OK;
}

template <typename T, uint32_t BLOCK>
gf_status launch_quantize(const void* data, uint64_t ld, uint32_t n, uint32_t dim, float alpha, uint8_t* packed, cudaStream_t s) {
    const Fp4Layout Lo = fp4_layout(n, dim, BLOCK);
    const T* x = static_cast<const T*>(data);
    const uint32_t w = row_alignment(data, ld, sizeof(T));
    auto pick = [&](auto fold, auto rows) {
        constexpr bool F = decltype(fold)::value;
        constexpr uint32_t R = decltype(rows)::value;
        return w == 16 ? fp4_quantize_kernel<T, BLOCK, 16, F, R>
               : w == 8 ? fp4_quantize_kernel<T, BLOCK, 8, F, R>
                        : fp4_quantize_kernel<T, BLOCK, sizeof(T), F, R>;
    };
    auto pick_rows = [&](auto fold) {
        if constexpr (sizeof(T) == 4)
            if (dim > 2 * kFp4Col) return pick(fold, std::integral_constant<uint32_t, 4>{});
        return pick(fold, std::integral_constant<uint32_t, 2>{});
    };
    auto* k = fold_alpha(alpha, BLOCK) ? pick_rows(std::true_type{}) : pick_rows(std::false_type{});
    return launch(k, grid_of(n, Lo), s, x, ld, n, dim, alpha, packed, Lo);
}
template <typename T, uint32_t BLOCK>
gf_status launch_dequantize(const uint8_t* packed, uint32_t n, uint32_t dim, float alpha, void* out, uint64_t ld, cudaStream_t s) {
    const Fp4Layout Lo = fp4_layout(n, dim, BLOCK);
    T* y = static_cast<T*>(out);
    const uint32_t w = row_alignment(out, ld, sizeof(T));
    const float inv = 1.0f / alpha;
    auto pick = [&](auto small) {
        constexpr bool S = decltype(small)::value;
        return w == 16 ? fp4_dequantize_kernel<T, BLOCK, 16, S>
               : w == 8 ? fp4_dequantize_kernel<T, BLOCK, 8, S>
                        : fp4_dequantize_kernel<T, BLOCK, sizeof(T), S>;
    };
    auto* k = pick(std::true_type{});
    if constexpr (BLOCK == 16)
        if (inv >= 0x1p9f * kNormal) k = pick(std::false_type{});
    return launch(k, grid_of(n, Lo), s, packed, n, dim, inv, y, ld, Lo);
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
    if (!fp4_alpha(alpha)) return fail(GF_ERR_ARG, "alpha must lie in [2^-126, 2^126]");
    if (ld < dim) return fail(GF_ERR_ARG, "row stride below dim");
    if (n == 0) return GF_OK;
    if (!data || !packed_out) return fail(GF_ERR_ARG, "null argument");
    if (!aligned(data, dtype_bytes(dtype)) || !aligned(packed_out, 16)) return fail(GF_ERR_ARG, "misaligned pointer");
    cudaStream_t s = (cudaStream_t)stream;
    uint8_t* out = static_cast<uint8_t*>(packed_out);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        return block == 16 ? launch_quantize<T, 16>(data, ld, n, dim, alpha, out, s)
                           : launch_quantize<T, 32>(data, ld, n, dim, alpha, out, s);
    };
    return dtype == GF_F32 ? go(float{}) : dtype == GF_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

extern "C" gf_status gf_dequantize_fp4(const void* packed, uint32_t n, uint32_t dim, uint32_t block, float alpha, void* out,
                                       uint32_t dtype, uint64_t ld, void* stream) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!dtype_bytes(dtype)) return fail(GF_ERR_ARG, "unknown dtype");
    if (!fp4_alpha(alpha)) return fail(GF_ERR_ARG, "alpha must lie in [2^-126, 2^126]");
    if (ld < dim) return fail(GF_ERR_ARG, "row stride below dim");
    if (n == 0) return GF_OK;
    if (!packed || !out) return fail(GF_ERR_ARG, "null argument");
    if (!aligned(out, dtype_bytes(dtype)) || !aligned(packed, 16)) return fail(GF_ERR_ARG, "misaligned pointer");
    cudaStream_t s = (cudaStream_t)stream;
    const uint8_t* in = static_cast<const uint8_t*>(packed);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        return block == 16 ? launch_dequantize<T, 16>(in, n, dim, alpha, out, ld, s)
                           : launch_dequantize<T, 32>(in, n, dim, alpha, out, ld, s);
    };
    return dtype == GF_F32 ? go(float{}) : dtype == GF_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

extern "C" gf_status gf_quantize_fp4_host(const float* data, uint32_t n, uint32_t dim, float alpha, uint32_t block,
                                          void* packed_out) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!fp4_alpha(alpha)) return fail(GF_ERR_ARG, "alpha must lie in [2^-126, 2^126]");
    if (n == 0) return GF_OK;
    if (!data || !packed_out) return fail(GF_ERR_ARG, "null argument");
    quantize_host(data, n, dim, alpha, block, static_cast<uint8_t*>(packed_out));
    return GF_OK;
}

extern "C" gf_status gf_dequantize_fp4_host(const void* packed, uint32_t n, uint32_t dim, uint32_t block, float alpha,
                                            float* out) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!fp4_alpha(alpha)) return fail(GF_ERR_ARG, "alpha must lie in [2^-126, 2^126]");
    if (n == 0) return GF_OK;
    if (!packed || !out) return fail(GF_ERR_ARG, "null argument");
    dequantize_host(static_cast<const uint8_t*>(packed), n, dim, block, alpha, out);
    return GF_OK;
}
