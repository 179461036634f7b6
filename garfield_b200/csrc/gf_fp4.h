// Layout of rows held in 4-bit block floating point (gf_fp4.cu, gf_fp4_tc.cu).
//
// Rows are cut into panels of 128 (fewer than 128 rows: one panel of their number rounded up to 16),
// their elements into groups of 128 and columns of 32.  A panel of h rows holds
//   scales   for each group, 128 rows x (128 / block) bytes, as `128 / (4 block)` sub-blocks of 512
//            bytes: byte b of row r in a sub-block (4 consecutive blocks b of the row) is at
//            (r % 32) * 16 + (r / 32) * 4 + b -- the order in which one tcgen05.cp (32x128b,
//            warpx4) spreads the scales of 128 rows over 4 TMEM columns
//   codes    for each column that has elements, h rows x 16 bytes, row r at r * 16, element 2i in
//            the low half of byte i -- 8 rows of a column are one tcgen05 core matrix (K-major,
//            no swizzle), so a column needs no rearranging between HBM and the MMA
// The scales of consecutive groups and the codes of consecutive columns are one run each: two bulk
// copies bring any number of groups into shared memory, one a whole panel.  Codes and scales
// past the end of a row are 0; what stands in the rows past n of the last panel is unspecified
// (a row's bytes reach only that row's outputs).
#pragma once

#include <stdint.h>

#include "gf_internal.h"

namespace gf {

constexpr uint32_t kFp4Rows = 128;              // rows of a panel
constexpr uint32_t kFp4Group = 128;             // elements of a group
constexpr uint32_t kFp4Col = 32;                // elements of a column
constexpr uint32_t kFp4ColBytes = kFp4Rows * 16;  // a column of a full panel
constexpr uint32_t kFp4ScaleSub = 512;          // bytes of one scale sub-block

struct Fp4Layout {
    uint32_t groups, cols, scale_bytes, col_bytes;  // groups and columns of a row, bytes of a group's scales and of a column
    uint64_t panel_bytes;
    __host__ __device__ uint64_t scales_at(uint32_t p, uint32_t g) const { return p * panel_bytes + (uint64_t)g * scale_bytes; }
    __host__ __device__ uint64_t col_at(uint32_t p, uint32_t c) const {
        return p * panel_bytes + (uint64_t)groups * scale_bytes + (uint64_t)c * col_bytes;
    }
};
__host__ __device__ inline Fp4Layout fp4_layout(uint32_t n, uint32_t dim, uint32_t block) {
    Fp4Layout L;
    L.col_bytes = (n < kFp4Rows ? (n + 15) / 16 * 16 : kFp4Rows) * 16;
    L.groups = (uint32_t)(((uint64_t)dim + kFp4Group - 1) / kFp4Group);
    L.cols = (uint32_t)(((uint64_t)dim + kFp4Col - 1) / kFp4Col);
    L.scale_bytes = block == 16 ? 2 * kFp4ScaleSub : kFp4ScaleSub;
    L.panel_bytes = (uint64_t)L.groups * L.scale_bytes + (uint64_t)L.cols * L.col_bytes;
    return L;
}
__host__ __device__ inline uint32_t fp4_panels(uint32_t n) { return (uint32_t)(((uint64_t)n + kFp4Rows - 1) / kFp4Rows); }
// Byte of row r's scale of block b (0 .. 128 / block - 1) in a group's scales.
__host__ __device__ inline uint32_t fp4_scale_at(uint32_t r, uint32_t b) {
    return (b >> 2) * kFp4ScaleSub + (r & 31u) * 16 + (r >> 5) * 4 + (b & 3u);
}

inline bool fp4_shape(uint32_t dim, uint32_t block) { return dim > 0 && (block == 16 || block == 32); }
inline bool fp4_alpha(float alpha) { return alpha >= 0x1p-126f && alpha <= 0x1p126f; }  // 1 / alpha is normal too
inline uint32_t dtype_bytes(uint32_t dtype) { return dtype == GF_F32 ? 4u : dtype == GF_F16 || dtype == GF_BF16 ? 2u : 0u; }
inline bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace gf
