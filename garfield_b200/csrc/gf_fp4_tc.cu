// Products of rows held in 4-bit block floating point (gf_fp4.h) on the tensor cores:
//   out[i][j] = scale * sum_b sq[i][b] sr[j][b] sum_{k in block b} q[i][k] r[j][k]
// with the block-scaled tcgen05.mma, which multiplies E2M1 codes exactly, applies both blocks' scales
// and accumulates in fp32.
//
// The rows r are the M side (128 rows of a panel = 128 TMEM lanes), the queries q the N side, so
// an accumulator's lanes are consecutive j: a warp's store of one column is a contiguous
// run of out, whatever the number of queries, and few queries cost few columns.  A CTA walks tiles
// (panel, nt queries), queries fastest, so a panel's bytes leave HBM once.  Warp 0 copies, per group of
// 128 elements, the panel's group (one run) and the query columns and scales into a ring of stages;
// one thread of warp 1 spreads the scales into TMEM (tcgen05.cp) and issues the
// group's two MMAs (64 elements each); eight warps read finished accumulators and write out.
//
// Every wait is bounded.  When one runs out the CTA stops and the outputs it still owes become NaN.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "gf_device.cuh"
#include "gf_fp4.h"

namespace gf {
namespace {

using namespace dev;

constexpr uint32_t kThreads = 320;    // producer warp, MMA warp, 8 epilogue warps
constexpr uint32_t kMaxStages = 8;
constexpr uint32_t kMaxAcc = 8;
constexpr uint32_t kMaxNt = 256;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kPolls = 1u << 20;
constexpr uint32_t kSmemLimit = 227 * 1024;

// Zeros for the second column of an MMA step that the row's last group lacks: with zero codes on the
// query side, what the other side's column holds from earlier stages adds nothing.
__device__ __align__(16) uint8_t g_zero[kMaxNt * 16];

struct ProdArgs {
    const uint8_t *r, *q;
    Fp4Layout Lo;
    uint32_t m, n, nt, acc, stages, qtiles;
    uint32_t stage_bytes, b_off, sfb_off;  // within a stage: query columns, query scales (the panel's group is at 0)
    uint32_t npan;                         // query panels a tile can touch
    uint32_t sf_cols;                      // TMEM columns of one stage's scales
    uint64_t tiles;
    void* out;
    uint64_t ld;
    float scale;
    uint32_t polls, extra_tx;
};

__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {  // K-major, no swizzle
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
           (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46;
}
// 32 rows x 16 bytes of scales from shared memory (four 128-byte core matrices) to 4 TMEM
// columns, repeated in each quarter of the lanes.
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint32_t saddr) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(smem_desc(saddr, 128, 128)) : "memory");
}
template <uint32_t BLOCK>
__device__ __forceinline__ void mma_fp4(uint32_t tmem, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t acc) {
    if (BLOCK == 16)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(tmem),
            "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(tmem),
            "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc));
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 16 consecutive TMEM columns of this warp's 32 lanes, and the wait that orders their use.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
// True in one lane of the warp.  Loops and addresses around it stay warp-uniform, so the compiler
// keeps them in uniform registers, which is what the asynchronous instructions read.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
// Bounded wait on a phase; false when it ran out or the CTA is stopping.
__device__ __forceinline__ bool bwait(uint64_t* bar, uint32_t par, const volatile uint32_t* stop, uint32_t polls) {
    for (uint32_t p = 0; p < polls; ++p) {
        if (mbar_try_wait(bar, par, 1000)) return true;
        if (*stop) return false;
    }
    return false;
}

// Position in a ring of barriers: slot and the parity of its current use.
struct Ring {
    uint32_t i = 0, par = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++i == n) {
            i = 0;
            par ^= 1u;
        }
    }
};

__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, uint32_t BLOCK>
__global__ void __launch_bounds__(kThreads, 1) fp4_product_kernel(const __grid_constant__ ProdArgs A) {
    extern __shared__ __align__(1024) unsigned char sm[];
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + A.stages * A.stage_bytes);
    uint64_t* empty = full + kMaxStages;
    uint64_t* tfull = empty + kMaxStages;
    uint64_t* tempty = tfull + kMaxAcc;
    uint64_t* drain = tempty + kMaxAcc;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile uint32_t* stop = tmem_slot + 1;
    const uint32_t warp = threadIdx.x >> 5, lane = lane_id();
    const bool split = A.nt >= 64;  // both epilogue halves share a tile's columns, else they take alternate tiles

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kMaxStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (uint32_t i = 0; i < kMaxAcc; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], split ? 8 : 4);
        }
        mbar_init(drain, 1);
        *stop = 0;
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t G = A.Lo.groups, ntc = A.nt * 16;

    if (warp == 0) {
        // -------------------------------------------------------------- producer warp
        bool ok = true;
        Ring ring;
        uint64_t filled = 0;
        for (uint64_t t = blockIdx.x; ok && t < A.tiles; t += gridDim.x) {
            const uint32_t panel = (uint32_t)(t / A.qtiles), q0 = (uint32_t)(t % A.qtiles) * A.nt;
            const uint32_t rows = min(A.nt, A.m - q0);
            const uint32_t pq0 = q0 / kFp4Rows, np = (q0 + rows - 1) / kFp4Rows - pq0 + 1;  // query panels of the tile
            const uint8_t* src_r = A.r + panel * A.Lo.panel_bytes;
            for (uint32_t g = 0; g < G; ++g, ring.next(A.stages), ++filled) {
                const uint32_t st = ring.i;
                // (a barrier's first wait, for the use before its first, returns at once)
                if (!(ok = __all_sync(kFull, bwait(&empty[st], ring.par ^ 1u, stop, A.polls)))) break;
                unsigned char* stg = sm + st * A.stage_bytes;
                const uint32_t cols = g + 1 == G ? A.Lo.last_cols : 4u;
                const uint32_t a_bytes = A.Lo.scale_bytes + cols * kFp4ColBytes;
                const uint32_t pad = cols & 1u;
                const uint64_t at = (uint64_t)g * A.Lo.group_bytes;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&full[st], a_bytes + np * A.Lo.scale_bytes + cols * rows * 16 + pad * ntc + A.extra_tx);
                    bulk_g2s(stg, src_r + at, a_bytes, &full[st]);
                    for (uint32_t j = 0; j < np; ++j) {
                        // the tile's rows of query panel pq0 + j: its scales, then a run of each column
                        const uint8_t* src = A.q + (uint64_t)(pq0 + j) * A.Lo.panel_bytes + at;
                        const uint32_t a = max(q0, (pq0 + j) * kFp4Rows), b = min(q0 + rows, (pq0 + j + 1) * kFp4Rows);
                        bulk_g2s(stg + A.sfb_off + j * A.Lo.scale_bytes, src, A.Lo.scale_bytes, &full[st]);
                        src += A.Lo.scale_bytes + (a % kFp4Rows) * 16;
                        unsigned char* dst = stg + A.b_off + (a - q0) * 16;
#pragma unroll
                        for (uint32_t c = 0; c < 4; ++c)
                            if (c < cols) bulk_g2s(dst + c * ntc, src + c * kFp4ColBytes, (b - a) * 16, &full[st]);
                    }
                    if (pad) bulk_g2s(stg + A.b_off + cols * ntc, g_zero, ntc, &full[st]);
                }
                __syncwarp();
            }
        }
        if (!ok) *stop = 1u;
        // every copy issued lands before the CTA exits (in normal operation they completed long ago)
        if (lane == 0)
            for (uint32_t st = 0; st < A.stages && st < filled; ++st) {
                const uint32_t use = (uint32_t)((filled - 1 - st) / A.stages);  // the slot's last
                uint32_t p = 0;
                while (!mbar_try_wait(&full[st], use & 1u, 1000) && ++p < A.polls) {
                }
            }
        __syncwarp();
    } else if (warp == 1) {
        // -------------------------------------------------------------- MMA warp
        // E2M1 x E2M1, K-major, N = nt, M = 128, scales UE8M0 (block 32) or UE4M3 (block 16)
        const uint32_t idesc = (1u << 7) | (1u << 10) | ((A.nt >> 3) << 17) | ((BLOCK == 32 ? 1u : 0u) << 23) | ((128u >> 4) << 24);
        const uint32_t sf0 = tmem + A.acc * A.nt;
        constexpr uint32_t kSub = BLOCK == 16 ? 2 : 1;  // scale sub-blocks of a group
        bool ok = true;
        Ring ring, accs;
        for (uint64_t t = blockIdx.x; t < A.tiles; t += gridDim.x, accs.next(A.acc)) {
            const uint32_t b = accs.i;
            const uint32_t q0 = (uint32_t)(t % A.qtiles) * A.nt, rows = min(A.nt, A.m - q0);
            const uint32_t np = (q0 + rows - 1) / kFp4Rows - q0 / kFp4Rows + 1;
            const uint32_t lead = (q0 % kFp4Rows) / 32;  // the tile's first row in its first panel's scales
            if (!(ok = __all_sync(kFull, bwait(&tempty[b], accs.par ^ 1u, stop, A.polls)))) break;
            tc_fence_after();
            for (uint32_t g = 0; g < G; ++g, ring.next(A.stages)) {
                const uint32_t st = ring.i;
                if (!(ok = __all_sync(kFull, bwait(&full[st], ring.par, stop, A.polls)))) break;
                tc_fence_after();
                const uint32_t stg = smem_u32(sm + st * A.stage_bytes);
                const uint32_t cols = g + 1 == G ? A.Lo.last_cols : 4u;
                // this stage's scales; their slot was last read by MMAs that the stage's empty barrier covers
                const uint32_t sfa = sf0 + st * A.sf_cols, sfb = sfa + 4 * kSub;
                const uint32_t a0 = stg + A.Lo.scale_bytes, b0 = stg + A.b_off;
                if (elect_one()) {
#pragma unroll
                    for (uint32_t h = 0; h < kSub; ++h) {
                        scales_to_tmem(sfa + h * 4, stg + h * kFp4ScaleSub);
                        for (uint32_t j = 0; j < np; ++j)
                            scales_to_tmem(sfb + (h * A.npan + j) * 4, stg + A.sfb_off + j * A.Lo.scale_bytes + h * kFp4ScaleSub);
                    }
#pragma unroll
                    for (uint32_t s = 0; s < 2; ++s) {
                        if (s * 2 >= cols) break;
                        const uint64_t ad = smem_desc(a0 + s * 2 * kFp4ColBytes, kFp4ColBytes, 128);
                        const uint64_t bd = smem_desc(b0 + s * 2 * ntc, ntc, 128);
                        // block 16: step s uses sub-block s; block 32: bytes 2s, 2s + 1 of the one sub-block
                        const uint32_t id = BLOCK == 16 ? idesc : idesc | (2 * s) << 4 | (2 * s) << 29;
                        const uint32_t h = BLOCK == 16 ? s : 0;
                        mma_fp4<BLOCK>(tmem + b * A.nt, ad, bd, id, sfa + h * 4, sfb + h * A.npan * 4 + lead, (g | s) ? 1u : 0u);
                    }
                    mma_commit(&empty[st]);  // the stage is free once these MMAs have read it
                    if (g + 1 == G) mma_commit(&tfull[b]);
                }
                __syncwarp();
            }
            if (!ok) break;
        }
        if (!ok) *stop = 1u;
        // every MMA has completed before TMEM is released
        if (elect_one()) mma_commit(drain);
        __syncwarp();
        uint32_t p = 0;
        while (!mbar_try_wait(drain, 0, 1000) && ++p < A.polls) {
        }
        if (p >= A.polls) *stop = 1u;
        __syncwarp();
    } else {
        // -------------------------------------------------------------- epilogue warps
        const uint32_t qq = warp & 3u, h = (warp - 2) >> 2;  // lane quarter, half
        T* out = static_cast<T*>(A.out);
        bool ok = true;
        uint32_t u = 0;
        Ring accs;
        for (uint64_t t = blockIdx.x; t < A.tiles; t += gridDim.x, ++u, accs.next(A.acc)) {
            if (!split && (u & 1u) != h) continue;
            const uint32_t b = accs.i;
            const uint32_t panel = (uint32_t)(t / A.qtiles), q0 = (uint32_t)(t % A.qtiles) * A.nt;
            const uint32_t rows = min(A.nt, A.m - q0);
            const uint64_t j = (uint64_t)panel * kFp4Rows + qq * 32 + lane;
            if (ok) {
                ok = __all_sync(kFull, bwait(&tfull[b], accs.par, stop, A.polls));
                tc_fence_after();
            }
            T* dst = out + q0 * A.ld + j;
            for (uint32_t c = split ? h * 16 : 0; c < rows; c += split ? 32 : 16) {
                uint32_t v[16];
                __syncwarp();  // tcgen05.ld is warp-collective
                if (ok) {
                    tmem_ld16(tmem + (qq * 32 << 16) + b * A.nt + c, v);
                    tmem_wait_ld16(v);
                }
                if (j < A.n)
#pragma unroll
                    for (uint32_t e = 0; e < 16; ++e)
                        if (c + e < rows) store(dst + (uint64_t)(c + e) * A.ld, ok ? __uint_as_float(v[e]) * A.scale : __int_as_float(0x7FC00000));
            }
            tc_fence_before();
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&tempty[b]);
        }
        if (!ok) *stop = 1u;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <typename T, uint32_t BLOCK>
gf_status launch_product(ProdArgs A, uint32_t grid, uint32_t smem, cudaStream_t s) {
    GF_CUDA(cudaFuncSetAttribute(fp4_product_kernel<T, BLOCK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    fp4_product_kernel<T, BLOCK><<<grid, kThreads, smem, s>>>(A);
    GF_CUDA(cudaGetLastError());
    return GF_OK;
}

gf_status product(const void* q, uint32_t m, const void* r, uint32_t n, uint32_t dim, uint32_t block, float scale, void* out,
                  uint32_t dtype, uint64_t ld, uint32_t test_wait, cudaStream_t s) {
    int dev = 0, sms = 0;
    GF_CUDA(cudaGetDevice(&dev));
    GF_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    ProdArgs A = {};
    A.r = static_cast<const uint8_t*>(r);
    A.q = static_cast<const uint8_t*>(q);
    A.Lo = fp4_layout(dim, block);
    A.m = m;
    A.n = n;
    A.out = out;
    A.ld = ld;
    A.scale = scale;
    A.polls = test_wait ? test_wait : kPolls;
    A.extra_tx = test_wait ? 16u : 0u;
    // queries of a tile: all of them up to 256, else equal tiles of a multiple of 64 (a tile then starts
    // at the first or the middle of the 4 TMEM columns of its panel's scales)
    const uint32_t nq = (uint32_t)(((uint64_t)m + kMaxNt - 1) / kMaxNt);
    const uint32_t per = (uint32_t)(((uint64_t)m + nq - 1) / nq), step = nq > 1 ? 64 : 16;
    A.nt = (per + step - 1) / step * step;
    A.qtiles = (uint32_t)(((uint64_t)m + A.nt - 1) / A.nt);
    A.npan = A.qtiles == 1 ? fp4_panels(A.nt) : (A.nt + (A.nt % kFp4Rows ? 64 : 0) + kFp4Rows - 1) / kFp4Rows;
    A.tiles = (uint64_t)fp4_panels(n) * A.qtiles;
    A.b_off = A.Lo.group_bytes;
    A.sfb_off = A.b_off + 4 * A.nt * 16;
    A.stage_bytes = A.sfb_off + A.npan * A.Lo.scale_bytes;
    A.sf_cols = (1 + A.npan) * 4 * (block == 16 ? 2 : 1);
    // two accumulators or more when they leave room for four stages' scales; then as many stages as fit
    A.acc = std::min(kMaxAcc, std::max(1u, (kTmemCols - 4 * A.sf_cols) / A.nt));
    A.stages = std::min({kMaxStages, (kSmemLimit - 1024) / A.stage_bytes, (kTmemCols - A.acc * A.nt) / A.sf_cols});
    const uint32_t smem = A.stages * A.stage_bytes + (2 * kMaxStages + 2 * kMaxAcc + 1) * 8 + 16;
    const uint32_t grid = (uint32_t)std::min<uint64_t>(A.tiles, (uint64_t)sms);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        return block == 16 ? launch_product<T, 16>(A, grid, smem, s) : launch_product<T, 32>(A, grid, smem, s);
    };
    return dtype == GF_F32 ? go(float{}) : dtype == GF_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

}  // namespace
}  // namespace gf

using namespace gf;

extern "C" gf_status gf_product_fp4(const void* q_packed, uint32_t m, const void* r_packed, uint32_t n, uint32_t dim,
                                    uint32_t block, float scale, void* out, uint32_t dtype, uint64_t ld, uint32_t test_wait,
                                    void* stream) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!dtype_bytes(dtype)) return fail(GF_ERR_ARG, "unknown dtype");
    if (!std::isfinite(scale)) return fail(GF_ERR_ARG, "scale must be finite");
    if (ld < n) return fail(GF_ERR_ARG, "row stride below n");
    if (m == 0 || n == 0) return GF_OK;
    if (!q_packed || !r_packed || !out) return fail(GF_ERR_ARG, "null argument");
    if (!aligned(q_packed, 16) || !aligned(r_packed, 16) || !aligned(out, dtype_bytes(dtype)))
        return fail(GF_ERR_ARG, "misaligned pointer");
    return product(q_packed, m, r_packed, n, dim, block, scale, out, dtype, ld, test_wait, (cudaStream_t)stream);
}
