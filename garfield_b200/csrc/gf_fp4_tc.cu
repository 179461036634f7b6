// Products of rows held in 4-bit block floating point (gf_fp4.h) on the tensor cores:
//   out[i][j] = scale * sum_b sq[i][b] sr[j][b] sum_{k in block b} q[i][k] r[j][k]
// with the block-scaled tcgen05.mma, which multiplies E2M1 codes exactly, applies both blocks' scales
// and accumulates in fp32.
//
// The rows r are the M side (128 rows of a panel = 128 TMEM lanes), the queries q the N side, so
// an accumulator's lanes are consecutive j: a warp's store of one column is a contiguous
// run of out, whatever the number of queries, and few queries cost few columns.  A CTA walks tiles
// (pb panels, a panel of queries), queries fastest, so a panel's bytes leave HBM once.  Warp 0
// copies the panels' groups and the query panel's, one run each, into a ring of stages; warp 1
// spreads the scales into TMEM (tcgen05.cp) and issues two MMAs of 64 elements per panel and
// group; eight warps read finished accumulators and write out.  A stage holds two groups of a
// panel or, for rows of one group, up to four panels: an asynchronous copy costs its issuing warp some 80
// cycles, and at the HBM rate a group of a panel passes in 200.
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
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kPolls = 1u << 20;
constexpr uint32_t kSmemLimit = 227 * 1024;

// Zeros for the second column of an MMA step that the rows' last group lacks: with zero codes on the
// query side, whatever codes stand in the other side's place add nothing.
__device__ __align__(16) uint8_t g_zero[kFp4ColBytes];

struct ProdArgs {
    const uint8_t *r, *q;
    Fp4Layout Lr, Lq;
    uint32_t m, n, panels, batches, qtiles;  // batches: tiles along the rows
    uint32_t nt;                        // columns of an accumulator: the rows of a query panel
    uint32_t pb, gs;                    // panels of a tile and groups of a stage (one of them 1)
    uint32_t acc, stages, stage_bytes;
    uint32_t b_off;                     // within a stage: the query panel's groups (the row panels' are at 0)
    uint32_t sf_cols;                   // TMEM columns of one stage's scales
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
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
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
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t par) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(smem_u32(bar)), "r"(par)
                 : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bwait(uint64_t* bar, uint32_t par, const volatile uint32_t* stop, uint32_t polls) {
    for (uint32_t p = 0; p < 16; ++p)
        if (mbar_test(bar, par)) return true;
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

// This CTA's tiles: blockIdx.x, + gridDim.x, ...; query tiles vary fastest.
struct Tiles {
    uint32_t p, q, dp, dq, qtiles, batches;
    __device__ __forceinline__ Tiles(uint32_t batches_, uint32_t qtiles_)
        : p(blockIdx.x / qtiles_), q(blockIdx.x % qtiles_), dp(gridDim.x / qtiles_), dq(gridDim.x % qtiles_), qtiles(qtiles_),
          batches(batches_) {}
    __device__ __forceinline__ bool more() const { return p < batches; }
    __device__ __forceinline__ void next() {
        p += dp;
        q += dq;
        if (q >= qtiles) {
            q -= qtiles;
            ++p;
        }
    }
};

__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, uint32_t BLOCK>
__global__ void __launch_bounds__(kThreads, 1) fp4_product_kernel(const __grid_constant__ ProdArgs A) {
    extern __shared__ __align__(1024) unsigned char sm[];
    constexpr uint32_t kSub = BLOCK == 16 ? 2 : 1;  // scale sub-blocks of a group
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + A.stages * A.stage_bytes);
    uint64_t* empty = full + kMaxStages;
    uint64_t* tfull = empty + kMaxStages;
    uint64_t* tempty = tfull + kMaxAcc;
    uint64_t* drain = tempty + kMaxAcc;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile uint32_t* stop = tmem_slot + 1;
    const uint32_t warp = threadIdx.x >> 5, lane = lane_id();
    const uint32_t cpp = A.nt / 16;     // 16-column chunks of a panel's accumulator
    const bool split = A.pb * cpp > 1;  // both epilogue halves share a tile's chunks, else they take alternate tiles

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
    const uint32_t G = A.Lr.groups;

    if (warp == 0) {
        // -------------------------------------------------------------- producer warp
        bool ok = true;
        Ring ring;
        uint64_t filled = 0;
        const uint32_t pad = (A.Lq.last_cols & 1u) * A.nt * 16;  // bytes of the zero column of the last group
        for (Tiles t(A.batches, A.qtiles); ok && t.more(); t.next()) {
            const uint32_t p0 = t.p * A.pb, np = min(A.pb, A.panels - p0);
            const uint8_t* src_r = A.r + p0 * A.Lr.panel_bytes;
            const uint8_t* src_q = A.q + t.q * A.Lq.panel_bytes;
            for (uint32_t g = 0; g < G; g += A.gs, ring.next(A.stages), ++filled) {
                // (a barrier's first wait, for the use before its first, returns at once)
                if (!(ok = __all_sync(kFull, bwait(&empty[ring.i], ring.par ^ 1u, stop, A.polls)))) break;
                unsigned char* stg = sm + ring.i * A.stage_bytes;
                uint64_t* bar = &full[ring.i];
                const bool last = g + A.gs >= G;
                const uint32_t whole = last ? G - 1 - g : A.gs;  // full groups of the stage
                const uint32_t a_bytes = (whole * A.Lr.group_bytes + (last ? A.Lr.last_bytes : 0u)) * np;
                const uint32_t b_bytes = whole * A.Lq.group_bytes + (last ? A.Lq.last_bytes : 0u);
                if (elect_one()) {
                    mbar_arrive_expect_tx(bar, a_bytes + b_bytes + (last ? pad : 0u) + A.extra_tx);
                    bulk_g2s(stg, src_r, a_bytes, bar);
                    bulk_g2s(stg + A.b_off, src_q, b_bytes, bar);
                    if (last && pad) bulk_g2s(stg + A.b_off + b_bytes, g_zero, pad, bar);
                }
                __syncwarp();
                src_r += a_bytes;
                src_q += b_bytes;
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
        const uint32_t acc_cols = A.pb * A.nt, sf0 = tmem + A.acc * acc_cols;
        // everything below in 16-byte units of shared memory, added to a descriptor's address field
        constexpr uint32_t kScales = kSub * kFp4ScaleSub / 16;
        const uint32_t a_item = (A.pb > 1 ? (uint32_t)A.Lr.panel_bytes : A.Lr.group_bytes) / 16, b_item = A.Lq.group_bytes / 16;
        const uint32_t a_step = A.Lr.col_bytes / 8, b_step = A.Lq.col_bytes / 8;
        const uint32_t sm0 = smem_u32(sm) / 16, st16 = A.stage_bytes / 16, b_off = A.b_off / 16;
        const uint64_t ad0 = smem_desc(0, A.Lr.col_bytes, 128) + kScales, bd0 = smem_desc(0, A.Lq.col_bytes, 128) + kScales;
        const uint64_t cd0 = smem_desc(0, 128, 128);
        const uint32_t sfb_off = A.pb * A.gs * 4 * kSub;
        bool ok = true;
        Ring ring, accs;
        for (Tiles t(A.batches, A.qtiles); t.more(); t.next(), accs.next(A.acc)) {
            const uint32_t np = min(A.pb, A.panels - t.p * A.pb);
            const uint32_t d0 = tmem + accs.i * acc_cols;
            if (!(ok = __all_sync(kFull, bwait(&tempty[accs.i], accs.par ^ 1u, stop, A.polls)))) break;
            tc_fence_after();
            for (uint32_t g = 0; g < G; g += A.gs, ring.next(A.stages)) {
                if (!(ok = __all_sync(kFull, bwait(&full[ring.i], ring.par, stop, A.polls)))) break;
                tc_fence_after();
                const uint32_t as = sm0 + ring.i * st16, bs = as + b_off;
                // this stage's scales; their slot was last read by MMAs that the stage's empty barrier covers
                const uint32_t sfa = sf0 + ring.i * A.sf_cols, sfb = sfa + sfb_off;
                const bool last = g + A.gs >= G;
                const uint32_t items = A.pb > 1 ? np : min(A.gs, G - g);
                // (panel, group) pair x of the stage: its scales, and its MMA step s of 64 elements
                auto scales = [&](uint32_t x, bool q) {
#pragma unroll
                    for (uint32_t h = 0; h < kSub; ++h) {
                        scales_to_tmem(sfa + (x * kSub + h) * 4, cd0 + (as + x * a_item + h * (kFp4ScaleSub / 16)));
                        if (q) scales_to_tmem(sfb + (x * kSub + h) * 4, cd0 + (bs + x * b_item + h * (kFp4ScaleSub / 16)));
                    }
                };
                auto step = [&](uint32_t x, uint32_t s, uint32_t gx, uint32_t d, uint32_t acc) {
                    // block 16: step s uses sub-block s; block 32: bytes 2s, 2s + 1 of the one sub-block
                    const uint32_t h = BLOCK == 16 ? s * 4 : 0;
                    mma_fp4<BLOCK>(d, ad0 + (as + x * a_item + s * a_step), bd0 + (bs + gx * b_item + s * b_step),
                                   BLOCK == 16 ? idesc : idesc | (2 * s) << 4 | (2 * s) << 29, sfa + x * 4 * kSub + h,
                                   sfb + gx * 4 * kSub + h, acc);
                };
                if (elect_one()) {
                    if (A.pb == 1 && (!last || (items == 2 && A.Lr.last_cols > 2))) {  // two groups, both steps
                        scales(0, true);
                        scales(1, true);
                        step(0, 0, 0, d0, g);
                        step(0, 1, 0, d0, 1);
                        step(1, 0, 1, d0, 1);
                        step(1, 1, 1, d0, 1);
                    } else if (items == 4 && A.Lr.last_cols > 2) {  // four panels, both steps
#pragma unroll
                        for (uint32_t x = 0; x < 4; ++x) scales(x, x == 0);
#pragma unroll
                        for (uint32_t x = 0; x < 4; ++x) {
                            step(x, 0, 0, d0 + x * A.nt, 0);
                            step(x, 1, 0, d0 + x * A.nt, 1);
                        }
                    } else {
                        for (uint32_t x = 0; x < items; ++x) {
                            const uint32_t gx = A.pb > 1 ? 0 : x, d = A.pb > 1 ? d0 + x * A.nt : d0;
                            scales(x, x == 0 || A.pb == 1);
                            step(x, 0, gx, d, g + gx);
                            if (g + gx + 1 < G || A.Lr.last_cols > 2) step(x, 1, gx, d, 1);
                        }
                    }
                    mma_commit(&empty[ring.i]);  // the stage is free once these MMAs have read it
                    if (last) mma_commit(&tfull[accs.i]);
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
        constexpr uint32_t kBatch = 4;  // chunks read before any is stored
        const uint32_t qq = warp & 3u, h = (warp - 2) >> 2;  // lane quarter, half
        const uint32_t acc_cols = A.pb * A.nt;
        T* out = static_cast<T*>(A.out);
        bool ok = true;
        uint32_t u = 0;
        Ring accs;
        for (Tiles t(A.batches, A.qtiles); t.more(); t.next(), ++u, accs.next(A.acc)) {
            if (!split && (u & 1u) != h) continue;
            const uint32_t p0 = t.p * A.pb, q0 = t.q * A.nt;
            const uint32_t rows = min(A.nt, A.m - q0);
            const uint32_t chunks = min(A.pb, A.panels - p0) * cpp, x0 = split ? h : 0, dx = split ? 2 : 1;
            const uint32_t addr = tmem + (qq * 32 << 16) + accs.i * acc_cols;
            if (ok) {
                ok = __all_sync(kFull, bwait(&tfull[accs.i], accs.par, stop, A.polls));
                tc_fence_after();
            }
            for (uint32_t x = x0; x < chunks || x == x0; x += kBatch * dx) {
                uint32_t v[kBatch][16];
                __syncwarp();  // tcgen05.ld is warp-collective
                if (ok) {
#pragma unroll
                    for (uint32_t y = 0; y < kBatch; ++y)
                        if (x + y * dx < chunks) tmem_ld16(addr + (x + y * dx) * 16, v[y]);
#pragma unroll
                    for (uint32_t y = 0; y < kBatch; ++y) tmem_wait_ld16(v[y]);
                    if (x + kBatch * dx >= chunks) {  // the accumulator's last read by this warp
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&tempty[accs.i]);
                    }
                }
#pragma unroll
                for (uint32_t y = 0; y < kBatch; ++y) {
                    const uint32_t xy = x + y * dx;
                    if (xy >= chunks) break;
                    const uint32_t p = xy / cpp, c = (xy - p * cpp) * 16;
                    const uint64_t j = (uint64_t)(p0 + p) * kFp4Rows + qq * 32 + lane;
                    T* dst = out + (uint64_t)(q0 + c) * A.ld + j;
                    if (j < A.n)
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e)
                            if (c + e < rows)
                                store(dst + e * A.ld, ok ? __uint_as_float(v[y][e]) * A.scale : __int_as_float(0x7FC00000));
                }
            }
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
    A.Lr = fp4_layout(n, dim, block);
    A.Lq = fp4_layout(m, dim, block);
    A.m = m;
    A.n = n;
    A.panels = fp4_panels(n);
    A.qtiles = fp4_panels(m);
    A.out = out;
    A.ld = ld;
    A.scale = scale;
    A.polls = test_wait ? test_wait : kPolls;
    A.extra_tx = test_wait ? 16u : 0u;
    A.nt = A.Lq.col_bytes / 16;
    A.pb = A.gs = 1;
    if (A.Lr.groups > 1)
        A.gs = 2;
    else  // several panels to a tile while two accumulators fit and every SM still has a tile
        while (A.pb < 4 && 2 * A.pb * A.nt <= 128 && (uint64_t)A.panels * A.qtiles >= 2ull * A.pb * sms) A.pb *= 2;
    const uint32_t sub = block == 16 ? 2 : 1;
    A.batches = (A.panels + A.pb - 1) / A.pb;
    const uint64_t tiles = (uint64_t)A.batches * A.qtiles;
    // the panels' part has room for whole groups: an MMA reads 128 rows of two columns whatever the panel has
    A.b_off = A.pb * A.gs * (sub * kFp4ScaleSub + kFp4Group / kFp4Col * kFp4ColBytes);
    A.stage_bytes = A.b_off + A.gs * A.Lq.group_bytes;
    A.sf_cols = (A.pb + 1) * A.gs * 4 * sub;
    A.stages = std::min(kMaxStages, (kSmemLimit - 1024) / A.stage_bytes);
    A.acc = std::min(kMaxAcc, (kTmemCols - A.stages * A.sf_cols) / (A.pb * A.nt));
    const uint32_t smem = A.stages * A.stage_bytes + (2 * kMaxStages + 2 * kMaxAcc + 1) * 8 + 16;
    const uint32_t grid = (uint32_t)std::min<uint64_t>(tiles, (uint64_t)sms);
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
