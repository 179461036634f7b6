// Products of rows held in 4-bit block floating point (gf_fp4.h) on the tensor cores:
//   out[i][j] = scale * sum_b sq[i][b] sr[j][b] sum_{k in block b} q[i][k] r[j][k]
// with the block-scaled tcgen05.mma, which multiplies E2M1 codes exactly, applies both blocks' scales
// and accumulates in fp32.
//
// The rows r are the M side (128 rows of a panel = 128 TMEM lanes), the queries q the N side, so
// an accumulator's lanes are consecutive j: a warp's store of one column is a contiguous
// run of out, whatever the number of queries, and few queries cost few columns.
//
// One kernel in three modes.
//   kRing: a CTA walks tiles of pb row panels by one query panel (up to 128 queries).
//   kFew:  the same for a single query panel small enough to stay in shared memory; up to 16 queries
//          may come as they are and are quantised there, which saves a launch.
//   kPair: a cluster of two CTAs walks tiles of two row panels by two query panels, each CTA holding
//          one of either and the tcgen05.mma of the pair (M = N = 256) reading both, so that a byte
//          copied into shared memory feeds twice the products.
// Tiles too few to occupy the SMs are split along the elements over clusters of up to 8 CTAs (kRing,
// kFew): each sums its share, the others send theirs to the first through distributed shared
// memory and it adds them in order.  Query tiles vary slowest within a band of row panels: a
// panel's bytes leave HBM once.
//
// Warp 0 copies scales and codes, one run each, into a ring of stages of up to four groups (of a
// panel, or of several panels that fit whole); warp 1 spreads the stage's scales into TMEM
// (tcgen05.cp) and issues two MMAs of 64 elements per panel and group; the other warps read
// finished accumulators and write out.  The stages are this long because a warp pays some 450
// cycles a stage whatever it holds (waiting, committing, the first instruction's way), while a group's
// MMAs take 128 cycles at N = 128 and its panel's bytes 200 at the HBM rate.
//
// Every wait on a barrier in shared memory is bounded.  When one runs out the CTA stops, is counted, and the outputs
// it still owes become NaN.  The waits for TMEM, for the kernel before and at cluster barriers have no bound of their own:
// the SM's holder of TMEM and the kernel before run to their ends without this CTA, and every CTA of a cluster
// reaches every one of its barriers.
#include <algorithm>
#include <cmath>

#include "gf_fp4_dev.cuh"

namespace gf {
namespace {

using namespace dev;
using namespace fp4;

// Epilogue groups of four warps, one per TMEM lane quarter.  A pair's two share a tile's columns: its one
// accumulator is free sooner.  Otherwise they take tiles in turn, so that one stores while another waits and
// reads (10000 x 100000 x 128 in fp16: 643 us when two shared each tile, 593 with two and 490 with three in
// turn).  A group that waits for a tile has seen the one before its last, so with as many
// accumulators as groups it has seen that accumulator's previous use, and a phase's parity is unambiguous.
constexpr uint32_t epi_groups(uint32_t ctas) { return ctas == 2 ? 2 : 3; }
constexpr uint32_t threads_of(uint32_t ctas) { return 64 + 128 * epi_groups(ctas); }  // and a producer and an MMA warp
constexpr uint32_t kMaxStages = 8;
constexpr uint32_t kMaxAcc = 8;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kPolls = 1u << 20;           // of 3.9 us each
constexpr uint64_t kBandBytes = 64u << 20;  // of row panels, half of L2
constexpr uint32_t kSmemLimit = 227 * 1024;

// Zeros for the second column of an MMA step that the rows' last group lacks: with zero codes on the
// query side, whatever codes stand in the other side's place add nothing.
__device__ __align__(16) uint8_t g_zero[kFp4ColBytes];
// CTAs of this device's products that stopped because a wait ran out.
__device__ unsigned long long g_timeouts;

enum Mode : uint32_t { kRing = 0, kFew = 1, kPair = 2 };
constexpr uint32_t ctas_of(uint32_t mode) { return mode == kPair ? 2 : 1; }
constexpr uint32_t kResident = 128 * 1024;  // bytes of queries kept in shared memory, at most
constexpr uint32_t kMaxSplit = 8;           // CTAs of a cluster that share a tile

// Groups of a full stage: four; three for a pair, whose fourth stage is worth more (8192^3, blocks of 32: 186 us
// against 191) and whose two query panels' scales of 16-element blocks take most of TMEM.
constexpr uint32_t stage_groups(uint32_t ctas) { return ctas == 2 ? 3 : 4; }

struct ProdArgs {
    const uint8_t *r, *q;
    Fp4Layout Lr, Lq;
    uint32_t m, n, panels, qpanels, batches, qtiles;  // batches: tiles along the rows
    uint32_t band;                      // tiles along the rows that are walked for every query tile in turn
    uint32_t nt;                        // columns of an accumulator
    uint32_t pb, gs;                    // row panels of a CTA's tile and groups of a stage (pb > 1: gs is all groups)
    uint32_t acc, stages, stage_bytes;
    uint32_t b_off, bc_off;             // within a stage: the query panels' scales, and the query panel's codes
    uint32_t sf_cols;                   // TMEM columns of one stage's scales
    uint32_t split, per;                // CTAs that share a tile, and groups of each
    uint32_t res_off, resc_off;         // kFew: scales and codes of the queries' share
    const void* raw;                    // kFew: queries as they are (else q), quantised with q_alpha
    uint64_t raw_ld;
    uint32_t raw_dtype;
    float q_alpha;
    void* out;
    uint64_t ld;
    float scale;
    uint32_t torn;                      // 1: store16_torn, with the groups' buffers at torn_off
    uint32_t dim, bar_off, torn_off, polls;
    uint32_t hold;                      // test hook: 1 keeps every stage from being reported full until its CTA has given up
};

__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {  // K-major, no swizzle
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
           (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46;
}
// 32 rows x 16 bytes of scales from shared memory (four 128-byte core matrices) to 4 TMEM
// columns, repeated in each quarter of the lanes (of both CTAs of a pair, each from its own).
template <uint32_t CTAS>
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint64_t desc) {
    if (CTAS == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
#define GF_MMA_FP4(group, kind)                                                                                 \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::" group ".kind::" kind  \
                 " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(tmem),                                        \
                 "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc))
template <uint32_t BLOCK, uint32_t CTAS>
__device__ __forceinline__ void mma_fp4(uint32_t tmem, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t acc) {
    if (BLOCK == 16 && CTAS == 1) GF_MMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
    if (BLOCK == 32 && CTAS == 1) GF_MMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
    if (BLOCK == 16 && CTAS == 2) GF_MMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
    if (BLOCK == 32 && CTAS == 2) GF_MMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
}
#undef GF_MMA_FP4
// Arrival on the barrier (of both CTAs of a pair, at the same offset) once the MMAs issued so far are done.
template <uint32_t CTAS>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    if (CTAS == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                         smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
}
template <uint32_t CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
    if (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    }
}
template <uint32_t CTAS>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
    if (CTAS == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Arrival on the same barrier of the cluster's CTA 0.  (A release at cluster scope would hold the arrival
// until this thread's stores to out have landed, and the tile's MMAs with it.  What the arrival reports is
// done by then: bulk copies that completed on this CTA's barrier, or TMEM reads that were waited for.)
__device__ __forceinline__ void arrive_at_leader(uint64_t* bar) {
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n mbarrier.arrive.shared::cluster.b64 _, [a];\n}\n" ::"r"(
            smem_u32(bar))
        : "memory");
}
// Every thread of the cluster has arrived; its earlier writes, to other CTAs' shared memory too, are seen.
__device__ __forceinline__ void sync_cluster() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
// Every thread of the CTA, or of the pair, has arrived.
template <uint32_t CTAS>
__device__ __forceinline__ void sync_all() {
    tc_fence_before();
    if (CTAS == 1)
        __syncthreads();
    else
        sync_cluster();
    tc_fence_after();
}
// v at the same shared-memory place of the cluster's CTA 0.
__device__ __forceinline__ void store_at_leader(const void* p, float v) {
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n st.shared::cluster.f32 [a], %1;\n}\n" ::"r"(smem_u32(p)),
                 "f"(v)
                 : "memory");
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
// Bounded wait on a phase; false when it ran out or the CTA is stopping.  (The suspending form of
// the test takes longer to answer than the plain one, so a few of those come first.)
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t par) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(par)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t par) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, "
        "p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(par), "r"(1000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bwait(uint64_t* bar, uint32_t par, const volatile uint32_t* stop, uint32_t polls) {
    for (uint32_t p = 0; p < 16; ++p)
        if (mbar_test(bar, par)) return true;
    for (uint32_t p = 0; p < polls; ++p) {
        if (mbar_try(bar, par)) return true;
        if (*stop) return false;
    }
    return false;
}

// A warp's wait ran out: the CTA stops, and is counted by the first such warp.  (A call, so that the code around it
// stays as it is: 10000 x 99977 x 128 in fp32 takes 1115 us, 1127 with this inlined and 1206 with a look at
// *stop at the kernel's end.)
__device__ __noinline__ void give_up(volatile uint32_t* stop) {
    if (lane_id() == 0 && atomicExch(const_cast<uint32_t*>(stop), 1u) == 0) atomicAdd(&g_timeouts, 1ull);
}

// Wait for asynchronous work that is under way (copies, MMAs), before the CTA gives up what it uses.
__device__ __forceinline__ void land(uint64_t* bar, uint32_t par) {
    for (uint32_t p = 0; p < kPolls && !mbar_try(bar, par); ++p) {
    }
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

// The tiles of worker i of w: i, i + w, ...  The row panels are cut into bands; within a band the panels
// vary fastest, then the query tiles, so that the tiles in flight write long runs of the same rows of out
// while a band's panels, read once for every query tile, stay in L2.
struct Tiles {
    uint32_t p, q = 0, w, band, width, batches, qtiles;  // (here p counts from the band's first panel)
    uint32_t first = 0;
    __device__ __forceinline__ Tiles(uint32_t i, uint32_t w_, uint32_t band_, uint32_t batches_, uint32_t qtiles_)
        : p(i), w(w_), band(band_), width(min(band_, batches_)), batches(batches_), qtiles(qtiles_) {
        settle();
    }
    __device__ __forceinline__ void settle() {
        while (first < batches && p >= width) {
            p -= width;
            if (++q == qtiles) {
                q = 0;
                first += width;
                width = min(band, batches - first);
            }
        }
    }
    __device__ __forceinline__ bool more() const { return first < batches; }
    __device__ __forceinline__ uint32_t batch() const { return first + p; }
    __device__ __forceinline__ void next() {
        p += w;
        settle();
    }
};

__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Sixteen columns' values of one j: rows i .. i + 15 of out, the first `rows` of them.  With registers to
// spare, four addresses step by four rows: one that steps by a row is a chain of 16 dependent 64-bit additions.
template <typename T, bool SPARE>
__device__ __forceinline__ void store16(T* d0, uint64_t ld, const uint32_t* v, float scale, uint32_t rows) {
    if (!SPARE) {
        if (rows >= 16) {
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e, d0 += ld) store(d0, __uint_as_float(v[e]) * scale);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e, d0 += ld)
                if (e < rows) store(d0, __uint_as_float(v[e]) * scale);
        }
        return;
    }
    T *d1 = d0 + ld, *d2 = d1 + ld, *d3 = d2 + ld;
    const uint64_t ld4 = 4 * ld;
    if (rows >= 16) {
#pragma unroll
        for (uint32_t e = 0; e < 16; e += 4, d0 += ld4, d1 += ld4, d2 += ld4, d3 += ld4) {
            store(d0, __uint_as_float(v[e]) * scale);
            store(d1, __uint_as_float(v[e + 1]) * scale);
            store(d2, __uint_as_float(v[e + 2]) * scale);
            store(d3, __uint_as_float(v[e + 3]) * scale);
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 16; e += 4, d0 += ld4, d1 += ld4, d2 += ld4, d3 += ld4) {
            if (e >= rows) break;
            store(d0, __uint_as_float(v[e]) * scale);
            if (e + 1 < rows) store(d1, __uint_as_float(v[e + 1]) * scale);
            if (e + 2 < rows) store(d2, __uint_as_float(v[e + 2]) * scale);
            if (e + 3 < rows) store(d3, __uint_as_float(v[e + 3]) * scale);
        }
    }
}

// fp32 rows of out that do not start on 32-byte sectors ("torn"): a warp's 32 elements of a row then leave a
// sector half written at either end, which costs where they reach HBM so.  Where out is far larger than L2, a group's
// four warps gather kTornCols rows' 128 elements in shared memory instead, and a warp writes whole rows, each
// store within one 128-byte line: 10000 x 99977 x 128 1114 us against 1227, 4000 x 99977 x 128 (1.5 GB) 450 against
// 455, but 2000 x 99977 x 128 229 against 208 and 300 x 77777 x 200 (in L2) 37 against 25.5.
constexpr uint32_t kTornCols = 8;
constexpr uint32_t kTornPitch = kFp4Rows + 4;                       // floats
constexpr uint32_t kTornBytes = 2 * kTornCols * kTornPitch * 4;     // of a group: two buffers in turn

// The four warps of an epilogue group.
__device__ __forceinline__ void group_sync(uint32_t gid) {
    __syncwarp();
    asm volatile("bar.sync %0, 128;" ::"r"(gid + 1) : "memory");
}

// Sixteen columns' values (v: those of this lane's row of the panel) into rows dst, dst + ld, ...; `rows` and n: rows
// and elements that exist.  All four warps of the group call it alike.
__device__ __forceinline__ void store16_torn(float* dst, uint64_t ld, const uint32_t* v, float scale, uint32_t rows, uint32_t n,
                                             float* buf, uint32_t& turn, uint32_t qq, uint32_t lane, uint32_t gid) {
#pragma unroll
    for (uint32_t c0 = 0; c0 < 16; c0 += kTornCols) {
        if (c0 >= rows) break;
        float* b = buf + turn * (kTornCols * kTornPitch);
        turn ^= 1u;
#pragma unroll
        for (uint32_t e = 0; e < kTornCols; ++e) b[e * kTornPitch + qq * 32 + lane] = __uint_as_float(v[c0 + e]) * scale;
        group_sync(gid);
        // (the buffer's next use follows the next such barrier, which follows these reads)
#pragma unroll
        for (uint32_t e = 0; e < kTornCols; e += 4) {
            if (c0 + e + qq >= rows) continue;
            float* row = dst + (c0 + e + qq) * ld;
            const uint32_t skew = (uint32_t)(reinterpret_cast<uintptr_t>(row) >> 2) & 31u;  // elements into the line
#pragma unroll
            for (uint32_t k = 0; k < 5; ++k) {
                const uint32_t w = k * 32 + lane - skew;  // (a large number before the row)
                if (w < n) row[w] = b[(e + qq) * kTornPitch + w];
            }
        }
    }
}

// Eight elements of a row from index k on, as floats; `left` of them exist.
template <typename T>
__device__ __forceinline__ void load8(const void* base, uint64_t at, uint32_t left, float* x) {
    const T* p = static_cast<const T*>(base) + at;
#pragma unroll
    for (uint32_t e = 0; e < kOct; ++e) x[e] = e < left ? to_f32(p[e]) : 0.0f;
}

// This CTA's share of the queries (groups gb .. ge - 1), quantised into shared memory in the packed
// panel's form by the epilogue's threads (t: this one's number).
template <uint32_t BLOCK, uint32_t THREADS>
__device__ __forceinline__ void quantize_queries(const ProdArgs& A, uint32_t gb, uint32_t ge, uint32_t dim, unsigned char* scales,
                                                 unsigned char* codes, uint32_t t) {
    const uint32_t octs = (ge - gb) * (kFp4Group / kOct), total = A.m * octs;
    const uint32_t cols = min(4 * ge, (A.Lq.cols + 1) & ~1u) - 4 * gb;  // with the zeros that complete an MMA step
    for (uint32_t i0 = t & ~31u; i0 < total; i0 += THREADS) {
        const uint32_t i = i0 + (t & 31u);  // (a row's octs are a multiple of 16: a block's threads share a row)
        const bool in = i < total;
        const uint32_t row = in ? i / octs : 0, o = in ? i - row * octs : 0;
        const uint32_t k = gb * kFp4Group + o * kOct, left = in && k < dim ? dim - k : 0u;
        float x[kOct];
        const uint64_t at = row * A.raw_ld + k;
        if (A.raw_dtype == GF_F32)
            load8<float>(A.raw, at, left, x);
        else if (A.raw_dtype == GF_F16)
            load8<__half>(A.raw, at, left, x);
        else
            load8<__nv_bfloat16>(A.raw, at, left, x);
        float mx = __fmul_rn(amax8(x), A.q_alpha);
        if (BLOCK == 32) mx = amax2(mx, __shfl_xor_sync(kFull, mx, 2));
        mx = amax2(mx, __shfl_xor_sync(kFull, mx, 1));
        uint32_t c;
        const uint32_t s8 = encode8<BLOCK, false>(x, mx, A.q_alpha, c);
        if (!in) continue;
        if (o / 4 < cols) *reinterpret_cast<uint32_t*>(codes + (o / 4) * A.Lq.col_bytes + row * 16 + (o & 3u) * 4) = c;
        if (o % (BLOCK / kOct) == 0)
            scales[(o / 16) * A.Lq.scale_bytes + fp4_scale_at(row, (o % 16) / (BLOCK / kOct))] = (uint8_t)s8;
    }
    fence_proxy_async_smem();  // the MMAs read these through the asynchronous proxy
    __syncwarp();
}

template <typename T, uint32_t BLOCK, uint32_t MODE>
__global__ void __launch_bounds__(threads_of(ctas_of(MODE)), 1) fp4_product_kernel(const __grid_constant__ ProdArgs A) {
    extern __shared__ __align__(1024) unsigned char sm[];
    constexpr uint32_t CTAS = ctas_of(MODE);
    constexpr uint32_t kSub = BLOCK == 16 ? 2 : 1;  // scale sub-blocks of a group
    constexpr uint32_t kGs = stage_groups(CTAS);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + A.bar_off);
    uint64_t* pfull = full + kMaxStages;  // CTA 0 of a pair: the other CTA's stage is full
    uint64_t* empty = pfull + kMaxStages;
    uint64_t* tfull = empty + kMaxStages;
    uint64_t* tempty = tfull + kMaxAcc;
    uint64_t* drain = tempty + kMaxAcc;
    uint64_t* qfull = drain + 1;  // kFew: the queries are in place
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(qfull + 1);
    volatile uint32_t* stop = tmem_slot + 1;
    const uint32_t warp = threadIdx.x >> 5, lane = lane_id();
    const uint32_t rank = CTAS == 2 ? (blockIdx.x & 1u) : 0u;  // in the pair (clusters are consecutive blocks)
    const uint32_t share = CTAS == 2 ? 0u : blockIdx.x % A.split;  // of the elements
    const uint32_t worker = CTAS == 2 ? blockIdx.x / 2 : blockIdx.x / A.split;
    const uint32_t workers = CTAS == 2 ? gridDim.x / 2 : gridDim.x / A.split;
    const uint32_t G = A.Lr.groups, gb = share * A.per, ge = min(G, gb + A.per);
    const uint32_t cpp = A.nt / 16;     // 16-column chunks of a panel's accumulator

    if (warp == 0) tmem_alloc<CTAS>(tmem_slot);
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kMaxStages; ++i) {
            mbar_init(&full[i], 1 + A.hold);
            mbar_init(&pfull[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (uint32_t i = 0; i < kMaxAcc; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], CTAS == 2 ? 4 * 2 * epi_groups(2) : 4);
        }
        mbar_init(drain, 1);
        mbar_init(qfull, A.raw ? 4 * epi_groups(CTAS) : 1);
        *stop = 0;
        fence_mbar_init();
    }
    sync_all<CTAS>();
    const uint32_t tmem = *tmem_slot;
    wait_for_previous();  // (nothing above touches global memory)

    bool done = true;  // epilogue warps of a split tile: the sums are in TMEM
    if (warp == 0) {
        // -------------------------------------------------------------- producer warp
        bool ok = true;
        Ring ring;
        uint64_t filled = 0;
        const uint32_t pad = A.Lq.cols & 1u;  // the last group lacks the second column of an MMA step
        if (MODE == kFew && !A.raw && elect_one()) {
            const uint32_t as = (ge - gb) * A.Lq.scale_bytes, bc = min(4 * (ge - gb), A.Lq.cols - 4 * gb) * A.Lq.col_bytes;
            const uint32_t z = ge == G && pad ? A.Lq.col_bytes : 0u;
            mbar_arrive_expect_tx(qfull, as + bc + z);
            bulk_g2s(sm + A.res_off, A.q + A.Lq.scales_at(0, gb), as, qfull);
            bulk_g2s(sm + A.resc_off, A.q + A.Lq.col_at(0, 4 * gb), bc, qfull);
            if (z) bulk_g2s(sm + A.resc_off + bc, g_zero, z, qfull);
        }
        __syncwarp();
        for (Tiles t(worker, workers, A.band, A.batches, A.qtiles); ok && t.more(); t.next()) {
            const uint32_t p0 = t.batch() * A.pb * CTAS + rank, np = p0 < A.panels ? min(A.pb, A.panels - p0) : 0u;
            const uint32_t qp = t.q * CTAS + rank;
            for (uint32_t g = gb; g < ge; g += A.gs, ring.next(A.stages), ++filled) {
                // (a barrier's first wait, for the use before its first, returns at once)
                if (!(ok = __all_sync(kFull, bwait(&empty[ring.i], ring.par ^ 1u, stop, A.polls)))) break;
                unsigned char* stg = sm + ring.i * A.stage_bytes;
                uint64_t* bar = &full[ring.i];
                const uint32_t ng = min(A.gs, ge - g), nc = min(4 * ng, A.Lr.cols - 4 * g);  // groups and columns
                const uint32_t as = ng * A.Lr.scale_bytes, ac = nc * A.Lr.col_bytes, bc = nc * A.Lq.col_bytes;
                const uint32_t z = g + ng == G && pad ? A.Lq.col_bytes : 0u;
                const uint32_t a_bytes = A.pb > 1 ? np * (uint32_t)A.Lr.panel_bytes : np * (as + ac);
                // query panels of the tile that exist: their scales all come, the codes of this CTA's
                const uint32_t nq = MODE == kFew ? 0u : min(CTAS, A.qpanels - t.q * CTAS);
                const uint32_t b_bytes = MODE == kFew ? 0u : nq * as + (qp < A.qpanels ? bc + z : 0u);
                if (elect_one()) {
                    mbar_arrive_expect_tx(bar, a_bytes + b_bytes);
                    if (A.pb > 1) {  // whole panels
                        bulk_g2s(stg, A.r + A.Lr.scales_at(p0, 0), a_bytes, bar);
                    } else if (np) {
                        bulk_g2s(stg, A.r + A.Lr.scales_at(p0, g), as, bar);
                        bulk_g2s(stg + A.gs * A.Lr.scale_bytes, A.r + A.Lr.col_at(p0, 4 * g), ac, bar);
                    }
                    if (MODE != kFew) {
                        bulk_g2s(stg + A.b_off, A.q + A.Lq.scales_at(t.q * CTAS, g), as, bar);
                        if (CTAS == 2 && nq == 2)
                            bulk_g2s(stg + A.b_off + A.gs * A.Lq.scale_bytes, A.q + A.Lq.scales_at(t.q * CTAS + 1, g), as, bar);
                        if (qp < A.qpanels) {
                            bulk_g2s(stg + A.bc_off, A.q + A.Lq.col_at(qp, 4 * g), bc, bar);
                            if (z) bulk_g2s(stg + A.bc_off + bc, g_zero, z, bar);
                        }
                    }
                }
                __syncwarp();
            }
        }
        if (!ok) give_up(stop);
        // Every copy issued lands before the CTA exits (in normal operation they completed long ago), whatever
        // A.polls is.  With A.hold no stage was emptied, so each was filled once at most; what kept it from being
        // full arrives once the MMA warp (of a pair, CTA 0's) has given up.
        if (lane == 0) {
            if (A.hold) land(drain, 0);
            for (uint32_t st = 0; st < A.stages && st < filled; ++st) {
                const uint32_t use = (uint32_t)((filled - 1 - st) / A.stages);  // the slot's last
                if (A.hold) mbar_arrive(&full[st]);
                land(&full[st], use & 1u);
            }
            if (MODE == kFew && !A.raw) land(qfull, 0);
        }
        __syncwarp();
    } else if (warp == 1 && rank != 0) {
        // ------------------------- the other CTA of a pair: tells CTA 0 which of its stages are full
        bool ok = true;
        Ring ring;
        for (Tiles t(worker, workers, A.band, A.batches, A.qtiles); ok && t.more(); t.next())
            for (uint32_t g = 0; g < G; g += A.gs, ring.next(A.stages)) {
                if (!(ok = __all_sync(kFull, bwait(&full[ring.i], ring.par, stop, A.polls)))) break;
                if (lane == 0) arrive_at_leader(&pfull[ring.i]);
                __syncwarp();
            }
        if (!ok) give_up(stop);
        // CTA 0's last commit, which follows all its others, has arrived here before this CTA can exit
        land(drain, 0);
        __syncwarp();
    } else if (warp == 1) {
        // -------------------------------------------------------------- MMA warp
        // E2M1 x E2M1, K-major, N = nt (256 for a pair), M = 128 (256), scales UE8M0 (block 32) or UE4M3 (block 16)
        const uint32_t idesc = (1u << 7) | (1u << 10) | ((A.nt >> 3) << 17) | ((BLOCK == 32 ? 1u : 0u) << 23) |
                               ((CTAS * 128u >> 4) << 24);
        const uint32_t acc_cols = A.pb * A.nt, sf0 = tmem + A.acc * acc_cols;
        // everything below in 16-byte units of shared memory, added to a descriptor's 14-bit address field (in a
        // cluster, a shared-memory address has the CTA's rank in its upper bits)
        constexpr uint32_t kScales = kSub * kFp4ScaleSub / 16;  // a group's scales
        const uint32_t a_item = (uint32_t)A.Lr.panel_bytes / 16;
        const uint32_t a_step = A.Lr.col_bytes / 8, b_step = A.Lq.col_bytes / 8;  // two columns
        const uint32_t sm0 = (smem_u32(sm) >> 4) & 0x3FFFu, st16 = A.stage_bytes / 16;
        const uint64_t ad0 = smem_desc(0, A.Lr.col_bytes, 128) + A.gs * kScales;
        const uint64_t bd0 = smem_desc(0, A.Lq.col_bytes, 128);
        const uint64_t cd0 = smem_desc(0, 128, 128);
        const uint32_t sfb_off = A.pb * A.gs * 4 * kSub, q2 = A.gs * kScales;
        bool ok = MODE != kFew || __all_sync(kFull, bwait(qfull, 0, stop, A.polls));
        Ring ring, accs;
        for (Tiles t(worker, workers, A.band, A.batches, A.qtiles); ok && t.more(); t.next(), accs.next(A.acc)) {
            const uint32_t np = CTAS == 2 ? 1u : min(A.pb, A.panels - t.batch() * A.pb);
            const uint32_t d0 = tmem + accs.i * acc_cols;
            if (!(ok = __all_sync(kFull, bwait(&tempty[accs.i], accs.par ^ 1u, stop, A.polls)))) break;
            tc_fence_after();
            for (uint32_t g = gb; g < ge; g += A.gs, ring.next(A.stages)) {
                ok = bwait(&full[ring.i], ring.par, stop, A.polls);
                if (CTAS == 2) ok = ok && bwait(&pfull[ring.i], ring.par, stop, A.polls);
                if (!(ok = __all_sync(kFull, ok))) break;
                tc_fence_after();
                const uint32_t st = sm0 + ring.i * st16;
                // the queries' scales and codes of the stage's first group
                const uint32_t bs = MODE == kFew ? sm0 + A.res_off / 16 + (g - gb) * kScales : st + A.b_off / 16;
                const uint32_t bc = MODE == kFew ? sm0 + A.resc_off / 16 + (g - gb) * 2 * b_step : st + A.bc_off / 16;
                // this stage's scales; their slot was last read by MMAs that the stage's empty barrier covers
                const uint32_t sfa = sf0 + ring.i * A.sf_cols, sfb = sfa + sfb_off;
                const uint32_t ng = min(A.gs, ge - g), steps = min(2 * ng, (A.Lr.cols - 4 * g + 1) / 2);
                const uint32_t acc0 = g - gb;
                // scales of panel x's group y, and of the query panels' group y
                auto row_scales = [&](uint32_t x, uint32_t y) {
#pragma unroll
                    for (uint32_t h = 0; h < kSub; ++h)
                        scales_to_tmem<CTAS>(sfa + ((x * A.gs + y) * kSub + h) * 4, cd0 + (st + x * a_item + (y * kSub + h) * 32));
                };
                auto query_scales = [&](uint32_t y) {
#pragma unroll
                    for (uint32_t h = 0; h < kSub; ++h)
#pragma unroll
                        for (uint32_t j = 0; j < CTAS; ++j)
                            scales_to_tmem<CTAS>(sfb + ((y * kSub + h) * CTAS + j) * 4, cd0 + (bs + j * q2 + (y * kSub + h) * 32));
                };
                // MMA step s of 64 elements of panel x (two steps to a group)
                auto step = [&](uint32_t x, uint32_t s, uint32_t acc) {
                    // block 16: a step has its own sub-block; block 32: bytes 2s, 2s + 1 of the group's
                    const uint32_t sub = BLOCK == 16 ? s : s / 2, byte = BLOCK == 16 ? 0u : 2 * (s & 1u);
                    mma_fp4<BLOCK, CTAS>(d0 + x * A.nt, ad0 + (st + x * a_item + s * a_step), bd0 + (bc + s * b_step),
                                         idesc | byte << 4 | byte << 29, sfa + (x * A.gs * kSub + sub) * 4,
                                         sfb + sub * CTAS * 4, acc);
                };
                if (elect_one()) {
                    // the usual full stages as straight code: kGs groups of a panel, one group of four panels
                    if (np == 1 && steps == 2 * kGs) {
#pragma unroll
                        for (uint32_t y = 0; y < kGs; ++y) {
                            row_scales(0, y);
                            query_scales(y);
                        }
                        step(0, 0, acc0);
#pragma unroll
                        for (uint32_t s = 1; s < 2 * kGs; ++s) step(0, s, 1);
                    } else if (CTAS == 1 && np == 4 && steps == 2) {
                        query_scales(0);
#pragma unroll
                        for (uint32_t x = 0; x < 4; ++x) row_scales(x, 0);
#pragma unroll
                        for (uint32_t x = 0; x < 4; ++x) {
                            step(x, 0, 0);
                            step(x, 1, 1);
                        }
                    } else {
                        for (uint32_t y = 0; y < ng; ++y) query_scales(y);
                        for (uint32_t x = 0; x < np; ++x) {
                            for (uint32_t y = 0; y < ng; ++y) row_scales(x, y);
                            for (uint32_t s = 0; s < steps; ++s) step(x, s, acc0 | s);
                        }
                    }
                    mma_commit<CTAS>(&empty[ring.i]);  // the stage is free once these MMAs have read it
                    if (g + ng == ge) mma_commit<CTAS>(&tfull[accs.i]);
                }
                __syncwarp();
            }
            if (!ok) break;
        }
        if (!ok) give_up(stop);
        // every MMA has completed before TMEM is released
        if (elect_one()) mma_commit<CTAS>(drain);
        __syncwarp();
        land(drain, 0);
        __syncwarp();
    } else {
        // -------------------------------------------------------------- epilogue warps
        constexpr uint32_t kBatch = CTAS == 2 ? 8 : 2;  // chunks read before any is stored
        const uint32_t qq = warp & 3u, h = (warp - 2) >> 2;  // lane quarter, group
        const uint32_t acc_cols = A.pb * A.nt;
        T* out = static_cast<T*>(A.out);
        if (MODE == kFew && A.raw) {
            quantize_queries<BLOCK, 128 * epi_groups(CTAS)>(A, gb, ge, A.dim, sm + A.res_off, sm + A.resc_off, threadIdx.x - 64);
            if (lane == 0) mbar_arrive(qfull);
        }
        bool ok = true;
        uint32_t u = 0, turn = 0;
        Ring accs;
        for (Tiles t(worker, workers, A.band, A.batches, A.qtiles); t.more(); t.next(), accs.next(A.acc)) {
            if (CTAS == 1 && A.split > 1) {  // the cluster's one tile, stored below
                done = __all_sync(kFull, bwait(&tfull[0], 0, stop, A.polls));
                ok = done;
                break;
            }
            if (CTAS == 1) {  // the groups take tiles in turn
                const bool mine = u == h;
                u = u + 1 == epi_groups(CTAS) ? 0 : u + 1;
                if (!mine) continue;
            }
            const uint32_t p0 = t.batch() * A.pb * CTAS + rank, q0 = t.q * A.nt;
            const uint32_t np = CTAS == 2 ? 1u : min(A.pb, A.panels - p0);
            const uint32_t rows = min(A.nt, A.m - q0);
            const uint32_t chunks = np * cpp, x0 = CTAS == 2 ? h : 0, dx = CTAS == 2 ? epi_groups(2) : 1;
            const uint32_t addr = tmem + (qq * 32 << 16) + accs.i * acc_cols;
            if (ok) {
                ok = __all_sync(kFull, bwait(&tfull[accs.i], accs.par, stop, A.polls));
                tc_fence_after();
            }
            uint32_t p = 0, c = x0 * 16;  // panel and column of chunk x
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
                        if (lane == 0) {
                            if (rank == 0)
                                mbar_arrive(&tempty[accs.i]);
                            else
                                arrive_at_leader(&tempty[accs.i]);
                        }
                    }
                }
#pragma unroll
                for (uint32_t y = 0; y < kBatch; ++y) {
                    if (x + y * dx >= chunks) break;
                    // in step, the group's warps write the 512 bytes of a row at about the same time, which fp32 rows
                    // on their way to HBM gain from (10000 x 100000 x 128: 816 us against 845; in fp16 541
                    // against 500)
                    if (sizeof(T) == 4 && !(CTAS == 1 && A.torn)) group_sync(h);
                    if (!ok)
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e) v[y][e] = 0x7FC00000u;
                    if (CTAS == 2) c = (x + y * dx) * 16;
                    const uint64_t j0 = (uint64_t)(p0 + p) * kFp4Rows, j = j0 + qq * 32 + lane;
                    if (CTAS == 1 && sizeof(T) == 4 && A.torn) {
                        if (c < rows)
                            store16_torn(reinterpret_cast<float*>(out + (uint64_t)(q0 + c) * A.ld + j0), A.ld, v[y], A.scale, rows - c,
                                         (uint32_t)min((uint64_t)kFp4Rows, A.n - j0),
                                         reinterpret_cast<float*>(sm + A.torn_off + h * kTornBytes), turn, qq, lane, h);
                    } else if (j < A.n && c < rows) {
                        store16<T, CTAS == 1>(out + (uint64_t)(q0 + c) * A.ld + j, A.ld, v[y], A.scale, rows - c);
                    }
                    if (CTAS == 1) {  // the next chunk of this warp's, perhaps of the next panel
                        c += 16;
                        if (c == A.nt) {
                            c = 0;
                            ++p;
                        }
                    }
                }
            }
        }
        if (!ok) give_up(stop);
    }
    if (CTAS == 1 && A.split > 1) {
        // ------------------------------------------- the shares of a tile, added in CTA 0 of the cluster
        // All of the cluster's MMAs are done, so CTA 0's stages are free: share i > 0 writes its sums there as
        // [i - 1][column][row] floats.
        const uint32_t qq = warp & 3u, row = qq * 32 + lane;
        const uint32_t addr = tmem + (qq * 32 << 16);
        Tiles t(worker, workers, A.band, A.batches, A.qtiles);
        const uint32_t q0 = t.q * A.nt, rows = min(A.nt, A.m - q0);
        float* sums = reinterpret_cast<float*>(sm);
        tc_fence_before();
        sync_cluster();
        tc_fence_after();
        for (uint32_t pass = 0; pass < 2; ++pass) {
            if (warp >= 2 && (pass == 0) == (share != 0))
                for (uint32_t c = ((warp - 2) >> 2) * 16; c < rows; c += 16 * epi_groups(CTAS)) {
                    uint32_t v[16];
                    __syncwarp();
                    tmem_ld16(addr + c, v);
                    tmem_wait_ld16(v);
                    if (!done)
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e) v[e] = 0x7FC00000u;
                    if (pass == 0) {
                        float* dst = sums + ((share - 1) * A.nt + c) * kFp4Rows + row;
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e) store_at_leader(dst + e * kFp4Rows, __uint_as_float(v[e]));
                    } else {
                        for (uint32_t i = 1; i < A.split; ++i) {
                            const float* src = sums + ((i - 1) * A.nt + c) * kFp4Rows + row;
#pragma unroll
                            for (uint32_t e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + src[e * kFp4Rows]);
                        }
                        const uint64_t j = (uint64_t)t.batch() * kFp4Rows + row;
                        if (j < A.n)
                            store16<T, true>(static_cast<T*>(A.out) + (uint64_t)(q0 + c) * A.ld + j, A.ld, v, A.scale, rows - c);
                    }
                }
            if (pass == 0) sync_cluster();
        }
    }
    sync_all<CTAS>();
    if (warp == 0) tmem_free<CTAS>(tmem);
}

template <typename T, uint32_t BLOCK, uint32_t MODE>
gf_status launch_product(const ProdArgs& A, uint32_t grid, uint32_t smem, cudaStream_t s) {
    // (the limit, not this call's size: calls of other sizes may be on their way in other threads)
    GF_CUDA(cudaFuncSetAttribute(fp4_product_kernel<T, BLOCK, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads_of(ctas_of(MODE)));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0] = early_start();
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {MODE == kPair ? 2 : A.split, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = at[1].val.clusterDim.x > 1 ? 2 : 1;
    GF_CUDA(cudaLaunchKernelEx(&cfg, fp4_product_kernel<T, BLOCK, MODE>, A));
    return GF_OK;
}

// Queries that a product quantises itself (their number and size let every CTA do it in passing).
bool quantised_in_passing(uint32_t m, uint32_t dim) { return m <= 16 && dim <= 8192 && (uint64_t)m * dim <= 32768; }

// q: packed queries, or NULL with raw ones in A (quantised_in_passing).
gf_status product(ProdArgs A, const void* q, uint32_t m, const void* r, uint32_t n, uint32_t dim, uint32_t block, float scale,
                  void* out, uint32_t dtype, uint64_t ld, uint32_t test_wait, cudaStream_t s) {
    int dev = 0, sms = 0;
    GF_CUDA(cudaGetDevice(&dev));
    GF_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    A.r = static_cast<const uint8_t*>(r);
    A.q = static_cast<const uint8_t*>(q);
    A.Lr = fp4_layout(n, dim, block);
    A.Lq = fp4_layout(m, dim, block);
    A.m = m;
    A.n = n;
    A.dim = dim;
    A.panels = fp4_panels(n);
    A.qpanels = fp4_panels(m);
    A.out = out;
    A.ld = ld;
    A.scale = scale;
    A.polls = test_wait ? test_wait : kPolls;
    A.hold = test_wait ? 1u : 0u;
    const uint32_t sub = block == 16 ? 2 : 1, scales = sub * kFp4ScaleSub, group = scales + 4 * kFp4ColBytes, G = A.Lr.groups;
    // Pairs of CTAs once their tiles, of 256 x 256, occupy every SM (of one row panel, or the last of an odd number,
    // half a tile is empty and counts all the same), where the rows are long enough for
    // their arithmetic to show (8192 x 16384 in bf16: 96 us against 78 at 512 elements, 86 against 97 at 768,
    // 117 against 151 at 2048), and where out is far larger than L2 and its rows are of 16 bits and torn, or of
    // 32 and not: a pair writes twice as long a run of each row at a time (10000 x 99999 x 128 in fp16 744 us
    // against 1066; 10000 x 100000 x 128 in fp32 822 against 848, but in fp16 704 against 492; torn fp32 rows
    // are put together as store16_torn says).
    const uint64_t pair_tiles = ((uint64_t)A.panels + 1) / 2 * ((A.qpanels + 1) / 2);
    const uint32_t es = dtype_bytes(dtype);
    const bool torn = (reinterpret_cast<uintptr_t>(out) | (m > 1 ? ld * es : 0u)) % 32 != 0;
    const bool past_l2 = (uint64_t)m * n >= (1ull << 30) / es;
    const bool large = m >= 1024 && past_l2 && torn == (es == 2);
    uint32_t mode = (G >= 6 || large) && A.qpanels >= 2 && pair_tiles >= (uint64_t)sms / 2 ? kPair : kRing;
    const uint32_t ctas = ctas_of(mode);
    A.nt = mode == kPair ? 256 : A.Lq.col_bytes / 16;
    A.gs = std::min(G, stage_groups(ctas));
    A.pb = 1;
    A.qtiles = (A.qpanels + ctas - 1) / ctas;
    A.split = 1;
    if (mode == kRing) {
        // tiles that leave SMs idle are split along the elements, at least four groups to a share
        const uint64_t tiles = (uint64_t)A.panels * A.qtiles;
        uint32_t want = 1;
        while (want < kMaxSplit && tiles * want * 2 <= (uint64_t)sms && G >= 8 * want) want *= 2;
        while (want > 1 && (want - 1) * A.nt * kFp4Rows * 4 > 96 * 1024) want /= 2;  // the shares' sums, in CTA 0's stages
        A.per = (G + want - 1) / want;
        A.split = (G + A.per - 1) / A.per;
        const uint64_t resident = (uint64_t)A.per * (scales + 4 * A.Lq.col_bytes);
        if (A.qpanels == 1 && (resident <= kResident / 2 || (A.raw && resident <= kResident))) mode = kFew;
        // several short panels to a tile, while every SM still has a tile
        if (A.gs == G && A.split == 1)
            while (2 * A.pb * A.gs <= 4 && 2 * A.pb * A.nt <= 128 && tiles >= 2ull * A.pb * sms) A.pb *= 2;
    } else {
        A.per = G;
    }
    A.gs = std::min(A.gs, A.per);
    A.torn = torn && es == 4 && past_l2 && m >= 16 && mode != kPair && A.split == 1;
    const uint32_t bars = (3 * kMaxStages + 2 * kMaxAcc + 2) * 8 + 16;
    const uint32_t fixed = bars + (A.torn ? epi_groups(1) * kTornBytes : 0u);
    const uint32_t resident = mode == kFew ? A.per * (scales + 4 * A.Lq.col_bytes) : 0u;
    const uint32_t accs = mode == kPair ? 1 : epi_groups(1);  // accumulators that there have to be
    for (;;) {
        // the panels' part has room for whole groups: an MMA reads 128 rows of two columns whatever the panel has
        A.b_off = A.pb * A.gs * group;
        A.bc_off = A.b_off + (mode == kFew ? 0u : ctas * A.gs * scales);
        A.stage_bytes = A.bc_off + (mode == kFew ? 0u : A.gs * 4 * A.Lq.col_bytes);
        A.sf_cols = (A.pb + ctas) * A.gs * 4 * sub;
        const uint32_t by_smem = (kSmemLimit - fixed - resident) / A.stage_bytes;
        const uint32_t by_tmem = (kTmemCols - accs * A.pb * A.nt) / A.sf_cols;
        A.stages = std::min({kMaxStages, by_smem, by_tmem});
        // two long stages are better than more short ones (8192 x 16384 x 512, blocks of 16: 76 us against 101),
        // unless it is shared memory that leaves no third: then shorter ones keep more bytes in flight
        if (A.stages >= 3 || (A.stages == 2 && A.gs >= 3 && by_smem > 2)) break;
        if (A.pb > 1)  // fewer panels to a tile, else fewer groups to a stage
            A.pb /= 2;
        else if (A.gs > 1)
            A.gs /= 2;
        else
            break;
    }
    A.batches = (A.panels + A.pb * ctas - 1) / (A.pb * ctas);
    A.acc = std::min(kMaxAcc, (kTmemCols - A.stages * A.sf_cols) / (A.pb * A.nt));
    A.res_off = A.stages * A.stage_bytes;
    A.resc_off = A.res_off + (resident ? A.per * scales : 0u);
    A.bar_off = A.res_off + resident;
    A.torn_off = A.bar_off + bars;
    // CTAs that wait for others of their cluster hold all of an SM's TMEM meanwhile: more than half of its shared
    // memory each, so that two never share an SM and no two clusters can hold what the other waits for
    const uint32_t smem = std::max(A.bar_off + fixed, mode == kPair || A.split > 1 ? 116u * 1024 : 0u);
    A.band = (uint32_t)std::min<uint64_t>(A.batches, std::max<uint64_t>(8, kBandBytes / (A.Lr.panel_bytes * A.pb * ctas)));
    const uint64_t tiles = (uint64_t)A.batches * A.qtiles;
    const uint32_t per_tile = ctas * A.split;
    const uint32_t grid = per_tile * (uint32_t)std::min<uint64_t>(tiles, (uint64_t)sms / per_tile);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (mode == kPair) return block == 16 ? launch_product<T, 16, kPair>(A, grid, smem, s) : launch_product<T, 32, kPair>(A, grid, smem, s);
        if (mode == kFew) return block == 16 ? launch_product<T, 16, kFew>(A, grid, smem, s) : launch_product<T, 32, kFew>(A, grid, smem, s);
        return block == 16 ? launch_product<T, 16, kRing>(A, grid, smem, s) : launch_product<T, 32, kRing>(A, grid, smem, s);
    };
    return dtype == GF_F32 ? go(float{}) : dtype == GF_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

gf_status check_product(uint32_t m, const void* r_packed, uint32_t n, uint32_t dim, uint32_t block, float scale, const void* out,
                        uint32_t dtype, uint64_t ld, uint32_t test_wait) {
    if (!fp4_shape(dim, block)) return fail(GF_ERR_ARG, "dim must be positive and block 16 or 32");
    if (!dtype_bytes(dtype)) return fail(GF_ERR_ARG, "unknown dtype");
    if (!std::isfinite(scale)) return fail(GF_ERR_ARG, "scale must be finite");
    if (ld < n) return fail(GF_ERR_ARG, "row stride below n");
    if (test_wait > kPolls) return fail(GF_ERR_ARG, "test_wait above 2^20");  // (it would hold the GPU for hours)
    if (m == 0 || n == 0) return GF_OK;
    if (!r_packed || !out) return fail(GF_ERR_ARG, "null argument");
    if (!aligned(r_packed, 16) || !aligned(out, dtype_bytes(dtype))) return fail(GF_ERR_ARG, "misaligned pointer");
    return GF_OK;
}

}  // namespace
}  // namespace gf

using namespace gf;

extern "C" gf_status gf_product_fp4(const void* q_packed, uint32_t m, const void* r_packed, uint32_t n, uint32_t dim,
                                    uint32_t block, float scale, void* out, uint32_t dtype, uint64_t ld, uint32_t test_wait,
                                    void* stream) {
    const gf_status st = check_product(m, r_packed, n, dim, block, scale, out, dtype, ld, test_wait);
    if (st != GF_OK || m == 0 || n == 0) return st;
    if (!q_packed) return fail(GF_ERR_ARG, "null argument");
    if (!aligned(q_packed, 16)) return fail(GF_ERR_ARG, "misaligned pointer");
    return product(ProdArgs{}, q_packed, m, r_packed, n, dim, block, scale, out, dtype, ld, test_wait, (cudaStream_t)stream);
}

extern "C" gf_status gf_product_fp4_raw(const void* q, uint32_t q_dtype, uint64_t q_ld, uint32_t m, float q_alpha,
                                        const void* r_packed, uint32_t n, uint32_t dim, uint32_t block, float scale, void* out,
                                        uint32_t dtype, uint64_t ld, void* workspace, uint32_t test_wait, void* stream) {
    const gf_status st = check_product(m, r_packed, n, dim, block, scale, out, dtype, ld, test_wait);
    if (st != GF_OK) return st;
    if (!dtype_bytes(q_dtype)) return fail(GF_ERR_ARG, "unknown dtype");
    if (!fp4_alpha(q_alpha)) return fail(GF_ERR_ARG, "alpha must lie in [2^-126, 2^126]");
    if (q_ld < dim) return fail(GF_ERR_ARG, "row stride below dim");
    if (m == 0 || n == 0) return GF_OK;
    if (!q) return fail(GF_ERR_ARG, "null argument");
    if (!aligned(q, dtype_bytes(q_dtype))) return fail(GF_ERR_ARG, "misaligned pointer");
    ProdArgs A = {};
    if (quantised_in_passing(m, dim)) {
        A.raw = q;
        A.raw_ld = q_ld;
        A.raw_dtype = q_dtype;
        A.q_alpha = q_alpha;
        return product(A, nullptr, m, r_packed, n, dim, block, scale, out, dtype, ld, test_wait, (cudaStream_t)stream);
    }
    if (!workspace) return fail(GF_ERR_ARG, "null argument: this many queries need a workspace");
    const gf_status sq = gf_quantize_fp4(q, q_dtype, q_ld, m, dim, q_alpha, block, workspace, stream);
    if (sq != GF_OK) return sq;
    return product(A, workspace, m, r_packed, n, dim, block, scale, out, dtype, ld, test_wait, (cudaStream_t)stream);
}

extern "C" gf_status gf_product_fp4_timeouts(uint64_t* count) {
    if (!count) return fail(GF_ERR_ARG, "null argument");
    unsigned long long v = 0;
    GF_CUDA(cudaMemcpyFromSymbol(&v, g_timeouts, sizeof v));
    *count = v;
    return GF_OK;
}
