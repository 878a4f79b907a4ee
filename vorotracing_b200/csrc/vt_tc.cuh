// vt_tc.cuh -- tensor-core plumbing for sm_100a: mbarriers, TMA tile loads,
// tensor memory and tcgen05 products.  Thin wrappers over PTX; one kernel file
// decides what they move.
//
// Every wait has an end.  A wait that lasts a second gives up, marks the CTA as
// failed in shared memory and writes VT_ERR_CUDA to the caller's error word; all
// other waits of that CTA then return too, its roles run to their ends, the
// producer waits (as long again at most) for the copies it has in flight, and
// tensor memory is freed.  The outputs of such a launch are not valid.
#pragma once

#include <cuda.h>

#include <atomic>

#include "vt_abi.cuh"
#include "vt_ring.cuh"
#include "vt_wait.cuh"

namespace vt {
namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- mbarriers ----

struct Fail {  // in shared memory, one a CTA
    volatile uint32_t failed;
};

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(uint64_t *bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok;
}
// Waits are timed by the SM's clock (vt_wait.cuh).  Reading %globaltimer instead takes about a microsecond, which
// every wait that is not over at once would pay.
static __device__ __noinline__ bool mbar_wait_slow(uint64_t *bar, uint32_t parity, Fail *fail, uint32_t *err, bool last)
{
    WaitTime time(clock64());
    for (;;) {
        for (int i = 0; i < 64; ++i)
            if (mbar_try(bar, parity)) return true;
        if (fail->failed && !last) return false;
        if (time.over(clock64())) {
            fail->failed = 1;
            if (err) *(volatile uint32_t *)err = VT_ERR_CUDA;  // a plain store: the word may be the host's
            return false;
        }
    }
}
// Waits for the phase of that parity to end; false: given up.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, Fail *fail, uint32_t *err)
{
    for (int i = 0; i < 16; ++i)
        if (mbar_try(bar, parity)) return true;
    return mbar_wait_slow(bar, parity, fail, err, false);
}

// Far longer than a copy takes: for copies in flight that no barrier tells of.
__device__ __forceinline__ void outlast_copies()
{
    const long long began = clock64();
    while (clock64() - began < WAIT_LIMIT / 100) {}
}

// ---- TMA ----

__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
// Contiguous bytes: addresses and size multiples of 16
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap *map)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// Shared-memory writes of this thread before, reads by TMA or tcgen05 after.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory ----

template <uint32_t COLS> __device__ __forceinline__ void tmem_alloc(uint32_t *slot)  // one warp
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <uint32_t COLS> __device__ __forceinline__ void tmem_free(uint32_t base)  // the same warp
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: lane l gets row l of its quadrant.  The load and its wait are
// one statement: arithmetic on the results could be moved before a wait of its own.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t *r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of a converged warp, the same each time.  Roles run with their whole warp and only
// their asynchronous instructions under it, so that addresses and descriptors stay in uniform
// registers, where those instructions want them.
__device__ __forceinline__ bool elect()
{
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p;
}
// The warp's number in its block, known to be the same in all its lanes
__device__ __forceinline__ uint32_t warp_number() { return __shfl_sync(~0u, threadIdx.x / 32u, 0); }

// ---- products ----

// Shared-memory operand in the 128-byte swizzle.  Atoms are 8 rows of 128 bytes (1024-byte
// aligned).  K-major operand: rows are the operand's rows, stride = bytes from 8 rows to the
// next 8, lead unused.  MN-major operand: rows are steps of k, stride = bytes from 8 steps of k
// to the next 8, lead = bytes from 64 rows of the operand to the next 64.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride)
{
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}
// Instruction descriptor of kind::f16, binary32 accumulators.  mn: the operand is MN-major.
template <bool BF16> __host__ __device__ constexpr uint32_t idesc_f16(uint32_t m, uint32_t n, bool a_mn, bool b_mn)
{
    return 1u << 4 | (BF16 ? 1u : 0u) << 7 | (BF16 ? 1u : 0u) << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 |
           (n >> 3) << 17 | (m >> 4) << 24;
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
// Shared-memory source of tmem_copy_scales: 32 rows of 16 bytes, unswizzled.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr)
{
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(128u >> 4) << 32 | 1ull << 46;
}
// 512 bytes of shared memory to 4 columns of tensor memory, the same 32 lanes four times: the
// scales of 128 rows of an operand and 4 blocks of k.  Row r and block b are byte b of word r / 32
// of the 16 bytes at 16 (r % 32).  Copies and products of one thread run in the order of issue.
__device__ __forceinline__ void tmem_copy_scales(uint32_t d, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(d), "l"(desc) : "memory");
}
// Instruction descriptor of kind::mxf4: e2m1 operands, power-of-two scales for blocks of 32,
// binary32 accumulators.  pair: which two of a word's four scales the product's 64 steps of k take.
__host__ __device__ constexpr uint32_t idesc_mxf4(uint32_t m, uint32_t n, uint32_t pair)
{
    return (2u * pair) << 4 | 1u << 7 | 1u << 10 | (n >> 3) << 17 | 1u << 23 | (m >> 7) << 27 | (2u * pair) << 29;
}
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b,
                                         bool accumulate)
{
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"((uint32_t)accumulate) : "memory");
}
// The same with A (M rows in the lanes, two 16-bit steps of k a column) in tensor memory.
__device__ __forceinline__ void mma_f16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
// The same for one half of the lanes of D (0..63 or 64..127); the other half keeps its values.
__device__ __forceinline__ void mma_f16_tmem_half(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool upper, bool accumulate)
{
    const uint32_t off01 = upper ? ~0u : 0u, off23 = ~off01;  // a set bit: this lane is not written
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %6, %6}, p;\n}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(off01), "r"(off23) : "memory");
}
// The barrier gets one arrival when the products issued so far by this thread are done.
__device__ __forceinline__ void commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// ---- pairs of CTAs (clusters of two): one product of 256 rows over both SMs ----
//
// Each CTA stages its 128 rows of A and its half of B's columns; the leader (rank 0) issues the
// products, which read both CTAs' shared memory at the same offsets and leave each CTA its own
// 128 rows of the result.

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// This CTA's shared-memory word, read in the cluster's CTA of that rank
__device__ __forceinline__ float load_cluster(const float *p, uint32_t rank)
{
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
// Address of the leader's copy of a shared-memory object
__device__ __forceinline__ uint32_t leader_addr(const void *p)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
    return a;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Into this CTA's shared memory; the bytes are counted by a barrier of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <uint32_t COLS> __device__ __forceinline__ void tmem_alloc_pair(uint32_t *slot)  // one warp of each CTA
{
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
template <uint32_t COLS> __device__ __forceinline__ void tmem_free_pair(uint32_t base)
{
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS));
}
__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
// Block-scaled 4-bit products of a pair: each CTA's tensor memory has the scales of its own 128 rows of A
// and of all of B's columns.  The copy runs in both CTAs, from and to the same places of each.
__device__ __forceinline__ void tmem_copy_scales_pair(uint32_t d, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(d), "l"(desc) : "memory");
}
__device__ __forceinline__ void mma_mxf4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b,
                                              bool accumulate)
{
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"((uint32_t)accumulate) : "memory");
}
// One arrival at the barrier of this offset in both CTAs when the leader's products so far are done.
__device__ __forceinline__ void commit_pair(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

// ---- host: tensor maps ----

// A row-major matrix (rows, cols) of `bytes`-wide elements with a row pitch in bytes, read in
// boxes of (box_rows, box_cols), by default with 128-byte swizzle; outside of the matrix zeros are read.
vt_status make_map(CUtensorMap *map, CUtensorMapDataType type, const void *p, uint64_t rows, uint64_t cols,
                   uint64_t pitch, uint32_t box_rows, uint32_t box_cols, bool swizzle = true);

// The same matrix as column chunks of `box_cols` side by side, all of them in one box, which
// lie one behind the other in shared memory.  The chunks have to make up whole rows.
vt_status make_chunk_map(CUtensorMap *map, CUtensorMapDataType type, const void *p, uint64_t rows, uint32_t chunks,
                         uint64_t pitch, uint32_t box_rows, uint32_t box_cols, uint32_t bytes);

// Lets a kernel have more shared memory than 48 KB, once a device.
template <typename K> inline vt_status allow_smem(K kernel, uint32_t bytes, std::atomic<uint64_t> &done)
{
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return VT_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(VT_ERR_CUDA, "%u bytes of shared memory: %s", bytes, cudaGetErrorString(e));
    }
    done.fetch_or(bit, std::memory_order_relaxed);
    return VT_OK;
}

}  // namespace tc
}  // namespace vt
