// Building blocks of the matrix-product kernels: mbarriers in a cluster, tensor-map loads that a CTA pair shares, the
// fifth-generation tensor-core instructions (tcgen05) and their descriptors.  sm_100a only, no TMA multicast.
#pragma once

#include "tkq_async.cuh"

namespace tkq {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Address, in the cluster's shared window, of the same variable in CTA `rank`.
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}

// Arrival at a barrier of any CTA of the cluster (address from map_to_rank).  What it announces is shared or tensor memory
// of the arriving thread's own SM, ordered by a proxy or tcgen05 fence before it.  Its scope is the default one, the CTA; with
// .release.cluster the same arrival waits for the thread's global loads and costs about a microsecond (16384 x 4096 x 7168 MXFP4:
// 511 us with it, 377 us without).  So for the other CTA of a pair the order rests on those fences and on how the hardware carries
// them out, which PTX's memory model does not spell out for this scope; test_many_waves compares every result that depends on it.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t addr, uint32_t parity) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done)
                 : "r"(addr), "r"(parity)
                 : "memory");
    return done != 0;
}

__device__ __forceinline__ void prefetch_tensor_map(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Tile loads of a three-dimensional tensor; x * element size is a multiple of 16 bytes.  With CG = 2 the barrier may
// belong to either CTA of the pair.
template <int CG>
__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* tmap, int32_t x, int32_t y, int32_t z, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                smem_dst),
            "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst),
            "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}

// ---------------------------------------------------------------------------
// Tensor memory
// ---------------------------------------------------------------------------
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, uint32_t columns) {  // one whole warp
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}

template <int CG>
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t columns) {  // the warp that allocated
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(columns));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(columns));
}

__device__ __forceinline__ void tcgen05_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 lanes x 32 columns of 32 bits: register c of lane l is column c of the warp's l-th lane.
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// 16 lanes x 32 columns as 8 x 8 matrices: registers 4x and 4x + 1 of lane l are columns 8x + 2 (l % 4) and the next of
// lane l / 4, registers 4x + 2 and 4x + 3 those of lane 8 + l / 4.
__device__ __forceinline__ void tmem_load_16x32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---------------------------------------------------------------------------
// Descriptors
// ---------------------------------------------------------------------------
constexpr uint64_t kSwizzle128 = uint64_t{2} << 61;
constexpr uint64_t kDescVersion = uint64_t{1} << 46;

// Shared-memory operand: `lbo` and `sbo` in bytes.
//   K-major, 128-byte swizzle: rows of 128 bytes, 8-row atoms `sbo` apart (lbo unused)
//   MN-major, 128-byte swizzle: 64 16-bit elements of the M or N axis per 128-byte row, `lbo` to the next 64, `sbo` to
//   the next 8 values of K
//   no swizzle (scale factors): 16-byte rows, 8-row groups `sbo` apart
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo, uint64_t swizzle) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | (static_cast<uint64_t>((lbo >> 4) & 0x3fffu) << 16) |
           (static_cast<uint64_t>((sbo >> 4) & 0x3fffu) << 32) | kDescVersion | swizzle;
}

// Instruction descriptor, kind::f16 with bf16 operands and fp32 accumulation.
__device__ __forceinline__ constexpr uint32_t idesc_bf16(uint32_t m, uint32_t n, bool a_mn_major, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_mn_major) << 15) | (static_cast<uint32_t>(b_mn_major) << 16) |
           ((n >> 3) << 17) | ((m >> 4) << 24);
}

// Instruction descriptor of the block-scaled kinds, without the scale ids.  `fmt`: 0 e4m3 (kind mxf8f6f4), 1 e2m1 (the
// four-bit kinds); `ue8m0`: type of the scales.
__device__ __forceinline__ constexpr uint32_t idesc_scaled(uint32_t m, uint32_t n, uint32_t fmt, bool ue8m0) {
    return (fmt << 7) | (fmt << 10) | ((n >> 3) << 17) | (static_cast<uint32_t>(ue8m0) << 23) | ((m >> 7) << 27);
}

// Which byte of the 32-bit scale cells an instruction starts at.
__device__ __forceinline__ uint32_t idesc_scale_ids(uint32_t a_id, uint32_t b_id) { return (b_id << 4) | (a_id << 29); }

// ---------------------------------------------------------------------------
// Matrix instructions; one thread issues them
// ---------------------------------------------------------------------------
constexpr int kKindBf16 = 0, kKindMxf8 = 1, kKindMxf4 = 2, kKindNvf4 = 3;

// The issuing functions are called by whole warps, with `one` true in a single lane: predicated instructions in
// uniform control flow take their descriptors from uniform registers as they are, where a branch for one lane moves every
// operand there first (about 60 cycles per instruction: 390 against 290 cycles for the four products of a bf16 stage).
template <int KIND, int CG>
__device__ __forceinline__ void tcgen05_mma(bool one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate) {
    const uint32_t acc = accumulate ? 1u : 0u, e = one ? 1u : 0u;
#define TKQ_MMA_PLAIN(CGS, KINDS)                                                                                                     \
    asm volatile("{ .reg .pred e, p; setp.ne.b32 p, %4, 0; setp.ne.b32 e, %5, 0; @e tcgen05.mma.cta_group::" CGS ".kind::" KINDS     \
                 " [%0], %1, %2, %3, p; }" ::"r"(d),                                                                                  \
                 "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(e)                                                                         \
                 : "memory")
#define TKQ_MMA_SCALED(CGS, KINDS)                                                                                                    \
    asm volatile("{ .reg .pred e, p; setp.ne.b32 p, %6, 0; setp.ne.b32 e, %7, 0; @e tcgen05.mma.cta_group::" CGS ".kind::" KINDS     \
                 " [%0], %1, %2, %3, [%4], [%5], p; }" ::"r"(d),                                                                      \
                 "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc), "r"(e)                                                     \
                 : "memory")
    if constexpr (KIND == kKindBf16) {
        if constexpr (CG == 2) TKQ_MMA_PLAIN("2", "f16");
        else TKQ_MMA_PLAIN("1", "f16");
    } else if constexpr (KIND == kKindMxf8) {
        if constexpr (CG == 2) TKQ_MMA_SCALED("2", "mxf8f6f4.block_scale.scale_vec::1X");
        else TKQ_MMA_SCALED("1", "mxf8f6f4.block_scale.scale_vec::1X");
    } else if constexpr (KIND == kKindMxf4) {
        if constexpr (CG == 2) TKQ_MMA_SCALED("2", "mxf4.block_scale.scale_vec::2X");
        else TKQ_MMA_SCALED("1", "mxf4.block_scale.scale_vec::2X");
    } else {
        if constexpr (CG == 2) TKQ_MMA_SCALED("2", "mxf4nvf4.block_scale.scale_vec::4X");
        else TKQ_MMA_SCALED("1", "mxf4nvf4.block_scale.scale_vec::4X");
    }
#undef TKQ_MMA_PLAIN
#undef TKQ_MMA_SCALED
}

// 512 bytes of scales (32 rows of 16 bytes) -> 4 columns x 32 lanes, repeated for the four lane quarters.  With CG = 2
// each CTA of the pair copies from its own shared memory into its own tensor memory.
template <int CG>
__device__ __forceinline__ void tcgen05_copy_scales(bool one, uint32_t taddr, uint64_t desc) {
    const uint32_t e = one ? 1u : 0u;
    if constexpr (CG == 2)
        asm volatile("{ .reg .pred e; setp.ne.b32 e, %2, 0; @e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1; }" ::"r"(taddr), "l"(desc), "r"(e)
                     : "memory");
    else
        asm volatile("{ .reg .pred e; setp.ne.b32 e, %2, 0; @e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1; }" ::"r"(taddr), "l"(desc), "r"(e)
                     : "memory");
}

// One arrival at `bar` (CG = 2: at the same barrier of both CTAs of the pair) once every tcgen05 operation this thread
// has issued so far is complete.
template <int CG>
__device__ __forceinline__ void tcgen05_commit(bool one, uint32_t bar) {
    const uint32_t e = one ? 1u : 0u;
    if constexpr (CG == 2)
        asm volatile(
            "{ .reg .pred e; setp.ne.b32 e, %2, 0; @e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], "
            "%1; }" ::"r"(bar),
            "h"(static_cast<uint16_t>(3)), "r"(e)
            : "memory");
    else
        asm volatile("{ .reg .pred e; setp.ne.b32 e, %1, 0; @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar),
                     "r"(e)
                     : "memory");
}

}  // namespace tkq
