// The matrix-product kernel behind tkq_block_scaled_gemm, tkq_grouped_gemm and tkq_grouped_gemm_wgrad.
//
//     out[j, i] = sum_k B[j, k] * A[i, k]          i = contiguous axis of the output
//
//   forward     i = output feature, j = row (token), k = input feature     A = weight of the row's expert, B = rows
//   rows' grad  i = input feature,  j = row,         k = output feature    A = the same weight read along its rows
//   weight grad i = input feature,  j = output feature, k = row            A = rows, B = their gradients
//
// The tensor core's M axis (128 lanes of tensor memory per CTA) carries i and its N axis carries j, whichever operand is
// the weight.  Two things follow: a thread of the epilogue owns one i, so a warp's store of one row of the output is a
// contiguous segment and needs no staging; and the ragged axis (rows of an expert) lies on N, whose extent an
// instruction chooses in steps of 16, so that a group of a few rows costs no full tile.
//
// A block: warp 0 loads operand tiles by TMA into a ring of stages, warp 1 issues the matrix instructions (accumulators in
// tensor memory, two of them, so that one is drained while the other fills), warps 2 and 3 bring scale factors into the
// layout the tensor core copies them from (or, for the weight gradient, clear the rows behind a group's end), warps 4 to
// 7 store results.  Blocks are persistent and take tiles in turn.  With CG = 2 two CTAs on neighbouring SMs work on one
// tile of 256 x N: each holds half of A's and half of B's rows, which halves the shared-memory fill per product.
#pragma once

#include <cuda_bf16.h>

#include "tkq_launch.cuh"
#include "tkq_tcgen05.cuh"

namespace tkq {

constexpr int kGemmThreads = 256;
constexpr int kMaxGroups = 1024;
constexpr uint32_t kGemmSmemBudget = 232448 - 1024 /* alignment */ - 512 /* barriers */ - 12 * (kMaxGroups + 1);

// Scale factors of one operand: the 32-bit word with the scales of row r and K-words k of group e is
// base[e * group_stride + (r >> row_shift) * row_stride + k * k_stride].
struct ScaleView {
    const uint32_t* base;
    int64_t group_stride, row_stride, k_stride;
    uint32_t row_shift;
    uint32_t words;      // words along K
    uint32_t k_shift;    // 2: a byte covers 128 values (one word per four stages), 0: 32 or 16 values
    uint32_t vec;        // the words of a row lie together on 16-byte boundaries
};

struct GemmParams {
    const int32_t* start;  // [groups] or null: one group of all rows
    const int32_t* end;
    const float* alpha;    // factor of the result, or null
    void* out;
    ScaleView sfa, sfb;
    int64_t out_stride;        // elements between rows of out
    int64_t out_group_stride;  // weight gradient: elements between the groups' results
    uint32_t groups, rows;     // rows: of the operand with the ragged axis
    uint32_t i_size, j_size;   // j_size: weight gradient only
    uint32_t i_tiles;
    uint32_t k_blocks, last_units;  // forward: stages along K, matrix instructions of the last one
    uint32_t alpha_stride;
    uint32_t out_f32, accumulate, zero_gaps, pair_stores;
};

template <int KIND_, int CG_, int NMAX_, bool WGRAD_, bool A_MN_>
struct GemmConfig {
    static constexpr int KIND = KIND_, CG = CG_, NMAX = NMAX_;
    static constexpr bool WGRAD = WGRAD_, A_MN = A_MN_, SCALED = KIND_ != kKindBf16;
    static constexpr uint32_t kBRows = NMAX / CG;
    static constexpr uint32_t kABytes = 128 * 128, kBBytes = kBRows * 128;
    static constexpr uint32_t kWords = KIND == kKindMxf8 ? 1 : KIND == kKindMxf4 ? 2 : KIND == kKindNvf4 ? 4 : 0;
    static constexpr uint32_t kSfbBlocks = (NMAX + 127) / 128;
    static constexpr uint32_t kSfaBytes = 512 * kWords, kSfbBytes = 512 * kWords * kSfbBlocks;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
    static constexpr uint32_t kStages = kGemmSmemBudget / kStageBytes < 12 ? kGemmSmemBudget / kStageBytes : 12;
    static constexpr uint32_t kSfCols = 4 * kWords * (1 + kSfbBlocks);  // tensor-memory columns of one stage's scales
    static constexpr uint32_t kSfBase = 2 * NMAX;
    static constexpr uint32_t kColsNeeded = 2 * NMAX + 2 * kSfCols;
    static constexpr uint32_t kCols = kColsNeeded <= 64 ? 64 : kColsNeeded <= 128 ? 128 : kColsNeeded <= 256 ? 256 : 512;
    static constexpr uint32_t kElems = KIND == kKindBf16 ? 64 : 128;  // tensor-map elements of a 128-byte row
    static constexpr uint32_t kNStep = CG == 2 ? 32 : 16;
    static_assert(kColsNeeded <= 512, "tensor memory");
    static_assert(!WGRAD || (A_MN && kBRows % 64 == 0), "weight gradient reads both operands along their rows");
    static_assert(kBBytes % 1024 == 0 && kStages >= 4, "stage layout");
};

struct GemmTile {
    uint32_t e, i0, j0, jn, n_mma, k0, k_blocks, k_rows;
};

__device__ unsigned int g_gemm_wait_failed = 0;

// Waits with a limit; once any role of the block has given up, the others follow within a few hundred polls.
struct GemmWait {
    volatile uint32_t* abort;
    __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
        for (uint32_t i = 0; i < kDefaultPollLimit; ++i) {
            if (mbar_try_wait_cluster(bar, parity)) return true;
            if ((i & 255u) == 255u && *abort) return false;
        }
        *abort = 1;
        atomicExch(&g_gemm_wait_failed, 1u);
        return false;
    }
};

// Rows of a group are dealt to ceil(rows / NMAX) tiles of about equal size, a multiple of the instruction's N step.
template <class C>
__device__ __forceinline__ uint32_t rows_per_tile(uint32_t rows) {
    const uint32_t t = (rows + C::NMAX - 1) / C::NMAX;
    return t == 0 ? C::kNStep : ((rows + t - 1) / t + C::kNStep - 1) / C::kNStep * C::kNStep;
}

template <class C>
struct GemmSchedule {
    const uint32_t* prefix;  // shared memory: tiles before group e
    const uint32_t* start;
    const uint32_t* rows;
    uint32_t total;

    __device__ __forceinline__ GemmTile tile(const GemmParams& p, uint32_t t) const {
        GemmTile r;
        uint32_t local, j_tiles, per;
        if constexpr (C::WGRAD) {
            per = C::NMAX;
            j_tiles = (p.j_size + per - 1) / per;
            r.e = t / (j_tiles * p.i_tiles);
            local = t - r.e * j_tiles * p.i_tiles;
        } else {
            uint32_t lo = 0, hi = p.groups;  // prefix[lo] <= t < prefix[hi]
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (prefix[mid] <= t) lo = mid;
                else hi = mid;
            }
            r.e = lo;
            local = t - prefix[lo];
            per = rows_per_tile<C>(rows[lo]);
            j_tiles = (rows[lo] + per - 1) / per;
        }
        // bands of eight tiles along j: the tiles in flight share few rows of either operand, which stay in L2
        const uint32_t band = local / (8 * p.i_tiles), rem = local - band * 8 * p.i_tiles;
        const uint32_t width = min(8u, j_tiles - band * 8);
        const uint32_t i = rem / width, j = band * 8 + rem - i * width;
        r.i0 = i * 128 * C::CG;
        const uint32_t limit = C::WGRAD ? p.j_size : rows[r.e];
        r.jn = min(per, limit - j * per);
        r.j0 = j * per + (C::WGRAD ? 0 : start[r.e]);
        r.n_mma = (r.jn + C::kNStep - 1) / C::kNStep * C::kNStep;
        r.k0 = C::WGRAD ? start[r.e] : 0;
        r.k_rows = C::WGRAD ? rows[r.e] : 0;
        r.k_blocks = C::WGRAD ? (rows[r.e] + 63) / 64 : p.k_blocks;
        return r;
    }
};

// Scale words of ROWBLK * 32 rows for one stage: lane l holds rows l, l + 32, ...
template <class C, int ROWBLK>
struct ScaleRegs {
    uint32_t w[ROWBLK][C::kWords > 0 ? C::kWords : 1];

    __device__ __forceinline__ void load(const ScaleView& v, const uint32_t* group, uint32_t row0, uint32_t row_end, uint32_t kb, uint32_t lane) {
        const uint32_t word0 = C::KIND == kKindMxf8 ? kb >> v.k_shift : kb * C::kWords;
#pragma unroll
        for (int c = 0; c < ROWBLK; ++c) {
            const uint32_t row = row0 + lane + 32u * c;
            const uint32_t* at = group + static_cast<int64_t>(row >> v.row_shift) * v.row_stride + static_cast<int64_t>(word0) * v.k_stride;
            const bool valid = row < row_end;
            if constexpr (C::kWords == 4) {
                if (v.vec && word0 + 4 <= v.words) {
                    uint4 q = valid ? __ldg(reinterpret_cast<const uint4*>(at)) : make_uint4(0, 0, 0, 0);
                    w[c][0] = q.x, w[c][1] = q.y, w[c][2] = q.z, w[c][3] = q.w;
                    continue;
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < C::kWords; ++k) w[c][k] = valid && word0 + k < v.words ? __ldg(at + k * v.k_stride) : 0u;
        }
    }

    // The tensor core copies 512-byte blocks of 128 rows: row r at (r % 32) * 16 + (r / 32) * 4.
    __device__ __forceinline__ void store(uint32_t smem, uint32_t lane) const {
        constexpr int kBlocks = (ROWBLK + 3) / 4;
#pragma unroll
        for (uint32_t k = 0; k < C::kWords; ++k)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                uint32_t q[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) q[i] = 4 * b + i < ROWBLK ? w[4 * b + i < ROWBLK ? 4 * b + i : 0][k] : 0u;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem + (k * kBlocks + b) * 512u + lane * 16u), "r"(q[0]), "r"(q[1]),
                             "r"(q[2]), "r"(q[3])
                             : "memory");
            }
    }
};

template <class C>
__global__ void __launch_bounds__(kGemmThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GemmParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[C::kStages], empty_bar[C::kStages], ready_bar[C::kStages], acc_full[2], acc_empty[2], drain_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t abort_flag;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = C::CG == 2 ? cluster_rank() : 0;
    const uint32_t unit = blockIdx.x / C::CG, units = gridDim.x / C::CG;

    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t a_base = base, b_base = a_base + C::kStages * C::kABytes, sf_base = b_base + C::kStages * C::kBBytes;
    uint32_t* group_mem = reinterpret_cast<uint32_t*>(smem_raw + (base - smem_u32(smem_raw)) + C::kStages * C::kStageBytes);
    uint32_t* s_prefix = group_mem;
    uint32_t* s_start = s_prefix + p.groups + 1;
    uint32_t* s_rows = s_start + p.groups;

    if (warp == 0) {
        if (lane == 0) {
            prefetch_tensor_map(&map_a);
            prefetch_tensor_map(&map_b);
        }
        // group table: start and rows clamped to the tensor, tiles before each group
        uint32_t before = 0;
        for (uint32_t e0 = 0; e0 < p.groups; e0 += 32) {
            const uint32_t e = e0 + lane;
            uint32_t tiles = 0;
            if (e < p.groups) {
                int64_t s = 0, t = p.rows;
                if (p.start != nullptr) {
                    s = min(max(static_cast<int64_t>(p.start[e]), int64_t{0}), static_cast<int64_t>(p.rows));
                    t = min(max(static_cast<int64_t>(p.end[e]), s), static_cast<int64_t>(p.rows));
                }
                const uint32_t rows = static_cast<uint32_t>(t - s), per = rows_per_tile<C>(rows);
                s_start[e] = static_cast<uint32_t>(s);
                s_rows[e] = rows;
                tiles = (rows + per - 1) / per * p.i_tiles;
            }
            uint32_t sum = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(kFullMask, sum, o);
                if (lane >= o) sum += up;
            }
            if (e < p.groups) s_prefix[e] = before + sum - tiles;
            before += __shfl_sync(kFullMask, sum, 31);
        }
        if (lane == 0) s_prefix[p.groups] = before;
    } else if (warp == 1) {
        if (lane == 0) {
            abort_flag = 0;
            for (uint32_t s = 0; s < C::kStages; ++s) {
                // scale loaders of every CTA arrive beside the TMA bytes; the weight gradient signals through ready_bar
                mbar_init(&full_bar[s], 1 + (C::SCALED ? 2 * C::CG : 0));
                mbar_init(&empty_bar[s], 1);
                mbar_init(&ready_bar[s], C::CG);
            }
            for (int a = 0; a < 2; ++a) {
                mbar_init(&acc_full[a], 1);
                mbar_init(&acc_empty[a], 4 * C::CG);
            }
            mbar_init(&drain_bar, 1);
        }
        __syncwarp();
        tmem_alloc<C::CG>(smem_u32(&tmem_slot), C::kCols);
    }
    tcgen05_fence_before();
    __syncthreads();
    if constexpr (C::CG == 2) cluster_sync();
    tcgen05_fence_after();

    const uint32_t tmem = tmem_slot;
    const GemmWait wait{&abort_flag};
    GemmSchedule<C> sched{s_prefix, s_start, s_rows, 0};
    sched.total = C::WGRAD ? p.groups * p.i_tiles * ((p.j_size + C::NMAX - 1) / C::NMAX) : s_prefix[p.groups];
    auto bar = [](uint64_t* b) { return smem_u32(b); };
    auto leader_bar = [&](uint64_t* b) { return C::CG == 2 ? map_to_rank(smem_u32(b), 0) : smem_u32(b); };

    if (warp == 0) {
        if (lane == 0) {
            // ---- operand tiles ----
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t t = unit; ok && t < sched.total; t += units) {
                const GemmTile tile = sched.tile(p, t);
                const int32_t i0 = static_cast<int32_t>(tile.i0 + rank * 128u);
                const int32_t j0 = static_cast<int32_t>(tile.j0 + (C::CG == 2 ? rank * (tile.n_mma / 2) : 0));
                for (uint32_t kb = 0; kb < tile.k_blocks; ++kb, ++it) {
                    const uint32_t s = it % C::kStages;
                    if (!(ok = wait(bar(&empty_bar[s]), ((it / C::kStages) & 1u) ^ 1u))) break;
                    uint32_t full;
                    if constexpr (C::WGRAD) {
                        full = bar(&full_bar[s]);
                        mbar_arrive_expect_tx(&full_bar[s], C::kABytes + C::kBBytes);
                    } else {
                        full = leader_bar(&full_bar[s]);
                        if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], C::CG * (C::kABytes + C::kBBytes));
                    }
                    const uint32_t a = a_base + s * C::kABytes, b = b_base + s * C::kBBytes;
                    const int32_t k = static_cast<int32_t>(tile.k0 + kb * C::kElems);
                    if constexpr (C::A_MN) {
                        const int32_t z = C::WGRAD ? 0 : static_cast<int32_t>(tile.e);
                        tma_load_3d<C::CG>(a, &map_a, i0, k, z, full);
                        tma_load_3d<C::CG>(a + 8192, &map_a, i0 + 64, k, z, full);
                    } else {
                        tma_load_3d<C::CG>(a, &map_a, k, i0, static_cast<int32_t>(tile.e), full);
                    }
                    if constexpr (C::WGRAD) {
#pragma unroll
                        for (uint32_t q = 0; q < C::kBRows / 64; ++q)
                            tma_load_3d<C::CG>(b + q * 8192, &map_b, j0 + static_cast<int32_t>(64 * q), k, 0, full);
                    } else {
                        tma_load_3d<C::CG>(b, &map_b, k, j0, 0, full);
                    }
                }
            }
            // every stage that was filled has been read before the block may end
            for (uint32_t n = 0; n < C::kStages && n < it; ++n) {
                const uint32_t q = it - 1 - n;
                if (ok) ok = wait(bar(&empty_bar[q % C::kStages]), (q / C::kStages) & 1u);
                else if (C::WGRAD || rank == 0) mbar_wait(&full_bar[q % C::kStages], (q / C::kStages) & 1u, 1u << 16);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && lane == 0) {
            // ---- matrix instructions ----
            constexpr uint32_t kM = 128 * C::CG;
            uint32_t it = 0, acc_it = 0;
            bool ok = true;
            for (uint32_t t = unit; ok && t < sched.total; t += units) {
                const GemmTile tile = sched.tile(p, t);
                if (tile.k_blocks == 0) continue;
                const uint32_t a = acc_it & 1u;
                if (!(ok = wait(bar(&acc_empty[a]), ((acc_it >> 1) & 1u) ^ 1u))) break;
                ++acc_it;
                tcgen05_fence_after();
                const uint32_t d = tmem + a * C::NMAX;
                uint32_t idesc;
                if constexpr (C::SCALED) idesc = idesc_scaled(kM, tile.n_mma, C::KIND == kKindMxf8 ? 0 : 1, C::KIND != kKindNvf4);
                else idesc = idesc_bf16(kM, tile.n_mma, C::A_MN, C::WGRAD);
                for (uint32_t kb = 0; kb < tile.k_blocks; ++kb, ++it) {
                    const uint32_t s = it % C::kStages, phase = (it / C::kStages) & 1u;
                    if (!(ok = wait(bar(C::WGRAD ? &ready_bar[s] : &full_bar[s]), phase))) break;
                    tcgen05_fence_after();
                    const uint32_t sfa = tmem + C::kSfBase + (it & 1u) * C::kSfCols, sfb = sfa + 4 * C::kWords;
                    if constexpr (C::SCALED) {
                        // the copies overwrite the scales of two stages ago: its products have to be finished
                        if (it >= 2) {
                            const uint32_t q = it - 2;
                            if (!(ok = wait(bar(&empty_bar[q % C::kStages]), (q / C::kStages) & 1u))) break;
                            tcgen05_fence_after();
                        }
                        const uint32_t sf = sf_base + s * (C::kSfaBytes + C::kSfbBytes);
#pragma unroll
                        for (uint32_t w = 0; w < C::kWords; ++w) {
                            tcgen05_copy_scales<C::CG>(sfa + 4 * w, smem_desc(sf + 512 * w, 16, 128, 0));
#pragma unroll
                            for (uint32_t b = 0; b < C::kSfbBlocks; ++b)
                                tcgen05_copy_scales<C::CG>(sfb + 4 * (w * C::kSfbBlocks + b),
                                                           smem_desc(sf + C::kSfaBytes + 512 * (w * C::kSfbBlocks + b), 16, 128, 0));
                        }
                    }
                    const uint32_t sa = a_base + s * C::kABytes, sb = b_base + s * C::kBBytes;
                    uint64_t da, db;
                    if constexpr (C::A_MN) da = smem_desc(sa, 8192, 1024, kSwizzle128);
                    else da = smem_desc(sa, 16, 1024, kSwizzle128);
                    if constexpr (C::WGRAD) db = smem_desc(sb, 8192, 1024, kSwizzle128);
                    else db = smem_desc(sb, 16, 1024, kSwizzle128);
                    // a step along K: 32 bytes of a K-major row, or 16 rows of 128 bytes
                    constexpr uint32_t kStepA = (C::A_MN ? 2048 : 32) >> 4, kStepB = (C::WGRAD ? 2048 : 32) >> 4;
                    uint32_t n_units = 4;
                    if (kb + 1 == tile.k_blocks) n_units = C::WGRAD ? (tile.k_rows - kb * 64 + 15) / 16 : p.last_units;
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) {
                        if (u >= n_units) break;
                        uint32_t id = idesc, fa = sfa, fb = sfb;
                        if constexpr (C::KIND == kKindMxf8)
                            id |= idesc_scale_ids(p.sfa.k_shift ? kb & 3u : u, p.sfb.k_shift ? kb & 3u : u);
                        if constexpr (C::KIND == kKindMxf4) {
                            id |= idesc_scale_ids((u & 1u) * 2, (u & 1u) * 2);
                            fa += 4 * (u >> 1);
                            fb += 4 * C::kSfbBlocks * (u >> 1);
                        }
                        if constexpr (C::KIND == kKindNvf4) {
                            fa += 4 * u;
                            fb += 4 * C::kSfbBlocks * u;
                        }
                        tcgen05_mma<C::KIND, C::CG>(d, da + u * kStepA, db + u * kStepB, id, fa, fb, kb > 0 || u > 0);
                    }
                    tcgen05_commit<C::CG>(bar(&empty_bar[s]));
                }
                if (ok) tcgen05_commit<C::CG>(bar(&acc_full[a]));
            }
            if (!ok) {  // products in flight end before the memory they use is given up
                tcgen05_commit<C::CG>(bar(&drain_bar));
                mbar_wait(&drain_bar, 0, 1u << 16);
            }
        }
    } else if (warp < 4) {
        if constexpr (C::SCALED) {
            // ---- scale factors: warp 2 those of A, warp 3 those of B; two stages of loads ahead of the stores ----
            auto run = [&](auto regs_tag, const ScaleView& v, uint32_t smem_off, bool is_a) {
                using Regs = decltype(regs_tag);
                uint32_t it = 0;
                bool ok = true;
                for (uint32_t t = unit; ok && t < sched.total; t += units) {
                    const GemmTile tile = sched.tile(p, t);
                    const uint32_t* group = v.base + (is_a ? static_cast<int64_t>(tile.e) * v.group_stride : 0);
                    const uint32_t row0 = is_a ? tile.i0 + rank * 128u : tile.j0, row_end = is_a ? p.i_size : tile.j0 + tile.jn;
                    Regs r[3];
                    r[0].load(v, group, row0, row_end, 0, lane);
                    if (tile.k_blocks > 1) r[1].load(v, group, row0, row_end, 1, lane);
                    for (uint32_t kb = 0; kb < tile.k_blocks; kb += 3) {
#pragma unroll
                        for (uint32_t u = 0; u < 3; ++u) {
                            if (kb + u >= tile.k_blocks) break;
                            if (kb + u + 2 < tile.k_blocks) r[(u + 2) % 3].load(v, group, row0, row_end, kb + u + 2, lane);
                            const uint32_t s = it % C::kStages;
                            ok = wait(bar(&empty_bar[s]), ((it / C::kStages) & 1u) ^ 1u);
                            if (!__all_sync(kFullMask, ok)) return;
                            r[u].store(sf_base + s * (C::kSfaBytes + C::kSfbBytes) + smem_off, lane);
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) mbar_arrive_cluster(C::CG == 2 ? map_to_rank(bar(&full_bar[s]), 0) : bar(&full_bar[s]));
                            ++it;
                        }
                    }
                }
            };
            if (warp == 2) run(ScaleRegs<C, 4>{}, p.sfa, 0, true);
            else run(ScaleRegs<C, (C::NMAX + 31) / 32>{}, p.sfb, C::kSfaBytes, false);
        } else if constexpr (C::WGRAD) {
            // ---- rows behind the group's end: the last stage's tail belongs to another group (or to nobody) and is cleared in
            // both operands, so that not even an infinity there can reach the sum ----
            if (warp == 2) {
                uint32_t it = 0;
                for (uint32_t t = unit; t < sched.total; t += units) {
                    const GemmTile tile = sched.tile(p, t);
                    for (uint32_t kb = 0; kb < tile.k_blocks; ++kb, ++it) {
                        const uint32_t s = it % C::kStages;
                        const bool ok = wait(bar(&full_bar[s]), (it / C::kStages) & 1u);
                        if (!__all_sync(kFullMask, ok)) goto done;
                        const uint32_t valid = min(64u, tile.k_rows - kb * 64), padded = (valid + 15) / 16 * 16;
                        if (valid < padded) {
                            const uint32_t chunks = (padded - valid) * 8;
                            for (uint32_t box = 0; box < 2 + C::kBRows / 64; ++box) {
                                const uint32_t at = (box < 2 ? a_base + s * C::kABytes + box * 8192 : b_base + s * C::kBBytes + (box - 2) * 8192) + valid * 128;
                                for (uint32_t q = lane; q < chunks; q += 32)
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + q * 16), "r"(0) : "memory");
                            }
                            fence_proxy_async_smem();
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(C::CG == 2 ? map_to_rank(bar(&ready_bar[s]), 0) : bar(&ready_bar[s]));
                    }
                }
            done:;
            }
        }
    } else {
        // ---- results ----
        const uint32_t quarter = warp & 3u;
        uint32_t acc_it = 0;
        for (uint32_t t = unit; t < sched.total; t += units) {
            const GemmTile tile = sched.tile(p, t);
            const uint32_t a = acc_it & 1u;
            const bool have = tile.k_blocks > 0;
            if (!have && p.accumulate) continue;
            if (have) {
                const bool ok = wait(bar(&acc_full[a]), (acc_it >> 1) & 1u);
                if (!__all_sync(kFullMask, ok)) break;
                ++acc_it;
                tcgen05_fence_after();
            }
            const float alpha = p.alpha == nullptr ? 1.0f : __ldg(p.alpha + static_cast<int64_t>(tile.e) * p.alpha_stride);
            const uint32_t iw = tile.i0 + rank * 128u + quarter * 32u;  // the warp's first column of the output
            const uint32_t taddr = tmem + a * C::NMAX + (quarter << 21);
            for (uint32_t c = 0; c < tile.jn; c += 32) {
                uint32_t v[32];
                if (have) {
                    tmem_load32(taddr + c, v);
                    tmem_load_wait();
                } else {
#pragma unroll
                    for (int q = 0; q < 32; ++q) v[q] = 0;
                }
                const int64_t off = static_cast<int64_t>(tile.e) * p.out_group_stride + static_cast<int64_t>(tile.j0 + c) * p.out_stride;
                const uint32_t n = min(32u, tile.jn - c);
                if (C::WGRAD && p.out_f32) {
                    float* o = static_cast<float*>(p.out) + off + iw + lane;
                    if (iw + lane < p.i_size) {
#pragma unroll
                        for (uint32_t q = 0; q < 32; ++q)
                            if (q < n) {
                                float x = __uint_as_float(v[q]);
                                if (p.accumulate) x += o[q * p.out_stride];
                                o[q * p.out_stride] = x;
                            }
                    }
                } else {
                    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + off;
                    if (p.pair_stores) {
                        // two rows per step: lanes 0..15 store pairs of columns of row q, lanes 16..31 of row q + 1
                        const uint32_t col = iw + 2 * (lane & 15u), src = 2 * (lane & 15u), upper = lane >> 4;
#pragma unroll
                        for (uint32_t q = 0; q < 32; q += 2) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(__fmul_rn(__uint_as_float(v[q]), alpha), __fmul_rn(__uint_as_float(v[q + 1]), alpha));
                            const uint32_t mine = *reinterpret_cast<const uint32_t*>(&h);
                            const uint32_t x = __shfl_sync(kFullMask, mine, src), y = __shfl_sync(kFullMask, mine, src + 1);
                            const uint32_t w = __byte_perm(x, y, upper ? 0x7632 : 0x5410);
                            if (q + upper < n && col < p.i_size) *reinterpret_cast<uint32_t*>(o + (q + upper) * p.out_stride + col) = w;
                        }
                    } else if (iw + lane < p.i_size) {
#pragma unroll
                        for (uint32_t q = 0; q < 32; ++q)
                            if (q < n) o[q * p.out_stride + iw + lane] = __float2bfloat16_rn(__fmul_rn(__uint_as_float(v[q]), alpha));
                    }
                }
            }
            if (have) {
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(C::CG == 2 ? map_to_rank(bar(&acc_empty[a]), 0) : bar(&acc_empty[a]));
            }
        }
        if (!C::WGRAD && p.zero_gaps) {
            // rows of no group: before the first, between two, behind the last
            const uint32_t w0 = blockIdx.x * 4 + quarter, nw = gridDim.x * 4;
            const bool wide = (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0 && (p.out_stride & 7) == 0;
            const uint32_t full8 = wide ? p.i_size / 8 : 0;
            for (uint32_t g = 0; g <= p.groups; ++g) {
                const uint32_t lo = g == 0 ? 0 : s_start[g - 1] + s_rows[g - 1], hi = g == p.groups ? p.rows : s_start[g];
                for (uint32_t r = lo + w0; r < hi; r += nw) {
                    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(r) * p.out_stride;
                    for (uint32_t q = lane; q < full8; q += 32) *reinterpret_cast<uint4*>(o + 8 * q) = make_uint4(0, 0, 0, 0);
                    for (uint32_t q = full8 * 8 + lane; q < p.i_size; q += 32) o[q] = __float2bfloat16_rn(0.0f);
                }
            }
        }
    }

    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if constexpr (C::CG == 2) cluster_sync();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc<C::CG>(tmem, C::kCols);
    }
    if constexpr (C::CG == 2) cluster_sync();
}

}  // namespace tkq
