// The matrix-product kernel behind tkq_block_scaled_gemm, tkq_grouped_gemm and tkq_grouped_gemm_wgrad.
//
//     out[j, i] = sum_k B[j, k] * A[i, k]          i = contiguous axis of the output
//
//   forward     i = output feature, j = row (token), k = input feature     A = weight of the row's expert, B = rows
//   rows' grad  i = input feature,  j = row,         k = output feature    A = the same weight read along its rows
//   weight grad i = input feature,  j = output feature, k = row            A = rows, B = their gradients
//
// The tensor core's M axis (128 lanes of tensor memory per CTA) carries i and its N axis carries j, whichever operand is
// the weight, so that the ragged axis (rows of an expert) lies on N, whose extent an instruction chooses in steps of 16: a
// group of a few rows costs no full tile.  A warp of the epilogue has 32 neighbouring columns of the output in its lanes.
//
// A block: warp 0 loads operand tiles by TMA into a ring of stages, warp 1 issues the matrix instructions (accumulators in
// tensor memory, two of them, so that one is drained while the other fills), the next warps bring scale factors into the
// layout the tensor core copies them from (or, for the weight gradient, clear the rows behind a group's end), the last four
// or eight store results.  Blocks are persistent and take tiles in turn.  With CG = 2 two CTAs on neighbouring SMs work on
// one tile of 256 x N: each holds half of A's and half of B's rows, which halves the shared-memory fill per product.
//
// With few tiles (one token through one matrix, the gradient of a small weight) K is split over a cluster of CTAs: each multiplies its part of K, hands
// its sums to the CTAs that own the columns, through their shared memory, and those add them in the order of the parts.
#pragma once

#include <cuda_bf16.h>

#include "tkq_launch.cuh"
#include "tkq_tcgen05.cuh"

namespace tkq {

constexpr int kMaxGroups = 1024;
constexpr uint32_t kGemmSmemBudget = 232448 - 1024 /* alignment */ - 512 /* barriers */;

// Scale factors of one operand: the 32-bit word with the scales of row r and K-words k of group e is
// base[e * group_stride + (r >> row_shift) * row_stride + k * k_stride].
struct ScaleView {
    const uint32_t* base;
    int64_t group_stride, row_stride, k_stride;
    uint32_t row_shift;
    uint32_t words;      // words along K
    uint32_t k_shift;    // 2: a byte covers 128 values (one word for two stages), 0: 32 or 16 values
    uint32_t vec;        // the words of a row lie together on 32-byte boundaries
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
    uint32_t k_stages, last_units;  // forward: stages along K, matrix instructions of the last one
    uint32_t alpha_stride;
    uint32_t split;  // CTAs of a cluster that share a tile along K
    uint32_t accumulate, zero_gaps;
    uint32_t out_bf16;  // weight gradient split along K: bf16 results
    uint32_t wide_out;  // rows of out on 16-byte boundaries and i_size a multiple of 8
};

// Where the weight gradient's sums go on in registers (see add_f32), and what becomes of them
constexpr int kSumsNone = 0, kSumsF32 = 1, kSumsAccumulate = 2, kSumsBf16 = 3;

template <int KIND_, int CG_, int NMAX_, bool WGRAD_, bool A_MN_, bool SPLIT_ = false, int SUMS_ = kSumsNone>
struct GemmConfig {
    static constexpr int KIND = KIND_, CG = CG_, NMAX = NMAX_;
    static constexpr bool WGRAD = WGRAD_, A_MN = A_MN_, SCALED = KIND_ != kKindBf16, SPLIT = SPLIT_;
    static constexpr int SUMS = SUMS_;
    static constexpr bool F32 = SUMS != kSumsNone;
    // stages whose products the tensor core adds up before the sum goes on in registers
    static constexpr uint32_t kChunk = !F32 ? 1u << 30 : SUMS == kSumsBf16 ? 64 : 4;
    // A stage holds kSub blocks of 128 bytes along K.  Waiting for a stage and handing it back costs the issuing warp some
    // 200 cycles: two thirds of a block's products in 4 or 8 bits (448 cycles at N = 224), which therefore come in pairs
    static constexpr uint32_t kSub = SCALED ? 2 : 1;
    static constexpr uint32_t kBRows = NMAX / CG;
    static constexpr uint32_t kABytes = 128 * 128, kBBytes = kBRows * 128;  // of one block
    static constexpr uint32_t kWords = KIND == kKindMxf8 ? 1 : KIND == kKindMxf4 ? 2 : KIND == kKindNvf4 ? 4 : 0;
    static constexpr uint32_t kSfbBlocks = (NMAX + 127) / 128;
    static constexpr uint32_t kSfaBytes = 512 * kWords, kSfbBytes = 512 * kWords * kSfbBlocks;
    static constexpr uint32_t kStageBytes = kSub * (kABytes + kBBytes + kSfaBytes + kSfbBytes);
    // Scale loaders: one warp per block of 128 rows (of A, and one or two of B), in sets that take stages in turn
    static constexpr uint32_t kScaleBlocks = SCALED ? 1 + (NMAX + 127) / 128 : 1, kScaleSets = SCALED ? 6 / kScaleBlocks : 1;
    static constexpr uint32_t kLoaders = SCALED ? 6 : 2;  // warps between the two issuing ones and those that store results
    static constexpr uint32_t kFirstResultWarp = 2 + kLoaders, kResultWarps = F32 ? 8 : 4;
    static constexpr uint32_t kThreads = 32 * (kFirstResultWarp + kResultWarps);
    static constexpr uint32_t kStagingPerWarp = F32 ? 0 : SCALED ? 2048 : 4096, kStagingBytes = kStagingPerWarp * kResultWarps;
    // split products: the parts' sums as [part][own column][row], columns padded so that 16-byte accesses meet no bank twice
    static constexpr uint32_t kPartialPitch = NMAX + 4, kPartialBytes = SPLIT ? 128 * kPartialPitch * 4 : 0;
    // (NVFP4 with 224 rows: the scales leave room for three stages and a table of fewer groups)
    static constexpr uint32_t kGroups = KIND == kKindNvf4 && NMAX > 192 ? 96 : kMaxGroups;
    static constexpr uint32_t kFits = (kGemmSmemBudget - kStagingBytes - kPartialBytes - 12 * (kGroups + 1)) / kStageBytes;
    static constexpr uint32_t kStages = kFits < 10 ? kFits : 10;
    static constexpr uint32_t kSfCols = 4 * kWords * (1 + kSfbBlocks);  // tensor-memory columns of one block's scales
    static constexpr uint32_t kSfBase = 2 * NMAX;
    // two sets of scale columns that blocks take in turn, or one where two do not fit beside the accumulators
    static constexpr uint32_t kSfSets = 2 * NMAX + kSub * kSfCols <= 512 ? kSub : 1;
    static constexpr uint32_t kColsNeeded = 2 * NMAX + kSfSets * kSfCols;
    static constexpr uint32_t kCols = kColsNeeded <= 64 ? 64 : kColsNeeded <= 128 ? 128 : kColsNeeded <= 256 ? 256 : 512;
    static constexpr uint32_t kBoxes = NMAX >= 96 && !WGRAD ? 3 : 1;
    static constexpr uint32_t kElems = KIND == kKindBf16 ? 64 : 128;  // tensor-map elements of a 128-byte row
    static constexpr uint32_t kNStep = CG == 2 ? 32 : 16;
    static_assert(kColsNeeded <= 512, "tensor memory");
    static_assert(kFirstResultWarp % 4 == 0, "a warp reads the quarter of tensor memory of its number modulo four");
    static_assert(!SPLIT || (CG == 1 && (!WGRAD || F32)), "the cluster of a split product is one along K");
    static_assert(!WGRAD || (A_MN && kBRows % 64 == 0 && kSub == 1), "weight gradient reads both operands along their rows");
    static_assert(kBBytes % 1024 == 0, "stage layout");
    // A scale loader goes from stage `it` to `it` + kScaleSets.  It waits by parity, so the slot it comes to has to be at most one
    // phase behind: MMA(it - kStages) is done by then, MMA(it + kScaleSets - 2 kStages) has to be.
    static_assert(kStages >= 3 && kStages >= kScaleSets, "a slot's parity would be ambiguous");
};

// A tile's rows of B come in one box.  The last tile of a group often has few rows, and loads, which bound the products of
// 256 x N tiles as much as the tensor core does, then take a box of a half or a quarter (16 experts of skewed sizes, bf16:
// 386 -> 383 us, NVFP4 55.8 -> 55.5).  Several small boxes instead of a large one are slower (312 -> 360 us on 8192 x 4096 x 7168).
struct GemmMapsB {
    CUtensorMap box[3];
};

struct GemmTile {
    uint32_t e, i0, j0, jn, n_mma, k0, k_stages, k_rows;
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
            per = C::NMAX;
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
        r.k_stages = C::WGRAD ? (rows[r.e] + 63) / 64 : p.k_stages;
        return r;
    }
};

// Scale words of 128 rows for one stage: lane l holds rows l, l + 32, l + 64 and l + 96.
template <class C>
struct ScaleRegs {
    static constexpr uint32_t kStageWords = C::kSub * C::kWords;
    uint32_t w[4][kStageWords];

    __device__ __forceinline__ void load(const ScaleView& v, const uint32_t* group, uint32_t row0, uint32_t row_end, uint32_t stage, uint32_t lane) {
        const uint32_t word0 = v.k_shift ? stage >> 1 : stage * kStageWords;  // scales of 128 values: one word for two stages
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t row = row0 + lane + 32u * c;
            const uint32_t* at = group + static_cast<int64_t>(row >> v.row_shift) * v.row_stride + static_cast<int64_t>(word0) * v.k_stride;
            const bool valid = row < row_end;
            if constexpr (C::KIND == kKindNvf4) {
                if (v.vec && word0 + kStageWords <= v.words) {  // the 32 bytes of a row in one load
#pragma unroll
                    for (uint32_t k = 0; k < kStageWords; ++k) w[c][k] = 0;
                    if (valid)
                        asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                                     : "=r"(w[c][0]), "=r"(w[c][1]), "=r"(w[c][2]), "=r"(w[c][3]), "=r"(w[c][4]), "=r"(w[c][5]), "=r"(w[c][6]), "=r"(w[c][7])
                                     : "l"(at));
                    continue;
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < kStageWords; ++k)
                w[c][k] = valid && word0 + k < v.words && (k == 0 || !v.k_shift) ? __ldg(at + k * v.k_stride) : 0u;
        }
    }

    // The tensor core copies 512-byte blocks of 128 rows, row r at (r % 32) * 16 + (r / 32) * 4; `pitch` between words.
    __device__ __forceinline__ void store(uint32_t smem, uint32_t pitch, uint32_t lane) const {
#pragma unroll
        for (uint32_t k = 0; k < kStageWords; ++k)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem + k * pitch + lane * 16u), "r"(w[0][k]), "r"(w[1][k]), "r"(w[2][k]), "r"(w[3][k])
                         : "memory");
    }
};

// A scale loader's place: stage `stage` of tile `tile`.
template <class C>
struct ScaleWalk {
    GemmTile tile;
    uint32_t t, stage, it;
    bool valid;

    uint32_t first, last;  // the block's part of K

    __device__ __forceinline__ void begin(const GemmParams& p, const GemmSchedule<C>& sched, uint32_t unit, uint32_t k_first, uint32_t k_end) {
        t = unit;
        first = stage = k_first;
        last = k_end;
        valid = t < sched.total;
        if (valid) tile = sched.tile(p, t);
    }
    __device__ __forceinline__ void advance(const GemmParams& p, const GemmSchedule<C>& sched, uint32_t units, uint32_t stages) {
        stage += stages;
        while (valid && stage >= last) {
            stage -= last - first;
            t += units;
            valid = t < sched.total;
            if (valid) tile = sched.tile(p, t);
        }
    }
};

// 32 columns of the accumulator (rows j of the output) of a warp's 32 lanes (its columns i) -> bf16.  The fragments of a
// 16-lane load are those of an 8 x 8 matrix store, which transposes them on the way into shared memory (64-byte rows, 16-byte
// chunks permuted so that neither side meets a bank twice); from there every lane moves 16 bytes of a row at a time.
template <class C>
__device__ __forceinline__ void store_bf16(const GemmParams& p, const GemmTile& tile, uint32_t (&v)[32], bool have, uint32_t taddr, uint32_t iw,
                                           uint32_t c, uint32_t n, float alpha, uint32_t smem, uint32_t lane) {
    if (have) {
        tmem_load_16x32(taddr, v);
        tmem_load_16x32(taddr + (16u << 16), v + 16);
        tmem_load_wait();
    } else {
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] = 0;
    }
#pragma unroll
    for (uint32_t half = 0; half < 2; ++half)
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            uint32_t m[4];
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x) {
                const float lo = __uint_as_float(v[16 * half + 4 * x + 2 * h]), hi = __uint_as_float(v[16 * half + 4 * x + 2 * h + 1]);
                const __nv_bfloat162 b = __floats2bfloat162_rn(__fmul_rn(lo, alpha), __fmul_rn(hi, alpha));
                m[x] = *reinterpret_cast<const uint32_t*>(&b);
            }
            const uint32_t chunk = (half * 2 + h) ^ ((lane >> 1) & 3u);
            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem + lane * 64u + chunk * 16u), "r"(m[0]),
                         "r"(m[1]), "r"(m[2]), "r"(m[3])
                         : "memory");
        }
    __syncwarp();
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(tile.e) * p.out_group_stride +
                         static_cast<int64_t>(tile.j0 + c) * p.out_stride + iw;
    if (p.wide_out) {
        const uint32_t chunk = lane & 3u;
        const bool in = iw + chunk * 8 < p.i_size;
        __nv_bfloat16* o = out + static_cast<int64_t>(lane >> 2) * p.out_stride + chunk * 8;
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
            const uint32_t row = q * 8 + (lane >> 2);
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(smem + row * 64u + ((chunk ^ ((row >> 1) & 3u)) * 16u)));
            if (in && row < n) *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
            o += 8 * p.out_stride;
        }
    } else if (iw + lane < p.i_size) {
        for (uint32_t row = 0; row < n; ++row) {
            uint16_t w;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(smem + row * 64u + (((lane >> 3) ^ ((row >> 1) & 3u)) * 16u) + (lane & 7u) * 2u));
            reinterpret_cast<uint16_t*>(out + static_cast<int64_t>(row) * p.out_stride)[lane] = w;
        }
    }
}

__device__ __forceinline__ uint32_t as_bits(uint32_t x) { return x; }
__device__ __forceinline__ uint32_t as_bits(float x) { return __float_as_uint(x); }

// Sums of the weight gradient in registers.  The tensor core cuts off what an addition to its accumulator shifts out instead of
// rounding, so a long sum drifts towards zero, by less than one unit (2^-23 of itself) per step of 16 rows; over groups of some
// 900 rows 1.3e-6 was measured, over 300000 rows of one sign 1.9e-3.  Every kChunk stages its sum is therefore added to one in
// registers, with rounding: eight warps hold 128 columns of the tile each, and the accumulators take turns, so that this goes on
// beside the products.  fp32 results: every 16 steps (16 experts, 8192 rows, 4096 x 7168: 2.4e-7 off and 560 us; 4.8e-7 and 552 us
// with 32 steps; 1.3e-6 and 540 us without).  bf16 results: every 256 steps, 2^-15 at most (half a step of bf16 is 2^-9 or more).
__device__ __forceinline__ void add_f32(float (&sum)[128], uint32_t taddr, uint32_t columns) {
#pragma unroll
    for (uint32_t g = 0; g < 8; ++g) {
        if (16 * g < columns) {
            uint32_t v[16];
            tmem_load16(taddr + 16 * g, v);
            tmem_load_wait();
#pragma unroll
            for (uint32_t q = 0; q < 16; ++q) sum[16 * g + q] = __fadd_rn(sum[16 * g + q], __uint_as_float(v[q]));
        }
    }
}

// Rows FROM .. FROM + N of a lane's column: what `out` holds plus the sum, N loads in flight.
template <uint32_t FROM, uint32_t N>
__device__ __forceinline__ void accumulate_rows(const float (&sum)[128], float*& o, int64_t stride, uint32_t rows) {
    if (FROM >= rows) return;
    const float* from = o;
    float old[N];
#pragma unroll
    for (uint32_t q = 0; q < N; ++q) {
        old[q] = 0.0f;
        if (FROM + q < rows) asm volatile("ld.global.f32 %0, [%1];" : "=f"(old[q]) : "l"(from) : "memory");
        from += stride;
    }
#pragma unroll
    for (uint32_t q = 0; q < N; ++q) {
        if (FROM + q < rows) asm volatile("st.global.f32 [%0], %1;" ::"l"(o), "f"(__fadd_rn(old[q], sum[FROM + q])) : "memory");
        o += stride;
    }
}

// A warp's 32 lanes hold 32 neighbouring columns, 128 bytes of a row, so every store is a whole line as it is.  (Shared memory
// is what the products are short of: staged rows and TMA stores took 600 us where these took 540, 16 experts, 8192 rows,
// 4096 x 7168.)
__device__ __forceinline__ void store_f32(const GemmParams& p, const float (&sum)[128], float* o, uint32_t rows) {
    if (rows >= 128) {
#pragma unroll
        for (uint32_t q = 0; q < 128; ++q) {
            asm volatile("st.global.L1::no_allocate.f32 [%0], %1;" ::"l"(o), "f"(sum[q]) : "memory");
            o += p.out_stride;
        }
    } else {
#pragma unroll
        for (uint32_t q = 0; q < 128; ++q) {
            if (q < rows) *o = sum[q];
            o += p.out_stride;
        }
    }
}

// An accumulating call reads, adds and writes: each element has one owner.  Registers of sums that are stored take later loads.
// (Additions in L2 by red.global.add.f32 would flush subnormals of either side to zero.)
__device__ __forceinline__ void accumulate_f32(const GemmParams& p, const float (&sum)[128], float* o, uint32_t rows) {
    accumulate_rows<0, 8>(sum, o, p.out_stride, rows);
    accumulate_rows<8, 16>(sum, o, p.out_stride, rows);
    accumulate_rows<24, 16>(sum, o, p.out_stride, rows);
    accumulate_rows<40, 24>(sum, o, p.out_stride, rows);
    accumulate_rows<64, 32>(sum, o, p.out_stride, rows);
    accumulate_rows<96, 32>(sum, o, p.out_stride, rows);
}

// bf16: 64 bytes of a row per warp.
__device__ __forceinline__ void store_long_bf16(const GemmParams& p, const float (&sum)[128], __nv_bfloat16* o, uint32_t rows) {
#pragma unroll
    for (uint32_t q = 0; q < 128; ++q) {
        if (q < rows) *o = __float2bfloat16_rn(sum[q]);
        o += p.out_stride;
    }
}

// N rows from row j on of a lane's column i of the tile go to the CTA of the cluster that owns the column.  (Rows behind the
// tile's last are never read.)
template <class C, uint32_t N, class T>
__device__ __forceinline__ void hand_over(const T (&v)[N], uint32_t j, uint32_t i, uint32_t split, uint32_t part, uint32_t partial) {
    const uint32_t own = 128 / split;
    const uint32_t to = map_to_rank(partial + ((part * own + i % own) * C::kPartialPitch + j) * 4, i / own);
#pragma unroll
    for (uint32_t q = 0; q < N; q += 4)
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + q * 4), "r"(as_bits(v[q])), "r"(as_bits(v[q + 1])),
                     "r"(as_bits(v[q + 2])), "r"(as_bits(v[q + 3]))
                     : "memory");
}

template <class C>
__global__ void __launch_bounds__(C::kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ GemmMapsB maps_b, const GemmParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[C::kStages], empty_bar[C::kStages], ready_bar[C::kStages], acc_full[2], acc_empty[2], drain_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t abort_flag;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = C::CG == 2 ? cluster_rank() : 0;
    const uint32_t unit = blockIdx.x / (C::SPLIT ? p.split : C::CG), units = gridDim.x / (C::SPLIT ? p.split : C::CG);
    // this CTA's part of K
    const uint32_t part = C::SPLIT ? cluster_rank() : 0;
    const uint32_t k_first = C::SPLIT && !C::WGRAD ? part * p.k_stages / p.split : 0;
    const uint32_t k_end = C::SPLIT ? (part + 1) * p.k_stages / p.split : p.k_stages;

    auto k_begin = [&](const GemmTile& tile) { return C::WGRAD && C::SPLIT ? part * tile.k_stages / p.split : k_first; };
    auto k_stop = [&](const GemmTile& tile) { return !C::WGRAD ? k_end : C::SPLIT ? (part + 1) * tile.k_stages / p.split : tile.k_stages; };

    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t a_base = base, b_base = a_base + C::kStages * C::kSub * C::kABytes, staging = b_base + C::kStages * C::kSub * C::kBBytes;
    const uint32_t partial = staging + C::kStagingBytes, sf_base = partial + C::kPartialBytes;
    uint32_t* group_mem =
        reinterpret_cast<uint32_t*>(smem_raw + (base - smem_u32(smem_raw)) + C::kStages * C::kStageBytes + C::kStagingBytes + C::kPartialBytes);
    uint32_t* s_prefix = group_mem;
    uint32_t* s_start = s_prefix + p.groups + 1;
    uint32_t* s_rows = s_start + p.groups;

    if (warp == 0) {
        if (lane == 0) {
            prefetch_tensor_map(&map_a);
            prefetch_tensor_map(&maps_b.box[0]);
        }
        // Group table: start and rows, clamped to the tensor and to what lies behind all earlier groups (so that every row is in one
        // group at most, whatever the bounds say), and the tiles before each group.  A group without rows ends nothing.
        uint32_t before = 0, taken = 0;
        for (uint32_t e0 = 0; e0 < p.groups; e0 += 32) {
            const uint32_t e = e0 + lane;
            uint32_t tiles = 0, first = 0, last = 0;
            if (e < p.groups) {
                last = p.rows;
                if (p.start != nullptr) {
                    first = static_cast<uint32_t>(min(max(static_cast<int64_t>(p.start[e]), int64_t{0}), static_cast<int64_t>(p.rows)));
                    last = static_cast<uint32_t>(min(max(static_cast<int64_t>(p.end[e]), int64_t{0}), static_cast<int64_t>(p.rows)));
                    if (last <= first) last = 0;
                }
            }
            uint32_t end = max(last, taken);  // the largest end so far
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(kFullMask, end, o);
                if (lane >= o) end = max(end, up);
            }
            uint32_t earlier = __shfl_up_sync(kFullMask, end, 1);
            if (lane == 0) earlier = taken;
            taken = __shfl_sync(kFullMask, end, 31);
            if (e < p.groups) {
                first = max(first, earlier);
                const uint32_t rows = last > first ? last - first : 0;
                s_start[e] = min(first, end);
                s_rows[e] = rows;
                tiles = (rows + C::NMAX - 1) / C::NMAX * p.i_tiles;
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
                mbar_init(&full_bar[s], 1 + (C::SCALED ? C::kScaleBlocks * C::CG : 0));
                mbar_init(&empty_bar[s], 1);
                mbar_init(&ready_bar[s], C::CG);
            }
            for (int a = 0; a < 2; ++a) {
                mbar_init(&acc_full[a], 1);
                mbar_init(&acc_empty[a], C::kResultWarps * C::CG);
            }
            mbar_init(&drain_bar, 1);
        }
        __syncwarp();
        tmem_alloc<C::CG>(smem_u32(&tmem_slot), C::kCols);
    }
    tcgen05_fence_before();
    __syncthreads();
    if constexpr (C::CG == 2 || C::SPLIT) cluster_sync();  // (a split product's CTAs write to one another)
    tcgen05_fence_after();

    const uint32_t tmem = tmem_slot;
    const GemmWait wait{&abort_flag};
    GemmSchedule<C> sched{s_prefix, s_start, s_rows, 0};
    sched.total = C::WGRAD ? p.groups * p.i_tiles * ((p.j_size + C::NMAX - 1) / C::NMAX) : s_prefix[p.groups];
    auto bar = [](uint64_t* b) { return smem_u32(b); };
    auto leader_bar = [&](uint64_t* b) { return C::CG == 2 ? map_to_rank(smem_u32(b), 0) : smem_u32(b); };

    // The two issuing warps run their loops whole, with one lane elected for the waits and the instructions: in a branch that
    // a lane enters alone, every operand of every instruction is moved into uniform registers first.  Per stage of four
    // bf16 products of 256 x 256 x 16 (512 cycles): 875 cycles with the loop in one lane's branch, 600 with a branch around the
    // instructions, 518 with predicated instructions and one polling lane that looks at the next stage ahead of time.
    if (warp == 0) {
        // ---- operand tiles ----
        const bool one = elect_one();
        uint32_t s = 0, phase = 1, filled = 0;
        bool ok = true;
        for (uint32_t t = unit; ok && t < sched.total; t += units) {
            const GemmTile tile = sched.tile(p, t);
            const int32_t i0 = static_cast<int32_t>(tile.i0 + rank * 128u);
            const int32_t j0 = static_cast<int32_t>(tile.j0 + (C::CG == 2 ? rank * (tile.n_mma / 2) : 0));
            const uint32_t k_from = k_begin(tile), k_last = k_stop(tile);
            const uint32_t small = C::kBoxes == 1 ? 0 : 4 * tile.n_mma <= C::NMAX ? 2 : 2 * tile.n_mma <= C::NMAX ? 1 : 0;
            const CUtensorMap* map_b = &maps_b.box[small];
            for (uint32_t kb = k_from; kb < k_last; ++kb) {
                ok = __any_sync(kFullMask, one && wait(bar(&empty_bar[s]), phase));
                if (!ok) break;
                const uint32_t a = a_base + s * (C::kSub * C::kABytes), b = b_base + s * (C::kSub * C::kBBytes);
                const int32_t k = static_cast<int32_t>(tile.k0 + kb * (C::kSub * C::kElems));
                const uint32_t full = C::WGRAD ? bar(&full_bar[s]) : leader_bar(&full_bar[s]);
                if (one) {
                    if (C::WGRAD) mbar_arrive_expect_tx(&full_bar[s], C::kABytes + C::kBBytes);
                    else if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], C::CG * C::kSub * (C::kABytes + (C::kBBytes >> small)));
#pragma unroll
                    for (uint32_t u = 0; u < C::kSub; ++u) {
                        const int32_t ku = k + static_cast<int32_t>(u * C::kElems);
                        if constexpr (C::A_MN) {
                            const int32_t z = C::WGRAD ? 0 : static_cast<int32_t>(tile.e);
                            tma_load_3d<C::CG>(a, &map_a, i0, ku, z, full);
                            tma_load_3d<C::CG>(a + 8192, &map_a, i0 + 64, ku, z, full);
                        } else {
                            tma_load_3d<C::CG>(a + u * C::kABytes, &map_a, ku, i0, static_cast<int32_t>(tile.e), full);
                        }
                        if constexpr (C::WGRAD) {
#pragma unroll
                            for (uint32_t q = 0; q < C::kBRows / 64; ++q)
                                tma_load_3d<C::CG>(b + q * 8192, map_b, j0 + static_cast<int32_t>(64 * q), ku, 0, full);
                        } else {
                            tma_load_3d<C::CG>(b + u * C::kBBytes, map_b, ku, j0, 0, full);
                        }
                    }
                }
                __syncwarp();
                filled = min(filled + 1, C::kStages);
                if (++s == C::kStages) s = 0, phase ^= 1;
            }
        }
        // every stage that was filled has been read before the block may end
        for (; filled > 0; --filled) {
            const uint32_t back = filled;  // the stage filled `back` fills ago
            const uint32_t q = s >= back ? s - back : s + C::kStages - back;
            const uint32_t q_phase = s >= back ? phase ^ 1u : phase;  // parity of that fill's own phase
            if (ok) ok = __any_sync(kFullMask, one && wait(bar(&empty_bar[q]), q_phase));
            else if (C::WGRAD || rank == 0) mbar_wait(&full_bar[q], q_phase, 1u << 16);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            // ---- matrix instructions ----
            constexpr uint32_t kM = 128 * C::CG;
            // a step along K: 32 bytes of a K-major row, or 16 rows of 128 bytes
            constexpr uint32_t kStepA = (C::A_MN ? 2048 : 32) >> 4, kStepB = (C::WGRAD ? 2048 : 32) >> 4;
            const uint64_t desc_a = smem_desc(a_base, C::A_MN ? 8192 : 16, 1024, kSwizzle128);
            const uint64_t desc_b = smem_desc(b_base, C::WGRAD ? 8192 : 16, 1024, kSwizzle128);
            const uint64_t desc_sf = smem_desc(sf_base, 16, 128, 0);
            // scale bytes of successive instructions: the next one (32 values each) or the same one (128 values)
            const uint32_t id_step = idesc_scale_ids(p.sfa.k_shift ? 0 : 1, p.sfb.k_shift ? 0 : 1);
            const uint32_t id_block = idesc_scale_ids(p.sfa.k_shift ? 1 : 0, p.sfb.k_shift ? 1 : 0);
            const bool one = elect_one();
            uint32_t s = 0, phase = 0, acc_it = 0;
            bool ok = true, ready = false;  // ready: the next stage's operands have been seen to be there
            for (uint32_t t = unit; ok && t < sched.total; t += units) {
                const GemmTile tile = sched.tile(p, t);
                const uint32_t k_from = k_begin(tile), k_last = k_stop(tile);
                if (k_last <= k_from) continue;
                uint32_t a = 0, d = 0;
                uint32_t idesc;
                if constexpr (C::SCALED) idesc = idesc_scaled(kM, tile.n_mma, C::KIND == kKindMxf8 ? 0 : 1, C::KIND != kKindNvf4);
                else idesc = idesc_bf16(kM, tile.n_mma, C::A_MN, C::WGRAD);
                for (uint32_t kb = k_from; kb < k_last; ++kb) {
                    const bool opens = kb == k_from || (C::F32 && (kb - k_from) % C::kChunk == 0);
                    const bool closes = kb + 1 == k_last || (C::F32 && (kb + 1 - k_from) % C::kChunk == 0);
                    if (opens) {
                        a = acc_it & 1u;
                        ok = __any_sync(kFullMask, one && wait(bar(&acc_empty[a]), ((acc_it >> 1) & 1u) ^ 1u));
                        if (!ok) break;
                        ++acc_it;
                        tcgen05_fence_after();
                        d = tmem + a * C::NMAX;
                    }
                    if (!ready) ok = __any_sync(kFullMask, one && wait(bar(C::WGRAD ? &ready_bar[s] : &full_bar[s]), phase));
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t now = s;
                    if (++s == C::kStages) s = 0, phase ^= 1;
                    bool seen = false;
                    if (one) seen = mbar_try_wait_cluster(bar(C::WGRAD ? &ready_bar[s] : &full_bar[s]), phase);
                    uint32_t n_units = 4 * C::kSub;
                    if (kb + 1 == (C::WGRAD ? tile.k_stages : p.k_stages)) n_units = C::WGRAD ? (tile.k_rows - kb * 64 + 15) / 16 : p.last_units;
#pragma unroll
                    for (uint32_t h = 0; h < C::kSub; ++h) {
                        if (h > 0 && 4 * h >= n_units) break;
                        const uint64_t da = desc_a + (now * C::kSub + h) * (C::kABytes >> 4), db = desc_b + (now * C::kSub + h) * (C::kBBytes >> 4);
                        const uint32_t sfa = tmem + C::kSfBase + h % C::kSfSets * C::kSfCols, sfb = sfa + 4 * C::kWords;
                        uint32_t id0 = idesc;
                        if constexpr (C::SCALED) {
                            // The copies go over the scales of an earlier block, whose products may still be under way.  Nothing is waited
                            // for: PTX promises that a product sees the copies issued before it, and the hardware has been seen to keep
                            // the order of issue the other way too, for which there is no such promise (test_many_waves compares products
                            // whose scales differ from block to block).
                            const uint64_t dfa = desc_sf + now * ((C::kSub * (C::kSfaBytes + C::kSfbBytes)) >> 4);
                            const uint64_t dfb = dfa + ((C::kSub * C::kSfaBytes) >> 4);
                            const uint32_t ha = C::KIND == kKindMxf8 && p.sfa.k_shift ? 0 : h, hb = C::KIND == kKindMxf8 && p.sfb.k_shift ? 0 : h;
#pragma unroll
                            for (uint32_t w = 0; w < C::kWords; ++w) {
                                tcgen05_copy_scales<C::CG>(one, sfa + 4 * w, dfa + 32 * (ha * C::kWords + w));
#pragma unroll
                                for (uint32_t b = 0; b < C::kSfbBlocks; ++b)
                                    tcgen05_copy_scales<C::CG>(one, sfb + 4 * (w * C::kSfbBlocks + b), dfb + 32 * ((hb * C::kWords + w) * C::kSfbBlocks + b));
                            }
                            if constexpr (C::KIND == kKindMxf8) id0 += id_block * ((kb & 1u) * 2 + h);
                        }
#pragma unroll
                        for (uint32_t u = 0; u < 4; ++u) {
                            if (u > 0 && 4 * h + u >= n_units) break;
                            uint32_t id = id0, fa = sfa, fb = sfb;
                            if constexpr (C::KIND == kKindMxf8) id += u * id_step;
                            if constexpr (C::KIND == kKindMxf4) {
                                id |= idesc_scale_ids((u & 1u) * 2, (u & 1u) * 2);
                                fa += 4 * (u >> 1);
                                fb += 4 * C::kSfbBlocks * (u >> 1);
                            }
                            if constexpr (C::KIND == kKindNvf4) {
                                fa += 4 * u;
                                fb += 4 * C::kSfbBlocks * u;
                            }
                            tcgen05_mma<C::KIND, C::CG>(one, d, da + u * kStepA, db + u * kStepB, id, fa, fb, !opens || h > 0 || u > 0);
                        }
                    }
                    tcgen05_commit<C::CG>(one, bar(&empty_bar[now]));
                    if (closes) tcgen05_commit<C::CG>(one, bar(&acc_full[a]));
                    ready = __any_sync(kFullMask, seen);
                }
            }
            if (!ok) {  // products in flight end before the memory they use is given up
                tcgen05_commit<C::CG>(one, bar(&drain_bar));
                mbar_wait(&drain_bar, 0, 1u << 16);
            }
        }
    } else if (warp < C::kFirstResultWarp) {
        if constexpr (C::SCALED) {
            // ---- scale factors.  A warp keeps the words of its next two stages on their way: they come from L2 while TMA loads
            // keep its ports busy, and take about a microsecond.  (8192 x 4096 x 7168 in MXFP4 took 136 us with one warp per
            // operand and loads two blocks ahead, NVFP4 143 us with loads one stage ahead and 126 us so.) ----
            const uint32_t block = (warp - 2) % C::kScaleBlocks, set = (warp - 2) / C::kScaleBlocks;
            const bool is_a = block == 0;
            const ScaleView& v = is_a ? p.sfa : p.sfb;
            const uint32_t to = sf_base + (is_a ? 0 : C::kSub * C::kSfaBytes + (block - 1) * 512u), pitch = is_a ? 512u : C::kSfbBlocks * 512u;
            ScaleRegs<C> r[3];
            ScaleWalk<C> ahead;  // the stage to load next; the stages to pass on follow two behind
            ahead.begin(p, sched, unit, k_first, k_end);
            ahead.advance(p, sched, units, set);
            auto load = [&](ScaleRegs<C>& regs) {
                const GemmTile& tile = ahead.tile;
                regs.load(v, v.base + (is_a ? static_cast<int64_t>(tile.e) * v.group_stride : 0), is_a ? tile.i0 + rank * 128u : tile.j0 + (block - 1) * 128u,
                          is_a ? p.i_size : tile.j0 + tile.jn, ahead.stage, lane);
                ahead.advance(p, sched, units, C::kScaleSets);
            };
            uint32_t it = set, loaded = 0;
            if (ahead.valid) load(r[0]), ++loaded;
            if (ahead.valid) load(r[1]), ++loaded;
            bool ok = true;
            while (ok && loaded > 0) {
#pragma unroll
                for (int h = 0; h < 3; ++h) {
                    if (loaded == 0) break;
                    if (ahead.valid) load(r[(h + 2) % 3]), ++loaded;
                    const uint32_t s = it % C::kStages;
                    ok = __all_sync(kFullMask, wait(bar(&empty_bar[s]), ((it / C::kStages) & 1u) ^ 1u));
                    if (!ok) break;
                    r[h].store(to + s * (C::kSub * (C::kSfaBytes + C::kSfbBytes)), pitch, lane);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(leader_bar(&full_bar[s]));
                    it += C::kScaleSets;
                    --loaded;
                }
            }
        } else if constexpr (C::WGRAD) {
            // ---- rows behind the group's end: the last stage's tail belongs to another group (or to nobody) and is cleared in
            // both operands, so that not even an infinity there can reach the sum ----
            if (warp == 2) {
                uint32_t s = 0, phase = 0;
                bool ok = true;
                for (uint32_t t = unit; ok && t < sched.total; t += units) {
                    const GemmTile tile = sched.tile(p, t);
                    for (uint32_t kb = k_begin(tile); kb < k_stop(tile); ++kb) {
                        ok = __any_sync(kFullMask, lane == 0 && wait(bar(&full_bar[s]), phase));
                        if (!ok) break;
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
                        if (lane == 0) mbar_arrive_cluster(leader_bar(&ready_bar[s]));
                        if (++s == C::kStages) s = 0, phase ^= 1;
                    }
                }
            }
        }
    } else {
        // ---- results ----
        const uint32_t quarter = warp & 3u, rw = warp - C::kFirstResultWarp;
        const uint32_t stage_mem = staging + rw * C::kStagingPerWarp;
        uint32_t acc_it = 0, turn = 0;
        if constexpr (C::F32) {
            bool ok = true;
            for (uint32_t t = unit; ok && t < sched.total; t += units) {
                const GemmTile tile = sched.tile(p, t);
                if (tile.k_stages == 0 && p.accumulate) continue;
                const uint32_t c = rw / 4 * 128, columns = tile.jn > c ? tile.jn - c : 0;  // the warp's 128 columns of the tile
                if constexpr (C::SUMS == kSumsAccumulate && !C::SPLIT) {
                    // What the sums are added to comes to L2 meanwhile; one lane per row, and its last column where a row's 128 bytes
                    // end in another line (16 experts, 8192 rows, 4096 x 7168, accumulating: 1175 us without, 826 us so).
                    const uint32_t iw = tile.i0 + rank * 128u + quarter * 32u, width = iw < p.i_size ? min(32u, p.i_size - iw) : 0;
                    const float* row = static_cast<const float*>(p.out) + static_cast<int64_t>(tile.e) * p.out_group_stride +
                                       static_cast<int64_t>(tile.j0 + c + lane) * p.out_stride + iw;
                    for (uint32_t q = lane; width > 0 && q < min(columns, 128u); q += 32) {
                        prefetch_l2(row);
                        prefetch_l2(row + width - 1);
                        row += 32 * p.out_stride;
                    }
                }
                float sum[128];
#pragma unroll
                for (uint32_t q = 0; q < 128; ++q) sum[q] = 0.0f;
                for (uint32_t kb = k_begin(tile); kb < k_stop(tile); kb += C::kChunk) {
                    const uint32_t a = acc_it & 1u;
                    ok = __all_sync(kFullMask, wait(bar(&acc_full[a]), (acc_it >> 1) & 1u));
                    if (!ok) break;
                    ++acc_it;
                    tcgen05_fence_after();
                    add_f32(sum, tmem + a * C::NMAX + c + (quarter << 21), columns);
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(leader_bar(&acc_empty[a]));
                }
                const uint32_t i = tile.i0 + rank * 128u + quarter * 32u + lane;
                if constexpr (C::SPLIT) {
                    if (ok && c < C::NMAX) hand_over<C>(sum, 0, quarter * 32 + lane, p.split, part, partial);
                } else if (ok && i < p.i_size) {
                    const int64_t at = static_cast<int64_t>(tile.e) * p.out_group_stride + static_cast<int64_t>(tile.j0 + c) * p.out_stride + i;
                    if constexpr (C::SUMS == kSumsBf16) store_long_bf16(p, sum, static_cast<__nv_bfloat16*>(p.out) + at, columns);
                    else if constexpr (C::SUMS == kSumsAccumulate) accumulate_f32(p, sum, static_cast<float*>(p.out) + at, columns);
                    else store_f32(p, sum, static_cast<float*>(p.out) + at, columns);
                }
            }
        }
        if (!C::WGRAD && p.zero_gaps) {
            // Rows of no group: before the first, between two, behind the last.  All warps of the grid take them in turn, counted
            // across the gaps, while the first products are on their way (50 experts, 1640 rows and 6400 of gaps, 6456 x 384, MXFP4:
            // 75 us gap by gap after the products, 40 us so).
            const uint32_t nw = gridDim.x * C::kResultWarps;
            const uint32_t full8 = p.wide_out ? p.i_size / 8 : 0;
            uint32_t ahead = blockIdx.x * C::kResultWarps + rw;  // rows of gaps until this warp's next one
            for (uint32_t g = 0; g <= p.groups; ++g) {
                const uint32_t lo = g == 0 ? 0 : s_start[g - 1] + s_rows[g - 1], hi = g == p.groups ? p.rows : s_start[g];
                for (; ahead < hi - lo; ahead += nw) {
                    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(lo + ahead) * p.out_stride;
                    for (uint32_t q = lane; q < full8; q += 32) *reinterpret_cast<uint4*>(o + 8 * q) = make_uint4(0, 0, 0, 0);
                    for (uint32_t q = full8 * 8 + lane; q < p.i_size; q += 32) o[q] = __float2bfloat16_rn(0.0f);
                }
                ahead -= hi - lo;
            }
        }
        for (uint32_t t = unit; !C::F32 && t < sched.total; t += units) {
            const GemmTile tile = sched.tile(p, t);
            const uint32_t a = acc_it & 1u;
            const bool have = tile.k_stages > 0;
            if (have) {
                const bool ok = wait(bar(&acc_full[a]), (acc_it >> 1) & 1u);
                if (!__all_sync(kFullMask, ok)) break;
                ++acc_it;
                tcgen05_fence_after();
            }
            const float alpha = p.alpha == nullptr ? 1.0f : __ldg(p.alpha + static_cast<int64_t>(tile.e) * p.alpha_stride);
            const uint32_t iw = tile.i0 + rank * 128u + quarter * 32u;  // the warp's first column of the output
            const uint32_t taddr = tmem + a * C::NMAX + (quarter << 21);
            for (uint32_t c = rw / 4 * 32; c < tile.jn; c += 8 * C::kResultWarps) {
                const uint32_t n = min(32u, tile.jn - c);
                uint32_t v[32];
                if constexpr (C::SPLIT) {
                    tmem_load32(taddr + c, v);
                    tmem_load_wait();
                    hand_over<C>(v, c, quarter * 32 + lane, p.split, part, partial);
                } else {
                    store_bf16<C>(p, tile, v, have, taddr + c, iw, c, n, alpha, stage_mem + (turn & 1u) * 2048u, lane);
                    if (C::kStagingPerWarp > 2048) ++turn;
                    else __syncwarp();
                }
            }
            if (have) {
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(leader_bar(&acc_empty[a]));
            }
        }
    }

    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if constexpr (C::CG == 2 || C::SPLIT) cluster_sync();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc<C::CG>(tmem, C::kCols);
    }
    if constexpr (C::CG == 2) cluster_sync();
    if constexpr (C::SPLIT) {
        if (unit < sched.total) {
            const GemmTile tile = sched.tile(p, unit);
            if (C::WGRAD && tile.k_stages == 0 && p.accumulate) return;
            const float alpha = p.alpha == nullptr ? 1.0f : __ldg(p.alpha + static_cast<int64_t>(tile.e) * p.alpha_stride);
            const uint32_t own = 128 / p.split, log_own = 31 - __clz(own);
            for (uint32_t q = threadIdx.x; q < (tile.jn + 3) / 4 << log_own; q += C::kThreads) {
                const uint32_t col = q & (own - 1), j = (q >> log_own) * 4, i = tile.i0 + part * own + col;
                if (i >= p.i_size) continue;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t from = 0; from < 8; ++from) {
                    if (from >= p.split) break;
                    float x[4];
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                                 : "r"(partial + ((from * own + col) * C::kPartialPitch + j) * 4));
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum[r] = __fadd_rn(sum[r], x[r]);
                }
                int64_t at = (C::WGRAD ? static_cast<int64_t>(tile.e) * p.out_group_stride : 0) + static_cast<int64_t>(tile.j0 + j) * p.out_stride + i;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (j + r >= tile.jn) break;
                    if (C::WGRAD && !p.out_bf16) {
                        float* o = static_cast<float*>(p.out) + at;
                        *o = p.accumulate ? __fadd_rn(*o, sum[r]) : sum[r];
                    } else {
                        static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(__fmul_rn(sum[r], alpha));
                    }
                    at += p.out_stride;
                }
            }
        }
    }
}

}  // namespace tkq
