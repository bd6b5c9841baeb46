// C entry points of the matrix products: argument checks, tensor maps, choice of the tile variant, launch.
#include <cudaTypedefs.h>

#include "tkq_gemm.cuh"

namespace tkq {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();  // tkq_tile.cu

int gemm_wait_flag() {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_gemm_wait_failed, sizeof(v)) != cudaSuccess) return -1;
    if (v) {
        const unsigned int zero = 0;
        if (cudaMemcpyToSymbol(g_gemm_wait_failed, &zero, sizeof(zero)) != cudaSuccess) return -1;
    }
    return v ? 1 : 0;
}

// One operand as a three-dimensional tensor (inner axis, rows, groups); strides in bytes.
struct Operand {
    const void* base;
    int64_t inner, rows, groups;
    int64_t row_bytes, group_bytes;
    bool bf16;
};

static int encode(CUtensorMap* map, const Operand& o, uint32_t box_inner, uint32_t box_rows) {
    auto fn = tensor_map_encoder();
    if (fn == nullptr) return set_error(TKQ_E_UNSUPPORTED, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(o.inner), static_cast<cuuint64_t>(o.rows), static_cast<cuuint64_t>(o.groups)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.row_bytes), static_cast<cuuint64_t>(o.group_bytes)};
    const cuuint32_t box[3] = {box_inner, box_rows, 1};
    const cuuint32_t steps[3] = {1, 1, 1};
    const CUresult r = fn(map, o.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(o.base), dims,
                          strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(TKQ_E_UNSUPPORTED, "cuTensorMapEncodeTiled rejected an operand (alignment or size)");
    return 0;
}

// Strides a tensor map accepts: positive multiples of 16 bytes.  The stride of an axis of length one is never used, so any stands in.
static int fix_strides(Operand& o, const char* expanded, const char* unaligned) {
    const int64_t tight = (o.inner * (o.bf16 ? 2 : 1) + 15) / 16 * 16;
    if (o.rows == 1) o.row_bytes = tight;
    if (o.groups == 1) o.group_bytes = o.row_bytes * o.rows;
    if (o.row_bytes <= 0 || o.group_bytes <= 0) return set_error(TKQ_E_UNSUPPORTED, expanded);
    if (o.row_bytes % 16 || o.group_bytes % 16 || !aligned16(o.base)) return set_error(TKQ_E_ALIGNMENT, unaligned);
    return 0;
}

template <class C>
static int launch_gemm(const Operand& a, const Operand& b, GemmParams p, const char* what, cudaStream_t stream) {
    alignas(64) CUtensorMap map_a;
    alignas(64) GemmMapsB maps_b{};
    if (int rc = encode(&map_a, a, C::A_MN ? 64 : C::kElems, C::A_MN ? 64 : 128)) return rc;
    for (uint32_t i = 0; i < C::kBoxes; ++i)
        if (int rc = encode(&maps_b.box[i], b, C::WGRAD ? 64 : C::kElems, C::WGRAD ? 64 : C::kBRows >> i)) return rc;
    p.wide_out = p.i_size % 8 == 0 && p.out_stride % 8 == 0 && p.out_group_stride % 8 == 0 && aligned16(p.out);
    p.i_tiles = (p.i_size + 128 * C::CG - 1) / (128 * C::CG);
    const int64_t j_tiles = C::WGRAD ? int64_t{p.groups} * ((p.j_size + C::NMAX - 1) / C::NMAX) : int64_t{p.rows} / C::NMAX + p.groups;
    if (j_tiles * p.i_tiles >= (int64_t{1} << 31)) return set_error(TKQ_E_UNSUPPORTED, "matrix product: more than 2^31 tiles");
    // CTAs of a cluster: a pair on one tile, or those that share a tile along K
    const int cluster = C::SPLIT ? static_cast<int>(p.split) : C::CG;
    if (p.groups > C::kGroups) return set_error(TKQ_E_UNSUPPORTED, "matrix product: more groups than the tile variant's table holds");
    const int64_t units = std::min<int64_t>(j_tiles * p.i_tiles, device_sm_count() / cluster);
    const int smem = static_cast<int>(1024 + C::kStages * C::kStageBytes + C::kStagingBytes + C::kPartialBytes + 4 * (3 * p.groups + 1));
    auto kernel = gemm_kernel<C>;
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(units * cluster));
    config.blockDim = dim3(C::kThreads);
    config.dynamicSmemBytes = static_cast<size_t>(smem);
    config.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = cluster > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, map_a, maps_b, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(static_cast<int>(e), cudaGetErrorString(e));
    }
    return check_launch(what);
}

// At most so many tiles along j: exact for one group, else with a partial tile in each.
static int64_t row_tiles(const GemmParams& p, int nmax) {
    return p.groups == 1 ? (int64_t{p.rows} + nmax - 1) / nmax : int64_t{p.rows} / nmax + p.groups;
}

// CTAs that share a tile along K: as many as there are SMs for, with at least `part` stages each.  Clusters of eight take half
// the SMs at most: they have to fit into groups of SMs, and of sixteen the last ones run after the others (one row of bf16 through
// 2048 x 7168: 18.5 us with sixteen clusters of eight, 13.7 of four).
static uint32_t split_of(int64_t tiles, int64_t stages, int64_t part) {
    const int64_t sms = device_sm_count();
    uint32_t split = 1;
    while (split < 8 && tiles * split * 2 <= (split == 4 ? sms / 2 : sms) && stages >= 2 * part * split) split *= 2;
    return split;
}

// Tiles that leave most SMs idle are split along K; a cluster takes one tile.  One row of FP8 through 4096 x 7168: 14.9 us whole,
// 10.5 us split by 4; of NVFP4 through 7168 x 2048 (eight stages): 7.8 us whole, 8.4 us split by 2, so a part has at least six.
template <int KIND, int NMAX, bool A_MN>
static bool launch_split(const Operand& a, const Operand& b, GemmParams p, const char* what, cudaStream_t stream, int* rc) {
    const int64_t tiles = row_tiles(p, NMAX) * ((p.i_size + 127) / 128);
    p.split = split_of(tiles, p.k_stages, 6);
    if (p.split == 1) return false;
    *rc = launch_gemm<GemmConfig<KIND, 1, NMAX, false, A_MN, true>>(a, b, p, what, stream);
    return true;
}

// Tile variant by the mean number of rows per group (over all rows: which of them belong to a group, and how evenly, is known on
// the device only).  Measured (us; 32 groups, 4096 x 7168, MXFP4 and bf16, groups of one size):
//   mean rows           4          20          32          34          64         100         200
//   128 x 32       80, 271     83, 275     84, 277    120, 427    146, 540    198, 746   358, 1394
//   128 x 128      83, 284     85, 288     86, 289     88, 292     93, 306    106, 361    148, 510
//   pair x 224/256 87, 289     89, 293     89, 295     90, 297     92, 294     97, 315    124, 406
// Groups of skewed sizes (the longest three times the mean) reach the second tile, and read their weight again, at a smaller mean:
//   mean rows           4           8          16          20          24          32
//   128 x 32       60, 200     71, 238     81, 275     83, 274     90, 309    100, 345
//   128 x 128      63, 209     74, 247     78, 262     81, 271     83, 280     84, 282
// so several groups take 128 x 32 up to a mean of 16, one group while its rows are one such tile.
// One group whose smaller tiles all run at once uses more SMs with them (200 rows of MXFP4: 13.0 against 16.3 us for the
// pair, 256 of FP8: 20.8 against 22.3).
template <int KIND, int NMID, int NLARGE, bool A_MN>
static int launch_rows(const Operand& a, const Operand& b, const GemmParams& p, const char* what, cudaStream_t stream) {
    const int64_t mean = p.rows / p.groups;
    int rc;
    if (mean <= (p.groups == 1 ? 32 : 16)) {
        if (launch_split<KIND, 32, A_MN>(a, b, p, what, stream, &rc)) return rc;
        return launch_gemm<GemmConfig<KIND, 1, 32, false, A_MN>>(a, b, p, what, stream);
    }
    if (mean <= 128 && launch_split<KIND, 64, A_MN>(a, b, p, what, stream, &rc)) return rc;
    if (mean <= 48 || row_tiles(p, NMID) * ((p.i_size + 127) / 128) <= device_sm_count())
        return launch_gemm<GemmConfig<KIND, 1, NMID, false, A_MN>>(a, b, p, what, stream);
    // NVFP4: 224 rows a tile where the group table fits beside them (8192 x 4096 x 7168: 121 us with 192, 111 us with 224)
    if constexpr (KIND == kKindNvf4)
        if (p.groups > GemmConfig<KIND, 2, NLARGE, false, A_MN>::kGroups) return launch_gemm<GemmConfig<KIND, 2, 192, false, A_MN>>(a, b, p, what, stream);
    return launch_gemm<GemmConfig<KIND, 2, NLARGE, false, A_MN>>(a, b, p, what, stream);
}

static int check_sizes(int64_t num_experts, int64_t num_rows, int64_t n, int64_t k) {
    if (num_experts <= 0 || num_rows < 0 || n <= 0 || k <= 0) return set_error(TKQ_E_BAD_ARG, "matrix product: bad size");
    if (num_experts > kMaxGroups) return set_error(TKQ_E_UNSUPPORTED, "matrix product: more than 1024 groups");
    if (num_rows >= (int64_t{1} << 30) || n >= (int64_t{1} << 30) || k >= (int64_t{1} << 30))
        return set_error(TKQ_E_UNSUPPORTED, "matrix product: an axis of 2^30 or more");
    return 0;
}

}  // namespace tkq

using namespace tkq;

extern "C" int tkq_block_scaled_gemm(const tkq_block_scaled_gemm_args* args, void* stream) {
    static_assert(sizeof(tkq_block_scaled_gemm_args) == 29 * 8, "8-byte fields only");
    if (args == nullptr) return set_error(TKQ_E_BAD_ARG, "block_scaled_gemm: null pointer");
    const auto [x, x_row_stride, x_sf, x_sf_row_stride, x_sf_k_stride, x_block_m, x_block_k, w, w_expert_stride, w_row_stride, w_sf,
                w_sf_expert_stride, w_sf_row_stride, w_sf_k_stride, w_block_m, w_block_k, fmt, sf_fmt, expert_start, expert_end, num_experts, num_rows,
                n, k, alpha, alpha_stride, out, out_row_stride, flags] = *args;
    if (int rc = check_sizes(num_experts, num_rows, n, k)) return rc;
    if ((fmt != TKQ_FMT_E4M3 && fmt != TKQ_FMT_E2M1) || (sf_fmt != TKQ_SFMT_UE8M0 && sf_fmt != TKQ_SFMT_E4M3))
        return set_error(TKQ_E_BAD_ARG, "block_scaled_gemm: unknown format");
    if (flags & ~int64_t{TKQ_ZERO_GAPS}) return set_error(TKQ_E_UNSUPPORTED, "block_scaled_gemm: only TKQ_ZERO_GAPS applies");
    if (num_rows == 0) return 0;
    if (x == nullptr || x_sf == nullptr || w == nullptr || w_sf == nullptr || out == nullptr || (expert_start == nullptr) != (expert_end == nullptr) ||
        (expert_start == nullptr && num_experts != 1))
        return set_error(TKQ_E_BAD_ARG, "block_scaled_gemm: null pointer");
    const bool fp8 = fmt == TKQ_FMT_E4M3, nv = sf_fmt == TKQ_SFMT_E4M3;
    auto shift_of = [](int64_t v) { return v == 1 ? 0 : v == 32 ? 5 : v == 128 ? 7 : -1; };
    const int xs = shift_of(x_block_m), ws = shift_of(w_block_m);
    bool group_ok;
    if (fp8) group_ok = !nv && (x_block_k == 32 || x_block_k == 128) && (w_block_k == 32 || w_block_k == 128);
    else group_ok = x_block_k == (nv ? 16 : 32) && w_block_k == (nv ? 16 : 32);
    if (!group_ok || xs < 0 || ws < 0)
        return set_error(TKQ_E_UNSUPPORTED, "block_scaled_gemm: scale blocks are 1, 32 or 128 rows by 32 or 128 (e4m3), 32 (e2m1) or 16 (e2m1 with e4m3 scales) values");
    if (k % (fp8 ? 32 : 64) != 0) return set_error(TKQ_E_UNSUPPORTED, "block_scaled_gemm: k must be a multiple of 32 (e4m3) or 64 (e2m1)");
    const int64_t per_byte = fp8 ? 1 : 2;
    if (x_row_stride % per_byte || w_row_stride % per_byte || w_expert_stride % per_byte)
        return set_error(TKQ_E_ALIGNMENT, "block_scaled_gemm: strides of packed e2m1 data are even");
    Operand a{w, k / per_byte, n, num_experts, w_row_stride / per_byte, w_expert_stride / per_byte, false};
    Operand b{x, k / per_byte, num_rows, 1, x_row_stride / per_byte, 0, false};
    constexpr const char* expanded = "block_scaled_gemm: data whose rows or matrices have stride 0 (an expanded tensor); make it contiguous";
    constexpr const char* unaligned = "block_scaled_gemm: data rows on 16-byte boundaries, scales on 4-byte boundaries";
    if (int rc = fix_strides(a, expanded, unaligned)) return rc;
    if (int rc = fix_strides(b, expanded, unaligned)) return rc;
    if ((reinterpret_cast<uintptr_t>(x_sf) & 3u) || (reinterpret_cast<uintptr_t>(w_sf) & 3u) || (reinterpret_cast<uintptr_t>(out) & 1u))
        return set_error(TKQ_E_ALIGNMENT, unaligned);
    GemmParams p{};
    p.start = expert_start;
    p.end = expert_end;
    p.alpha = alpha;
    p.alpha_stride = static_cast<uint32_t>(alpha_stride);
    p.out = out;
    p.out_stride = out_row_stride;
    p.groups = static_cast<uint32_t>(num_experts);
    p.rows = static_cast<uint32_t>(num_rows);
    p.i_size = static_cast<uint32_t>(n);
    const int64_t row_bytes = k / per_byte;
    p.k_stages = static_cast<uint32_t>((row_bytes + 255) / 256);
    p.last_units = static_cast<uint32_t>((row_bytes - (int64_t{p.k_stages} - 1) * 256) / 32);
    p.zero_gaps = (flags & TKQ_ZERO_GAPS) ? 1 : 0;
    auto view = [k = k](const void* sf, int64_t e, int64_t r, int64_t q, int shift, int64_t block_k) {
        ScaleView v{};
        v.base = static_cast<const uint32_t*>(sf);
        v.group_stride = e;
        v.row_stride = r;
        v.k_stride = q;
        v.row_shift = static_cast<uint32_t>(shift);
        v.words = static_cast<uint32_t>((k + 4 * block_k - 1) / (4 * block_k));
        v.k_shift = block_k == 128 ? 2 : 0;
        v.vec = q == 1 && r % 8 == 0 && e % 8 == 0 && reinterpret_cast<uintptr_t>(sf) % 32 == 0;
        return v;
    };
    p.sfa = view(w_sf, w_sf_expert_stride, w_sf_row_stride, w_sf_k_stride, ws, w_block_k);
    p.sfb = view(x_sf, 0, x_sf_row_stride, x_sf_k_stride, xs, x_block_k);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (fp8) return launch_rows<kKindMxf8, 128, 224, false>(a, b, p, "block_scaled_gemm", s);
    if (!nv) return launch_rows<kKindMxf4, 128, 224, false>(a, b, p, "block_scaled_gemm", s);
    return launch_rows<kKindNvf4, 96, 224, false>(a, b, p, "block_scaled_gemm", s);
}

extern "C" int tkq_grouped_gemm(const tkq_grouped_gemm_args* args, void* stream) {
    static_assert(sizeof(tkq_grouped_gemm_args) == 15 * 8, "8-byte fields only");
    if (args == nullptr) return set_error(TKQ_E_BAD_ARG, "grouped_gemm: null pointer");
    const auto [x, x_row_stride, w, w_expert_stride, w_row_stride, transpose_w, expert_start, expert_end, num_experts, num_rows, n, k, out,
                out_row_stride, flags] = *args;
    if (int rc = check_sizes(num_experts, num_rows, n, k)) return rc;
    if (flags & ~int64_t{TKQ_ZERO_GAPS}) return set_error(TKQ_E_UNSUPPORTED, "grouped_gemm: only TKQ_ZERO_GAPS applies");
    if (num_rows == 0) return 0;
    if (x == nullptr || w == nullptr || out == nullptr || expert_start == nullptr || expert_end == nullptr)
        return set_error(TKQ_E_BAD_ARG, "grouped_gemm: null pointer");
    Operand a{w, transpose_w ? n : k, transpose_w ? k : n, num_experts, w_row_stride * 2, w_expert_stride * 2, true};
    Operand b{x, k, num_rows, 1, x_row_stride * 2, 0, true};
    constexpr const char* expanded = "grouped_gemm: rows or matrices of stride 0 (an expanded tensor); make it contiguous";
    constexpr const char* unaligned = "grouped_gemm: rows of x and w on 16-byte boundaries";
    if (int rc = fix_strides(a, expanded, unaligned)) return rc;
    if (int rc = fix_strides(b, expanded, unaligned)) return rc;
    if (reinterpret_cast<uintptr_t>(out) & 1u) return set_error(TKQ_E_ALIGNMENT, unaligned);
    GemmParams p{};
    p.start = expert_start;
    p.end = expert_end;
    p.out = out;
    p.out_stride = out_row_stride;
    p.groups = static_cast<uint32_t>(num_experts);
    p.rows = static_cast<uint32_t>(num_rows);
    p.i_size = static_cast<uint32_t>(n);
    p.k_stages = static_cast<uint32_t>((k + 63) / 64);
    p.last_units = static_cast<uint32_t>((k - (int64_t{p.k_stages} - 1) * 64 + 15) / 16);
    p.zero_gaps = (flags & TKQ_ZERO_GAPS) ? 1 : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (transpose_w) return launch_rows<kKindBf16, 128, 256, true>(a, b, p, "grouped_gemm", s);
    return launch_rows<kKindBf16, 128, 256, false>(a, b, p, "grouped_gemm", s);
}

extern "C" int tkq_grouped_gemm_wgrad(const tkq_grouped_gemm_wgrad_args* args, void* stream) {
    static_assert(sizeof(tkq_grouped_gemm_wgrad_args) == 13 * 8, "8-byte fields only");
    if (args == nullptr) return set_error(TKQ_E_BAD_ARG, "grouped_gemm_wgrad: null pointer");
    const auto [grad, grad_row_stride, x, x_row_stride, expert_start, expert_end, num_experts, num_rows, n, k, out_dtype, out, flags] = *args;
    if (int rc = check_sizes(num_experts, num_rows, n, k)) return rc;
    if (out_dtype != TKQ_DT_BF16 && out_dtype != TKQ_DT_FP32) return set_error(TKQ_E_BAD_ARG, "grouped_gemm_wgrad: unknown output type");
    if (flags & ~int64_t{TKQ_ACCUMULATE}) return set_error(TKQ_E_UNSUPPORTED, "grouped_gemm_wgrad: only TKQ_ACCUMULATE applies");
    if ((flags & TKQ_ACCUMULATE) && out_dtype != TKQ_DT_FP32)
        return set_error(TKQ_E_UNSUPPORTED, "grouped_gemm_wgrad: accumulation needs a float32 output");
    if (out == nullptr || expert_start == nullptr || expert_end == nullptr || (num_rows > 0 && (grad == nullptr || x == nullptr)))
        return set_error(TKQ_E_BAD_ARG, "grouped_gemm_wgrad: null pointer");
    if (num_rows == 0) {  // every group is empty: gradients of zero
        if (flags & TKQ_ACCUMULATE) return 0;
        const cudaError_t e = cudaMemsetAsync(out, 0, static_cast<size_t>(num_experts * n * k) * (out_dtype == TKQ_DT_FP32 ? 4 : 2),
                                              static_cast<cudaStream_t>(stream));
        return e == cudaSuccess ? 0 : set_error(static_cast<int>(e), "grouped_gemm_wgrad: memset failed");
    }
    Operand a{x, k, num_rows, 1, x_row_stride * 2, 0, true};
    Operand b{grad, n, num_rows, 1, grad_row_stride * 2, 0, true};
    constexpr const char* expanded = "grouped_gemm_wgrad: rows of stride 0 (an expanded tensor); make it contiguous";
    constexpr const char* unaligned = "grouped_gemm_wgrad: rows of grad and x on 16-byte boundaries";
    if (int rc = fix_strides(a, expanded, unaligned)) return rc;
    if (int rc = fix_strides(b, expanded, unaligned)) return rc;
    if (reinterpret_cast<uintptr_t>(out) & (out_dtype == TKQ_DT_FP32 ? 3u : 1u)) return set_error(TKQ_E_ALIGNMENT, unaligned);
    GemmParams p{};
    p.start = expert_start;
    p.end = expert_end;
    p.out = out;
    p.out_stride = k;
    p.out_group_stride = n * k;
    p.groups = static_cast<uint32_t>(num_experts);
    p.rows = static_cast<uint32_t>(num_rows);
    p.i_size = static_cast<uint32_t>(k);
    p.j_size = static_cast<uint32_t>(n);
    p.accumulate = (flags & TKQ_ACCUMULATE) ? 1 : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // Small results whose 128 x 128 tiles leave SMs idle: the rows of a group are split over a cluster.  Whole (pairs on 256 x
    // 256) against split: 20000 rows, 128 x 128: 102, 22 us; 4096 rows, 512 x 512: 27.5, 14.5; 8 experts, 16000 rows, 256 x 512:
    // 25.5, 21.6.  Parts of five or six stages gained nothing (700 rows, 512 x 512: 10.6, 10.9), so a part has at least eight.
    // The mean decides here too: one long group among empty ones is not split.
    p.split = split_of(num_experts * ((n + 127) / 128) * ((k + 127) / 128), num_rows / num_experts / 64, 8);
    if (p.split > 1) {
        p.out_bf16 = out_dtype == TKQ_DT_BF16;
        return launch_gemm<GemmConfig<kKindBf16, 1, 128, true, true, true, kSumsF32>>(a, b, p, "grouped_gemm_wgrad", s);
    }
    if (p.accumulate) return launch_gemm<GemmConfig<kKindBf16, 2, 256, true, true, false, kSumsAccumulate>>(a, b, p, "grouped_gemm_wgrad", s);
    if (out_dtype == TKQ_DT_FP32) return launch_gemm<GemmConfig<kKindBf16, 2, 256, true, true, false, kSumsF32>>(a, b, p, "grouped_gemm_wgrad", s);
    // bf16: up to 16384 rows what the tensor core cuts off (2^-23 per 16 rows, together 2^-13) is little beside the rounding to bf16.
    // Longer calls have their sums go on in registers every 4096 rows: groups can be long, and their bounds are known on the device
    // only.  (Without against with, 4096 x 7168: 16 experts of 1024 rows 685, 703 us; one of 32768 rows 1395, 1407.)
    if (num_rows > 16384) return launch_gemm<GemmConfig<kKindBf16, 2, 256, true, true, false, kSumsBf16>>(a, b, p, "grouped_gemm_wgrad", s);
    return launch_gemm<GemmConfig<kKindBf16, 2, 256, true, true>>(a, b, p, "grouped_gemm_wgrad", s);
}
