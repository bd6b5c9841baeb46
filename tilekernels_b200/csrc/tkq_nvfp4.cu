// NVFP4: e2m1 codes with one e4m3 scale per 16 values and one fp32 scale per tensor, and the way back.
//
//     s = nearest e4m3 of (max |x| over the block) / (6 ts), at most 448      d = s * ts
//     q = nearest e2m1 of x / d, ties to the even code, 0 where d = 0          value = q * s * ts
//
// Both roundings are those of the exact quotients.  A block's values are ratios of short numbers, so quotients on or next
// to a border between two codes are common enough to matter, and an fp32 quotient that is half an ulp off would take the
// other code.  The quotient is therefore formed with a reciprocal (relative error below 2^-22), rounded twice, from
// just below and just above (factors 1 -+ 2^-21): if both give the same code, so does the exact one.  If not, |x| is
// compared with T * d for the border T between the two codes (or max |x| with 6 B ts for a border B of e4m3): T * s has at
// most seven significant bits, so fma(T * s, ts, -|x|) has the sign of the exact difference.  In bf16 tensors scaled by
// their own maximum that is no rarity: deciding all 16 codes of a block anew took 126 us on [20001, 7168], the open ones alone 62 us.
//
// Streaming kernels bound by HBM: 2 + 0.5625 bytes per bf16 value in either direction.  A lane owns one block of 16 values
// (one 256-bit load, one 64-bit store, one scale byte), a warp 512 values of a row, as in the other per-token casts.
#include <cuda_bf16.h>

#include "tkq_launch.cuh"
#include "tkq_token_kernels.cuh"

namespace tkq {

struct Nvfp4Params {
    const void* x;
    const float* tensor_scale;
    uint8_t* codes;
    uint8_t* sf;
    void* out;
    int64_t x_stride;
    uint32_t hidden, items_per_row, total_items, stride_rows, stride_items;
    bool wide;
};

constexpr int kNvThreads = 256;

// Walks the (row, 512-value step) items of a grid-stride warp without a division per item.
struct NvItems {
    uint32_t row, sub;
    __device__ __forceinline__ NvItems(const Nvfp4Params& p, uint32_t warp) : row(warp / p.items_per_row), sub(warp - row * p.items_per_row) {}
    __device__ __forceinline__ void next(const Nvfp4Params& p) {
        sub += p.stride_items;
        row += p.stride_rows;
        if (sub >= p.items_per_row) {
            sub -= p.items_per_row;
            ++row;
        }
    }
};

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kBelow = 1.0f - 0x1p-21f, kAbove = 1.0f + 0x1p-21f;

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    uint32_t f16x2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f16x2) : "h"(static_cast<uint16_t>(byte)));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(f16x2 & 0xffffu)));
}

__device__ __forceinline__ uint32_t block_scale(float amax, float ts, float inv6) {
    if (amax == 0.0f) return 0;
    const float r = __fmul_rn(amax, inv6);
    const uint32_t both = cvt_e4m3x2(__fmul_rn(r, kBelow), __fmul_rn(r, kAbove)), lo = both & 0xffu, hi = both >> 8;
    if (lo == hi) return lo;
    const float border = __fmul_rn(__fadd_rn(e4m3_value(lo), e4m3_value(hi)), 3.0f);  // six times the middle, exact
    const float above = __fmaf_rn(border, ts, -amax);
    return above < 0.0f || (above == 0.0f && (hi & 1u) == 0) ? hi : lo;
}

// The codes of eight values whose quotients, rounded from below and from above, are the codes `lo` and `hi`: where these
// differ (by one), the exact comparison with the border between them decides.
__device__ __forceinline__ uint32_t settle_codes(const float* v, uint32_t lo, uint32_t hi, float s, float ts) {
    uint32_t open = lo ^ hi;
    while (open) {
        const uint32_t shift = (__ffs(open) - 1) & ~3u;
        open &= ~(0xfu << shift);
        const uint32_t cl = (lo >> shift) & 7u, ch = (hi >> shift) & 7u;
        uint32_t f16x2;
        asm("{ .reg .b8 t; cvt.u8.u32 t, %1; cvt.rn.f16x2.e2m1x2 %0, t; }" : "=r"(f16x2) : "r"(cl | (ch << 4)));
        const float2 values = __half22float2(*reinterpret_cast<const __half2*>(&f16x2));
        const float border = __fmul_rn(__fadd_rn(values.x, values.y), 0.5f);
        const float above = __fmaf_rn(__fmul_rn(border, s), ts, -fabsf(v[shift >> 2]));
        if (above < 0.0f || (above == 0.0f && (ch & 1u) == 0)) lo ^= (cl ^ ch) << shift;
    }
    return lo;
}

template <int DT>
__global__ void __launch_bounds__(kNvThreads) nvfp4_cast_kernel(const Nvfp4Params p) {
    using Src = PlainSource<DT>;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, nwarps = (gridDim.x * blockDim.x) >> 5;
    // A tensor scale near the ends of fp32's range is moved to its middle, and the values with it (both exact, but for
    // values that round to zero anyway), so that no product below under- or overflows.
    float ts = __ldg(p.tensor_scale);
    const float shift = ts < 0x1p-60f ? 0x1p60f : ts > 0x1p60f ? 0x1p-60f : 1.0f;
    ts = __fmul_rn(ts, shift);
    const float inv6 = __fdiv_rn(1.0f, __fmul_rn(6.0f, ts));
    const uint8_t* xb = static_cast<const uint8_t*>(p.x);
    NvItems at(p, warp);
    for (uint32_t item = warp; item < p.total_items; item += nwarps, at.next(p)) {
        const uint32_t col = at.sub * 512u + lane * 16u;
        if (col >= p.hidden) continue;
        typename Src::Raw raw;
        Src::issue(raw, xb + Src::bytes(static_cast<int64_t>(at.row) * p.x_stride + col), p.wide);
        float v[16];
        Src::unpack(raw, v);
        if (shift != 1.0f) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __fmul_rn(v[i], shift);
        }
        const uint32_t byte = block_scale(absmax16(v), ts, inv6);
        const float s = e4m3_value(byte), d = __fmul_rn(s, ts);
        uint2 codes = make_uint2(0, 0);
        if (d > 0.0f) {
            const float inv = rcp_approx(d);
            uint32_t below[2], above[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float lo[8], hi[8];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float2 x = mul2(make_float2(v[8 * q + i], v[8 * q + i + 1]), splat2(inv));
                    const float2 a = mul2(x, splat2(kBelow)), b = mul2(x, splat2(kAbove));
                    lo[i] = a.x, lo[i + 1] = a.y, hi[i] = b.x, hi[i + 1] = b.y;
                }
                below[q] = cvt_e2m1x8(lo);
                above[q] = cvt_e2m1x8(hi);
            }
            codes = make_uint2(below[0], below[1]);
            if (below[0] != above[0] || below[1] != above[1]) {
                float copy[16];  // the values themselves stay in registers
#pragma unroll
                for (int i = 0; i < 16; ++i) copy[i] = v[i];
                codes.x = settle_codes(copy, below[0], above[0], s, ts);
                codes.y = settle_codes(copy + 8, below[1], above[1], s, ts);
            }
        }
        const int64_t block = (static_cast<int64_t>(at.row) * p.hidden + col) >> 4;
        stg64(p.codes + block * 8, codes.x, codes.y);
        p.sf[block] = static_cast<uint8_t>(byte);
    }
}

// The values leave as lines that L2 gives up first: without the hint they are still being written to DRAM while the next
// kernel reads (cast and way back in turn, [20001, 7168] bf16: 150.6 us, with it 128.5; either alone is the same).
__device__ __forceinline__ void stg256_evict_first(void* p, const uint32_t* w) {
    asm volatile("st.global.L1::no_allocate.L2::evict_first.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// q * s is exact in fp32 (at most six significant bits), so a value is rounded once, by the product with the tensor scale.
template <int OUT_DT>
__global__ void __launch_bounds__(kNvThreads) nvfp4_cast_back_kernel(const Nvfp4Params p) {
    using Src = QuantSource<TKQ_FMT_E2M1>;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, nwarps = (gridDim.x * blockDim.x) >> 5;
    const float ts = __ldg(p.tensor_scale);
    NvItems at(p, warp);
    for (uint32_t item = warp; item < p.total_items; item += nwarps, at.next(p)) {
        const uint32_t col = at.sub * 512u + lane * 16u;
        if (col >= p.hidden) continue;
        const int64_t first = static_cast<int64_t>(at.row) * p.hidden + col;
        typename Src::Raw raw;
        Src::issue(raw, p.codes + first / 2, false);
        const float s = e4m3_value(p.sf[first >> 4]);
        float v[16];
        Src::unpack(raw, v, s);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float2 t = mul2(make_float2(v[i], v[i + 1]), splat2(ts));
            v[i] = t.x, v[i + 1] = t.y;
        }
        uint32_t w[16];
        if constexpr (OUT_DT == TKQ_DT_FP32) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
        }
        constexpr int kWords = OUT_DT == TKQ_DT_FP32 ? 16 : 8;
        uint32_t* dst = static_cast<uint32_t*>(p.out) + first * kWords / 16;
#pragma unroll
        for (int q = 0; q < kWords; q += 8) {
            if (p.wide) {
                stg256_evict_first(dst + q, w + q);
            } else {
                stg128(dst + q, w[q], w[q + 1], w[q + 2], w[q + 3]);
                stg128(dst + q + 4, w[q + 4], w[q + 5], w[q + 6], w[q + 7]);
            }
        }
    }
}

template <class Kernel>
static int launch_nvfp4(Kernel kernel, Nvfp4Params p, int64_t num_tokens, int max_per_sm, const char* what, cudaStream_t stream) {
    p.items_per_row = (p.hidden + 511) / 512;
    const int64_t items = num_tokens * p.items_per_row;
    if (items >= (int64_t{1} << 31)) return set_error(TKQ_E_UNSUPPORTED, "nvfp4: more than 2^31 work items; split the token dimension");
    p.total_items = static_cast<uint32_t>(items);
    constexpr int kWarps = kNvThreads / 32;
    int grid = grid_size(kernel, kNvThreads, (items + kWarps - 1) / kWarps, 0);
    grid = std::min(grid, device_sm_count() * max_per_sm);
    const uint32_t nwarps = static_cast<uint32_t>(grid) * kWarps;
    p.stride_rows = nwarps / p.items_per_row;
    p.stride_items = nwarps % p.items_per_row;
    kernel<<<grid, kNvThreads, 0, stream>>>(p);
    return check_launch(what);
}

static int check_nvfp4(int64_t num_tokens, int64_t hidden, int dtype, const char* bad) {
    if (num_tokens < 0 || hidden <= 0 || (dtype != TKQ_DT_BF16 && dtype != TKQ_DT_FP32)) return set_error(TKQ_E_BAD_ARG, bad);
    if (hidden % 16 != 0 || hidden >= (int64_t{1} << 30)) return set_error(TKQ_E_UNSUPPORTED, "nvfp4: hidden must be a multiple of 16, below 2^30");
    return 0;
}

}  // namespace tkq

using namespace tkq;

extern "C" int tkq_per_token_cast_nvfp4(const void* x, int x_dtype, int64_t num_tokens, int64_t hidden, int64_t x_row_stride,
                                        const float* tensor_scale, void* out, void* sf, void* stream) {
    if (int rc = check_nvfp4(num_tokens, hidden, x_dtype, "per_token_cast_nvfp4: bad size or input type")) return rc;
    if (num_tokens == 0) return 0;
    if (x == nullptr || tensor_scale == nullptr || out == nullptr || sf == nullptr)
        return set_error(TKQ_E_BAD_ARG, "per_token_cast_nvfp4: null pointer");
    const int64_t width = x_dtype == TKQ_DT_BF16 ? 2 : 4;
    if (num_tokens == 1) x_row_stride = hidden;
    if (!aligned16(x) || x_row_stride * width % 16 != 0 || (reinterpret_cast<uintptr_t>(out) & 7u) || (reinterpret_cast<uintptr_t>(tensor_scale) & 3u))
        return set_error(TKQ_E_ALIGNMENT, "per_token_cast_nvfp4: rows of x on 16-byte boundaries, out on 8-byte boundaries");
    Nvfp4Params p{};
    p.x = x;
    p.tensor_scale = tensor_scale;
    p.codes = static_cast<uint8_t*>(out);
    p.sf = static_cast<uint8_t*>(sf);
    p.x_stride = x_row_stride;
    p.hidden = static_cast<uint32_t>(hidden);
    p.wide = reinterpret_cast<uintptr_t>(x) % 32 == 0 && x_row_stride * width % 32 == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x_dtype == TKQ_DT_BF16) return launch_nvfp4(nvfp4_cast_kernel<TKQ_DT_BF16>, p, num_tokens, 6, "per_token_cast_nvfp4", s);
    return launch_nvfp4(nvfp4_cast_kernel<TKQ_DT_FP32>, p, num_tokens, 6, "per_token_cast_nvfp4", s);
}

extern "C" int tkq_cast_back_nvfp4(const void* x, const void* sf, const float* tensor_scale, int64_t num_tokens, int64_t hidden, int out_dtype,
                                   void* out, void* stream) {
    if (int rc = check_nvfp4(num_tokens, hidden, out_dtype, "cast_back_nvfp4: bad size or output type")) return rc;
    if (num_tokens == 0) return 0;
    if (x == nullptr || sf == nullptr || tensor_scale == nullptr || out == nullptr) return set_error(TKQ_E_BAD_ARG, "cast_back_nvfp4: null pointer");
    if ((reinterpret_cast<uintptr_t>(x) & 7u) || !aligned16(out) || (reinterpret_cast<uintptr_t>(tensor_scale) & 3u))
        return set_error(TKQ_E_ALIGNMENT, "cast_back_nvfp4: x on an 8-byte, out on a 16-byte boundary");
    Nvfp4Params p{};
    p.tensor_scale = tensor_scale;
    p.codes = const_cast<uint8_t*>(static_cast<const uint8_t*>(x));
    p.sf = const_cast<uint8_t*>(static_cast<const uint8_t*>(sf));
    p.out = out;
    p.hidden = static_cast<uint32_t>(hidden);
    p.wide = reinterpret_cast<uintptr_t>(out) % 32 == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_dtype == TKQ_DT_BF16) return launch_nvfp4(nvfp4_cast_back_kernel<TKQ_DT_BF16>, p, num_tokens, 6, "cast_back_nvfp4", s);
    return launch_nvfp4(nvfp4_cast_back_kernel<TKQ_DT_FP32>, p, num_tokens, 6, "cast_back_nvfp4", s);
}
