"""block_scaled_gemm: product of two quantized matrices on the tensor cores.  The reference has the casts but no product
that reads them; the operand forms are those its casts write."""
from typing import Optional

import torch

from .. import _lib
from .common import current_stream_ptr, device_guard, empty_matrix
from .types import QuantTensor


class ScaledOperand:
    """A checked quantized operand as tkq_block_scaled_gemm takes it: a matrix (rows, k), or with `num_groups` stacked
    matrices (num_groups, rows, k), whose scales may also come as one matrix of all rows."""
    __slots__ = ('data', 'sf', 'rows', 'k', 'block_m', 'block_k', 'fmt', 'sf_fmt', 'group_stride', 'row_stride', 'sf_strides')

    def __init__(self, x: QuantTensor, block_size: tuple[int, int], num_groups: Optional[int]):
        data, sf = x
        block_m, block_k = block_size
        assert data.is_cuda and sf.is_cuda and data.get_device() == sf.get_device()
        assert data.dim() == (2 if num_groups is None else 3)
        shape, strides = data.shape, data.stride()
        rows, physical = shape[-2], shape[-1]
        assert physical <= 1 or strides[-1] == 1
        assert block_m in (1, 32, 128)
        if data.dtype is torch.float8_e4m3fn:
            per_byte, self.fmt, k = 1, _lib.FMT_E4M3, physical
        else:
            assert data.dtype is torch.int8, 'data is float8_e4m3fn or int8 (two FP4 per byte)'
            per_byte, self.fmt, k = 2, _lib.FMT_E2M1, physical * 2
        blocks = rows if block_m == 1 else -(-rows // block_m)
        if sf.dtype is torch.float8_e4m3fn:
            # one e4m3 scale per 16 values, four bytes read at a time: the scales of a row lie together
            assert per_byte == 2 and block_k == 16 and block_m == 1, 'float8_e4m3fn scales go with FP4 data and blocks of (1, 16)'
            assert k % 64 == 0 and sf.stride(-1) == 1
            sf = sf.view(torch.int32)
            self.sf_fmt = _lib.SFMT_E4M3
        else:
            assert sf.dtype is torch.int32, 'scales are packed ue8m0 words (int32) or float8_e4m3fn'
            assert block_k == 32 or (block_k == 128 and per_byte == 1)
            self.sf_fmt = _lib.SFMT_UE8M0
        words = -(-k // (4 * block_k))
        sf_strides = sf.stride()
        if num_groups is None:
            assert sf.shape == (blocks, words), f'scales must be {(blocks, words)}, got {tuple(sf.shape)}'
            self.sf_strides = (0,) + sf_strides
            self.group_stride = 0
        else:
            if len(sf_strides) == 3:
                assert sf.shape == (num_groups, blocks, words), f'scales must be {(num_groups, blocks, words)}, got {tuple(sf.shape)}'
                self.sf_strides = sf_strides
            else:
                assert rows % block_m == 0, 'scales of all groups in one matrix need whole blocks of rows per group'
                assert sf.shape == (num_groups * blocks, words), f'scales must be {(num_groups * blocks, words)}, got {tuple(sf.shape)}'
                self.sf_strides = (blocks * sf_strides[0],) + sf_strides
            self.group_stride = per_byte * strides[0]
        self.data, self.sf, self.rows, self.k, self.block_m, self.block_k = data, sf, rows, k, block_m, block_k
        self.row_stride = per_byte * strides[-2]


def check_out(out: torch.Tensor, shape: tuple, like: torch.Tensor) -> None:
    assert out.dim() == 2 and out.shape == shape and out.dtype is torch.bfloat16 and out.get_device() == like.get_device()
    assert (shape[1] <= 1 or out.stride(1) == 1) and (shape[0] <= 1 or out.stride(0) >= shape[1])


def launch_block_scaled_gemm(x: ScaledOperand, w: ScaledOperand, expert_start, expert_end, num_experts: int, alpha, out: torch.Tensor,
                             flags: int) -> None:
    assert x.k > 0 and x.k == w.k, f'inner sizes differ: {x.k} and {w.k}'
    assert x.fmt == w.fmt and x.sf_fmt == w.sf_fmt, 'both operands must have the same format'
    assert x.data.get_device() == w.data.get_device()
    alpha_ptr, alpha_stride = 0, 0
    if alpha is not None:
        assert alpha.dtype is torch.float32 and alpha.get_device() == x.data.get_device() and alpha.dim() <= 1
        assert alpha.numel() in (1, num_experts)
        alpha_ptr = alpha.data_ptr()
        alpha_stride = alpha.stride(0) if alpha.numel() > 1 else 0
    if x.rows == 0 or w.rows == 0:
        return
    args = _lib.BLOCK_SCALED_GEMM_ARGS.pack(
        x.data.data_ptr(), x.row_stride, x.sf.data_ptr(), x.sf_strides[1], x.sf_strides[2], x.block_m, x.block_k, w.data.data_ptr(), w.group_stride,
        w.row_stride, w.sf.data_ptr(), *w.sf_strides, w.block_m, w.block_k, x.fmt, x.sf_fmt, 0 if expert_start is None else expert_start.data_ptr(),
        0 if expert_end is None else expert_end.data_ptr(), num_experts, x.rows, w.rows, x.k, alpha_ptr, alpha_stride, out.data_ptr(),
        out.stride(0), flags)
    device = out.device
    with device_guard(device):
        rc = _lib.lib().tkq_block_scaled_gemm(args, current_stream_ptr(device))
    if rc:
        _lib.check(rc, 'tkq_block_scaled_gemm')


def block_scaled_gemm(
    a: QuantTensor,
    b: QuantTensor,
    a_block_size: tuple[int, int],
    b_block_size: tuple[int, int],
    alpha: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """alpha * a @ b.T for two quantized matrices, in bfloat16.

    The data reach the tensor core in their 8- or 4-bit form; the block scales are applied there.  Its fp32 sums cut off what an
    addition shifts out (2^-23 of the sum at most per 32 values of k in FP8, 64 in FP4) and are rounded once to bfloat16.

    Args:
        a: (data, scales) of (m, k) values, b: of (n, k).  Both in one of the forms
            float8_e4m3fn data, packed ue8m0 scales (int32) per 32 or 128 values, as per_token_cast and per_block_cast
            return them with use_packed_ue8m0;
            int8 data (two FP4 per byte) with packed ue8m0 scales per 32 values;
            int8 data with float8_e4m3fn scales per 16 values (per_token_cast_to_nvfp4).
            k is a multiple of 32 (FP8) or 64 (FP4); rows of the data start on 16-byte boundaries and are not expanded.
        a_block_size, b_block_size: (rows, values) per scale; rows 1, 32 or 128.
        alpha: optional fp32 tensor of one element, e.g. the product of the tensor scales of two NVFP4 operands.
        out: optional (m, n) bfloat16 destination with unit column stride.

    Returns: (m, n) bfloat16.
    """
    x, w = ScaledOperand(a, a_block_size, None), ScaledOperand(b, b_block_size, None)
    shape = (x.rows, w.rows)
    if out is None:
        out = empty_matrix(x.rows, w.rows, torch.bfloat16, x.data.device)
    else:
        check_out(out, shape, x.data)
    launch_block_scaled_gemm(x, w, None, None, 1, alpha, out, 0)
    return out
