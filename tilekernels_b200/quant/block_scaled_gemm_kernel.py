"""block_scaled_gemm: product of two quantized matrices on the tensor cores.  The reference has the casts but no product
that reads them; the operand forms are those its casts write."""
from typing import Optional

import torch

from .. import _lib
from .common import FMT_TO_ENUM, current_stream_ptr, device_guard, get_logical_hidden
from .types import QuantTensor


def scaled_operand(x: QuantTensor, block_size: tuple[int, int], num_groups: Optional[int]) -> dict:
    """Checks a quantized operand and describes it for tkq_block_scaled_gemm.  `num_groups` None: a matrix
    (rows, k); else stacked matrices (num_groups, rows, k), whose scales may also come as one matrix of all rows."""
    data, sf = x
    assert isinstance(data, torch.Tensor) and isinstance(sf, torch.Tensor)
    assert data.dtype in (torch.float8_e4m3fn, torch.int8), 'data is float8_e4m3fn or int8 (two FP4 per byte)'
    assert data.is_cuda and sf.is_cuda and sf.device == data.device
    block_m, block_k = block_size
    rows = data.shape[-2]
    k = get_logical_hidden(data.shape[-1], data.dtype)
    assert data.dim() == (2 if num_groups is None else 3) and (data.shape[-1] <= 1 or data.stride(-1) == 1)
    assert block_m in (1, 32, 128)
    blocks = -(-rows // block_m)
    if sf.dtype == torch.float8_e4m3fn:
        # one e4m3 scale per 16 values, four bytes read at a time: the scales of a row lie together
        assert data.dtype == torch.int8 and block_k == 16 and block_m == 1, 'float8_e4m3fn scales go with FP4 data and blocks of (1, 16)'
        assert k % 64 == 0 and sf.stride(-1) == 1
        sf = sf.view(torch.int32)
    else:
        assert sf.dtype == torch.int32, 'scales are packed ue8m0 words (int32) or float8_e4m3fn'
        assert block_k in ((32, 128) if data.dtype == torch.float8_e4m3fn else (32,))
    words = -(-k // (4 * block_k))
    if num_groups is None:
        assert tuple(sf.shape) == (blocks, words), f'scales must be {(blocks, words)}, got {tuple(sf.shape)}'
        sf_strides = (0,) + sf.stride()
    elif sf.dim() == 3:
        assert tuple(sf.shape) == (num_groups, blocks, words), f'scales must be {(num_groups, blocks, words)}, got {tuple(sf.shape)}'
        sf_strides = sf.stride()
    else:
        assert rows % block_m == 0, 'scales of all groups in one matrix need whole blocks of rows per group'
        assert tuple(sf.shape) == (num_groups * blocks, words), f'scales must be {(num_groups * blocks, words)}, got {tuple(sf.shape)}'
        sf_strides = (blocks * sf.stride(0),) + sf.stride()
    per_byte = 2 if data.dtype == torch.int8 else 1
    return dict(data=data, sf=sf, rows=rows, k=k, block=(block_m, block_k), fmt='e2m1' if data.dtype == torch.int8 else 'e4m3',
                sf_fmt=_lib.SFMT_E4M3 if block_k == 16 else _lib.SFMT_UE8M0, strides=tuple(per_byte * s for s in data.stride()[:-1]),
                sf_strides=sf_strides)


def check_alpha(alpha: Optional[torch.Tensor], device: torch.device, count: int) -> tuple[Optional[int], int]:
    """Pointer and stride of the optional fp32 factors: one for all, or `count`."""
    if alpha is None:
        return None, 0
    assert alpha.dtype == torch.float32 and alpha.device == device and alpha.numel() in (1, count)
    assert alpha.dim() <= 1
    return alpha.data_ptr(), alpha.stride(0) if alpha.numel() > 1 else 0


def check_out(out: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> None:
    assert out.shape == shape and out.dtype == dtype and out.device == device
    assert out.dim() == 2 and (out.shape[1] <= 1 or out.stride(1) == 1) and (out.shape[0] <= 1 or out.stride(0) >= out.shape[1])


def launch_block_scaled_gemm(x: dict, w: dict, expert_start, expert_end, num_experts: int, alpha, out: torch.Tensor, flags: int) -> None:
    assert x['k'] == w['k'], f"inner sizes differ: {x['k']} and {w['k']}"
    assert x['fmt'] == w['fmt'] and x['sf_fmt'] == w['sf_fmt'], 'both operands must have the same format'
    assert x['data'].device == w['data'].device
    num_rows, n, k = x['rows'], w['rows'], x['k']
    alpha_ptr, alpha_stride = check_alpha(alpha, x['data'].device, num_experts)
    w_strides = w['strides'] if len(w['strides']) == 2 else (0,) + w['strides']
    if num_rows == 0 or n == 0:
        return
    with device_guard(out.device):
        rc = _lib.lib().tkq_block_scaled_gemm(
            x['data'].data_ptr(), x['strides'][-1], x['sf'].data_ptr(), x['sf_strides'][1], x['sf_strides'][2], x['block'][0],
            x['block'][1], w['data'].data_ptr(), w_strides[0], w_strides[1], w['sf'].data_ptr(), *w['sf_strides'], w['block'][0],
            w['block'][1], FMT_TO_ENUM[x['fmt']], x['sf_fmt'], None if expert_start is None else expert_start.data_ptr(),
            None if expert_end is None else expert_end.data_ptr(), num_experts, num_rows, n, k, alpha_ptr, alpha_stride, out.data_ptr(),
            out.stride(0), flags, current_stream_ptr(out.device))
    _lib.check(rc, 'tkq_block_scaled_gemm')


def block_scaled_gemm(
    a: QuantTensor,
    b: QuantTensor,
    a_block_size: tuple[int, int],
    b_block_size: tuple[int, int],
    alpha: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """alpha * a @ b.T for two quantized matrices, in bfloat16 (one rounding of the fp32 sums).

    The data reach the tensor core in their 8- or 4-bit form; the block scales are applied there.

    Args:
        a: (data, scales) of (m, k) values, b: of (n, k).  Both in one of the forms
            float8_e4m3fn data, packed ue8m0 scales (int32) per 32 or 128 values, as per_token_cast and per_block_cast
            return them with use_packed_ue8m0;
            int8 data (two FP4 per byte) with packed ue8m0 scales per 32 values;
            int8 data with float8_e4m3fn scales per 16 values (per_token_cast_to_nvfp4).
            k is a multiple of 32 (FP8) or 64 (FP4); rows of the data start on 16-byte boundaries.
        a_block_size, b_block_size: (rows, values) per scale; rows 1, 32 or 128.
        alpha: optional fp32 tensor of one element, e.g. the product of the tensor scales of two NVFP4 operands.
        out: optional (m, n) bfloat16 destination with unit column stride.

    Returns: (m, n) bfloat16.
    """
    x, w = scaled_operand(a, a_block_size, None), scaled_operand(b, b_block_size, None)
    assert x['k'] > 0 and x['k'] == w['k'], f"inner sizes differ: {x['k']} and {w['k']}"
    shape = (x['rows'], w['rows'])
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=x['data'].device)
    else:
        check_out(out, shape, torch.bfloat16, x['data'].device)
    launch_block_scaled_gemm(x, w, None, None, 1, alpha, out, 0)
    return out
