"""grouped_gemm, grouped_gemm_wgrad: products of rows sorted by expert with each expert's weight, and their gradients.  The
reference lays rows out for such products (expand_to_fused) and leaves the products to another library."""
from typing import Optional, Union

import torch

from .. import _lib
from ..quant.block_scaled_gemm_kernel import ScaledOperand, check_out, launch_block_scaled_gemm
from ..quant.common import DTYPE_TO_ENUM, current_stream_ptr, device_guard, empty_matrix
from ..quant.types import QuantTensor


def _check_groups(expert_start: torch.Tensor, expert_end: torch.Tensor, num_experts: int, like: torch.Tensor) -> None:
    for t in (expert_start, expert_end):
        assert t.dtype is torch.int32 and t.get_device() == like.get_device() and t.shape == (num_experts,) and t.is_contiguous()


def _check_matrix(x: torch.Tensor, dim: int) -> None:
    assert x.dtype is torch.bfloat16 and x.is_cuda and x.dim() == dim
    assert x.shape[-1] <= 1 or x.stride(-1) == 1


def grouped_gemm(
    x: Union[torch.Tensor, QuantTensor],
    w: Union[torch.Tensor, QuantTensor],
    expert_start: torch.Tensor,
    expert_end: torch.Tensor,
    x_block_size: Optional[tuple[int, int]] = None,
    w_block_size: Optional[tuple[int, int]] = None,
    alpha: Optional[torch.Tensor] = None,
    transpose_w: bool = False,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """out[r] = x[r] @ w[e].T for the rows r of every expert e, expert_start[e] <= r < expert_end[e].

    Args:
        x: (num_rows, k) bfloat16, or a quantized pair in a form of quant.block_scaled_gemm.
        w: (num_experts, n, k) bfloat16; with transpose_w (num_experts, k, n), which with the gradient of the output as x
            gives the gradient of the input.  Or a quantized pair: data (num_experts, n, k), scales
            (num_experts, blocks of rows, words) or, for whole blocks, one matrix of all experts' rows.
        expert_start, expert_end: int32 (num_experts,), ascending; segments may be empty, of any length and alignment, and
            need not touch.  Where they overlap or go back, an expert has no rows before the end of an earlier one.  At most
            1024 experts.
        x_block_size, w_block_size: (rows, values) per scale of quantized operands, as in quant.block_scaled_gemm.
        alpha: optional fp32 tensor with one factor for all or one per expert (quantized operands).
        out: optional (num_rows, n) bfloat16 destination with unit column stride.  Rows of no expert are left as they
            are; without `out` they are zero.

    Rows of bfloat16 operands start on 16-byte boundaries (k, and n with transpose_w, multiples of 8 when contiguous), and no
    axis of the data is expanded (stride 0).

    Returns: (num_rows, n) bfloat16, rounded once from the tensor core's fp32 sums.  Those cut off what an addition shifts out,
    2^-23 of the sum at most per 16 values of k (bfloat16), 32 (FP8) or 64 (FP4): 3.2e-5 of a sum of 9000 values of one sign, where
    the rounding to bfloat16 is up to 3.9e-3.
    """
    flags = _lib.ZERO_GAPS if out is None else 0
    quantized = isinstance(x, tuple)
    if quantized:
        assert isinstance(w, tuple) and x_block_size is not None and w_block_size is not None
        assert not transpose_w, 'transpose_w takes bfloat16 weights: quantize the transposed weight instead'
        num_experts = w[0].shape[0]
        xo, wo = ScaledOperand(x, x_block_size, None), ScaledOperand(w, w_block_size, num_experts)
        num_rows, n, like = xo.rows, wo.rows, xo.data
    else:
        assert isinstance(w, torch.Tensor) and x_block_size is None and w_block_size is None and alpha is None
        _check_matrix(x, 2)
        _check_matrix(w, 3)
        num_experts, n, k = (w.shape[0], w.shape[2], w.shape[1]) if transpose_w else w.shape
        num_rows, like = x.shape[0], x
        assert w.get_device() == x.get_device()
        assert k > 0 and x.shape[1] == k, f'inner sizes differ: {x.shape[1]} and {k}'
    assert num_experts >= 1
    _check_groups(expert_start, expert_end, num_experts, like)
    device = like.device
    if out is None:
        out = empty_matrix(num_rows, n, torch.bfloat16, device)
    else:
        check_out(out, (num_rows, n), like)
    if quantized:
        launch_block_scaled_gemm(xo, wo, expert_start, expert_end, num_experts, alpha, out, flags)
    elif num_rows > 0 and n > 0:
        args = _lib.GROUPED_GEMM_ARGS.pack(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), w.stride(1), int(transpose_w), expert_start.data_ptr(),
                                           expert_end.data_ptr(), num_experts, num_rows, n, k, out.data_ptr(), out.stride(0), flags)
        with device_guard(device):
            rc = _lib.lib().tkq_grouped_gemm(args, current_stream_ptr(device))
        if rc:
            _lib.check(rc, 'tkq_grouped_gemm')
    return out


def grouped_gemm_wgrad(
    grad: torch.Tensor,
    x: torch.Tensor,
    expert_start: torch.Tensor,
    expert_end: torch.Tensor,
    out_dtype: torch.dtype = torch.float32,
    out: Optional[torch.Tensor] = None,
    accumulate: bool = False,
) -> torch.Tensor:
    """The gradient of grouped_gemm's weight: dw[e] = grad[rows of e].T @ x[rows of e].

    Args:
        grad: (num_rows, n) bfloat16, gradient of the output.
        x: (num_rows, k) bfloat16, the input.  Rows of both start on 16-byte boundaries.
        expert_start, expert_end: as in grouped_gemm; rows of no expert are not read into any sum.
        out_dtype: torch.float32 or torch.bfloat16.
        out: optional contiguous (num_experts, n, k) destination of out_dtype.
        accumulate: add to `out` (float32 only), one fp32 addition; experts without rows leave their part alone.

    Returns: (num_experts, n, k); zeros for experts without rows.  The tensor core, which cuts off instead of rounding (see
    grouped_gemm), adds up 256 rows at a time for float32, up to 16384 for bfloat16; beyond that sums are rounded fp32 additions.
    """
    _check_matrix(grad, 2)
    _check_matrix(x, 2)
    assert grad.get_device() == x.get_device() and grad.shape[0] == x.shape[0]
    assert out_dtype is torch.float32 or out_dtype is torch.bfloat16
    num_rows, n, k = x.shape[0], grad.shape[1], x.shape[1]
    num_experts = expert_start.numel()
    assert num_experts >= 1
    _check_groups(expert_start, expert_end, num_experts, x)
    device = x.device
    if out is None:
        assert not accumulate, 'accumulate needs out'
        out = torch.empty_strided((num_experts, n, k), (max(n * k, 1), max(k, 1), 1), dtype=out_dtype, device=device)
    else:
        assert out.shape == (num_experts, n, k) and out.dtype is out_dtype and out.get_device() == x.get_device() and out.is_contiguous()
        assert not accumulate or out_dtype is torch.float32, 'accumulate needs a float32 destination'
    if n > 0 and k > 0:
        args = _lib.GROUPED_GEMM_WGRAD_ARGS.pack(grad.data_ptr(), grad.stride(0), x.data_ptr(), x.stride(0), expert_start.data_ptr(), expert_end.data_ptr(),
                                                 num_experts, num_rows, n, k, DTYPE_TO_ENUM[out_dtype], out.data_ptr(),
                                                 _lib.ACCUMULATE if accumulate else 0)
        with device_guard(device):
            rc = _lib.lib().tkq_grouped_gemm_wgrad(args, current_stream_ptr(device))
        if rc:
            _lib.check(rc, 'tkq_grouped_gemm_wgrad')
    return out
