"""per_token_cast_to_nvfp4: FP4 with an e4m3 scale per 16 values and one fp32 scale per tensor; and its way back, which
cast_back calls.  The reference's FP4 cast has power-of-two scales only (tile_kernels/quant/per_token_cast_kernel.py)."""
import torch

from .. import _lib
from .common import DTYPE_TO_ENUM, current_stream_ptr, device_guard, empty_matrix
from .types import QuantTensor


def _check_tensor_scale(tensor_scale: torch.Tensor, device: torch.device) -> None:
    assert isinstance(tensor_scale, torch.Tensor), 'tensor_scale is a CUDA tensor: its value is read on the device'
    assert tensor_scale.dtype is torch.float32 and tensor_scale.numel() == 1 and tensor_scale.get_device() == device.index


def per_token_cast_to_nvfp4(x: torch.Tensor, tensor_scale: torch.Tensor) -> QuantTensor:
    """Cast a matrix to FP4 e2m1 with one e4m3 scale per 16 values of a row.

    A value stands for code * scale * tensor_scale.  The scale of a block is the e4m3 number nearest to
    max|x| / (6 * tensor_scale), at most 448; the codes are the e2m1 numbers nearest to x / (scale * tensor_scale), both of
    the exact quotients with ties to even, 0 in blocks whose scale rounds to 0.  Values beyond the range saturate; NaN has
    no code of its own.

    Args:
        x: (num_tokens, hidden) bfloat16 or float32 CUDA tensor, hidden a multiple of 16, rows may be strided (16-byte
            boundaries).
        tensor_scale: fp32 CUDA tensor of one element, positive; usually max|x| / (6 * 448) of the tensor or of a
            calibration set.

    Returns: (out, out_sf): int8 (num_tokens, hidden / 2), even index in the low nibble; float8_e4m3fn
        (num_tokens, hidden / 16), row-major.
    """
    assert x.dim() == 2 and x.is_cuda and x.dtype in (torch.bfloat16, torch.float32)
    num_tokens, hidden = x.shape
    assert hidden > 0 and hidden % 16 == 0 and x.stride(1) == 1
    _check_tensor_scale(tensor_scale, x.device)
    device = x.device
    out = empty_matrix(num_tokens, hidden // 2, torch.int8, device)
    out_sf = empty_matrix(num_tokens, hidden // 16, torch.float8_e4m3fn, device)
    if num_tokens > 0:
        with device_guard(x.device):
            rc = _lib.lib().tkq_per_token_cast_nvfp4(x.data_ptr(), DTYPE_TO_ENUM[x.dtype], num_tokens, hidden, x.stride(0),
                                                     tensor_scale.data_ptr(), out.data_ptr(), out_sf.data_ptr(), current_stream_ptr(x.device))
        if rc:
            _lib.check(rc, 'tkq_per_token_cast_nvfp4')
    return out, out_sf


def cast_back_nvfp4(x: QuantTensor, fmt: str, tensor_scale: torch.Tensor) -> torch.Tensor:
    """Dequantise what per_token_cast_to_nvfp4 returns."""
    data, sf = x
    assert data.dim() == 2 and data.dtype == torch.int8 and data.is_contiguous() and data.is_cuda
    num_tokens, hidden = data.shape[0], data.shape[1] * 2
    assert hidden > 0 and hidden % 16 == 0
    assert sf.dtype == torch.float8_e4m3fn and sf.shape == (num_tokens, hidden // 16) and sf.is_contiguous() and sf.get_device() == data.get_device()
    _check_tensor_scale(tensor_scale, data.device)
    out = empty_matrix(num_tokens, hidden, torch.bfloat16 if fmt == 'bf16' else torch.float32, data.device)
    if num_tokens > 0:
        with device_guard(data.device):
            rc = _lib.lib().tkq_cast_back_nvfp4(data.data_ptr(), sf.data_ptr(), tensor_scale.data_ptr(), num_tokens, hidden,
                                                DTYPE_TO_ENUM[out.dtype], out.data_ptr(), current_stream_ptr(data.device))
        if rc:
            _lib.check(rc, 'tkq_cast_back_nvfp4')
    return out
