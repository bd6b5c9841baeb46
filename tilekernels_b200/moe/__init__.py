"""MoE entry points next to the quantization path: row expansion with scale factors (reference: tile_kernels/moe/__init__.py,
expand_to_fused_kernel.py) and the products grouped by expert that its rows are laid out for.  The rest of the reference's
moe package (gating, mapping, reduction) is outside this library."""
from .. import _lib as _lib_module

_lib_module.lib()  # fail at import when the CUDA library is missing

from .expand_to_fused_kernel import expand_to_fused, expand_to_fused_with_sf  # noqa: E402
from .grouped_gemm_kernel import grouped_gemm, grouped_gemm_wgrad  # noqa: E402
