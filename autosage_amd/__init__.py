"""MI355X-native (gfx950 HIP) implementation of AutoSAGE's sparse hot path.

Public names are those of the reference package (``autosage/__init__.py:1-17``),
and the operators it has no counterpart of: the learned position bias of edges
and the paged key-value cache with its attention.
"""

from ._auto import calibrate_full, csr_attention_forward, sddmm_csr_auto, spmm_csr_auto
from ._version import __version__
from .conv import AutoSAGEConv
from .ops import load_native, native_available, spmm_csr, validate_csr
from .paged import paged_attention, paged_cache_read, paged_cache_write
from .position import csr_position_bias

__all__ = [
    "AutoSAGEConv",
    "__version__",
    "calibrate_full",
    "csr_attention_forward",
    "csr_position_bias",
    "load_native",
    "native_available",
    "paged_attention",
    "paged_cache_read",
    "paged_cache_write",
    "sddmm_csr_auto",
    "spmm_csr",
    "spmm_csr_auto",
    "validate_csr",
]
