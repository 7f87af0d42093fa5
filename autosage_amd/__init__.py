"""MI355X-native (gfx950 HIP) implementation of AutoSAGE's sparse hot path.

Public names are those of the reference package (``autosage/__init__.py:1-17``),
and the operators it has no counterpart of: the learned position bias of edges,
rotary positions, and the paged key-value cache with its lists and its attention.
"""

from ._auto import calibrate_full, csr_attention_forward, sddmm_csr_auto, spmm_csr_auto
from ._version import __version__
from .conv import AutoSAGEConv
from .ops import load_native, native_available, spmm_csr, validate_csr
from .paged import paged_attention, paged_cache_read, paged_cache_write
from .paged_lists import paged_cache_resize
from .position import csr_position_bias
from .rotary import rotary_frequencies, rotary_positions

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
    "paged_cache_resize",
    "paged_cache_write",
    "rotary_frequencies",
    "rotary_positions",
    "sddmm_csr_auto",
    "spmm_csr",
    "spmm_csr_auto",
    "validate_csr",
]
