"""B200-native (sm_100a) VMonarch attention: a drop-in for ``video_monarch_attention``.

Exports the reference's three names (reference ``video_monarch_attention/__init__.py:1-4``) and, beside
them, attention over packed sequences of different lengths and over a paged key / value
cache (in 16 or 8 bits, with a book on the host or the GPU), and the gated residual norm between a transformer's blocks.
Importing loads the in-tree CUDA library through its C ABI and raises if it is missing.
"""
from .gated_norm import gated_residual_norm  # noqa: F401
from .kernel import flash_entropy_attention
from .page_tables import PageTables, reserve_pages, truncate_pages  # noqa: F401
from .packed import PackedSequences, packed_attention  # noqa: F401
from .paged import PagedKVCache, append_pages, copy_pages, paged_attention  # noqa: F401
from .vmonarch import VMonarchAttention, vmonarch_attention

# the drop-in names: `from vmonarch_b200 import *` brings in what the reference's package does
__all__ = ["VMonarchAttention", "vmonarch_attention", "flash_entropy_attention"]
