"""FlashAttention-2 style fused attention for AMD Instinct MI355X (gfx950), HIP kernels.

Drop-in for amaanmithani/triton-attn's `tattn` package (src/tattn/__init__.py:3-5).
"""

from tattn.api import attention, autotune_cache, configs, hip_available, set_autotune, triton_available
from tattn.cross import cross_attention, prefix_attention
from tattn.norm_rope import qk_norm_rope
from tattn.paged import Cache4, PageTables, cache4_attention, cache4_read, cache4_write, page_tables
from tattn.rope_axes import qk_rope_axes
from tattn.window import window_attention

__all__ = ["attention", "triton_available", "hip_available", "configs", "set_autotune", "autotune_cache",
           "page_tables", "PageTables", "Cache4", "cache4_write", "cache4_read", "cache4_attention", "qk_norm_rope",
           "window_attention", "cross_attention", "prefix_attention", "qk_rope_axes"]
