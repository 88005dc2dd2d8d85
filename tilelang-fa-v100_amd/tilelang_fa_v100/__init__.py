"""MI355X (gfx950) FlashAttention, drop-in for the tilelang_fa_v100 API.

The kernels are hand-written HIP in ../csrc, built into libfa355.so and called
through a C ABI (include/fa355.h).  Exports match the reference package
(tilelang_fa_v100/__init__.py:3-16), plus
  * reshape_and_cache, the KV-cache writer that produces the paged layout the
    paged kernels read;
  * set_backward_workspace_limit, the cap on the dense backward's optional dS
    workspace (above it the backward needs only the reference's memory);
  * qk_norm_rope, the norm and rotation of queries and keys before attention
    (with gradients), and norm_rope_and_cache, its serving form that writes
    the keys and values into the paged cache;
  * linear_attn_func (with gradients), linear_attn_prefill and
    linear_attn_decode: linear attention with a decay for each head.
"""

from ._cache_write import reshape_and_cache
from ._dense import set_backward_workspace_limit
from ._linear import linear_attn_decode, linear_attn_func, linear_attn_prefill
from ._rope import norm_rope_and_cache, qk_norm_rope
from .interface import (
    FlashAttnTileLangVFunc,
    tilelang_decode_forward,
    tilelang_flash_attn_func,
    tilelang_flash_attn_gpu,
    tilelang_paged_forward,
)

__version__ = "1.0.0"
__all__ = [
    "tilelang_flash_attn_func",
    "tilelang_flash_attn_gpu",
    "tilelang_paged_forward",
    "tilelang_decode_forward",
]
# Everything the reference does not have is importable by name; __all__ stays
# the reference's list.
