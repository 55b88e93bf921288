"""shard_amd — MI355X-native compressed-KV attention path of Shard.

Public API (same names as the reference package ``shard``):
    Cache, enable_llama_fused_attention, fused_attention_compressed
and, with no counterpart there, PagedCache: a paged cache held in 4 bits for
batches of uneven sequences, and token_logprobs.
The kernels live in libshard_hip.so (built in-tree by shard_amd.build).
"""
from .cache import Cache, CacheLayer
from .attention import enable_llama_fused_attention, fused_attention_compressed
from .ops import token_logprobs
from .paged import PagedCache

__all__ = ["Cache", "CacheLayer", "PagedCache", "enable_llama_fused_attention", "fused_attention_compressed",
           "token_logprobs"]
__version__ = "0.1.0"
