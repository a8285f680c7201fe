"""B200-native (sm_100a) implementation of the Kairos hybrid-attention hot path.

Public operators keep the reference's PyTorch signatures:

* :func:`chunk_gated_delta_rule`  -- ``fla/ops/gated_delta_rule/chunk.py:216``

Serving operators, without a counterpart in the reference:

* :func:`attention_prompt` -- causal attention over packed prompts with grouped heads
* :class:`KVCache`, :func:`kv_cache_append`, :func:`kv_cache_gather` -- an 8-bit paged key/value cache
* :func:`attention_cached` -- attention of the newest tokens over that cache
"""
from .attention import attention_prompt  # noqa: F401
from .gated_delta_rule import chunk_gated_delta_rule  # noqa: F401
from .kv_cache import KVCache, attention_cached, kv_cache_append, kv_cache_gather  # noqa: F401

__all__ = ['chunk_gated_delta_rule', 'attention_prompt', 'KVCache', 'kv_cache_append', 'kv_cache_gather',
           'attention_cached']
