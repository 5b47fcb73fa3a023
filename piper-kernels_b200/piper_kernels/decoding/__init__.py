"""Operators of one (speculative) decoding step over a quantised paged KV cache.

A step of a model's layer writes the new or drafted tokens' keys and values
into the cache (:func:`write_kv_cache`), then attends over it
(:func:`tree_attention`).  After the last layer the target's probabilities
decide which drafted nodes stay (:func:`verify_draft_tree`), and each layer's
cache moves their rows together (:func:`keep_draft_path`).
:func:`read_kv_cache` gives back keys and values, for instance to run
``piper_attention`` over a cached prefix.
"""

from .attention import tree_attention, tree_mask_from_parents
from .cache import QuantizedKVCache, keep_draft_path, read_kv_cache, write_kv_cache
from .verification import DraftVerification, verify_draft_tree

__all__ = [
    "DraftVerification",
    "QuantizedKVCache",
    "keep_draft_path",
    "read_kv_cache",
    "tree_attention",
    "tree_mask_from_parents",
    "verify_draft_tree",
    "write_kv_cache",
]
