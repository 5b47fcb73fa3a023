"""Piper Kernels -- B200 (sm_100a) backend of the attention operators.

Drop-in for the reference package's public entry points
(Piper Kernels 0.2.1, ``src/piper_kernels/__init__.py:3-6``): the same
``piper_kernels.piper_attention`` and ``piper_kernels.sage_attention_2pp``
functions and the same ``torch.ops.piper_kernels.*`` custom operators,
computed by hand-written sm_100a CUDA kernels behind the C ABI in
``include/piper_b200.h``.

Next to them, the operators of a (speculative) decoding step over a quantised
paged KV cache (:mod:`piper_kernels.decoding`), which the reference does not
have.
"""

from .attention.piper_attention import piper_attention
from .attention.sage_attention_2pp import sage_attention_2pp
from .decoding import DraftVerification as DraftVerification
from .decoding import QuantizedKVCache as QuantizedKVCache
from .decoding import keep_draft_path as keep_draft_path
from .decoding import read_kv_cache as read_kv_cache
from .decoding import tree_attention as tree_attention
from .decoding import tree_mask_from_parents as tree_mask_from_parents
from .decoding import verify_draft_tree as verify_draft_tree
from .decoding import write_kv_cache as write_kv_cache

# A star import gives the reference package's names and no others; the decoding
# operators are attributes of the package, and decoding.__all__ lists them.
__all__ = ["piper_attention", "sage_attention_2pp"]
