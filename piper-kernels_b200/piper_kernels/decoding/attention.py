"""Attention of a drafted tree's nodes over the quantised cache."""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch

from .. import _native
from ._common import DTYPE_CODES, MAX_NODES, check_half, check_tensor, direct, fits, launch, refuse_grad, require_device
from .cache import QuantizedKVCache, check_batch, check_cache_grad

OPERATOR = "tree_attention"


def tree_attention(
    query: torch.Tensor,
    cache: QuantizedKVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    tree_mask: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of the newest tokens of each request over its cached tokens.

    ``query`` is float16 or bfloat16 ``[batch, heads, nodes, head_dim]`` (a
    contiguous head dimension, any other strides) with 1 to 64 nodes; ``heads``
    is a multiple of the cache's KV heads, and query head ``h`` reads KV head
    ``h // (heads // kv_heads)``.  The nodes' own keys and values are in the
    cache already, at positions ``lengths[b] + node``
    (:func:`~piper_kernels.write_kv_cache`).

    Every node sees the ``lengths[b]`` committed tokens.  Of the nodes it sees
    those whose bit is set in its word of ``tree_mask`` (int64 ``[batch,
    nodes]``, or ``[nodes]`` for one tree for all;
    :func:`~piper_kernels.tree_mask_from_parents`); by default node ``t`` sees
    nodes 0 to ``t``, which for one node is plain decoding.  A node that sees
    nothing gets zeros.  ``scale`` defaults to ``head_dim ** -0.5`` (from 2**-126
    to 2**127).

    Returns a contiguous ``[batch, heads, nodes, head_dim]`` of ``query``'s
    type.  Inference only.
    """
    out = direct(
        "attend", "piper_b200_tree_attention", cache.buffers, query, block_table, lengths, tree_mask, scale
    )
    if out is not None:
        return out
    effective = _check(query, cache, block_table, lengths, tree_mask, scale)
    return torch.ops.piper_kernels.tree_attention(
        query, cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales, block_table, lengths,
        tree_mask, effective,
    )


def _check(
    query: torch.Tensor,
    cache: QuantizedKVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    tree_mask: torch.Tensor | None,
    scale: float | None,
) -> float:
    """Check a call's arguments; the scale that it uses."""
    cache.check()
    if query.ndim != 4:
        raise ValueError(
            f"{OPERATOR} query must have shape [batch, heads, sequence, head_dim], got {tuple(query.shape)}"
        )
    batch, heads, nodes, _ = query.shape
    device, dtype, head_dim = cache.device, query.dtype, cache.head_dim
    if dtype not in DTYPE_CODES:
        check_half(OPERATOR, "query", dtype)
    if not fits(query, (batch, heads, nodes, head_dim), dtype, device):
        check_tensor(OPERATOR, "query", query, (batch, heads, nodes, head_dim), dtype, device)
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"{OPERATOR} supports 1 to {MAX_NODES} nodes, got {nodes}")
    if heads == 0 or heads % cache.kv_heads != 0:
        raise ValueError(f"{OPERATOR} heads must be a multiple of the cache's {cache.kv_heads} KV heads, got {heads}")
    check_batch(OPERATOR, cache, batch, block_table, lengths)
    if tree_mask is not None:
        shape = (nodes,) if tree_mask.ndim == 1 else (batch, nodes)
        if not fits(tree_mask, shape, torch.int64, device):
            check_tensor(OPERATOR, "tree_mask", tree_mask, shape, torch.int64, device)
    if query.requires_grad and torch.is_grad_enabled():
        refuse_grad(OPERATOR)
    check_cache_grad(OPERATOR, cache, mean=False)
    effective = head_dim**-0.5 if scale is None else float(scale)
    if not math.isfinite(effective) or effective <= 0:
        raise ValueError(f"{OPERATOR} scale must be finite and positive, got {scale}")
    if not 2.0**-126 <= effective <= 2.0**127:
        raise ValueError(f"{OPERATOR} scale must be from 2**-126 to 2**127, got {scale}")
    require_device(OPERATOR, device)
    return effective


def workspace_bytes(batch: int, heads: int, kv_heads: int, nodes: int, head_dim: int, positions: int) -> int:
    """Workspace of one call on the current device, whose block table has room for ``positions`` tokens (0: none)."""
    size = ctypes.c_size_t(0)
    _native.check(
        _native.library().piper_b200_tree_attention_workspace_bytes(
            batch, heads, kv_heads, nodes, head_dim, positions, ctypes.byref(size)
        ),
        "piper_b200_tree_attention_workspace_bytes",
    )
    return int(size.value)


@lru_cache(maxsize=4096)  # the same few shapes come back every step
def _workspace_bytes(device: int, *sizes: int) -> int:
    with torch.cuda.device(device):  # (the plan goes by its SMs)
        return workspace_bytes(*sizes)


def _run(query, cache, block_table, lengths, tree_mask, scale) -> torch.Tensor:
    batch, heads, nodes, head_dim = query.shape
    device = query.device
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    nbytes = _workspace_bytes(
        device.index, batch, heads, cache.kv_heads, nodes, head_dim, block_table.shape[1] * cache.page_size
    )
    workspace = out.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    mask_ptr, mask_stride = None, 0
    if tree_mask is not None:
        mask_ptr, mask_stride = tree_mask.data_ptr(), tree_mask.stride(0) if tree_mask.ndim == 2 else 0
    launch(
        "piper_b200_tree_attention", device, _native.library().piper_b200_tree_attention,
        ctypes.byref(cache.native(block_table, lengths)), query.data_ptr(), _native.strides3(query), out.data_ptr(),
        DTYPE_CODES[query.dtype], heads, nodes, mask_ptr, mask_stride, scale,
        None if workspace is None else workspace.data_ptr(), nbytes,
    )
    return out


def tree_mask_from_parents(parents: torch.Tensor) -> torch.Tensor:
    """The words of ``tree_attention``'s ``tree_mask``: each node sees itself and its ancestors.

    ``parents`` is an integer tensor ``[nodes]`` or ``[batch, nodes]`` of at
    most 64 nodes; ``parents[..., i] < i`` names node ``i``'s parent, and a
    negative entry (the root's) means that it has none.  Plain torch
    operations, on any device; a tree that stays the same needs it once.
    """
    if parents.ndim not in (1, 2):
        raise ValueError(f"tree_mask_from_parents parents must have 1 or 2 dimensions, got {tuple(parents.shape)}")
    if parents.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tree_mask_from_parents parents must use int32 or int64, got {parents.dtype}")
    nodes = parents.shape[-1]
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"tree_mask_from_parents supports 1 to {MAX_NODES} nodes, got {nodes}")
    mask = torch.zeros(parents.shape, dtype=torch.int64, device=parents.device)
    for i in range(nodes):
        word = torch.full_like(mask[..., 0], 1 << i if i < 63 else -(1 << 63))
        if i:
            parent = parents[..., i].to(torch.int64)
            above = mask[..., :i].gather(-1, parent.clamp(0, i - 1).unsqueeze(-1)).squeeze(-1)
            word = torch.where((parent >= 0) & (parent < i), word | above, word)
        mask[..., i] = word
    return mask


@torch.library.custom_op("piper_kernels::tree_attention", mutates_args=())
def _tree_attention_op(
    query: torch.Tensor,
    key_codes: torch.Tensor,
    key_scales: torch.Tensor,
    value_codes: torch.Tensor,
    value_scales: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    tree_mask: torch.Tensor | None,
    scale: float,
) -> torch.Tensor:
    cache = QuantizedKVCache(key_codes, key_scales, value_codes, value_scales)
    _check(query, cache, block_table, lengths, tree_mask, scale)
    return _run(query, cache, block_table, lengths, tree_mask, scale)


@_tree_attention_op.register_fake
def _tree_attention_fake(query, *_args) -> torch.Tensor:
    return torch.empty_like(query, memory_format=torch.contiguous_format)
