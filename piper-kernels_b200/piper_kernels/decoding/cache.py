"""The quantised paged KV cache: its buffers, and writing, reading and moving rows.

A row is one token of one KV head.  Its ``head_dim`` values ``x`` (for keys
less ``key_mean``) are held as INT8 codes and one fp32 scale::

    scale = max|x| * fp32(1/127)      (1 for a row of zeros)
    code  = round half to even (x / scale)

and stand for ``code * scale`` (plus ``key_mean`` for keys).  A constant taken
off every key does not change a softmax over keys, so attention over the cache
does not need the mean; it only makes the codes finer, like the K smoothing of
``piper_attention``.

A request's tokens lie in the pages that its row of ``block_table`` names, in
order; ``lengths`` counts its committed tokens, and token ``i`` of a call has
position ``lengths[b] + i``.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _native
from ._common import (
    DTYPE_CODES,
    MAX_NODES,
    SUPPORTED_HEAD_DIMS,
    check_half,
    check_tensor,
    direct,
    fits,
    launch,
    refuse_grad,
    require_device,
)

PAGE_SIZES = (16, 32, 64, 128, 256)


class QuantizedKVCache:
    """Buffers of one layer's cache; a handle that a program keeps.

    ``key_codes`` and ``value_codes`` are int8 ``[pages, kv_heads, page_size,
    head_dim]``, ``key_scales`` and ``value_scales`` float32 ``[pages,
    kv_heads, page_size]``, all contiguous on one device.  ``key_mean`` is
    float32 ``[kv_heads, head_dim]`` or None; it belongs to the rows written
    with it.  ``page_size`` is 16, 32, 64, 128 or 256, ``head_dim`` 64 or 128.
    The buffers are read-only attributes (``buffers``: all five), like the
    sizes ``pages``, ``kv_heads``, ``page_size`` and ``head_dim`` and the
    ``device``; every call checks that they still belong together.
    """

    __slots__ = ("_buffers",)

    def __init__(
        self,
        key_codes: torch.Tensor,
        key_scales: torch.Tensor,
        value_codes: torch.Tensor,
        value_scales: torch.Tensor,
        key_mean: torch.Tensor | None = None,
    ) -> None:
        self._buffers = (key_codes, key_scales, value_codes, value_scales, key_mean)
        self.check()

    def check(self) -> None:
        """Raise ``ValueError`` unless the buffers are what the class says."""
        key_codes, key_scales, value_codes, value_scales, key_mean = self._buffers
        shape, device = key_codes.shape, key_codes.device
        if not (
            len(shape) == 4
            and shape[0] > 0
            and shape[1] > 0
            and shape[2] in PAGE_SIZES
            and shape[3] in SUPPORTED_HEAD_DIMS
            and key_codes.dtype is torch.int8
            and key_codes.is_contiguous()
            and fits(value_codes, shape, torch.int8, device)
            and value_codes.is_contiguous()
            and fits(key_scales, shape[:3], torch.float32, device)
            and key_scales.is_contiguous()
            and fits(value_scales, shape[:3], torch.float32, device)
            and value_scales.is_contiguous()
            and (key_mean is None or fits(key_mean, shape[1::2], torch.float32, device) and key_mean.is_contiguous())
        ):
            _refuse_buffers(key_codes, key_scales, value_codes, value_scales, key_mean)

    @classmethod
    def allocate(
        cls,
        pages: int,
        kv_heads: int,
        page_size: int,
        head_dim: int,
        *,
        device: torch.device | str | int | None = None,
        key_mean: torch.Tensor | None = None,
    ) -> "QuantizedKVCache":
        """A new cache whose rows all stand for zero."""
        shape = (pages, kv_heads, page_size, head_dim)
        if device is None:
            device = "cuda"
        return cls(
            torch.zeros(shape, dtype=torch.int8, device=device),
            torch.ones(shape[:3], dtype=torch.float32, device=device),
            torch.zeros(shape, dtype=torch.int8, device=device),
            torch.ones(shape[:3], dtype=torch.float32, device=device),
            key_mean=key_mean,
        )

    @property
    def buffers(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor | None]:
        return self._buffers

    @property
    def key_codes(self) -> torch.Tensor:
        return self._buffers[0]

    @property
    def key_scales(self) -> torch.Tensor:
        return self._buffers[1]

    @property
    def value_codes(self) -> torch.Tensor:
        return self._buffers[2]

    @property
    def value_scales(self) -> torch.Tensor:
        return self._buffers[3]

    @property
    def key_mean(self) -> torch.Tensor | None:
        return self._buffers[4]

    @property
    def device(self) -> torch.device:
        return self._buffers[0].device

    @property
    def pages(self) -> int:
        return self._buffers[0].shape[0]

    @property
    def kv_heads(self) -> int:
        return self._buffers[0].shape[1]

    @property
    def page_size(self) -> int:
        return self._buffers[0].shape[2]

    @property
    def head_dim(self) -> int:
        return self._buffers[0].shape[3]

    def native(self, block_table: torch.Tensor, lengths: torch.Tensor) -> _native.KVCache:
        """The C ABI's description of this cache for one batch."""
        key_codes, key_scales, value_codes, value_scales, key_mean = self.buffers
        batch, width = block_table.shape
        return _native.KVCache(
            key_codes.data_ptr(), key_scales.data_ptr(), value_codes.data_ptr(), value_scales.data_ptr(),
            None if key_mean is None else key_mean.data_ptr(), block_table.data_ptr(), lengths.data_ptr(),
            self.pages, block_table.stride(0), self.kv_heads, self.page_size, self.head_dim, batch, width,
        )


def _refuse_buffers(key_codes, key_scales, value_codes, value_scales, key_mean) -> None:
    """Say what is wrong with a cache's buffers."""
    name = "QuantizedKVCache"
    if key_codes.ndim != 4:
        raise ValueError(
            f"{name} key_codes must have shape [pages, kv_heads, page_size, head_dim], got {tuple(key_codes.shape)}"
        )
    pages, kv_heads, page_size, head_dim = key_codes.shape
    if head_dim not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"{name} supports head dimensions 64 and 128, got {head_dim}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"{name} page_size must be one of {PAGE_SIZES}, got {page_size}")
    if pages == 0 or kv_heads == 0:
        raise ValueError(f"{name} needs at least one page and one KV head")
    for label, tensor, shape, dtype in (
        ("key_codes", key_codes, key_codes.shape, torch.int8),
        ("value_codes", value_codes, key_codes.shape, torch.int8),
        ("key_scales", key_scales, key_codes.shape[:3], torch.float32),
        ("value_scales", value_scales, key_codes.shape[:3], torch.float32),
        ("key_mean", key_mean, (kv_heads, head_dim), torch.float32),
    ):
        if tensor is not None:
            check_tensor(name, label, tensor, shape, dtype, key_codes.device)
            if not tensor.is_contiguous():
                raise ValueError(f"{name} {label} must be contiguous")
    raise ValueError(f"{name} buffers do not belong together")


def check_batch(
    operator: str, cache: QuantizedKVCache, batch: int, block_table: torch.Tensor, lengths: torch.Tensor
) -> None:
    """Check the arguments that say where a batch's tokens lie."""
    table = block_table.shape
    if (
        batch > 0
        and len(table) == 2
        and table[1] > 0
        and fits(block_table, (batch, table[1]), torch.int32, cache.device)
        and fits(lengths, (batch,), torch.int32, cache.device)
    ):
        return
    if batch == 0:
        raise ValueError(f"{operator} does not accept an empty batch")
    check_tensor(operator, "block_table", block_table, (batch, None), torch.int32, cache.device)
    check_tensor(operator, "lengths", lengths, (batch,), torch.int32, cache.device)
    if block_table.shape[1] == 0:
        raise ValueError(f"{operator} block_table must have at least one column")


def check_cache_grad(operator: str, cache: QuantizedKVCache, *, mean: bool) -> None:
    """Refuse a cache whose scales (or key mean, if the call's result depends on it) want a gradient."""
    tensors = (cache.key_scales, cache.value_scales, cache.key_mean if mean else None)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        refuse_grad(operator)


def write_kv_cache(
    cache: QuantizedKVCache,
    key: torch.Tensor,
    value: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    counts: torch.Tensor | None = None,
) -> None:
    """Quantise new keys and values into the cache, in place.

    ``key`` and ``value`` are float16 or bfloat16 ``[batch, kv_heads, tokens,
    head_dim]`` with a contiguous head dimension and any other strides; token
    ``i`` of request ``b`` goes to position ``lengths[b] + i`` if ``i <
    counts[b]`` (int32; default: every token).  ``block_table`` is int32
    ``[batch, columns]``, ``lengths`` int32 ``[batch]``; ``lengths`` is not
    changed.  Tokens whose position has no page (a column past the table, or an
    entry that is no page of the cache, such as -1) are not written.  Pages
    that are written must not be shared between requests.
    """
    if direct(
        "write", "piper_b200_kv_cache_write", cache.buffers, key, value, block_table, lengths, counts
    ) is not None:
        return
    _check_write(cache, key, value, block_table, lengths, counts)
    torch.ops.piper_kernels.write_kv_cache(
        cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales, cache.key_mean, key, value,
        block_table, lengths, counts,
    )


def _check_write(cache, key, value, block_table, lengths, counts) -> None:
    operator = "write_kv_cache"
    cache.check()
    if key.ndim != 4:
        raise ValueError(f"{operator} key must have shape [batch, heads, sequence, head_dim], got {tuple(key.shape)}")
    batch, _, tokens, _ = key.shape
    device, dtype, shape = cache.device, key.dtype, (batch, cache.kv_heads, tokens, cache.head_dim)
    if dtype not in DTYPE_CODES:
        check_half(operator, "key", dtype)
    if not (fits(key, shape, dtype, device) and fits(value, shape, dtype, device)):
        check_tensor(operator, "key", key, shape, dtype, device)
        check_tensor(operator, "value", value, shape, dtype, device)
    if tokens == 0:
        raise ValueError(f"{operator} does not accept an empty sequence")
    check_batch(operator, cache, batch, block_table, lengths)
    if counts is not None and not fits(counts, (batch,), torch.int32, device):
        check_tensor(operator, "counts", counts, (batch,), torch.int32, device)
    if (key.requires_grad or value.requires_grad) and torch.is_grad_enabled():
        refuse_grad(operator)
    check_cache_grad(operator, cache, mean=True)
    require_device(operator, cache.device)


def _write(cache, key, value, block_table, lengths, counts) -> None:
    launch(
        "piper_b200_kv_cache_write", cache.device, _native.library().piper_b200_kv_cache_write,
        ctypes.byref(cache.native(block_table, lengths)), key.data_ptr(), _native.strides3(key), value.data_ptr(),
        _native.strides3(value), DTYPE_CODES[key.dtype], key.shape[2], None if counts is None else counts.data_ptr(),
    )


def read_kv_cache(
    cache: QuantizedKVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    tokens: int,
    *,
    counts: torch.Tensor | None = None,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of cached rows, as ``dtype`` ``[batch, kv_heads, tokens, head_dim]``.

    Token ``i`` of request ``b`` is the row at position ``lengths[b] + i``
    (``lengths`` of zeros reads from the start); tokens from ``counts[b]`` on
    (default: none), and positions without a page, read as zeros.
    """
    if dtype in DTYPE_CODES:
        out = direct(
            "read", "piper_b200_kv_cache_read", cache.buffers, block_table, lengths, counts, tokens,
            dtype is torch.float16,
        )
        if out is not None:
            return out
    tokens = int(tokens)
    _check_read(cache, block_table, lengths, counts, tokens, dtype)
    return torch.ops.piper_kernels.read_kv_cache(
        cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales, cache.key_mean, block_table,
        lengths, counts, tokens, dtype,
    )


def _check_read(cache, block_table, lengths, counts, tokens, dtype) -> None:
    operator = "read_kv_cache"
    cache.check()
    if dtype not in DTYPE_CODES:
        check_half(operator, "dtype", dtype)
    if tokens <= 0:
        raise ValueError(f"{operator} tokens must be positive, got {tokens}")
    if lengths.ndim != 1:
        raise ValueError(f"{operator} lengths must have shape [batch], got {tuple(lengths.shape)}")
    check_batch(operator, cache, lengths.shape[0], block_table, lengths)
    if counts is not None and not fits(counts, (lengths.shape[0],), torch.int32, cache.device):
        check_tensor(operator, "counts", counts, (lengths.shape[0],), torch.int32, cache.device)
    check_cache_grad(operator, cache, mean=True)
    require_device(operator, cache.device)


def _read(cache, block_table, lengths, counts, tokens, dtype) -> tuple[torch.Tensor, torch.Tensor]:
    shape = (lengths.shape[0], cache.kv_heads, tokens, cache.head_dim)
    key = cache.key_codes.new_empty(shape, dtype=dtype)
    value = torch.empty_like(key)
    launch(
        "piper_b200_kv_cache_read", cache.device, _native.library().piper_b200_kv_cache_read,
        ctypes.byref(cache.native(block_table, lengths)), key.data_ptr(), value.data_ptr(), DTYPE_CODES[dtype],
        tokens, None if counts is None else counts.data_ptr(),
    )
    return key, value


def keep_draft_path(
    cache: QuantizedKVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    path: torch.Tensor,
    counts: torch.Tensor,
) -> None:
    """Move the accepted drafted rows together, in place.

    ``path`` (int32 ``[batch, nodes]``) and ``counts`` (int32 ``[batch]``) are
    :func:`~piper_kernels.verify_draft_tree`'s: the row at position
    ``lengths[b] + path[b, j]`` moves to ``lengths[b] + j`` for ``1 <= j <
    counts[b]``.  ``lengths`` is not changed; the committed length is then
    ``lengths + counts``.
    """
    if direct("keep", "piper_b200_kv_cache_keep", cache.buffers, block_table, lengths, path, counts) is not None:
        return
    _check_keep(cache, block_table, lengths, path, counts)
    torch.ops.piper_kernels.keep_draft_path(
        cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales, block_table, lengths, path, counts
    )


def _check_keep(cache, block_table, lengths, path, counts) -> None:
    operator = "keep_draft_path"
    cache.check()
    if path.ndim != 2:
        raise ValueError(f"{operator} path must have shape [batch, nodes], got {tuple(path.shape)}")
    batch, nodes = path.shape
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"{operator} supports 1 to {MAX_NODES} nodes, got {nodes}")
    check_batch(operator, cache, batch, block_table, lengths)
    device = cache.device
    if not (fits(path, (batch, nodes), torch.int32, device) and fits(counts, (batch,), torch.int32, device)):
        check_tensor(operator, "path", path, (batch, nodes), torch.int32, device)
        check_tensor(operator, "counts", counts, (batch,), torch.int32, device)
    check_cache_grad(operator, cache, mean=False)
    require_device(operator, cache.device)


def _keep(cache, block_table, lengths, path, counts) -> None:
    launch(
        "piper_b200_kv_cache_keep", cache.device, _native.library().piper_b200_kv_cache_keep,
        ctypes.byref(cache.native(block_table, lengths)), path.data_ptr(), path.stride(0), path.shape[1],
        counts.data_ptr(),
    )


_BUFFERS = ("key_codes", "key_scales", "value_codes", "value_scales")


@torch.library.custom_op("piper_kernels::write_kv_cache", mutates_args=_BUFFERS)
def _write_op(
    key_codes: torch.Tensor,
    key_scales: torch.Tensor,
    value_codes: torch.Tensor,
    value_scales: torch.Tensor,
    key_mean: torch.Tensor | None,
    key: torch.Tensor,
    value: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    counts: torch.Tensor | None,
) -> None:
    cache = QuantizedKVCache(key_codes, key_scales, value_codes, value_scales, key_mean)
    _check_write(cache, key, value, block_table, lengths, counts)
    _write(cache, key, value, block_table, lengths, counts)


@_write_op.register_fake
def _write_fake(*_args) -> None:
    return None


@torch.library.custom_op("piper_kernels::read_kv_cache", mutates_args=())
def _read_op(
    key_codes: torch.Tensor,
    key_scales: torch.Tensor,
    value_codes: torch.Tensor,
    value_scales: torch.Tensor,
    key_mean: torch.Tensor | None,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    counts: torch.Tensor | None,
    tokens: int,
    dtype: torch.dtype,
) -> tuple[torch.Tensor, torch.Tensor]:
    cache = QuantizedKVCache(key_codes, key_scales, value_codes, value_scales, key_mean)
    _check_read(cache, block_table, lengths, counts, tokens, dtype)
    return _read(cache, block_table, lengths, counts, tokens, dtype)


@_read_op.register_fake
def _read_fake(
    key_codes, _key_scales, _value_codes, _value_scales, _key_mean, _block_table, lengths, _counts, tokens, dtype
):
    shape = (lengths.shape[0], key_codes.shape[1], tokens, key_codes.shape[3])
    return key_codes.new_empty(shape, dtype=dtype), key_codes.new_empty(shape, dtype=dtype)


@torch.library.custom_op("piper_kernels::keep_draft_path", mutates_args=_BUFFERS)
def _keep_op(
    key_codes: torch.Tensor,
    key_scales: torch.Tensor,
    value_codes: torch.Tensor,
    value_scales: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    path: torch.Tensor,
    counts: torch.Tensor,
) -> None:
    cache = QuantizedKVCache(key_codes, key_scales, value_codes, value_scales)
    _check_keep(cache, block_table, lengths, path, counts)
    _keep(cache, block_table, lengths, path, counts)


@_keep_op.register_fake
def _keep_fake(*_args) -> None:
    return None
