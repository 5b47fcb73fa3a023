"""Decoding operators on the GPU against plain implementations (B200 only).

Codes, scales, moved rows and verification decisions are compared exactly;
attention against float64 with a bound for each element (oracle/decoding.py)
beside the rounding of the output.
"""

from __future__ import annotations

import math

import pytest
import torch
from conftest import require_b200

import piper_kernels as pk
from oracle import decoding as oracle
from piper_kernels import _native

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # largest relative error of one rounding
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-133}  # and of one that ends subnormal


def _pool(g, pages, heads, page, d, *, mean=False):
    """A cache filled with random rows, on the CPU."""
    codes = [torch.randint(-127, 128, (pages, heads, page, d), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand((pages, heads, page), generator=g) * 0.03 + 0.001 for _ in range(2)]
    m = torch.randn((heads, d), generator=g) if mean else None
    return pk.QuantizedKVCache(codes[0], scales[0], codes[1], scales[1], key_mean=m)


def _on(cache, dev):
    mean = None if cache.key_mean is None else cache.key_mean.to(dev)
    return pk.QuantizedKVCache(*(getattr(cache, n).to(dev) for n in
                                 ("key_codes", "key_scales", "value_codes", "value_scales")), key_mean=mean)


def _table(g, pages, batch, width):
    """Distinct pages for every request, in scattered order."""
    assert batch * width <= pages
    return torch.randperm(pages, generator=g)[: batch * width].view(batch, width).to(torch.int32)


def _same(a, b):
    return torch.equal(a.cpu().nan_to_num(nan=123.0), b.cpu().nan_to_num(nan=123.0))


def _check_cache(actual, expected):
    for name in ("key_codes", "key_scales", "value_codes", "value_scales"):
        assert _same(getattr(actual, name), getattr(expected, name)), name


def _write_plain(cache, key, value, table, lengths, counts):
    pages, heads, page, _ = cache.key_codes.shape
    for b in range(key.shape[0]):
        for i in range(min(key.shape[2], int(counts[b]) if counts is not None else key.shape[2])):
            at = oracle.find_row(table, pages, page, b, int(lengths[b]) + i)
            if at is None:
                continue
            for x, codes, scales, mean in ((key, cache.key_codes, cache.key_scales, cache.key_mean),
                                           (value, cache.value_codes, cache.value_scales, None)):
                row = x[b, :, i].float()
                q, s = oracle.quantise(row if mean is None else row - mean)
                codes[at[0], :, at[1]] = q
                scales[at[0], :, at[1]] = s


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("d", "page", "heads", "tokens", "layout"), [
    (64, 16, 3, 1, "bhnd"), (128, 64, 2, 37, "bnhd"), (128, 16, 1, 50, "odd"), (64, 256, 5, 129, "odd"),
    (128, 32, 8, 2, "broadcast"),
])
def test_write_matches_the_definition(d, page, heads, tokens, layout, dtype) -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(tokens + d)
    batch, width = 3, 1 + (tokens + 20) // page
    cache = _pool(g, batch * width + 2, heads, page, d, mean=layout != "odd")
    table = _table(g, cache.key_codes.shape[0], batch, width)
    table[1, -1] = -1  # a request whose last page is missing
    table[2, 0] = 10**6  # an entry that is no page
    lengths = torch.tensor([0, page - 1, 5], dtype=torch.int32)
    counts = torch.tensor([tokens, tokens + 9, max(0, tokens - 2)], dtype=torch.int32)
    if layout == "broadcast":
        key, value = (torch.randn((1, 1, tokens, d), generator=g).to(dtype).expand(batch, heads, tokens, d)
                      for _ in range(2))
    elif layout == "odd":  # rows that start at any element
        key, value = (torch.randn((batch, heads, tokens, d + 3), generator=g).to(dtype)[..., 1 : d + 1]
                      for _ in range(2))
    else:
        shape = (batch, tokens, heads, d) if layout == "bnhd" else (batch, heads, tokens, d)
        key, value = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        if layout == "bnhd":
            key, value = key.transpose(1, 2), value.transpose(1, 2)
    there = _on(cache, dev)
    on_gpu = [torch.empty(0, dtype=dtype, device=dev).set_(
        x.untyped_storage().cuda(), x.storage_offset(), x.shape, x.stride()) for x in (key, value)]
    pk.write_kv_cache(there, *on_gpu, table.to(dev), lengths.to(dev), counts=counts.to(dev))
    _write_plain(cache, key, value, table, lengths, counts)
    _check_cache(there, cache)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_write_of_extreme_rows(dtype) -> None:
    dev = require_b200()
    d, info = 64, torch.finfo(dtype)
    rows = torch.zeros((6, d), dtype=dtype)
    rows[1] = info.max
    rows[1, ::2] = -info.max
    rows[2, 3] = info.smallest_normal * 2**-6  # subnormal
    rows[3, 5] = torch.inf
    rows[4, 7] = torch.nan
    rows[5] = torch.arange(d) + 0.5  # quotients that end in a half
    rows[5, 0] = 127
    key = rows.view(1, 1, 6, d)
    cache = pk.QuantizedKVCache.allocate(1, 1, 16, d, device=dev)
    table, lengths = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    pk.write_kv_cache(cache, key.to(dev), key.to(dev), table, lengths)
    q, s = oracle.quantise(rows.float())
    fine = [0, 1, 2, 5]
    assert torch.equal(cache.key_codes[0, 0, fine].cpu(), q[fine])
    assert torch.equal(cache.key_scales[0, 0, fine].cpu(), s[fine])
    k, v = pk.read_kv_cache(cache, table, lengths, 6, dtype=dtype)
    for x in (k.cpu()[0, 0], v.cpu()[0, 0]):
        assert not x[0].any() and torch.isnan(x[3:5]).all() and torch.isfinite(x[[0, 2, 5]]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("d", "page", "heads", "tokens"), [(64, 16, 3, 1), (128, 64, 2, 150), (128, 16, 5, 33)])
def test_read_gives_back_the_values(d, page, heads, tokens, dtype) -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(tokens)
    batch, width = 3, 1 + tokens // page
    cache = _pool(g, batch * width, heads, page, d, mean=True)
    table = _table(g, batch * width, batch, width)
    table[0, -1] = -7
    starts = torch.tensor([0, 3, -2], dtype=torch.int32)
    counts = torch.tensor([tokens, tokens - 1, tokens + 5], dtype=torch.int32)
    k, v = pk.read_kv_cache(_on(cache, dev), table.to(dev), starts.to(dev), tokens, counts=counts.to(dev), dtype=dtype)
    expected = torch.zeros((2, batch, heads, tokens, d), dtype=dtype)
    for b in range(batch):
        for i in range(min(tokens, int(counts[b]))):
            at = oracle.find_row(table, batch * width, page, b, int(starts[b]) + i)
            if at is None:
                continue
            p, o = at
            expected[0, b, :, i] = (cache.key_codes[p, :, o].float() * cache.key_scales[p, :, o, None]
                                    + cache.key_mean).to(dtype)
            expected[1, b, :, i] = (cache.value_codes[p, :, o].float() * cache.value_scales[p, :, o, None]).to(dtype)
    assert torch.equal(k.cpu(), expected[0]) and torch.equal(v.cpu(), expected[1])


@pytest.mark.parametrize(("d", "page", "nodes"), [(64, 16, 1), (128, 32, 9), (128, 64, 64), (64, 16, 64)])
def test_keep_moves_rows_as_if_read_first(d, page, nodes) -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(nodes + d)
    batch, heads, width = 5, 3, 2 + nodes // page
    cache = _pool(g, batch * width, heads, page, d)
    table = _table(g, batch * width, batch, width)
    lengths = torch.tensor([0, 1, page - 1, page, 7], dtype=torch.int32)
    path = torch.full((batch, nodes), -1, dtype=torch.int32)
    counts = torch.ones(batch, dtype=torch.int32)
    for b in range(batch):
        # A dense choice: most targets are sources of other moves too.
        chosen = [0] + [i for i in range(1, nodes) if torch.rand((), generator=g) < (0.9 if b != 3 else 0.2)]
        path[b, : len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        counts[b] = len(chosen)
    counts[4] = nodes + 3  # more than the path holds: the -1 entries move nothing
    there = _on(cache, dev)
    pk.keep_draft_path(there, table.to(dev), lengths.to(dev), path.to(dev), counts.to(dev))
    before = _on(cache, "cpu")
    for b in range(batch):
        for j in range(1, min(nodes, int(counts[b]))):
            if path[b, j] < 0:
                continue
            p, o = oracle.find_row(table, batch * width, page, b, int(lengths[b]) + int(path[b, j]))
            q, r = oracle.find_row(table, batch * width, page, b, int(lengths[b]) + j)
            for name in ("key_codes", "key_scales", "value_codes", "value_scales"):
                getattr(cache, name)[q, :, r] = getattr(before, name)[p, :, o].clone()
    _check_cache(there, cache)


# ------------------------------------------------------------------ attention
def _attend(g, dev, *, d, page, kv_heads, group, nodes, lengths, dtype, mask="tree", scale=None, garbage=True,
            gain=1.0):
    batch = len(lengths)
    width = max(1, -(-(max(lengths) + nodes) // page))
    cache = _pool(g, batch * width + 1, kv_heads, page, d)
    table = _table(g, batch * width + 1, batch, width)
    lens = torch.tensor(lengths, dtype=torch.int32)
    if garbage:  # what lies beyond a request's tokens has never been written
        for b, n in enumerate(lengths):
            for position in range(n + nodes, width * page):
                p, o = oracle.find_row(table, batch * width + 1, page, b, position)
                cache.key_scales[p, :, o] = torch.nan
                cache.value_scales[p, :, o] = torch.inf if position % 2 else torch.nan
    query = (gain * torch.randn((batch, nodes, kv_heads * group, d), generator=g)).to(dtype).transpose(1, 2)
    words = None
    if mask == "tree":
        parents = (torch.arange(nodes) - 1 - torch.randint(0, 3, (batch, nodes), generator=g)).clamp(min=0)
        parents[:, 0] = -1
        words = pk.tree_mask_from_parents(parents)
    elif mask == "random":  # any words, zeros among them
        words = torch.randint(-(2**62), 2**62, (batch, nodes), generator=g)
        words[:, ::3] = 0
    elif mask == "shared":
        words = pk.tree_mask_from_parents((torch.arange(nodes) - 1) // 2 - (torch.arange(nodes) == 0).long())
    out = pk.tree_attention(query.to(dev), _on(cache, dev), table.to(dev), lens.to(dev),
                            tree_mask=None if words is None else words.to(dev), scale=scale)
    assert out.shape == query.shape and out.is_contiguous() and out.dtype is dtype
    expected, bound = oracle.attention(query, cache.key_codes, cache.key_scales, cache.value_codes,
                                       cache.value_scales, table, lens, words, d**-0.5 if scale is None else scale)
    off = (out.cpu().double() - expected).abs()
    allowed = UNIT[dtype] * expected.abs() + (1 + UNIT[dtype]) * bound + TINY[dtype]
    assert bool((off <= allowed).all()), float((off / allowed).max())
    return out.cpu(), expected


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("d", "page", "kv_heads", "group", "nodes", "lengths", "mask"), [
    (64, 16, 2, 1, 1, [0, 1, 15, 16, 17], None),
    (128, 64, 2, 4, 1, [63, 64, 65, 127, 300], None),
    (128, 16, 1, 8, 1, [1000], None),
    (128, 32, 2, 5, 7, [0, 31, 32, 200], "tree"),
    (64, 64, 1, 3, 16, [0, 5, 129], "shared"),
    (64, 128, 3, 1, 33, [95, 96, 127], "tree"),
    (128, 256, 1, 8, 64, [0, 190, 257], "tree"),
    (128, 64, 1, 8, 64, [64, 321], None),
    (64, 16, 1, 16, 9, [0, 77], "random"),
    (128, 64, 2, 2, 64, [0, 130], "random"),
])
def test_attention_matches_float64(d, page, kv_heads, group, nodes, lengths, mask, dtype) -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(d + page + nodes)
    _attend(g, dev, d=d, page=page, kv_heads=kv_heads, group=group, nodes=nodes, lengths=lengths, dtype=dtype,
            mask=mask)
    assert _native.device_status(0) == 0


@pytest.mark.parametrize("nodes", [1, 12, 64])
def test_attention_over_a_long_ragged_batch(nodes) -> None:
    # Long enough that a request's keys are split over several CTAs, beside
    # requests of a token or none.
    dev = require_b200()
    g = torch.Generator().manual_seed(nodes)
    _attend(g, dev, d=128, page=64, kv_heads=1, group=2, nodes=nodes, lengths=[4001, 0, 1, 70, 2500],
            dtype=torch.bfloat16)


@pytest.mark.parametrize(("group", "nodes"), [
    (8, 1), (3, 3), (4, 4), (1, 17), (8, 3), (5, 5), (4, 8), (11, 3), (1, 31),
])
@pytest.mark.parametrize(("d", "page", "lengths", "mask"), [
    (64, 16, [2900, 0, 1, 70, 1500], "random"), (128, 32, [2900, 0, 1, 70, 1500], "tree"),
    (64, 64, [5, 200], None), (128, 64, [0, 333], "random"),
])
def test_attention_of_few_rows_on_both_sides_of_each_tile(group, nodes, d, page, lengths, mask) -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(group * 100 + nodes + d)
    _attend(g, dev, d=d, page=page, kv_heads=2, group=group, nodes=nodes, lengths=lengths, dtype=torch.bfloat16,
            mask=mask)


def test_attention_of_24_rows_with_sharp_scores() -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(4)
    for d in (64, 128):
        _attend(g, dev, d=d, page=64, kv_heads=1, group=6, nodes=4, lengths=[900, 3], dtype=torch.float16, scale=0.9,
                gain=4.0)


def test_attention_of_sharp_scores_and_explicit_scale() -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(3)
    _attend(g, dev, d=128, page=64, kv_heads=1, group=4, nodes=5, lengths=[500, 3], dtype=torch.float16, scale=0.9,
            gain=4.0)
    _attend(g, dev, d=64, page=32, kv_heads=1, group=4, nodes=5, lengths=[500, 3], dtype=torch.bfloat16, scale=1e-4)


def test_attention_rows_that_see_nothing_are_zero() -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(4)
    cache = _on(_pool(g, 4, 2, 16, 64), dev)
    cache.key_scales.fill_(torch.nan)
    cache.value_scales.fill_(torch.nan)
    query = torch.randn((2, 4, 3, 64), generator=g).half().to(dev)
    table = torch.tensor([[0, 1], [-1, 99]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([0, 20], dtype=torch.int32, device=dev)  # nothing committed; no pages at all
    out = pk.tree_attention(query, cache, table, lengths, tree_mask=torch.zeros(3, dtype=torch.int64, device=dev))
    assert not out.any()
    out = pk.tree_attention(query, cache, table, torch.full_like(lengths, -5),
                            tree_mask=torch.zeros((2, 3), dtype=torch.int64, device=dev))
    assert not out.any()


def test_attention_when_lengths_reach_past_the_table() -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(5)
    cache = _pool(g, 3, 1, 16, 64)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    query = torch.randn((1, 2, 4, 64), generator=g).half()
    for length in (30, 32, 1000):
        lengths = torch.tensor([length], dtype=torch.int32)
        out = pk.tree_attention(query.to(dev), _on(cache, dev), table.to(dev), lengths.to(dev)).cpu()
        expected, bound = oracle.attention(query, cache.key_codes, cache.key_scales, cache.value_codes,
                                           cache.value_scales, table, lengths, None, 64**-0.5)
        assert bool(((out.double() - expected).abs() <= 2.0**-11 * expected.abs() + 1.001 * bound).all())


def test_attention_with_value_scales_of_very_different_size() -> None:
    # Rows whose values are 2^60 apart: the smaller ones still count in the
    # softmax's total, and the larger ones do not push the others out where
    # their own weight is nothing.
    dev = require_b200()
    d, page = 64, 16
    cache = pk.QuantizedKVCache.allocate(1, 1, page, d, device=dev)
    cache.value_codes.fill_(100)
    cache.value_scales[0, 0, 0] = 2.0**40
    cache.value_scales[0, 0, 1:] = 2.0**-20
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    lengths = torch.tensor([3], dtype=torch.int32, device=dev)
    query = torch.ones((1, 1, 1, d), dtype=torch.bfloat16, device=dev)
    out = pk.tree_attention(query, cache, table, lengths)  # four equal scores
    assert torch.allclose(out.float(), torch.full_like(out.float(), 25 * 2.0**40), rtol=2.0**-7)
    cache.key_codes[0, 0, 0] = -127  # now the large row's weight vanishes
    cache.key_scales[0, 0, 0] = 1.0
    out = pk.tree_attention(query, cache, table, lengths, scale=1.0)
    assert torch.allclose(out.float(), torch.full_like(out.float(), 100 * 2.0**-20), rtol=2.0**-7)


def test_attention_propagates_non_finite_rows_it_sees() -> None:
    dev = require_b200()
    cache = pk.QuantizedKVCache.allocate(2, 1, 16, 64, device=dev)
    cache.key_scales[0, 0, 2] = torch.nan
    table = torch.tensor([[0], [1]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([5, 5], dtype=torch.int32, device=dev)
    out = pk.tree_attention(torch.ones((2, 1, 1, 64), dtype=torch.float16, device=dev), cache, table, lengths)
    assert torch.isnan(out[0]).all() and not out[1].any()


def test_rows_beyond_two_to_the_31_elements() -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(6)
    d, page, heads = 128, 256, 2
    pages = 2**31 // (page * heads * d) + 3
    cache = pk.QuantizedKVCache.allocate(pages, heads, page, d, device=dev)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    lengths = torch.zeros(1, dtype=torch.int32)
    key, value = (torch.randn((1, heads, 300, d), generator=g).bfloat16() for _ in range(2))
    pk.write_kv_cache(cache, key.to(dev), value.to(dev), table.to(dev), lengths.to(dev))
    k, v = pk.read_kv_cache(cache, table.to(dev), lengths.to(dev), 300)
    for x, y in ((k, key), (v, value)):
        q, s = oracle.quantise(y.float())
        assert torch.equal(x.cpu(), (q.float() * s[..., None]).bfloat16())
    query = torch.randn((1, 4, 1, d), generator=g).bfloat16()
    lengths = torch.tensor([299], dtype=torch.int32)
    out = pk.tree_attention(query.to(dev), cache, table.to(dev), lengths.to(dev)).cpu()
    low = pk.QuantizedKVCache(*(getattr(cache, n)[-2:].cpu() for n in
                                ("key_codes", "key_scales", "value_codes", "value_scales")))
    expected, bound = oracle.attention(query, low.key_codes, low.key_scales, low.value_codes, low.value_scales,
                                       table - (pages - 2), lengths, None, d**-0.5)
    assert bool(((out.double() - expected).abs() <= 2.0**-8 * expected.abs() + 1.01 * bound).all())


# --------------------------------------------------------------- verification
def _tree_inputs(g, batch, nodes, vocab, *, chain=False, sharp=2.0, differ=0.8):
    logits = sharp * torch.randn((batch, nodes, vocab), generator=g)
    draft = torch.softmax(logits, -1)
    target = torch.softmax(logits + differ * torch.randn((batch, nodes, vocab), generator=g), -1)
    back = torch.zeros((batch, nodes), dtype=torch.int64) if chain else torch.randint(0, 4, (batch, nodes), generator=g)
    parents = (torch.arange(nodes) - 1 - back).clamp(min=0).to(torch.int32)
    parents[:, 0] = -1
    tokens = torch.zeros((batch, nodes), dtype=torch.int64)
    for b in range(batch):
        for i in range(1, nodes):
            tokens[b, i] = torch.multinomial(draft[b, parents[b, i]], 1, generator=g)
    uniform = torch.rand((batch, nodes), generator=g)
    noise = torch.empty((batch, vocab)).exponential_(generator=g)
    return target, draft, tokens, parents, uniform, noise


@pytest.mark.parametrize(("batch", "nodes", "vocab", "chain"), [
    (1, 1, 1, True), (3, 1, 5, True), (2, 8, 1000, True), (5, 16, 257, False), (40, 64, 33, False),
    (4, 24, 50001, False), (2, 6, 131072, False), (3, 5, 32768, True),
])
def test_verification_matches_the_definition(batch, nodes, vocab, chain) -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(batch * 1000 + nodes)
    args = _tree_inputs(g, batch, nodes, vocab, chain=chain)
    if nodes > 4:
        args[2][:, 3] = -1  # an absent node, and one outside the vocabulary
        args[2][0, 4] = vocab
    got = pk.verify_draft_tree(*(x.to(dev) for x in args))
    path, count, following = oracle.verify(*args)
    assert torch.equal(got.path.cpu(), path)
    assert torch.equal(got.count.cpu(), count)
    assert torch.equal(got.next_token.cpu(), following)
    assert _native.device_status(0) == 0


def test_verification_of_strided_rows_and_ties() -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(8)
    target, draft, tokens, parents, uniform, noise = _tree_inputs(g, 3, 7, 1001)
    # Rows that start at any element, in a buffer with more nodes and words.
    wide_t, wide_d, wide_n = torch.rand((3, 9, 1100)), torch.rand((3, 9, 1100)), torch.rand((3, 1100))
    wide_t[:, 1:8, 3:1004], wide_d[:, 1:8, 5:1006], wide_n[:, 7:1008] = target, draft, noise
    got = pk.verify_draft_tree(
        wide_t.to(dev)[:, 1:8, 3:1004], wide_d.to(dev)[:, 1:8, 5:1006], tokens.to(dev), parents.to(dev),
        uniform.to(dev), wide_n.to(dev)[:, 7:1008])
    for x, y in zip(got, oracle.verify(target, draft, tokens, parents, uniform, noise)):
        assert torch.equal(x.cpu(), y)
    # Equal scores go to the lowest index; a row without any mass to index 0.
    flat = torch.full((2, 1, 5000), 1 / 5000)
    flat[0, 0, :1234] = 0
    flat[1] = 0
    got = pk.verify_draft_tree(flat.to(dev), flat.to(dev), tokens[:2, :1].to(dev), parents[:2, :1].to(dev),
                               uniform[:2, :1].to(dev), torch.ones((2, 5000), device=dev))
    assert got.next_token.tolist() == [1234, 0] and got.count.tolist() == [1, 1]


def test_verification_when_nothing_is_left() -> None:
    # A draft that covers the target everywhere leaves nothing: rest stays.
    dev = require_b200()
    target = torch.tensor([[[0.25, 0.0, 0.5, 0.25]] * 3])
    draft = torch.tensor([[[0.25, 0.0, 0.5, 0.25]] * 3])
    tokens, parents = torch.tensor([[0, 1, 1]]), torch.tensor([[-1, 0, 0]], dtype=torch.int32)
    args = (target, draft, tokens, parents, torch.zeros((1, 3)), torch.tensor([[1.0, 1.0, 4.0, 0.5]]))
    got = pk.verify_draft_tree(*(x.to(dev) for x in args))
    assert got.count.item() == 1 and got.next_token.item() == 3
    for x, y in zip(got, oracle.verify(*args)):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("left,scale", [(1e-30, 1e20), (1e-20, 1.0), (0.25, 1e38), (1e-37, 1e9)])
@pytest.mark.parametrize("children", [1, 2])
def test_verification_of_a_rest_that_is_nearly_nothing(left, scale, children) -> None:
    # One word is all that is left (everywhere else the target is at most the
    # draft, in the same bits), so the next token is that word whatever the
    # noise, even where left / noise is below the least fp32 number.
    dev = require_b200()
    g = torch.Generator().manual_seed(21)
    batch, vocab, word = 3, 5003, 4444
    nodes = 1 + children
    draft = torch.softmax(torch.randn((batch, 1, vocab), generator=g), -1).repeat(1, nodes, 1)
    draft[:, :, word] = 0.0
    target = draft.clone()
    tokens = torch.arange(nodes).repeat(batch, 1) + 10
    target[:, :, 11 : 11 + children] = 0.0
    target[:, :, word] = left
    parents = torch.zeros((batch, nodes), dtype=torch.int32)
    parents[:, 0] = -1
    uniform = torch.full((batch, nodes), 0.5)
    noise = torch.empty((batch, vocab)).exponential_(generator=g).clamp(0.1, 3.0) * scale
    args = (target, draft, tokens, parents, uniform, noise)
    got = pk.verify_draft_tree(*(x.to(dev) for x in args))
    assert got[2].tolist() == [word] * batch
    for x, y in zip(got, oracle.verify(*args)):
        assert torch.equal(x.cpu(), y)


def test_verification_follows_the_target_distribution() -> None:
    # Binomial counts within five standard deviations (plus one).
    dev = require_b200()
    g = torch.Generator().manual_seed(9)
    vocab, tries = 5, 20000
    target, draft = (torch.softmax(torch.randn(vocab, generator=g), -1) for _ in range(2))
    tokens = torch.zeros((tries, 4), dtype=torch.int64)
    tokens[:, 1:] = torch.multinomial(draft, 3 * tries, replacement=True, generator=g).view(tries, 3)
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=dev).expand(tries, 4)
    uniform = torch.rand((tries, 4), generator=g)
    noise = torch.empty((tries, vocab)).exponential_(generator=g)
    got = pk.verify_draft_tree(target.to(dev).expand(tries, 4, vocab), draft.to(dev).expand(tries, 4, vocab),
                               tokens.to(dev), parents, uniform.to(dev), noise.to(dev))
    path, count, following = (x.cpu() for x in got)
    first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].long().clamp(min=0))[:, 0], following)
    for x in range(vocab):
        p = float(target[x])
        assert abs(int((first == x).sum()) - tries * p) <= 5 * (tries * p * (1 - p)) ** 0.5 + 1


# ------------------------------------------------------- streams, graphs, step
def _step(dev, g, *, nodes=6, batch=3, d=128, page=16, kv_heads=2, group=3, dtype=torch.bfloat16):
    width = 12
    cache = _on(_pool(g, batch * width, kv_heads, page, d, mean=True), dev)
    table = _table(g, batch * width, batch, width).to(dev)
    lengths = torch.tensor([0, 65, 130][:batch], dtype=torch.int32, device=dev)
    key, value = (torch.randn((batch, kv_heads, nodes, d), generator=g).to(dtype).to(dev) for _ in range(2))
    query = torch.randn((batch, kv_heads * group, nodes, d), generator=g).to(dtype).to(dev)
    verify = [x.to(dev) for x in _tree_inputs(g, batch, nodes, 777)]
    mask = pk.tree_mask_from_parents(verify[3])

    def step():
        pk.write_kv_cache(cache, key, value, table, lengths)
        out = pk.tree_attention(query, cache, table, lengths, tree_mask=mask)
        verified = pk.verify_draft_tree(*verify)
        pk.keep_draft_path(cache, table, lengths, verified.path, verified.count)
        return (out, *verified, *pk.read_kv_cache(cache, table, lengths, nodes, counts=verified.count))

    return step


def test_a_step_gives_the_same_bits_on_any_stream_and_in_a_graph() -> None:
    dev = require_b200()
    step = _step(dev, torch.Generator().manual_seed(10))
    first = [x.clone() for x in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, third))


def test_a_compiled_step_traces_the_operators_whole() -> None:
    dev = require_b200()
    step = _step(dev, torch.Generator().manual_seed(11))
    expected = [x.clone() for x in step()]
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    assert all(torch.equal(a, b) for a, b in zip(expected, compiled()))


def test_attention_over_a_written_prompt_is_close_to_unquantised_attention() -> None:
    # 8-bit rows: each code is off by at most half a step of 1/127 of the row's
    # largest value.  The output is a weighted mean of values, so its error from
    # V is below max|v| / 254, and a score's from K below sum|q| max|k| / 254
    # times the scale; twice that, weighted by the spread of the values.
    dev = require_b200()
    g = torch.Generator().manual_seed(12)
    d, n = 128, 200
    mean = 3 * torch.randn((2, d), generator=g)
    key = (torch.randn((1, 2, n, d), generator=g) + mean[:, None]).bfloat16()
    value = torch.randn((1, 2, n, d), generator=g).bfloat16()
    query = (0.3 * torch.randn((1, 2, 1, d), generator=g)).bfloat16()
    cache = pk.QuantizedKVCache.allocate(4, 2, 64, d, device=dev, key_mean=mean.to(dev))
    table = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    pk.write_kv_cache(cache, key.to(dev), value.to(dev), table, zero)
    out = pk.tree_attention(query.to(dev), cache, table, zero + n - 1).cpu().double()
    s = query.double() @ key.double().transpose(-1, -2) * d**-0.5
    expected = torch.softmax(s, -1) @ value.double()
    most_k = (key.double() - mean[:, None].double()).abs().amax()
    off = float(query.double().abs().sum(-1).max() * most_k) / 254 * d**-0.5
    allowed = float(value.double().abs().max()) * (1 / 254 + 2 * off) + 2.0**-8 * float(expected.abs().max())
    assert float((out - expected).abs().max()) <= allowed


def test_the_example_keeps_every_layer_consistent_with_its_tokens() -> None:
    # After the last step the caches hold the rows of the prompt and of every
    # token but the last: the first layer's rows depend on the token alone, so
    # they are the quantised projections of the embeddings.
    from piper_kernels.decoding import example

    dev = require_b200()
    model = example.ToyModel()
    prompt = torch.randint(0, model.vocab, (3, 21), generator=torch.Generator().manual_seed(13)).to(dev)
    with torch.no_grad():
        generated, caches, table, lengths = example.generate(model, prompt, 5)
        for b, tokens in enumerate(generated):
            assert 6 <= len(tokens) <= 1 + 5 * 3 and all(0 <= t < model.vocab for t in tokens)
            assert int(lengths[b]) == prompt.shape[1] + len(tokens) - 1
            sequence = torch.cat([prompt[b], torch.tensor(tokens[:-1], device=dev)])[None]
            h = torch.nn.functional.normalize(model.embedding[sequence].float(), dim=-1).to(torch.bfloat16) * 8
            # (The projection of one row and of a batch of rows may round differently: one bf16 step and one code.)
            k, v = pk.read_kv_cache(caches[0], table[b : b + 1], torch.zeros_like(lengths[:1]), sequence.shape[1])
            for got, weight in ((k, model.key[0]), (v, model.value[0])):
                expected = model.heads_of(h, weight).float()
                step = expected.abs().amax(-1, keepdim=True) / 127
                assert bool(((got.float() - expected).abs() <= 1.6 * step + 2.0**-6 * expected.abs()).all())


@pytest.mark.parametrize("nodes", [1, 11, 40])
def test_attention_of_many_short_requests(nodes) -> None:
    # More requests than a warp has lanes, segments of a few tiles: runs hold
    # many of them whole and cut others.
    dev = require_b200()
    g = torch.Generator().manual_seed(nodes + 70)
    lengths = [int(x) for x in torch.randint(0, 1500, (70,), generator=g)]
    lengths[3], lengths[33], lengths[69] = 2600, 0, 2049
    _attend(g, dev, d=64, page=128, kv_heads=2, group=2, nodes=nodes, lengths=lengths, dtype=torch.float16)


@pytest.mark.parametrize("nodes", [1, 6, 50])
def test_attention_with_scales_of_either_sign(nodes) -> None:
    # The handle takes any scales; a negative one only turns its row around.
    dev = require_b200()
    g = torch.Generator().manual_seed(nodes + 80)
    cache = _pool(g, 20, 1, 64, 128)
    for name in ("key_scales", "value_scales"):
        getattr(cache, name).mul_(torch.randint(0, 2, (20, 1, 64), generator=g) * 2 - 1)
    table = torch.randperm(20, generator=g)[:18].view(1, 18).to(torch.int32)
    lengths = torch.tensor([1100], dtype=torch.int32)
    query = torch.randn((1, 4, nodes, 128), generator=g).bfloat16()
    out = pk.tree_attention(query.to(dev), _on(cache, dev), table.to(dev), lengths.to(dev)).cpu().double()
    expected, _ = oracle.attention(query, cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales,
                                   table, lengths, None, 128**-0.5)
    _, bound = oracle.attention(query, cache.key_codes, cache.key_scales, cache.value_codes,
                                cache.value_scales.abs(), table, lengths, None, 128**-0.5)
    assert bool(((out - expected).abs() <= 2.0**-8 * expected.abs() + 1.01 * bound).all())


@pytest.mark.parametrize("nodes", [1, 20, 64])
def test_attention_ends_before_what_follows_on_its_stream(nodes) -> None:
    # The joining kernel may be placed early; the next kernel on the stream must
    # still find attention done with the cache.
    dev = require_b200()
    g = torch.Generator().manual_seed(nodes + 90)
    cache = _on(_pool(g, 300, 2, 64, 128), dev)
    table = torch.randperm(300, generator=g)[:280].view(4, 70).to(torch.int32).to(dev)
    lengths = torch.tensor([4000, 17, 3000, 900], dtype=torch.int32, device=dev)
    query = torch.randn((4, 8, nodes, 128), generator=g).bfloat16().to(dev)
    saved = cache.value_codes.clone()
    expected = pk.tree_attention(query, cache, table, lengths).clone()
    torch.cuda.synchronize()
    for _ in range(20):
        out = pk.tree_attention(query, cache, table, lengths)
        cache.value_codes.zero_()
        cache.value_codes.copy_(saved)
        assert torch.equal(out, expected)


def test_calls_on_two_streams_at_once_do_not_share_anything() -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(95)
    cache = _on(_pool(g, 200, 2, 64, 128), dev)
    table = torch.randperm(200, generator=g)[:192].view(4, 48).to(torch.int32).to(dev)
    lengths = torch.tensor([3000, 2000, 1, 2900], dtype=torch.int32, device=dev)
    queries = [torch.randn((4, 8, n, 128), generator=g).bfloat16().to(dev) for n in (1, 1, 24, 50)]
    expected = [pk.tree_attention(q, cache, table, lengths) for q in queries]
    streams = [torch.cuda.Stream() for _ in queries]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for q, stream in zip(queries, streams):
            with torch.cuda.stream(stream):
                outs.append(pk.tree_attention(q, cache, table, lengths))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, expected[i % len(queries)])


def test_a_step_traced_from_real_tensors_computes_what_it_records() -> None:
    from torch.fx.experimental.proxy_tensor import make_fx

    dev = require_b200()
    step = _step(dev, torch.Generator().manual_seed(96))
    expected = [x.clone() for x in step()]
    traced = make_fx(lambda: step())()
    for out in (traced(), traced()):
        assert all(torch.equal(a, b) for a, b in zip(expected, out))


def test_attention_of_a_tensor_whose_memory_is_not_its_value() -> None:
    # A lazily negated view: the fast path may not read its memory.
    dev = require_b200()
    g = torch.Generator().manual_seed(97)
    cache = _on(_pool(g, 2, 2, 16, 64), dev)
    table, lengths = torch.tensor([[1, 0]], dtype=torch.int32, device=dev), torch.tensor([20], dtype=torch.int32, device=dev)
    query = torch.randn((1, 4, 3, 64), generator=g).half().to(dev)
    assert torch.equal(pk.tree_attention(torch._neg_view(query), cache, table, lengths),
                       pk.tree_attention(-query, cache, table, lengths))


# Query rows of a KV head (heads, nodes) that take each of the five tiles.
EACH_TILE = [(4, 1), (4, 4), (6, 4), (8, 5), (4, 47)]


@pytest.mark.parametrize(("group", "nodes"), EACH_TILE)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_factors_that_underflow_skips_unseen_keys(group, nodes, d) -> None:
    # A bf16 row of zeros counts every key it sees alike, whatever the scale; so
    # does any row at the least scale (its scores are below 2^-90).  The bound is
    # the oracle's; half of the keys of the last tile are unseen.
    dev = require_b200()
    g = torch.Generator().manual_seed(group + nodes + d)
    cache = _pool(g, 12, 1, 32, d)
    table = torch.randperm(12, generator=g).view(2, 6).to(torch.int32)
    lengths = torch.tensor([70, 3], dtype=torch.int32)
    words = torch.randint(0, 2**62, (2, nodes), generator=g)
    for dtype, gain, scale in ((torch.bfloat16, 0.0, 1e-9), (torch.bfloat16, 0.0, 2.0**-126),
                               (torch.float16, 1.0, 2.0**-126), (torch.bfloat16, 2.0**-60, 1e-20)):
        query = (gain * torch.randn((2, group, nodes, d), generator=g)).to(dtype)
        out = pk.tree_attention(query.to(dev), _on(cache, dev), table.to(dev), lengths.to(dev),
                                tree_mask=words.to(dev), scale=scale).cpu().double()
        expected, bound = oracle.attention(query, cache.key_codes, cache.key_scales, cache.value_codes,
                                           cache.value_scales, table, lengths, words, scale)
        allowed = UNIT[dtype] * expected.abs() + (1 + UNIT[dtype]) * bound + TINY[dtype]
        assert bool(((out - expected).abs() <= allowed).all())


def _check_rows(dev, cache, table, lengths, words, query, scale):
    """Attention against the oracle, within its bound; the output."""
    dtype = query.dtype
    out = pk.tree_attention(query.to(dev), _on(cache, dev), table.to(dev), lengths.to(dev),
                            tree_mask=None if words is None else words.to(dev), scale=scale).cpu()
    expected, bound = oracle.attention(query, cache.key_codes, cache.key_scales, cache.value_codes,
                                       cache.value_scales, table, lengths, words, scale)
    allowed = UNIT[dtype] * expected.abs() + (1 + UNIT[dtype]) * bound + TINY[dtype]
    off = (out.double() - expected).abs()
    assert bool((off <= allowed).all()), float((off / allowed).max())
    return out


@pytest.mark.parametrize(("group", "nodes"), EACH_TILE)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pages", [8, 40])  # one CTA a segment, and runs that are joined
def test_attention_of_scores_that_rise_along_the_keys(group, nodes, d, pages) -> None:
    # Scores rise by about a factor of 2 every 5 keys: a row's reference moves
    # several times within a tile and again in each later one, over weights and
    # numerators that are not zero.  Rows rise, fall and stay, by their first element.
    dev = require_b200()
    g = torch.Generator().manual_seed(1000 * group + nodes + d + pages)
    cache = _pool(g, 2 * pages, 1, 32, d)
    table = torch.randperm(2 * pages, generator=g).view(2, pages).to(torch.int32)
    most = 32 * pages - nodes
    lengths = torch.tensor([most, most // 2 + 3], dtype=torch.int32)
    cache.key_codes[..., 0] = 127
    cache.key_codes[..., 1:] = torch.randint(-3, 4, cache.key_codes[..., 1:].shape, generator=g, dtype=torch.int8)
    for b in range(2):
        for column in range(pages):
            rise = torch.arange(32) + 32 * column
            # A step down now and then: a tile's largest score is not always its last.
            cache.key_scales[table[b, column], 0] = (rise - 40 * (rise % 100 > 90)).clamp(min=0) / 127
    query = torch.randn((2, group, nodes, d), generator=g)
    query[..., 0] = torch.tensor([1.0, 0.6, -1.0, 0.0, 0.25])[torch.arange(group * nodes).view(group, nodes) % 5]
    _check_rows(dev, cache, table, lengths, None, query.to(torch.float16), 0.14)
    _check_rows(dev, cache, table, lengths, None, query.to(torch.bfloat16), 0.14)


@pytest.mark.parametrize(("group", "nodes"), EACH_TILE)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_with_value_scales_of_any_size_on_each_tile(group, nodes, d) -> None:
    dev = require_b200()
    g = torch.Generator().manual_seed(2000 * group + nodes + d)
    cache = _pool(g, 60, 1, 32, d)
    cache.value_scales.copy_(torch.exp2(torch.randint(-60, 40, cache.value_scales.shape, generator=g).float()))
    table = torch.randperm(60, generator=g)[:56].view(2, 28).to(torch.int32)
    lengths = torch.tensor([800, 37], dtype=torch.int32)
    query = (4 * torch.randn((2, group, nodes, d), generator=g)).to(torch.bfloat16)
    _check_rows(dev, cache, table, lengths, None, query, 0.3)


@pytest.mark.parametrize(("group", "nodes"), EACH_TILE)
@pytest.mark.parametrize("what", ["key", "value"])
def test_attention_propagates_non_finite_rows_on_each_tile(group, nodes, what) -> None:
    # The last node's row is not finite: the rows that see it are not, all others are as without it.
    dev = require_b200()
    g = torch.Generator().manual_seed(3000 * group + nodes)
    cache = _pool(g, 40, 1, 32, 64)
    table = torch.randperm(40, generator=g)[:38].view(1, 38).to(torch.int32)
    lengths = torch.tensor([1100], dtype=torch.int32)
    query = torch.randn((1, group, nodes, 64), generator=g).half()
    words = torch.randint(0, 2**62, (1, nodes), generator=g) & ~(1 << (nodes - 1))
    there = _on(cache, dev)
    page, offset = oracle.find_row(table, 40, 32, 0, 1100 + nodes - 1)
    getattr(there, what + "_scales")[page, 0, offset] = torch.nan
    bad = words.clone()
    bad[:, :: 2] |= 1 << (nodes - 1)
    args = (query.to(dev), there, table.to(dev), lengths.to(dev))
    out = pk.tree_attention(*args, tree_mask=bad.to(dev)).cpu()
    clean = _check_rows(dev, cache, table, lengths, words, query, 0.125)
    assert not torch.isfinite(out[:, :, ::2]).any() and torch.equal(out[:, :, 1::2], clean[:, :, 1::2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("group", "nodes"), EACH_TILE)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize(("kv_heads", "length", "bits"), [
    (300, 8200, 26),  # runs of about a request's keys, so that one reference serves nearly all of them
    (40, 900, 22),    # one CTA a segment
])
def test_attention_keeps_the_tail_of_a_peaked_softmax(kv_heads, length, bits, d, group, nodes, dtype) -> None:
    # One key has 2^bits times the weight of each other, and zeros for values in
    # the even channels: these come from the others alone.  A weight may be off
    # by 2^-11 of itself or, where fp16 holds it as a subnormal, by 2^-25, the
    # largest one standing at 2^10 (more than 24 or 32 rows: 2^6) or more: 2^-35
    # of it, all alike at worst, or 2^-31 of it at random (the others' value scales
    # are), which over N keys is 5 sqrt(N / 3) times that: both are below N 2^-33
    # here.  A value is below 127.  fp32 sums and exponentials add 2^-16, the scores
    # (bits * ln 2, in fp32) 2^-17 of a weight.
    dev = require_b200()
    g = torch.Generator(device=dev).manual_seed(group + nodes + d)
    page = 64
    pages = -(-(length + nodes) // page)
    shape = (pages, kv_heads, page, d)
    codes = torch.zeros(shape, dtype=torch.int8, device=dev)
    values = torch.randint(40, 128, shape, generator=g, dtype=torch.int8, device=dev)
    value_scales = torch.rand(shape[:3], generator=g, device=dev) * 0.5 + 0.5
    table = torch.randperm(pages, generator=g, device=dev).view(1, pages).to(torch.int32)
    at, offset = int(table[0, 70 // page]), 70 % page
    codes[at, :, offset, 0] = 127
    values[at, :, offset, ::2] = 0
    cache = pk.QuantizedKVCache(codes, torch.ones(shape[:3], device=dev), values, value_scales)
    query = torch.zeros((1, kv_heads * group, nodes, d), dtype=dtype, device=dev)
    query[..., 0] = 1.0
    out = pk.tree_attention(query, cache, table, torch.tensor([length], dtype=torch.int32, device=dev),
                            tree_mask=torch.zeros(nodes, dtype=torch.int64, device=dev),
                            scale=bits * math.log(2) / 127).double()
    order = table[0].long()
    total, sums = 0.0, 0.0
    for i in range(0, pages, 16):  # (a part at a time: the values in fp64 are large)
        position = torch.arange(i * page, min(pages, i + 16) * page, device=dev)
        p = torch.where(position == 70, 1.0, 2.0**-bits) * (position < length).double()
        v = (values[order[i : i + 16]].double() * value_scales[order[i : i + 16]].double()[..., None])
        v = v.transpose(0, 1).reshape(kv_heads, -1, d)
        total, sums = total + p.sum(), sums + torch.einsum("n,hnd->hd", p, v)
    expected = (sums / total).repeat_interleave(group, 0)[None, :, None]
    bound = (2.0**-11 + 2.0**-15) * expected.abs() + length * 2.0**-33 * 127
    assert bool(((out - expected).abs() <= (UNIT[dtype] + bound / expected.abs().clamp(min=1e-30)) * expected.abs()
                 + TINY[dtype]).all()), float(((out - expected).abs() / expected).max())


def test_a_cache_whose_buffers_were_resized_is_refused() -> None:
    # (Checked on the host, before anything is launched.)
    dev = require_b200()
    table = torch.zeros((2, 2), dtype=torch.int32, device=dev)
    lengths, ints = torch.zeros(2, dtype=torch.int32, device=dev), torch.zeros((2, 3), dtype=torch.int32, device=dev)
    x = torch.zeros((2, 2, 3, 64), dtype=torch.float16, device=dev)
    for name, shape in (("value_codes", (2, 2, 16, 64)), ("key_scales", (4, 2, 8)), ("key_mean", (2, 32))):
        for call in (lambda c: pk.write_kv_cache(c, x, x, table, lengths),
                     lambda c: pk.read_kv_cache(c, table, lengths, 2),
                     lambda c: pk.keep_draft_path(c, table, lengths, ints, lengths),
                     lambda c: pk.tree_attention(x, c, table, lengths)):
            cache = pk.QuantizedKVCache.allocate(4, 2, 16, 64, device=dev, key_mean=torch.zeros((2, 64), device=dev))
            getattr(cache, name).resize_(shape)
            with pytest.raises(ValueError, match="QuantizedKVCache"):
                call(cache)


@pytest.mark.parametrize("left", [1e-39, 1e-42, 1e-44])
@pytest.mark.parametrize("children", [1, 2, 3])
def test_verification_of_a_rest_whose_total_is_subnormal(left, children) -> None:
    # Two words are all that is left, the sum of both below the least normal fp32
    # number; the rest is normalised all the same, and the next token is one of them.
    dev = require_b200()
    g = torch.Generator().manual_seed(22)
    batch, vocab, words = 4, 5003, [1234, 4444]
    nodes = 1 + children
    draft = torch.softmax(torch.randn((batch, 1, vocab), generator=g), -1).repeat(1, nodes, 1)
    draft[:, :, words] = 0.0
    target = draft.clone()
    tokens = torch.arange(nodes).repeat(batch, 1) + 10
    target[:, :, 11 : 11 + children] = 0.0
    target[:, :, words] = torch.tensor([left, 2 * left])
    parents = torch.zeros((batch, nodes), dtype=torch.int32)
    parents[:, 0] = -1
    noise = torch.empty((batch, vocab)).exponential_(generator=g)
    noise[:, words[0]] = torch.tensor([1.0, 1.0, 0.01, 1.0])
    noise[:, words[1]] = torch.tensor([1.0, 3.0, 1.0, 1e-20])
    args = (target, draft, tokens, parents, torch.full((batch, nodes), 0.5), noise)
    got = pk.verify_draft_tree(*(x.to(dev) for x in args))
    assert got.next_token.tolist() == [words[1], words[0], words[0], words[1]]
    for x, y in zip(got, oracle.verify(*args)):
        assert torch.equal(x.cpu(), y)


def test_a_learned_key_mean_serves_without_gradients_only() -> None:
    dev = require_b200()
    mean = torch.zeros((2, 64), device=dev, requires_grad=True)
    cache = pk.QuantizedKVCache.allocate(2, 2, 16, 64, device=dev, key_mean=mean)
    table, lengths = torch.tensor([[1]], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    x = torch.ones((1, 2, 3, 64), dtype=torch.float16, device=dev)
    for call in (lambda: pk.write_kv_cache(cache, x, x, table, lengths), lambda: pk.read_kv_cache(cache, table, lengths, 2)):
        with pytest.raises(RuntimeError, match="autograd"):
            call()
        with torch.no_grad():
            call()
    assert torch.equal(pk.tree_attention(x, cache, table, lengths), x)


def test_writes_raise_the_version_of_the_buffers() -> None:
    dev = require_b200()
    table, lengths = torch.tensor([[1]], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    path = torch.zeros((1, 3), dtype=torch.int32, device=dev)
    x = torch.ones((1, 2, 3, 64), dtype=torch.float16, device=dev)
    with torch.inference_mode():
        inside = pk.QuantizedKVCache.allocate(2, 2, 16, 64, device=dev)
        pk.write_kv_cache(inside, x, x, table, lengths)  # (tensors without versions)
        pk.keep_draft_path(inside, table, lengths, path, lengths)
    cache = pk.QuantizedKVCache.allocate(2, 2, 16, 64, device=dev)

    def versions():
        return [t._version for t in cache.buffers[:4]]

    before = versions()
    pk.read_kv_cache(cache, table, lengths, 3)
    pk.tree_attention(x, cache, table, lengths)
    assert versions() == before
    pk.write_kv_cache(cache, x, x, table, lengths)
    pk.keep_draft_path(cache, table, lengths, path, lengths)
    assert all(now >= was + 2 for now, was in zip(versions(), before))
    # What autograd saved of a buffer is no longer what it was.
    weight = torch.ones((), device=dev, requires_grad=True)
    product = (weight * cache.key_scales).sum()
    pk.write_kv_cache(cache, 2 * x, x, table, lengths)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
