"""Cases of the decoding operators: the quantised KV cache, attention over it, and draft verification.

The operators serve one step of (speculative) decoding.  A paged cache holds
INT8 codes of keys and values, one fp32 scale for each row (token, KV head);
T drafted tokens form a tree whose node 0 is the last committed token.

``cache``   write N new tokens per request into the cache, read them back
``attend``  attention of the T nodes over the cached tokens and their ancestors
``verify``  walk the tree: which nodes the target accepts, and the next token
``keep``    move the accepted nodes' rows together, read them back

``run`` computes each in plain fp32 torch operations, or, with ``own``, through
``piper_kernels``.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parents[1]
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_MAX_NODES = 64


def _piper():
    path = str(_ROOT / "piper-kernels_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import piper_kernels

    return piper_kernels


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One user's chat at its start: a single token over a few pages.
        _attend("attend_single_256", 1, 1, 32, 8, 128, 64, 256, 256, "bf16"),
        # A serving batch, one token each, lengths ragged from one token up.
        _attend("attend_batch64_ragged", 64, 1, 32, 8, 128, 64, 1, 8192, "bf16"),
        # One long document (the longest sequence configured here), a drafted
        # tree over a group of five query heads per KV head.
        _attend("attend_tree16_131072", 1, 16, 40, 8, 128, 128, 131072, 131072, "fp16"),
        # A batch with wide trees: 188 query rows for each KV head.
        _attend("attend_tree47_batch16", 16, 47, 32, 8, 128, 64, 4000, 8191, "bf16"),
        # No shared heads, narrow heads, small pages, a short chain of drafts.
        _attend("attend_mha_d64", 32, 5, 24, 24, 64, 16, 333, 4097, "fp16"),
        # One token for each request of a batch.
        _cache("cache_step_batch64", 64, 1, 1, 8, 128, 64, 1, 8192, "bf16"),
        # A batch of ragged prompts into empty pages.
        _cache("cache_prompts_8192", 4, 5001, 8192, 32, 128, 64, 0, 0, "bf16"),
        # Chunks of prompts that start inside a page, narrow heads.
        _cache("cache_chunk_d64", 3, 777, 1000, 24, 64, 16, 37, 1001, "fp16"),
        # A single request's chain of seven drafts.
        _verify("verify_chain8", 1, 8, 32768, "chain"),
        # A batch with trees, a vocabulary whose size is odd.
        _verify("verify_tree16_odd", 16, 16, 50001, "tree"),
        # The widest batch, trees and vocabulary.
        _verify("verify_tree32_batch64", 64, 32, 131072, "tree"),
        # A batch's accepted paths moved together after verification.
        _keep("keep_batch64", 64, 64, 8, 128, 64, 1, 4096, "bf16"),
    ]


def _attend(name, batch, nodes, heads, kv_heads, head_dim, page, len_min, len_max, dtype):
    return {"name": name, "kind": "attend", "batch": batch, "nodes": nodes, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "len_min": len_min, "len_max": len_max, "dtype": dtype}


def _cache(name, batch, new_min, new_max, kv_heads, head_dim, page, len_min, len_max, dtype):
    return {"name": name, "kind": "cache", "batch": batch, "new_min": new_min, "new_max": new_max,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "len_min": len_min, "len_max": len_max,
            "dtype": dtype}


def _verify(name, batch, nodes, vocab, tree):
    return {"name": name, "kind": "verify", "batch": batch, "nodes": nodes, "vocab": vocab, "tree": tree}


def _keep(name, batch, nodes, kv_heads, head_dim, page, len_min, len_max, dtype):
    return {"name": name, "kind": "keep", "batch": batch, "nodes": nodes, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "len_min": len_min, "len_max": len_max, "dtype": dtype}


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case: sizes log-uniform over the listed cases' range, capped at the largest listed cost."""
    kind = rng.choice(["attend", "attend", "attend", "cache", "cache", "verify", "verify", "keep"])
    head_dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "attend":
        kv_heads = rng.choice([1, 2, 4, 8, 8, 24])
        heads = kv_heads * (1 if kv_heads == 24 else rng.choice([1, 2, 4, 4, 5, 8]))
        batch = _log_uniform(rng, 1, 64)
        nodes = rng.choice([1, 1, _log_uniform(rng, 2, _MAX_NODES)])
        # The batch's cached rows, and the products over them, stay below the
        # largest listed cases'.
        most = min(131072, 2_000_000 // (batch * kv_heads), 140_000_000 // (batch * heads * nodes))
        len_max = _log_uniform(rng, 1, max(1, most))
        return _unnamed(_attend("", batch, nodes, heads, kv_heads, head_dim, page,
                                rng.randint(max(0, len_max // 4), len_max), len_max, dtype))
    if kind == "cache":
        kv_heads = rng.choice([1, 2, 8, 24, 32])
        batch = _log_uniform(rng, 1, 64)
        new_max = _log_uniform(rng, 1, max(1, min(8192, 840_000 // (batch * kv_heads))))
        len_max = rng.choice([0, _log_uniform(rng, 1, 2048)])
        return _unnamed(_cache("", batch, rng.randint((new_max + 1) // 2, new_max), new_max, kv_heads, head_dim, page,
                               rng.randint(0, len_max), len_max, dtype))
    if kind == "verify":
        vocab = _log_uniform(rng, 1000, 131072)
        nodes = _log_uniform(rng, 1, _MAX_NODES)
        batch = _log_uniform(rng, 1, max(1, min(64, 268_000_000 // (vocab * nodes))))
        return _unnamed(_verify("", batch, nodes, vocab, rng.choice(["chain", "tree", "tree"])))
    len_max = _log_uniform(rng, 1, 4096)
    return _unnamed(_keep("", _log_uniform(rng, 1, 64), _log_uniform(rng, 4, _MAX_NODES), rng.choice([1, 8, 24]),
                          head_dim, page, rng.randint(0, len_max), len_max, dtype))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def _spread(low, high, count):
    """``count`` whole numbers from ``low`` to ``high``, evenly spaced, in a scattered order."""
    if count == 1:
        return [high]
    values = [low + (high - low) * i // (count - 1) for i in range(count)]
    random.Random(count).shuffle(values)
    return values


def _lengths(case):
    return _spread(case["len_min"], case["len_max"], case["batch"])


def _new_tokens(case):
    return _spread(case["new_min"], case["new_max"], case["batch"])


def _kept(case):
    """Accepted nodes of each request (root included), at most a third of the tree."""
    return _spread(1, max(1, case["nodes"] // 3), case["batch"])


def work(case):
    if case["kind"] == "verify":
        # The rows where the walk ends: the target's probabilities and the
        # noise (the draft's too where the walk ends in a rejection).
        return {"bytes": 8 * case["batch"] * case["vocab"], "flops": 2 * case["batch"] * case["vocab"]}
    d, kv_heads = case["head_dim"], case["kv_heads"]
    row = 2 * d + 8  # K and V codes and their scales
    if case["kind"] == "attend":
        keys = sum(n + case["nodes"] for n in _lengths(case))
        q_rows = case["batch"] * case["heads"] * case["nodes"]
        return {"bytes": keys * kv_heads * row + 2 * q_rows * d * 2,
                "flops": 4 * d * case["heads"] * case["nodes"] * keys}
    if case["kind"] == "cache":
        rows = sum(_new_tokens(case)) * kv_heads
        # Inputs read, rows written; rows read, outputs written.
        return {"bytes": rows * 2 * (4 * d + row), "flops": rows * 2 * d * 4}
    rows = sum(_kept(case)) * kv_heads
    return {"bytes": rows * (3 * row + 4 * d), "flops": rows * 2 * d}


# ------------------------------------------------------------------ inputs
def _quantise(x):
    """Codes and the scale of each row (last axis): the largest magnitude stands at code 127."""
    amax = x.abs().amax(-1)
    scale = torch.where(amax > 0, amax * (1.0 / 127.0), torch.ones_like(amax))
    return torch.round(x / scale[..., None]).clamp(-127, 127).to(torch.int8), scale


def _pool(case, tokens, g):
    """A paged pool filled with quantised rows, and a block table in scattered page order."""
    dev, page, kv_heads, d = "cuda", case["page"], case["kv_heads"], case["head_dim"]
    need = [-(-n // page) for n in tokens]
    pages = sum(need) + 3
    # Keys with channel offsets, as models have them; the cache subtracts them.
    mean = 2.0 * torch.randn((kv_heads, d), generator=g, device=dev)
    k_codes, k_scale = _quantise(torch.randn((pages, kv_heads, page, d), generator=g, device=dev))
    v_codes, v_scale = _quantise(
        torch.randn((pages, kv_heads, page, d), generator=g, device=dev)
        + torch.randn((kv_heads, 1, d), generator=g, device=dev))
    # The last page is in no request's table.
    order = torch.randperm(pages - 1, generator=g, device=dev, dtype=torch.int32)
    width = max(1, max(need))
    column = torch.arange(width, device=dev)
    need_t = torch.tensor(need, device=dev)
    first = torch.cumsum(need_t, 0) - need_t
    index = (first[:, None] + column).clamp(max=pages - 2)
    table = torch.where(column < need_t[:, None], order[index], -1).to(torch.int32).contiguous()
    return {"key_codes": k_codes, "key_scales": k_scale, "value_codes": v_codes, "value_scales": v_scale,
            "key_mean": mean, "table": table}


def _parents(case, g):
    """Each node's parent, one of the up to four nodes before it (a chain: the node before it)."""
    batch, nodes = case["batch"], case["nodes"]
    i = torch.arange(nodes, device="cuda")
    back = torch.zeros((batch, nodes), device="cuda")
    if case.get("tree") != "chain":
        back = torch.rand((batch, nodes), generator=g, device="cuda") * i.clamp(max=4)
    return (i - 1 - back.floor().to(torch.int64)).clamp(min=0).to(torch.int32) - (i == 0).to(torch.int32)


def _ancestors(parents):
    """Bit j of row i: node j is node i or one of its ancestors."""
    mask = torch.zeros(parents.shape, dtype=torch.int64, device=parents.device)
    for i in range(parents.shape[1]):
        bit = 1 << i if i < 63 else -(1 << 63)
        mask[:, i] = bit
        if i:
            mask[:, i] |= mask.gather(1, parents[:, i : i + 1].to(torch.int64))[:, 0]
    return mask


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["kind"] == "verify":
        return _prepare_verify(case, g)
    lengths = _lengths(case)
    state = {"kind": case["kind"], "dtype": _DTYPES[case["dtype"]],
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev)}
    kv_heads, d, batch = case["kv_heads"], case["head_dim"], case["batch"]
    if case["kind"] == "attend":
        nodes = case["nodes"]
        state.update(_pool(case, [n + nodes for n in lengths], g))
        # Laid out [batch, nodes, heads, head_dim], as a projection leaves them.
        q = 2.0 * torch.randn((batch, nodes, case["heads"], d), generator=g, device=dev)
        state["query"] = q.to(state["dtype"]).transpose(1, 2)
        state["mask"] = _ancestors(_parents(case, g))
    elif case["kind"] == "cache":
        new = _new_tokens(case)
        state.update(_pool(case, [n + m for n, m in zip(lengths, new)], g))
        shape = (batch, case["new_max"], kv_heads, d)
        key = torch.randn(shape, generator=g, device=dev) + state["key_mean"]
        value = torch.randn(shape, generator=g, device=dev)
        state["key"] = key.to(state["dtype"]).transpose(1, 2)
        state["value"] = value.to(state["dtype"]).transpose(1, 2)
        state["counts"] = torch.tensor(new, dtype=torch.int32, device=dev)
        state["new"] = case["new_max"]
    else:
        nodes, kept = case["nodes"], _kept(case)
        state.update(_pool(case, [n + nodes for n in lengths], g))
        count = torch.tensor(kept, dtype=torch.int32, device=dev)
        # An increasing choice of nodes beyond the places that they move to.
        weight = torch.rand((batch, nodes), generator=g, device=dev)
        column = torch.arange(nodes, device=dev)
        weight = torch.where(column < count[:, None], 2.0, weight)
        rank = weight.argsort(-1).argsort(-1)
        chosen = (rank < count[:, None] - 1) & (column >= count[:, None])
        place = torch.where(chosen, chosen.to(torch.int64).cumsum(-1), nodes)
        path = torch.full((batch, nodes + 1), -1, dtype=torch.int32, device=dev)
        path.scatter_(1, place, column.to(torch.int32).expand(batch, nodes).contiguous())
        path = path[:, :nodes].contiguous()
        path[:, 0] = 0
        state["path"], state["counts"], state["new"] = path, count, nodes
    return state


def _prepare_verify(case, g):
    dev, batch, nodes, vocab = "cuda", case["batch"], case["nodes"], case["vocab"]
    logits = 3.0 * torch.randn((batch, nodes, vocab), generator=g, device=dev)
    draft = torch.softmax(logits, -1)
    logits += 0.7 * torch.randn((batch, nodes, vocab), generator=g, device=dev)
    target = torch.softmax(logits, -1)
    del logits
    parents = _parents(case, g)
    tokens = torch.zeros((batch, nodes), dtype=torch.int64, device=dev)
    rows = torch.arange(batch, device=dev)
    for i in range(1, nodes):  # each node's token is drawn from its parent's draft distribution
        race = torch.empty((batch, vocab), device=dev).exponential_(generator=g)
        tokens[:, i] = (draft[rows, parents[:, i].to(torch.int64)] / race).argmax(-1)
    return {"kind": "verify", "target": target, "draft": draft, "tokens": tokens, "parents": parents,
            "uniform": torch.rand((batch, nodes), generator=g, device=dev),
            "noise": torch.empty((batch, vocab), device=dev).exponential_(generator=g)}


# ------------------------------------------------------------- plain forms
def _rows(state, position):
    """Page and offset of each position [B, N], and whether the table has a page for it."""
    page = state["key_codes"].shape[2]
    column = torch.div(position, page, rounding_mode="floor")
    found = state["table"].to(torch.int64).gather(1, column.clamp(0, state["table"].shape[1] - 1))
    ok = (position >= 0) & (column < state["table"].shape[1]) & (found >= 0)
    return found.clamp(min=0), position % page, ok


def _plain_attend(state):
    query, mask = state["query"], state["mask"]
    batch, heads, nodes, d = query.shape
    kv_heads, page = state["key_codes"].shape[1:3]
    pages = state["table"].to(torch.int64).clamp(min=0)
    length = pages.shape[1] * page

    def gathered(codes, scales):
        x = codes[pages].float() * scales[pages][..., None]  # [B, pages, H, page, D]
        return x.transpose(1, 2).reshape(batch, kv_heads, length, d)

    k = gathered(state["key_codes"], state["key_scales"])
    q = query.float().reshape(batch, kv_heads, heads // kv_heads * nodes, d)
    score = torch.matmul(q, k.transpose(-1, -2)) * d**-0.5
    del k
    lengths = state["lengths"].to(torch.int64)
    position = torch.arange(length, device=query.device)
    j = position - lengths[:, None]  # which drafted node a position holds
    bit = (mask[:, :, None] >> j.clamp(0, nodes - 1)[:, None, :]) & 1
    seen = (j[:, None, :] < 0) | ((bit == 1) & (j[:, None, :] < nodes))  # [B, T, L]
    score = score.view(batch, kv_heads, heads // kv_heads, nodes, length)
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = p.sum(-1)
    v = gathered(state["value_codes"], state["value_scales"])
    out = torch.matmul(p.view(batch, kv_heads, -1, length), v).view(batch, heads, nodes, d)
    total = total.view(batch, heads, nodes, 1)
    return torch.where(total > 0, out / total, 0.0).to(query.dtype)


def _plain_read(state, start, count, new):
    i = torch.arange(new, device=start.device)
    page, offset, ok = _rows(state, start.to(torch.int64)[:, None] + i)
    ok = (ok & (i < count[:, None]))[:, None, :, None]  # [B, 1, N, 1]

    def rows(codes, scales, mean):
        x = codes[page, :, offset].float() * scales[page, :, offset][..., None]  # [B, N, H, D]
        x = x if mean is None else x + mean
        return torch.where(ok, x.transpose(1, 2), 0.0).to(state["dtype"])

    return (rows(state["key_codes"], state["key_scales"], state["key_mean"]),
            rows(state["value_codes"], state["value_scales"], None))


def _plain_cache(state):
    new = state["new"]
    i = torch.arange(new, device="cuda")
    page, offset, ok = _rows(state, state["lengths"].to(torch.int64)[:, None] + i)
    ok = ok & (i < state["counts"][:, None])
    # What is not to be written goes to the page that no table names.
    page = torch.where(ok, page, state["key_codes"].shape[0] - 1)
    for name, x in (("key", state["key"].float().transpose(1, 2) - state["key_mean"]),
                    ("value", state["value"].float().transpose(1, 2))):
        codes, scales = _quantise(x)  # [B, N, H, D]
        state[name + "_codes"][page, :, offset] = codes
        state[name + "_scales"][page, :, offset] = scales
    return _plain_read(state, state["lengths"], state["counts"], new)


def _plain_keep(state):
    nodes = state["path"].shape[1]
    i = torch.arange(nodes, device="cuda")
    start = state["lengths"].to(torch.int64)[:, None]
    moved = (i > 0) & (i < state["counts"][:, None]) & (state["path"] >= 0)
    source, s_offset, _ = _rows(state, start + state["path"].clamp(min=0))
    target, t_offset, _ = _rows(state, start + i)
    # What is not to be moved goes to the page that no table names.
    target = torch.where(moved, target, state["key_codes"].shape[0] - 1)
    for name in ("key_codes", "key_scales", "value_codes", "value_scales"):
        state[name][target, :, t_offset] = state[name][source, :, s_offset]
    return _plain_read(state, state["lengths"], state["counts"], nodes)


def _plain_verify(state):
    target, draft, tokens, parents = state["target"], state["draft"], state["tokens"], state["parents"]
    batch, nodes, _ = target.shape
    b = torch.arange(batch, device=target.device)
    current = torch.zeros(batch, dtype=torch.int64, device=target.device)
    path = torch.full((batch, nodes), -1, dtype=torch.int32, device=target.device)
    path[:, 0] = 0
    count = torch.ones(batch, dtype=torch.int32, device=target.device)
    rest = target[:, 0]  # what is left of the target's distribution after the current node
    # Each node in order: a child of the current node is accepted, or its
    # draft's distribution is taken out of what is left.
    for i in range(1, nodes):
        child = (parents[:, i] == current) & (tokens[:, i] >= 0)
        x = tokens[:, i].clamp(min=0)
        accept = child & (state["uniform"][:, i] * draft[b, current, x] < rest[b, x])
        reject = child & ~accept
        left = (rest - draft[b, current]).clamp(min=0)
        total = left.sum(-1, keepdim=True)
        left = torch.where(total > 0, left / total, rest)
        current = torch.where(accept, i, current)
        rest = torch.where(accept[:, None], target[:, i], torch.where(reject[:, None], left, rest))
        place = torch.where(accept, count, nodes - 1).to(torch.int64)[:, None]
        kept = path.gather(1, place)[:, 0]
        path.scatter_(1, place, torch.where(accept, i, kept).to(torch.int32)[:, None])
        count = count + accept.to(torch.int32)
    return {"path": path, "count": count, "next": (rest / state["noise"]).argmax(-1)}


def run(state):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind == "attend":
        return _plain_attend(state)
    if kind == "cache":
        return _plain_cache(state)
    if kind == "verify":
        return _plain_verify(state)
    return _plain_keep(state)


# --------------------------------------------------------- framework calls
def _own(state):
    piper = _piper()
    if state["kind"] == "verify":
        verified = piper.verify_draft_tree(state["target"], state["draft"], state["tokens"], state["parents"],
                                           state["uniform"], state["noise"])
        return {"path": verified.path, "count": verified.count, "next": verified.next_token}
    cache = piper.QuantizedKVCache(state["key_codes"], state["key_scales"], state["value_codes"],
                                   state["value_scales"], key_mean=state["key_mean"])
    table, lengths = state["table"], state["lengths"]
    if state["kind"] == "attend":
        return piper.tree_attention(state["query"], cache, table, lengths, tree_mask=state["mask"])
    if state["kind"] == "cache":
        piper.write_kv_cache(cache, state["key"], state["value"], table, lengths, counts=state["counts"])
    else:
        piper.keep_draft_path(cache, table, lengths, state["path"], state["counts"])
    return piper.read_kv_cache(cache, table, lengths, state["new"], counts=state["counts"], dtype=state["dtype"])


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """What ``run`` returns from the definitions in fp64, one request at a time."""
    if case["kind"] == "verify":
        return None  # whole numbers only
    state = prepare(case, seed)
    table = state["table"].tolist()
    lengths = state["lengths"].tolist()
    page = case["page"]

    def at(name, b, position):
        """The row's (page, offset) entries of a buffer: [N, H, ...]."""
        pages = torch.tensor([table[b][p // page] for p in position], dtype=torch.int64, device="cuda")
        offsets = torch.tensor([p % page for p in position], dtype=torch.int64, device="cuda")
        return state[name][pages, :, offsets].double()

    def values(side, b, position):
        x = at(side + "_codes", b, position) * at(side + "_scales", b, position)[..., None]
        return x + state["key_mean"].double() if side == "key" else x

    if case["kind"] == "attend":
        nodes, group = case["nodes"], case["heads"] // case["kv_heads"]
        masks = state["mask"].tolist()
        out = []
        for b, n in enumerate(lengths):
            position = range(n + nodes)
            k = values("key", b, position).permute(1, 2, 0)  # [H, D, L]
            v = values("value", b, position).permute(1, 0, 2)
            q = state["query"][b].double().view(case["kv_heads"], group, nodes, case["head_dim"])
            s = torch.einsum("hgtd,hdl->hgtl", q, k) / math.sqrt(case["head_dim"])
            hidden = torch.tensor([[(masks[b][t] >> j) & 1 == 0 for j in range(nodes)] for t in range(nodes)],
                                  device="cuda")
            s[..., n:].masked_fill_(hidden, -math.inf)
            out.append(torch.einsum("hgtl,hld->hgtd", torch.softmax(s, -1), v).flatten(0, 1))
        return torch.stack(out)
    shape = (case["batch"], case["kv_heads"], state["new"], case["head_dim"])
    found = {side: torch.zeros(shape, dtype=torch.float64, device="cuda") for side in ("key", "value")}
    counts = state["counts"].tolist()
    for b, (n, count) in enumerate(zip(lengths, counts)):
        for side in found:
            if case["kind"] == "cache":
                x = state[side][b, :, :count].double()
                mean = state["key_mean"].double()[:, None] if side == "key" else 0.0
                x = x - mean
                step = x.abs().amax(-1, keepdim=True) / 127
                x = torch.round(x / step) * step + mean
            else:
                source = [n + p for p in state["path"][b, :count].tolist()]
                x = values(side, b, source).transpose(0, 1)
            found[side][b, :, :count] = x
    return found["key"], found["value"]
