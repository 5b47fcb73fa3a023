"""CPU oracle of the decoding operators, in plain torch -- TEST INFRASTRUCTURE ONLY.

Attention and read-back are computed in float64 from the stored codes and
scales; quantisation and verification follow their definitions in float32,
whose every operation rounds once, so that codes, scales and decisions can be
compared exactly.
"""

from __future__ import annotations

import math

import torch


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of float32 rows (last axis)."""
    amax = x.abs().amax(-1)
    scale = torch.where(amax == 0, torch.ones_like(amax), amax * torch.tensor(1.0 / 127.0, dtype=torch.float32))
    return torch.round(x / scale[..., None]).clamp(-127, 127).to(torch.int8), scale


def find_row(table: torch.Tensor, pages: int, page_size: int, b: int, position: int) -> tuple[int, int] | None:
    """(page, offset) of a request's position, or None where there is no page."""
    column = position // page_size
    if position < 0 or column >= table.shape[1]:
        return None
    page = int(table[b, column])
    return (page, position % page_size) if 0 <= page < pages else None


def attention(
    query: torch.Tensor,
    key_codes: torch.Tensor,
    key_scales: torch.Tensor,
    value_codes: torch.Tensor,
    value_scales: torch.Tensor,
    table: torch.Tensor,
    lengths: torch.Tensor,
    tree_mask: torch.Tensor | None,
    scale: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Output in float64 and a bound on a kernel's error beside the output's own rounding.

    Per element, with weights p (sum 1), A = sum p |v| and M the largest p *
    (V scale) * 127: probabilities rounded to fp16 give 2^-11 A (2^-25 M for
    each key whose weight is subnormal); a score is a sum of D fp32 products
    of fp16 numbers, off by at most D 2^-23 times the sum of magnitudes S
    (query rounding and fp32 sums), which moves weights and total by that
    fraction each; exponentials, sums and merges in fp32 get 2^-16 A.
    """
    batch, heads, nodes, d = query.shape
    pages, kv_heads, page_size, _ = key_codes.shape
    group = heads // kv_heads
    out = torch.zeros((batch, heads, nodes, d), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b in range(batch):
        length = max(0, int(lengths[b]))
        rows, drafted = [], []
        for position in range(length + nodes):
            at = find_row(table, pages, page_size, b, position)
            if at is not None:
                rows.append(at)
                drafted.append(position - length)
        if not rows:
            continue
        page = torch.tensor([r[0] for r in rows])
        offset = torch.tensor([r[1] for r in rows])
        j = torch.tensor(drafted)
        for t in range(nodes):
            word = (1 << (t + 1)) - 1 if tree_mask is None else int(
                tree_mask[t] if tree_mask.ndim == 1 else tree_mask[b, t])
            seen = torch.tensor([n < 0 or bool((word >> n) & 1) for n in drafted])
            if not bool(seen.any()):
                continue
            for h in range(heads):
                kv = h // group
                at = (page[seen], kv, offset[seen])
                k = key_codes[at].double() * key_scales[at].double()[:, None]
                vs = value_scales[at].double()
                v = value_codes[at].double() * vs[:, None]
                q = query[b, h, t].double()
                s = k @ q * scale
                p = torch.softmax(s, 0)
                o = p @ v
                a = p @ v.abs()
                out[b, h, t] = o
                off = d * 2.0**-23 * float((k.abs() @ q.abs()).max()) * scale
                most = float((p * vs).max()) * 127
                bound[b, h, t] = a * (2.0**-11 + 2 * math.expm1(off) + 2.0**-16) + len(vs) * 2.0**-25 * most
    return out, bound


def verify(
    target: torch.Tensor,
    draft: torch.Tensor,
    tokens: torch.Tensor,
    parents: torch.Tensor,
    uniform: torch.Tensor,
    noise: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Path, count and next token of each request, one node at a time in float32."""
    batch, nodes, vocab = target.shape
    path = torch.full((batch, nodes), -1, dtype=torch.int32)
    count = torch.zeros(batch, dtype=torch.int32)
    following = torch.zeros(batch, dtype=torch.int64)
    for b in range(batch):
        current, kept, rest = 0, [0], target[b, 0]
        for i in range(1, nodes):
            x = int(tokens[b, i])
            if int(parents[b, i]) != current or not 0 <= x < vocab:
                continue
            if bool(uniform[b, i] * draft[b, current, x] < rest[x]):
                current, rest = i, target[b, i]
                kept.append(i)
                continue
            left = (rest - draft[b, current]).clamp(min=0)
            total = left.sum()
            if total > 0:
                rest = left / total
        path[b, : len(kept)] = torch.tensor(kept, dtype=torch.int32)
        count[b] = len(kept)
        score = rest / noise[b]
        following[b] = int((score == score.max()).nonzero()[0, 0])
    return path, count, following
