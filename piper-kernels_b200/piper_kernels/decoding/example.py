"""Speculative decoding with the operators of this package, end to end on a toy model.

``python -m piper_kernels.decoding.example [--steps N] [--batch B]``

The model is a small attention-only transformer with random weights (grouped
heads, no training, no positions); the draft is the same model without its
layers.  What the
example shows is the order of the calls and who keeps what:

* the prompt runs through ``piper_attention`` and ``write_kv_cache``;
* a step drafts a tree from the last committed token, writes the nodes' keys
  and values into each layer's cache, attends with ``tree_attention``, lets
  ``verify_draft_tree`` walk the tree with the target's probabilities, and
  moves the accepted rows together with ``keep_draft_path``;
* ``lengths`` then grows by the number of accepted nodes, whose rows are
  committed; the next token becomes the next tree's root.
"""

from __future__ import annotations

import argparse
from dataclasses import dataclass

import torch

from ..attention.piper_attention import piper_attention
from .attention import tree_attention, tree_mask_from_parents
from .cache import QuantizedKVCache, keep_draft_path, write_kv_cache
from .verification import verify_draft_tree

# Two children of the root, two of each of them.
PARENTS = (-1, 0, 0, 1, 1, 2, 2)


@dataclass
class ToyModel:
    """``layers`` attention layers over ``heads`` query and ``kv_heads`` KV heads of 64."""

    vocab: int = 1000
    layers: int = 2
    heads: int = 4
    kv_heads: int = 2
    device: str = "cuda"
    seed: int = 0

    def __post_init__(self) -> None:
        g = torch.Generator(device=self.device).manual_seed(self.seed)

        def weight(*shape: int) -> torch.Tensor:
            w = torch.randn(shape, generator=g, device=self.device) * shape[-2] ** -0.5
            return w.to(torch.bfloat16)

        self.width = self.heads * 64
        self.embedding = torch.randn((self.vocab, self.width), generator=g, device=self.device).to(torch.bfloat16)
        self.readout = 3 * torch.randn((self.width, self.vocab), generator=g, device=self.device) * self.width**-0.5
        self.query, self.out = weight(self.layers, self.width, self.width), weight(self.layers, self.width, self.width)
        self.key, self.value = (weight(self.layers, self.width, self.kv_heads * 64) for _ in range(2))

    def heads_of(self, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        """``[batch, heads, tokens, 64]`` of a projection (a strided view)."""
        return (x @ weight).unflatten(-1, (-1, 64)).transpose(1, 2)

    def forward(self, tokens: torch.Tensor, attend) -> torch.Tensor:
        """Logits ``[batch, tokens, vocab]``; ``attend(layer, q, k, v)`` is the attention."""
        x = self.embedding[tokens]
        for layer in range(self.layers):
            h = torch.nn.functional.normalize(x.float(), dim=-1).to(x.dtype) * 8
            q, k, v = (self.heads_of(h, w[layer]) for w in (self.query, self.key, self.value))
            x = x + attend(layer, q, k, v).transpose(1, 2).flatten(-2) @ self.out[layer]
        return x.float() @ self.readout

    def draft(self, tokens: torch.Tensor) -> torch.Tensor:
        """Probabilities after each token without looking further back."""
        return torch.softmax(self.embedding[tokens].float() @ self.readout, -1)


def generate(
    model: ToyModel, prompt: torch.Tensor, steps: int, *, page_size: int = 16, seed: int = 0
) -> tuple[list[list[int]], list[QuantizedKVCache], torch.Tensor, torch.Tensor]:
    """``steps`` speculative steps after ``prompt`` (int64 ``[batch, tokens]``).

    Returns the generated tokens of each request, the layers' caches, the block
    table and the committed lengths.
    """
    device, (batch, prompt_length) = prompt.device, prompt.shape
    g = torch.Generator(device=device).manual_seed(seed)
    nodes = len(PARENTS)
    parents = torch.tensor(PARENTS, dtype=torch.int32, device=device).expand(batch, nodes).contiguous()
    tree_mask = tree_mask_from_parents(parents[0])
    columns = -(-(prompt_length + nodes * (steps + 1)) // page_size)
    table = torch.randperm(batch * columns, generator=g, device=device).view(batch, columns).to(torch.int32)
    caches = [QuantizedKVCache.allocate(batch * columns, model.kv_heads, page_size, 64, device=device)
              for _ in range(model.layers)]
    lengths = torch.zeros(batch, dtype=torch.int32, device=device)

    def prompt_attention(layer, q, k, v):
        write_kv_cache(caches[layer], k, v, table, lengths)
        group = model.heads // model.kv_heads
        return piper_attention(q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1), is_causal=True)

    def node_attention(layer, q, k, v):
        write_kv_cache(caches[layer], k, v, table, lengths)
        return tree_attention(q, caches[layer], table, lengths, tree_mask=tree_mask)

    def race(probs: torch.Tensor) -> torch.Tensor:
        return (probs / torch.empty_like(probs).exponential_(generator=g)).argmax(-1)

    root = race(torch.softmax(model.forward(prompt, prompt_attention)[:, -1], -1))
    lengths += prompt_length
    generated = [[int(t)] for t in root]
    for _ in range(steps):
        tokens = root[:, None].repeat(1, nodes)
        draft = torch.empty((batch, nodes, model.vocab), device=device)
        for i, parent in enumerate(PARENTS):
            if parent >= 0:
                tokens[:, i] = race(draft[:, parent])
            draft[:, i] = model.draft(tokens[:, i])
        target = torch.softmax(model.forward(tokens, node_attention), -1)
        accepted = verify_draft_tree(
            target, draft, tokens, parents, torch.rand((batch, nodes), generator=g, device=device),
            torch.empty((batch, model.vocab), device=device).exponential_(generator=g))
        for cache in caches:
            keep_draft_path(cache, table, lengths, accepted.path, accepted.count)
        lengths += accepted.count
        root = accepted.next_token
        path, count = accepted.path.tolist(), accepted.count.tolist()
        for b, (row, n) in enumerate(zip(path, count)):
            generated[b] += [int(tokens[b, i]) for i in row[1:n]] + [int(root[b])]
    return generated, caches, table, lengths


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=16)
    parser.add_argument("--batch", type=int, default=4)
    args = parser.parse_args()
    model = ToyModel()
    prompt = torch.randint(0, model.vocab, (args.batch, 40), device="cuda",
                           generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.no_grad():
        generated, *_ = generate(model, prompt, args.steps)
    for b, tokens in enumerate(generated):
        print(f"request {b}: {len(tokens)} tokens in {args.steps} steps: {tokens[:12]} ...")


if __name__ == "__main__":
    main()
