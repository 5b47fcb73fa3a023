"""Verification of a drafted tree against the target's probabilities."""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _native
from ._common import MAX_NODES, check_tensor, direct, fits, launch, refuse_grad, require_device

OPERATOR = "verify_draft_tree"


class DraftVerification(NamedTuple):
    """What the target accepts of each request's tree.

    ``path`` int32 ``[batch, nodes]``: the accepted nodes from the root on, then
    -1; ``count`` int32 ``[batch]``: how many they are (at least 1);
    ``next_token`` int64 ``[batch]``: the token that follows the last of them.
    """

    path: torch.Tensor
    count: torch.Tensor
    next_token: torch.Tensor


def verify_draft_tree(
    target_probs: torch.Tensor,
    draft_probs: torch.Tensor,
    tokens: torch.Tensor,
    parents: torch.Tensor,
    uniform: torch.Tensor,
    noise: torch.Tensor,
) -> DraftVerification:
    """Rejection sampling over drafted trees, from given random numbers.

    Node 0 of each tree is the last committed token.  Node ``i`` carries
    ``tokens[b, i]``, drawn from ``draft_probs[b, parents[b, i]]``; its parent
    precedes it, and a token outside the vocabulary (such as -1) means that
    the node is absent.  The walk starts at the root with ``rest`` =
    ``target_probs[b, 0]`` and looks at the nodes in order.  A child ``x`` of
    the current node is accepted if ``uniform[b, i] * draft[x] < rest[x]``,
    ``draft`` being the current node's row; it becomes the current node, and
    ``rest`` its row of ``target_probs``.  Otherwise ``rest`` becomes ``max(rest
    - draft, 0)``, normalised (and stays as it was where that is zero
    everywhere).  The next token is the lowest index of the largest ``rest /
    noise[b]``.

    With uniform numbers in [0, 1) and exponentially distributed noise
    (``torch.Tensor.exponential_``) the accepted tokens and the next one are
    distributed as the target's.

    ``target_probs`` and ``draft_probs`` are float32 ``[batch, nodes, vocab]``
    (finite and not negative; any strides but a contiguous vocabulary),
    ``tokens`` int64, ``parents`` int32 and ``uniform`` float32 ``[batch,
    nodes]``, ``noise`` float32 ``[batch, vocab]`` (positive); 1 to 64 nodes.
    """
    found = direct(
        "verify", "piper_b200_verify_draft_tree", target_probs, draft_probs, tokens, parents, uniform, noise
    )
    if found is not None:
        return DraftVerification(*found)
    _check(target_probs, draft_probs, tokens, parents, uniform, noise)
    return DraftVerification(
        *torch.ops.piper_kernels.verify_draft_tree(target_probs, draft_probs, tokens, parents, uniform, noise)
    )


def _check(target_probs, draft_probs, tokens, parents, uniform, noise) -> None:
    if target_probs.ndim != 3:
        raise ValueError(
            f"{OPERATOR} target_probs must have shape [batch, nodes, vocab], got {tuple(target_probs.shape)}"
        )
    batch, nodes, vocab = target_probs.shape
    device = target_probs.device
    rows, pair, single = (batch, nodes, vocab), (batch, nodes), torch.float32
    if not (
        fits(target_probs, rows, single, device)
        and fits(draft_probs, rows, single, device)
        and fits(tokens, pair, torch.int64, device)
        and fits(parents, pair, torch.int32, device)
        and fits(uniform, pair, single, device)
        and fits(noise, (batch, vocab), single, device)
    ):
        check_tensor(OPERATOR, "target_probs", target_probs, rows, single, device)
        check_tensor(OPERATOR, "draft_probs", draft_probs, rows, single, device)
        check_tensor(OPERATOR, "tokens", tokens, pair, torch.int64, device)
        check_tensor(OPERATOR, "parents", parents, pair, torch.int32, device)
        check_tensor(OPERATOR, "uniform", uniform, pair, single, device)
        check_tensor(OPERATOR, "noise", noise, (batch, vocab), single, device)
    if batch == 0 or vocab == 0:
        raise ValueError(f"{OPERATOR} does not accept an empty batch or vocabulary")
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"{OPERATOR} supports 1 to {MAX_NODES} nodes, got {nodes}")
    if (target_probs.requires_grad or draft_probs.requires_grad) and torch.is_grad_enabled():
        refuse_grad(OPERATOR)
    require_device(OPERATOR, device)


def _run(target, draft, tokens, parents, uniform, noise) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    batch, nodes, vocab = target.shape
    device = target.device
    path = parents.new_empty((batch, nodes))
    count = parents.new_empty(batch)
    next_token = tokens.new_empty(batch)
    launch(
        "piper_b200_verify_draft_tree", device, _native.library().piper_b200_verify_draft_tree,
        target.data_ptr(), _native.strides2(target), draft.data_ptr(), _native.strides2(draft),
        tokens.data_ptr(), tokens.stride(0), parents.data_ptr(), parents.stride(0), uniform.data_ptr(),
        uniform.stride(0), noise.data_ptr(), noise.stride(0), batch, nodes, vocab,
        path.data_ptr(), count.data_ptr(), next_token.data_ptr(),
    )
    return path, count, next_token


@torch.library.custom_op("piper_kernels::verify_draft_tree", mutates_args=())
def _verify_op(
    target_probs: torch.Tensor,
    draft_probs: torch.Tensor,
    tokens: torch.Tensor,
    parents: torch.Tensor,
    uniform: torch.Tensor,
    noise: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check(target_probs, draft_probs, tokens, parents, uniform, noise)
    return _run(target_probs, draft_probs, tokens, parents, uniform, noise)


@_verify_op.register_fake
def _verify_fake(target_probs, _draft_probs, _tokens, _parents, _uniform, _noise):
    batch, nodes, _vocab = target_probs.shape
    new = target_probs.new_empty
    return new((batch, nodes), dtype=torch.int32), new((batch,), dtype=torch.int32), new((batch,), dtype=torch.int64)
