"""Routing: the step before ``topk_ids``, with the balance loss and its gradient.

The pager's tables take a step's ``topk_ids`` and the MoE its ``topk_weights``
(``table.py``, ``moe.contributions``); the reference gets both from vLLM's
router.  Callers outside a vLLM model, and those who tune a router over paged
experts, get them here:

* ``route``: router logits to the top-k experts of every token, their softmax
  weights and the number of choices of every expert (which tells how many cache
  slots a layer needs); in training also the balance loss.
* ``balance_loss``: the same loss and counts for a routing chosen elsewhere.

Both are differentiable by the logits, once and backwards (a gradient with
``create_graph`` and a dual tensor of forward-mode derivatives are refused).  Each forward and backward pass is one or two launches of
``libxpager.so`` (routing.cu) on the current stream of the tensors' device,
without a host synchronisation, so they can be captured in a CUDA graph.
Arguments are checked in csrc/torch_ops.cpp; a refused call raises ValueError
and launches nothing.  To
capture a backward pass, keep no eager autograd graph of the same leaf alive:
autograd would tie the leaf's accumulation to the eager graph's stream, which a
capture does not allow.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from vllm_expert_pager import native


class Routing(NamedTuple):
    weights: torch.Tensor      # float32 [T, topk]
    ids: torch.Tensor          # int32 [T, topk], -1 where a token has no further expert
    counts: torch.Tensor       # int64 [E]
    loss: torch.Tensor | None  # float32 scalar with balance=True


def route(logits: torch.Tensor, topk: int, *, renormalize: bool = True,
          valid: torch.Tensor | None = None, balance: bool = False) -> Routing:
    """Choose every token's ``topk`` experts from its router logits ``[T, E]``.

    The experts with the largest logits, in descending order (equal logits: the
    lower expert first); a logit of -inf closes its expert, and where fewer than
    ``topk`` are open the remaining ids are -1 and their weights 0 (the pager's
    tables ignore ids out of range).  ``weights`` are the softmax probabilities of the
    chosen experts, divided by their sum with ``renormalize``.  A NaN logit is
    chosen first and makes its token's weights NaN.  ``valid`` (bool ``[T]``)
    marks the rows that hold a token: the others get ids -1 and weights 0, and
    nothing of them is read or counted.  A probability ``exp(l - max) / sum`` is exact to
    about ``10 + 2 (max - l)`` steps of 2^-23, and 0 below 2^-126.

    ``counts[e]`` is the number of tokens routed to expert ``e``.  ``balance``
    adds ``loss = E * sum_e f_e P_e``, ``f_e`` the share of choices that went to
    ``e`` and ``P_e`` its mean probability over the tokens: 1 when both are
    even, 0 without tokens.  Gradients flow to the logits through ``weights``
    (of the chosen experts) and through ``P_e``; ids and counts have none.
    """
    return Routing(*native.torch_ops().route(logits, topk, renormalize, valid, balance))


def balance_loss(logits: torch.Tensor, topk_ids: torch.Tensor, *,
                 valid: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, counts)`` as ``route`` gives them, for ids ``[T, topk]`` chosen elsewhere.

    Ids outside ``[0, E)`` are not counted.  The loss is differentiable by the
    logits.
    """
    return native.torch_ops().balance_loss(logits, topk_ids, valid)
