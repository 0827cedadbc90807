"""Routing: the step before ``topk_ids``, with the balance loss and its gradient.

The pager's tables take a step's ``topk_ids`` and the MoE its ``topk_weights``
(``table.py``, ``moe.contributions``); the reference gets both from vLLM's
router.  Callers outside a vLLM model, and those who tune a router over paged
experts, get them here:

* ``route``: router logits to the top-k experts of every token, their softmax
  weights and the number of choices of every expert (which tells how many cache
  slots a layer needs); in training also the balance loss.
* ``balance_loss``: the same loss and counts for a routing chosen elsewhere.

Both are differentiable by the logits, once.  Each forward and backward pass is
one or two launches of ``libxpager.so`` (routing.cu) on the current stream,
without a host synchronisation, so they can be captured in a CUDA graph.  To
capture a backward pass, keep no eager autograd graph of the same leaf alive:
autograd would tie the leaf's accumulation to the eager graph's stream, which a
capture does not allow.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from vllm_expert_pager import native


class Routing(NamedTuple):
    weights: torch.Tensor      # float32 [T, topk]
    ids: torch.Tensor          # int32 [T, topk], -1 where a token has no further expert
    counts: torch.Tensor       # int64 [E]
    loss: torch.Tensor | None  # float32 scalar with balance=True


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(T: int, E: int) -> int:
    return native.lib().xp_route_scratch_bytes(T, E)


def _check(logits: torch.Tensor, valid: torch.Tensor | None) -> None:
    native.require_cuda(logits, valid)
    if logits.dim() != 2 or logits.dtype not in native.DTYPES:
        raise ValueError("logits must be a float32, bfloat16 or float16 [tokens, experts] tensor, "
                         f"got {logits.dtype} {list(logits.shape)}")
    T, E = logits.shape
    if not 1 <= E <= native.MAX_EXPERTS:
        raise ValueError(f"between 1 and {native.MAX_EXPERTS} experts are supported, got {E}")
    if T > native.MAX_TOKENS:
        raise ValueError(f"at most {native.MAX_TOKENS} tokens are supported, got {T}")
    if valid is not None:
        if valid.dtype not in (torch.bool, torch.uint8) or valid.shape != (T,):
            raise ValueError(f"valid must be a bool or uint8 tensor of {T} tokens, got "
                             f"{valid.dtype} {list(valid.shape)}")
        if valid.device != logits.device:
            raise ValueError(f"valid is on {valid.device}, logits on {logits.device}")


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """Logits whose rows are contiguous (any distance between rows)."""
    return logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()


def _forward(logits, topk, renormalize, valid, balance, given, count_tokens):
    """One forward pass on checked arguments; ``given``: ids chosen elsewhere."""
    T, E = logits.shape
    dev = logits.device
    empty = torch.empty
    counts = empty((E,), dtype=torch.int64, device=dev)
    # Without padding the backward pass knows the number of tokens: all rows.
    tokens = (empty((1,), dtype=torch.int64, device=dev) if count_tokens and valid is not None
              else None)
    loss = empty((), dtype=torch.float32, device=dev) if balance else None
    need = _scratch_bytes(T, E)
    scratch = empty((need,), dtype=torch.uint8, device=dev) if need else None
    tail = (counts.data_ptr(), native.ptr(tokens), native.ptr(loss), native.ptr(scratch), need)
    head = (logits.data_ptr(), native.DTYPES[logits.dtype], T, E, logits.stride(0),
            native.ptr(valid))
    if given is None:
        weights = empty((T, topk), dtype=torch.float32, device=dev)
        ids = empty((T, topk), dtype=torch.int32, device=dev)
        native.launch(dev, "route", native.lib().xp_route, *head, topk, renormalize,
                      weights.data_ptr(), ids.data_ptr(), *tail)
        return weights, ids, counts, loss, tokens
    native.launch(dev, "balance_loss", native.lib().xp_balance, *head, given.data_ptr(),
                  given.element_size(), topk, *tail)
    return None, None, counts, loss, tokens


def _once() -> None:
    # Under create_graph the result would pass for a constant of the logits.
    if torch.is_grad_enabled():
        raise RuntimeError("vllm-expert-pager: routing is differentiable once; its gradient "
                           "cannot be taken with create_graph=True")


def _backward(logits, topk, renormalize, valid, ids, weights, grad_weights, counts, tokens, grad_loss):
    if grad_weights is not None:
        grad_weights = grad_weights.contiguous()
    T, E = logits.shape
    grad = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
    ptr = native.ptr
    native.launch(logits.device, "route_backward", native.lib().xp_route_backward,
                  logits.data_ptr(), native.DTYPES[logits.dtype], T, E, logits.stride(0),
                  ptr(valid), ptr(ids), ptr(weights), topk, renormalize, ptr(grad_weights), ptr(counts),
                  ptr(tokens), ptr(grad_loss), grad.data_ptr())
    return grad


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, renormalize, valid, balance):
        weights, ids, counts, loss, tokens = _forward(logits, topk, renormalize, valid, balance,
                                                      None, balance)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(ids, counts)
        ctx.save_for_backward(logits, valid, ids, weights, counts if balance else None, tokens)
        ctx.options = topk, renormalize
        return weights, ids, counts, loss

    @staticmethod
    def backward(ctx, grad_weights, _ids, _counts, grad_loss):
        _once()
        if grad_weights is None and grad_loss is None:
            return (None,) * 5
        logits, valid, ids, weights, counts, tokens = ctx.saved_tensors
        grad = _backward(logits, *ctx.options, valid, ids, weights, grad_weights, counts, tokens,
                         grad_loss)
        return grad, None, None, None, None


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, valid):
        _, _, counts, loss, tokens = _forward(logits, ids.shape[1], 0, valid, True, ids, True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(counts)
        ctx.save_for_backward(logits, valid, counts, tokens)
        ctx.topk = ids.shape[1]
        return loss, counts

    @staticmethod
    def backward(ctx, grad_loss, _counts):
        _once()
        if grad_loss is None:
            return None, None, None
        logits, valid, counts, tokens = ctx.saved_tensors
        return _backward(logits, ctx.topk, 0, valid, None, None, None, counts, tokens,
                         grad_loss), None, None


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
    nothing of them is read or counted.

    ``counts[e]`` is the number of tokens routed to expert ``e``.  ``balance``
    adds ``loss = E * sum_e f_e P_e``, ``f_e`` the share of choices that went to
    ``e`` and ``P_e`` its mean probability over the tokens: 1 when both are
    even, 0 without tokens.  Gradients flow to the logits through ``weights``
    (of the chosen experts) and through ``P_e``; ids and counts have none.
    """
    _check(logits, valid)
    if not 1 <= topk <= min(logits.shape[1], native.MAX_TOPK):
        raise ValueError(f"topk must be between 1 and {min(logits.shape[1], native.MAX_TOPK)} "
                         f"for {logits.shape[1]} experts, got {topk}")
    logits = _rows(logits)
    if valid is not None:
        valid = valid.contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        return Routing(*_Route.apply(logits, topk, bool(renormalize), valid, bool(balance)))
    return Routing(*_forward(logits, topk, bool(renormalize), valid, balance, None, False)[:4])


def balance_loss(logits: torch.Tensor, topk_ids: torch.Tensor, *,
                 valid: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, counts)`` as ``route`` gives them, for ids ``[T, topk]`` chosen elsewhere.

    Ids outside ``[0, E)`` are not counted.  The loss is differentiable by the
    logits.
    """
    _check(logits, valid)
    native.require_cuda(topk_ids)
    if topk_ids.dim() != 2 or topk_ids.shape[0] != logits.shape[0] or topk_ids.shape[1] < 1:
        raise ValueError(f"topk_ids must be [{logits.shape[0]}, topk], got "
                         f"{list(topk_ids.shape)}")
    if topk_ids.is_floating_point() or topk_ids.is_complex() or topk_ids.dtype == torch.bool:
        raise ValueError(f"topk_ids must be integers, got {topk_ids.dtype}")
    if topk_ids.device != logits.device:
        raise ValueError(f"topk_ids are on {topk_ids.device}, logits on {logits.device}")
    if topk_ids.dtype not in (torch.int32, torch.int64):
        topk_ids = topk_ids.to(torch.int64)
    topk_ids = topk_ids.contiguous()
    logits = _rows(logits)
    if valid is not None:
        valid = valid.contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        return _Balance.apply(logits, topk_ids, valid)
    _, _, counts, loss, _ = _forward(logits, topk_ids.shape[1], 0, valid, True, topk_ids, False)
    return loss, counts
