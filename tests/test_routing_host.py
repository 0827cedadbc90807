"""Refusals of the routing entry points: none of them reaches a GPU.

The C ABI checks its arguments before any CUDA call; the torch functions check
shapes and types before devices, so CPU tensors show both.
"""

import ctypes

import pytest
import torch

from vllm_expert_pager import native, routing

BUF = (ctypes.c_uint8 * 4096)()
P = ctypes.addressof(BUF)


def xp_route(logits=P, dtype=0, T=4, E=8, stride=8, valid=None, topk=2, renorm=1, weights=P,
             ids=P, counts=P, tokens=None, loss=None, scratch=None, scratch_bytes=0):
    return native.lib().xp_route(logits, dtype, T, E, stride, valid, topk, renorm, weights, ids,
                                 counts, tokens, loss, scratch, scratch_bytes, None)


def xp_balance(logits=P, dtype=0, T=4, E=8, stride=8, valid=None, ids=P, ids_bytes=4, topk=2,
               counts=P, tokens=None, loss=P, scratch=None, scratch_bytes=0):
    return native.lib().xp_balance(logits, dtype, T, E, stride, valid, ids, ids_bytes, topk,
                                   counts, tokens, loss, scratch, scratch_bytes, None)


def xp_backward(logits=P, dtype=0, T=4, E=8, stride=8, valid=None, ids=P, weights=P, topk=2, renorm=1,
                grad_weights=P, counts=P, tokens=P, grad_loss=P, grad=P):
    return native.lib().xp_route_backward(logits, dtype, T, E, stride, valid, ids, weights, topk, renorm,
                                          grad_weights, counts, tokens, grad_loss, grad, None)


@pytest.mark.parametrize("change, status", [
    ({"dtype": 3}, native.XP_EINVAL), ({"dtype": -1}, native.XP_EINVAL),
    ({"T": -1}, native.XP_EINVAL), ({"E": 0}, native.XP_EINVAL),
    ({"E": 4097}, native.XP_ERANGE), ({"T": (1 << 26) + 1}, native.XP_ERANGE),
    ({"stride": -8}, native.XP_EINVAL), ({"topk": 0}, native.XP_EINVAL),
    ({"topk": 9}, native.XP_EINVAL), ({"E": 64, "stride": 64, "topk": 33}, native.XP_ERANGE),
    ({"logits": None}, native.XP_EINVAL), ({"weights": None}, native.XP_EINVAL),
    ({"ids": None}, native.XP_EINVAL), ({"counts": None}, native.XP_EINVAL),
    # Several CTAs: the sum over them needs scratch.
    ({"T": 4096}, native.XP_EINVAL),
    ({"T": 4096, "scratch": P, "scratch_bytes": 64}, native.XP_EINVAL),
    ({"T": 4096, "scratch": P + 1, "scratch_bytes": 1 << 30}, native.XP_EINVAL),
])
def test_route_checks_its_arguments(change, status):
    assert xp_route(**change) == status


@pytest.mark.parametrize("change, status", [
    ({"ids_bytes": 2}, native.XP_EINVAL), ({"ids": None}, native.XP_EINVAL),
    ({"loss": None}, native.XP_EINVAL), ({"counts": None}, native.XP_EINVAL),
    ({"dtype": 7}, native.XP_EINVAL), ({"E": 5000}, native.XP_ERANGE),
    # A count of all choices would not fit 32 bits.
    ({"T": 1 << 20, "topk": 1 << 11}, native.XP_ERANGE), ({"T": 4096}, native.XP_EINVAL),
])
def test_balance_checks_its_arguments(change, status):
    assert xp_balance(**change) == status


@pytest.mark.parametrize("change, status", [
    ({"topk": 40}, native.XP_ERANGE), ({"ids": None}, native.XP_EINVAL),
    ({"weights": None}, native.XP_EINVAL),
    ({"grad": None}, native.XP_EINVAL), ({"counts": None}, native.XP_EINVAL),
    ({"tokens": None, "valid": P}, native.XP_EINVAL), ({"logits": None}, native.XP_EINVAL),
    ({"E": 0}, native.XP_EINVAL), ({"T": 0}, native.XP_OK),
])
def test_backward_checks_its_arguments(change, status):
    assert xp_backward(**change) == status


def test_scratch_size():
    need = native.lib().xp_route_scratch_bytes
    assert need(0, 256) == 0 and need(1, 256) == 0
    assert need(1 << 16, 256) % 4 == 0 and need(1 << 16, 256) > 0
    assert need(1 << 26, 256) == need(1 << 16, 256)  # the launch's CTAs are bounded
    assert need(-1, 256) == -1 and need(1, 0) == -1 and need(1, 5000) == -1


def test_cpu_tensors_are_refused():
    x = torch.zeros((4, 8))
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        routing.route(x, 2)
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        routing.balance_loss(x, torch.zeros((4, 2), dtype=torch.int32))


def test_route_refusals():
    x = torch.zeros((4, 8))
    for bad in (torch.zeros((4, 8), dtype=torch.float64), torch.zeros((4, 8), dtype=torch.int32),
                torch.zeros((8,)), torch.zeros((2, 4, 8))):
        with pytest.raises(ValueError, match="logits must be"):
            routing.route(bad, 2)
    with pytest.raises(ValueError, match="experts are supported"):
        routing.route(torch.zeros((2, 4097)), 2)
    with pytest.raises(ValueError, match="experts are supported"):
        routing.route(torch.zeros((2, 0)), 1)
    for k in (0, -1, 9):
        with pytest.raises(ValueError, match="topk must be between 1 and 8"):
            routing.route(x, k)
    with pytest.raises(ValueError, match="topk must be between 1 and 32"):
        routing.route(torch.zeros((2, 64)), 33)
    for bad in (torch.ones((5,), dtype=torch.bool), torch.ones((4, 1), dtype=torch.bool),
                torch.ones((4,))):
        with pytest.raises(ValueError, match="valid must be"):
            routing.route(x, 2, valid=bad)


def test_balance_refusals():
    x = torch.zeros((4, 8))
    for bad in (torch.zeros((4,), dtype=torch.int32), torch.zeros((3, 2), dtype=torch.int32),
                torch.zeros((4, 0), dtype=torch.int32)):
        with pytest.raises(ValueError, match="topk_ids must be"):
            routing.balance_loss(x, bad)
    for bad in (torch.zeros((4, 2)), torch.zeros((4, 2), dtype=torch.bool)):
        with pytest.raises(ValueError, match="must be integers"):
            routing.balance_loss(x, bad)
    with pytest.raises(ValueError, match="valid must be"):
        routing.balance_loss(x, torch.zeros((4, 2), dtype=torch.int32),
                             valid=torch.ones((3,), dtype=torch.bool))


def test_dual_tensors_are_refused():
    """A tangent would be lost in silence; where forward-mode derivatives are off it is no
    matter, and the call gets as far as the device."""
    from torch.autograd import forward_ad

    ids = torch.zeros((4, 2), dtype=torch.int32)
    with forward_ad.dual_level():
        for leaf in (torch.ones((4, 8)), torch.ones((4, 8), requires_grad=True)):
            x = forward_ad.make_dual(leaf, torch.ones((4, 8)))
            for call in (lambda: routing.route(x, 2), lambda: routing.balance_loss(x, ids)):
                with pytest.raises(ValueError, match="no forward-mode derivative"):
                    call()
                with forward_ad._set_fwd_grad_enabled(False):
                    with pytest.raises(ValueError, match="expected a CUDA tensor"):
                        call()
        with pytest.raises(ValueError, match="expected a CUDA tensor"):
            routing.route(torch.ones((4, 8)), 2)
