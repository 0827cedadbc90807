"""Refusals of the low-rank entry points: none of them reaches a GPU."""

import ctypes

import pytest
import torch

from vllm_expert_pager import adapters, native

BUF = (ctypes.c_uint8 * 4096)()
P = ctypes.addressof(BUF)


def xp_add(x=P, xs=64, y=P, ys=32, out=P, os=32, dtype=1, M=4, H=64, N=32, r=8, a=P, b=P, slots=4,
           scale=None, ids=P, ids_bytes=4, slot_of=None, slot_bytes=4, adapters_=0, scratch=None,
           scratch_bytes=0):
    return native.lib().xp_add_low_rank(x, xs, y, ys, out, os, dtype, M, H, N, r, a, b, slots,
                                        scale, ids, ids_bytes, slot_of, slot_bytes, adapters_, scratch,
                                        scratch_bytes, None)


@pytest.mark.parametrize("change, status", [
    ({"dtype": 0}, native.XP_EINVAL), ({"dtype": 3}, native.XP_EINVAL),
    ({"M": -1}, native.XP_EINVAL), ({"H": 0}, native.XP_EINVAL), ({"N": 0}, native.XP_EINVAL),
    ({"r": 0}, native.XP_EINVAL), ({"r": 129}, native.XP_ERANGE),
    ({"slots": 0}, native.XP_EINVAL), ({"slots": 8193}, native.XP_ERANGE),
    ({"H": 1 << 31}, native.XP_ERANGE), ({"N": 1 << 31}, native.XP_ERANGE), ({"M": (1 << 26) + 1}, native.XP_ERANGE),
    ({"ids_bytes": 2}, native.XP_EINVAL), ({"slot_of": P, "slot_bytes": 2}, native.XP_EINVAL),
    ({"xs": -1}, native.XP_EINVAL),
    ({"ys": -1}, native.XP_EINVAL), ({"os": 31}, native.XP_EINVAL),
    ({"adapters_": -1}, native.XP_EINVAL), ({"x": None}, native.XP_EINVAL),
    ({"y": None}, native.XP_EINVAL), ({"out": None}, native.XP_EINVAL),
    ({"a": None}, native.XP_EINVAL), ({"b": None}, native.XP_EINVAL),
    ({"ids": None}, native.XP_EINVAL), ({"M": 0, "x": None}, native.XP_OK),
])
def test_add_low_rank_checks_its_arguments(change, status):
    assert xp_add(**change) == status


def test_scratch_size():
    need = native.lib().xp_low_rank_scratch_bytes
    assert need(0, 4) >= 0 and need(1, 4) >= 0
    assert need(-1, 4) == -1 and need(1, 0) == -1 and need((1 << 26) + 1, 4) == -1
    assert need(1, 8193) == -1
    big = need(1 << 16, 8)
    if big:
        assert xp_add(M=1 << 16, slots=8) == native.XP_EINVAL  # no scratch
        assert xp_add(M=1 << 16, slots=8, scratch=P, scratch_bytes=big - 1) == native.XP_EINVAL
        assert xp_add(M=1 << 16, slots=8, scratch=P + 4, scratch_bytes=big) == native.XP_EINVAL


def test_cpu_tensors_are_refused():
    t = torch.bfloat16
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        adapters.add_low_rank(torch.zeros((2, 4), dtype=t), torch.zeros((2, 3), dtype=t),
                              torch.zeros((1, 2, 3), dtype=t), torch.zeros((1, 4, 2), dtype=t),
                              torch.zeros((2,), dtype=torch.int32))


def operands(M=6, H=16, N=24, r=4, S=3, t=torch.bfloat16):
    return dict(y=torch.zeros((M, N), dtype=t), x=torch.zeros((M, H), dtype=t),
                a=torch.zeros((S, r, H), dtype=t), b=torch.zeros((S, N, r), dtype=t),
                ids=torch.zeros((M,), dtype=torch.int32))


@pytest.mark.parametrize("change, words", [
    (dict(x=torch.zeros((6, 2, 8), dtype=torch.bfloat16)), "expected x"),
    (dict(ids=torch.zeros((6, 1), dtype=torch.int32)), "expected x"),
    (dict(x=torch.zeros((5, 16), dtype=torch.bfloat16)), "shapes do not fit"),
    (dict(x=torch.zeros((6, 15), dtype=torch.bfloat16)), "shapes do not fit"),
    (dict(ids=torch.zeros((5,), dtype=torch.int32)), "shapes do not fit"),
    (dict(b=torch.zeros((2, 24, 4), dtype=torch.bfloat16)), "shapes do not fit"),
    (dict(out=torch.zeros((6, 23), dtype=torch.bfloat16)), "shapes do not fit"),
    (dict(x=torch.zeros((6, 16))), "bfloat16 or all float16"),
    (dict(y=torch.zeros((6, 24), dtype=torch.float16)), "bfloat16 or all float16"),
    (dict(ids=torch.zeros((6,), dtype=torch.int16)), "ids must be"),
    (dict(ids=torch.zeros((6,))), "ids must be"),
    (dict(scale=torch.zeros((4,))), "scale must be"),
    (dict(scale=torch.zeros((3,), dtype=torch.float64)), "scale must be"),
    (dict(slot_map=torch.zeros((9,), dtype=torch.int16)), "slot_map must be"),
    (dict(slot_map=torch.zeros((9, 1), dtype=torch.int32)), "slot_map must be"),
    (dict(a=torch.zeros((3, 16, 4), dtype=torch.bfloat16).transpose(1, 2)), "contiguous"),
    (dict(out=torch.zeros((24, 6), dtype=torch.bfloat16).t()), "rows of out"),
    (dict(out=torch.zeros((1, 24), dtype=torch.bfloat16).expand(6, 24)), "rows of out"),
])
def test_add_low_rank_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        adapters.add_low_rank(**{**operands(), **change})


def test_rank_limit():
    with pytest.raises(ValueError, match="the rank at most 128"):
        adapters.add_low_rank(**operands(r=129))
    with pytest.raises(ValueError, match="the rank at most 128"):
        adapters.add_low_rank(**operands(r=0))


def test_gradients_are_refused():
    for name in ("x", "y", "a", "b"):
        o = operands()
        o[name].requires_grad_()
        with pytest.raises(ValueError, match="no gradient"):
            adapters.add_low_rank(**o)


def test_overlap_is_refused():
    o = operands(H=24)
    with pytest.raises(ValueError, match="overlap"):
        adapters.add_low_rank(**{**o, "out": o["x"]})
    buf = torch.zeros((7, 24), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):  # out one row behind y
        adapters.add_low_rank(**{**o, "y": buf[:6], "out": buf[1:]})
    slab = torch.zeros((3 * 24 * 4,), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap the adapter slabs"):
        adapters.add_low_rank(**{**o, "b": slab.view(3, 24, 4), "out": slab[:144].view(6, 24)})
    wide = torch.zeros((6, 40), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):  # columns of out run into x's
        adapters.add_low_rank(**{**o, "x": wide[:, :24], "out": wide[:, 16:]})


def test_columns_of_one_buffer_do_not_overlap():
    wide = torch.zeros((6, 64), dtype=torch.bfloat16)

    def share(u, v):
        return native.torch_ops().overlap(u.data_ptr(), u.stride(0), u.shape[1], v.data_ptr(),
                                 v.stride(0), v.shape[1], u.shape[0])

    assert not share(wide[:, :24], wide[:, 24:48])
    assert not share(wide[:, 40:], wide[:, :40])
    assert share(wide[:, :24], wide[:, 23:48])
    assert share(wide[:, 30:50], wide[:, 10:31])
    assert share(wide[:3], wide[2:5]) and share(wide, wide)
    assert not share(wide[:3], wide[3:])


@pytest.mark.parametrize("args, words", [
    ((0, 1, 8, 16, 16, torch.bfloat16), "num_adapters"),
    ((4097, 1, 8, 16, 16, torch.bfloat16), "num_adapters"),
    ((4, 0, 8, 16, 16, torch.bfloat16), "slots must be"),
    ((4, 5, 8, 16, 16, torch.bfloat16), "slots must be"),
    ((4000, 2049, 8, 16, 16, torch.bfloat16), "slots must be"),
    ((4, 2, 0, 16, 16, torch.bfloat16), "the rank must be"),
    ((4, 2, 129, 16, 16, torch.bfloat16), "the rank must be"),
    ((4, 2, 8, 0, 16, torch.bfloat16), "the rank must be"),
    ((4, 2, 8, 16, 0, torch.bfloat16), "the rank must be"),
    ((4, 2, 8, 16, 16, torch.float32), "bfloat16 or float16"),
    ((4, 2, 8, 16, 16, torch.bfloat16), "lives on a CUDA device"),
])
def test_pager_refuses_its_arguments(args, words):
    with pytest.raises(ValueError, match=words):
        adapters.AdapterPager(*args, torch.device("cpu"))


def test_dual_tensors_are_refused():
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        for name in ("x", "y", "a", "b", "scale", "out"):
            o = {**operands(), "scale": torch.ones((3,)), "out": torch.zeros((6, 24)).bfloat16()}
            o[name] = forward_ad.make_dual(o[name], torch.ones_like(o[name]))
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                adapters.add_low_rank(**o)
        with pytest.raises(ValueError, match="expected a CUDA tensor"):
            adapters.add_low_rank(**operands())


def test_one_row_may_be_updated_in_place_at_any_stride():
    """The distance to a row that is not there is no difference between out and y."""
    o = operands(M=1)
    wide = torch.zeros((2, 64), dtype=torch.bfloat16)
    for stride in (24, 64, 1000):
        with pytest.raises(ValueError, match="expected a CUDA tensor"):
            adapters.add_low_rank(**{**o, "y": wide[:1, :24],
                                     "out": wide.as_strided((1, 24), (stride, 1))})
    with pytest.raises(ValueError, match="overlap"):
        adapters.add_low_rank(**{**o, "y": wide[:1, :24], "out": wide[:1, 1:25]})


def test_wait_limit():
    limit = native.lib().xp_low_rank_wait_limit
    assert limit(-1) == 2 * 10**9
    try:
        assert limit(5) == 2 * 10**9 and limit(-7) == 5
        assert limit(1 << 40) == 5 and limit(-1) == 2 * 10**9
    finally:
        limit(2 * 10**9)
    assert native.lib().xp_low_rank_errors(None, None) == native.XP_EINVAL
