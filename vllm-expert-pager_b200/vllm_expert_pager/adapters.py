"""Low-rank adapters of many requests, paged into slots as experts are.

``add_low_rank`` adds every row's adapter to the output of a projection that all
rows share: ``out = y + scale[s] * (x a[s]^T) b[s]^T`` with ``s`` the slot of the
row's adapter, for any mix of adapters in a batch.  The adapters lie in slabs
``a [slots, rank, in]`` and ``b [slots, out, rank]`` in slot order, as the
experts of a layer do.

``AdapterPager`` keeps more adapters than the slabs hold: all of them in pinned
host memory, those in use in the slabs, with the slot table (``table.py``) and
the row copy (``gather.py``) that page experts.
"""

from __future__ import annotations

import functools

import torch

from vllm_expert_pager import native

_DTYPES = (torch.bfloat16, torch.float16)
_ID_DTYPES = {torch.int32: 4, torch.int64: 8}


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(rows: int, slots: int) -> int:
    return native.lib().xp_low_rank_scratch_bytes(rows, slots)


def _overlap(p: int, ps: int, pw: int, q: int, qs: int, qw: int, rows: int) -> bool:
    """Whether two operands of ``rows`` rows of 16-bit values have bytes in common: first address,
    row stride and width of each.  Columns of one buffer that lie apart have none."""
    if q + 2 * ((rows - 1) * qs + qw) <= p or p + 2 * ((rows - 1) * ps + pw) <= q:
        return False
    if ps == qs and ps > 0:
        off = (q - p) % (2 * ps)  # q's columns, counted from p's, in a row of the buffer
        if off >= 2 * pw and off + 2 * qw <= 2 * ps:
            return False
    return True


def add_low_rank(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                 ids: torch.Tensor, *, scale: torch.Tensor | None = None,
                 slot_map: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[m] = y[m] + scale[s] * (x[m] a[s]^T) b[s]^T``; returns ``out``.

    ``x`` is ``[M, in]``, ``y`` and ``out`` ``[M, out]`` (rows contiguous, any
    distance between rows), ``a`` ``[slots, rank, in]`` and ``b`` ``[slots, out,
    rank]``, all bfloat16 or all float16; ``scale`` float32 ``[slots]``, ones if
    None.  Row ``m`` uses slot ``s = ids[m]``, or ``slot_map[ids[m]]`` with
    ``slot_map`` (int32, an ``expert_map``); a row whose id or slot is out of
    range has no adapter and keeps ``y[m]``.  ``out`` defaults to ``y`` itself
    (the update in place) and may share no memory with the other operands.
    Ranks up to 128; pad an adapter of a lower rank with zeros.  The sums are
    held in 32 bits and the result is rounded once.  Not differentiable: a call
    that would need a gradient is refused.
    """
    if out is None:
        out = y
    native.require_cuda(y, x, a, b, ids, scale, slot_map, out)
    if x.dim() != 2 or y.dim() != 2 or a.dim() != 3 or b.dim() != 3 or ids.dim() != 1:
        raise ValueError("expected x [M, in], y [M, out], a [slots, rank, in], b [slots, out, "
                         f"rank] and ids [M], got {list(x.shape)}, {list(y.shape)}, "
                         f"{list(a.shape)}, {list(b.shape)} and {list(ids.shape)}")
    (M, H), N, (S, r, _) = x.shape, y.shape[1], a.shape
    if (y.shape[0] != M or ids.shape[0] != M or out.shape != y.shape or a.shape[2] != H
            or b.shape != (S, N, r)):
        raise ValueError(f"shapes do not fit: x {list(x.shape)}, y {list(y.shape)}, out "
                         f"{list(out.shape)}, a {list(a.shape)}, b {list(b.shape)}, ids "
                         f"{list(ids.shape)}")
    t, dev = x.dtype, x.device
    if t not in _DTYPES or not (y.dtype == a.dtype == b.dtype == out.dtype == t):
        raise ValueError("x, y, a, b and out must all be bfloat16 or all float16, got "
                         f"{t}, {y.dtype}, {a.dtype}, {b.dtype} and {out.dtype}")
    if not (y.device == a.device == b.device == ids.device == out.device == dev):
        raise ValueError("all operands must be on one device")
    if (H < 1 or N < 1 or not 1 <= S <= native.MAX_ADAPTER_SLOTS
            or not 1 <= r <= native.MAX_RANK):
        raise ValueError(f"sizes must be at least 1, the rank at most {native.MAX_RANK} and the "
                         f"slots at most {native.MAX_ADAPTER_SLOTS}, got in {H}, out {N}, rank "
                         f"{r}, slots {S}")
    if M > native.MAX_TOKENS:
        raise ValueError(f"at most {native.MAX_TOKENS} rows are supported, got {M}")
    if ids.dtype not in _ID_DTYPES:
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (S,)
                              or scale.device != dev):
        raise ValueError(f"scale must be float32 [{S}] on {dev}, got {scale.dtype} "
                         f"{list(scale.shape)} on {scale.device}")
    if slot_map is not None and (slot_map.dtype != torch.int32 or slot_map.dim() != 1
                                 or slot_map.device != dev):
        raise ValueError(f"slot_map must be an int32 vector on {dev}, got {slot_map.dtype} "
                         f"{list(slot_map.shape)} on {slot_map.device}")
    if ((x.requires_grad or y.requires_grad or a.requires_grad or b.requires_grad
         or out.requires_grad or scale is not None and scale.requires_grad)
            and torch.is_grad_enabled()):
        raise ValueError("add_low_rank has no gradient: call it under torch.no_grad() or on "
                         "detached tensors")
    if not (a.is_contiguous() and b.is_contiguous()):
        raise ValueError("adapter slabs must be contiguous")
    (xs, xe), (ys, ye), (os, oe) = x.stride(), y.stride(), out.stride()
    if oe != 1 and N > 1 or os < N and M > 1:
        raise ValueError("the rows of out must be contiguous and apart")
    if M == 0:
        return out
    xp, yp, op = x.data_ptr(), y.data_ptr(), out.data_ptr()
    if _overlap(op, os, N, xp, xs, H, M) or ((op, os) != (yp, ys)
                                             and _overlap(op, os, N, yp, ys, N, M)):
        raise ValueError("out may be y itself, and may not overlap x or other rows of y")
    if xe != 1:
        x = x.contiguous()
        xp, xs = x.data_ptr(), x.stride(0)
    if ye != 1:
        y = y.contiguous()
        yp, ys = y.data_ptr(), y.stride(0)
    ids = ids.contiguous()
    if scale is not None:
        scale = scale.contiguous()
    if slot_map is not None:
        slot_map = slot_map.contiguous()
    need = _scratch_bytes(M, S)
    scratch = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
    native.launch(dev, "add_low_rank", native.lib().xp_add_low_rank,
                  xp, xs, yp, ys, op, os, native.DTYPES[t], M, H, N, r, a.data_ptr(),
                  b.data_ptr(), S, native.ptr(scale), ids.data_ptr(), _ID_DTYPES[ids.dtype],
                  native.ptr(slot_map), 0 if slot_map is None else slot_map.shape[0],
                  native.ptr(scratch), need)
    return out
