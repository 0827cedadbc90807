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
from vllm_expert_pager.acquire import MAX_SLOTS
from vllm_expert_pager.gather import gather_rows
from vllm_expert_pager.store import PinnedBuffer, numa_node_of
from vllm_expert_pager.table import ExpertTable

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
    ``slot_map`` (int32 or int64: an ``expert_map``, or a table's ``slot_of``); a row whose id or slot is out of
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
    if slot_map is not None and (slot_map.dtype not in _ID_DTYPES or slot_map.dim() != 1
                                 or slot_map.device != dev):
        raise ValueError(f"slot_map must be an int32 or int64 vector on {dev}, got {slot_map.dtype} "
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
                  *((slot_map.data_ptr(), _ID_DTYPES[slot_map.dtype], slot_map.shape[0])
                    if slot_map is not None else (None, 0, 0)), native.ptr(scratch), need)
    return out


class AdapterPager:
    """The low-rank adapters of one projection: all in pinned host memory, some in VRAM slots.

    ``num_adapters`` adapters of ranks up to ``rank`` are kept in pinned memory on
    the GPU's NUMA node, ``slots`` of them in slabs on the GPU.  ``page`` brings a
    step's adapters into slots (least recently used ones make room), ``add`` adds
    the rows' updates; both only enqueue work on the current stream, so a step of
    them can be captured in a CUDA graph.  Adapters that were never written are
    zero.
    """

    def __init__(self, num_adapters: int, slots: int, rank: int, in_features: int,
                 out_features: int, dtype: torch.dtype, device: torch.device) -> None:
        if not 1 <= num_adapters <= native.MAX_EXPERTS:
            raise ValueError(f"num_adapters must be between 1 and {native.MAX_EXPERTS}, got "
                             f"{num_adapters}")
        if not 1 <= slots <= min(num_adapters, MAX_SLOTS):
            raise ValueError(f"slots must be between 1 and {min(num_adapters, MAX_SLOTS)}, got "
                             f"{slots}")
        if not 1 <= rank <= native.MAX_RANK or in_features < 1 or out_features < 1:
            raise ValueError(f"the rank must be between 1 and {native.MAX_RANK} and the features "
                             f"at least 1, got rank {rank}, in {in_features}, out {out_features}")
        if dtype not in _DTYPES:
            raise ValueError(f"adapters must be bfloat16 or float16, got {dtype}")
        # Ranks in whole 16-byte pieces: the rows of b then start on their boundaries.
        r = self.rank = -(-rank // 8) * 8
        self.num_adapters, self.slots = num_adapters, slots
        self.in_features, self.out_features, self.dtype = in_features, out_features, dtype
        self.table = ExpertTable(num_adapters, slots, device)  # refuses other than CUDA devices
        device = self.device = self.table.counters.device
        shapes = ((r, in_features), (out_features, r))
        numa = numa_node_of(device)
        self._buffers = [PinnedBuffer(num_adapters * m * n * dtype.itemsize, device, numa)
                         for m, n in shapes]
        self._host, self._rows = [], []
        for buf, (m, n) in zip(self._buffers, shapes):
            nbytes = num_adapters * m * n * dtype.itemsize
            self._host.append(buf.cpu[:nbytes].view(dtype).view(num_adapters, m, n))
            self._rows.append(buf.cuda[:nbytes].view(torch.int32).view(num_adapters, -1))
        self._scales = torch.zeros((num_adapters, 1), dtype=torch.float32, device=device)
        self.a = torch.zeros((slots, *shapes[0]), dtype=dtype, device=device)
        self.b = torch.zeros((slots, *shapes[1]), dtype=dtype, device=device)
        self.scale = torch.zeros((slots,), dtype=torch.float32, device=device)
        # The row copy takes a scale row for each of the two names; an adapter has one, and
        # both copies write it.
        self._scale_rows = [self._scales.view(torch.int32)] * 2
        self._scale_slots = [self.scale.view(torch.int32).view(slots, 1)] * 2
        self._slabs = [t.view(slots, -1).view(torch.int32) for t in (self.a, self.b)]

    def write(self, adapter: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Store adapter ``adapter``: ``a [r, in]``, ``b [out, r]`` with ``r`` up to the pager's rank.

        Waits for the device, which may still be reading the old rows, and
        takes the adapter out of its slot: the next ``page`` brings the new one.
        """
        if not self._buffers:
            raise RuntimeError("vllm-expert-pager: the adapters were released")
        if not 0 <= adapter < self.num_adapters:
            raise ValueError(f"adapter must be in [0, {self.num_adapters}), got {adapter}")
        r = a.shape[0] if a.dim() == 2 else -1
        if (not 1 <= r <= self.rank or a.shape != (r, self.in_features)
                or b.shape != (self.out_features, r)):
            raise ValueError(f"expected a [r, {self.in_features}] and b [{self.out_features}, r] "
                             f"with r up to {self.rank}, got {list(a.shape)} and {list(b.shape)}")
        if a.dtype != self.dtype or b.dtype != self.dtype:
            raise ValueError(f"adapters of this pager are {self.dtype}, got {a.dtype} and "
                             f"{b.dtype}")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("vllm-expert-pager: adapters cannot be written during a capture")
        torch.cuda.synchronize(self.device)
        host_a, host_b = (t[adapter] for t in self._host)
        host_a.zero_()
        host_b.zero_()
        host_a[:r].copy_(a.detach())
        host_b[:, :r].copy_(b.detach())
        self._scales[adapter] = float(scale)
        # Out of its slot; an adapter without one has -1, the arrays' sink element.
        t = self.table
        slot = t.slot_of[adapter : adapter + 1]
        t.expert_in[slot] = -1
        t.last_used[slot] = 0
        t.slot_of[adapter] = -1
        torch.cuda.synchronize(self.device)

    def page(self, ids: torch.Tensor) -> torch.Tensor:
        """Bring the adapters in ``ids`` (int32 or int64, at most ``slots`` of them) into slots.

        Ids out of range (requests without an adapter: -1) are ignored, equal
        ones counted once.  Returns every adapter's slot after the step, int64
        ``[num_adapters]``, -1 for those in host memory only.
        """
        if not self._buffers:
            raise RuntimeError("vllm-expert-pager: the adapters were released")
        if ids.numel() > self.slots:
            raise ValueError(f"a step pages at most {self.slots} adapters, got {ids.numel()} ids: "
                             "pass each request's adapter once, or split the batch")
        if ids.device.type == "cuda" and ids.device != self.device:
            raise ValueError(f"ids are on {ids.device}, the adapters on {self.device}")
        with torch.cuda.device(self.device):
            _, slot, todo = self.table.acquire(ids)
            if todo.numel():
                gather_rows(todo, slot, self.table.no_cache, self.table.experts, 0, self._rows,
                            self._slabs, self._slabs, None, self._scale_rows, self._scale_slots)
        self.slot_map = slot
        return slot

    def add(self, y: torch.Tensor, x: torch.Tensor, ids: torch.Tensor,
            out: torch.Tensor | None = None) -> torch.Tensor:
        """``add_low_rank`` with every row's adapter id, after ``page`` of the step's adapters.

        A row whose adapter is in no slot keeps ``y``, as a row without one does.
        """
        if not hasattr(self, "slot_map"):
            raise RuntimeError("vllm-expert-pager: page the step's adapters first")
        return add_low_rank(y, x, self.a, self.b, ids, scale=self.scale, slot_map=self.slot_map,
                            out=out)

    def release(self) -> None:
        """Wait for the device and free the pinned memory; the pager cannot page after it."""
        if not self._buffers:
            return
        torch.cuda.synchronize(self.device)
        self._host, self._rows = [], []
        for buf in self._buffers:
            buf.free()
        self._buffers = []
