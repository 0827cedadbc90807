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

import ctypes

import torch

from vllm_expert_pager import native
from vllm_expert_pager.acquire import MAX_SLOTS
from vllm_expert_pager.gather import gather_rows
from vllm_expert_pager.store import PinnedBuffer, numa_node_of
from vllm_expert_pager.table import ExpertTable

_DTYPES = (torch.bfloat16, torch.float16)


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
    that would need a gradient, or with a dual tensor of forward-mode
    derivatives, is refused, and a backward pass that saved the
    values which ``out`` had before raises, as after torch's own updates in place.
    Rows may hold NaN that the operands do not explain only if ``wait_errors`` has
    risen.
    """
    return native.torch_ops().add_low_rank(y, x, a, b, ids, scale, slot_map, out)


def wait_errors(device: torch.device | None = None) -> int:
    """Blocks of ``add_low_rank`` that gave up waiting on ``device`` (the current one) so far.

    The parts of a block of a call with more than 1024 rows wait for one another, 2
    seconds at most; a block that gives up fills its part of ``out`` with NaN.  Waits
    for the current stream; during its capture it raises ValueError.
    """
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    count = ctypes.c_uint32()
    with torch.cuda.device(device):
        native.check(native.lib().xp_low_rank_errors(ctypes.byref(count),
                                                     native.stream_of(device)), "wait_errors")
    return count.value


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
        # The table's own map, not this step's copy: it is current after any page, one
        # replayed from a graph too.  (Behind the adapters stands the table's sink.)
        self.slot_map = self.table.slot_of[: self.num_adapters]
        return slot

    def add(self, y: torch.Tensor, x: torch.Tensor, ids: torch.Tensor,
            out: torch.Tensor | None = None) -> torch.Tensor:
        """``add_low_rank`` with every row's adapter id, after ``page`` of the step's adapters.

        The slots are those of the last ``page`` on the device, called or replayed.  A row
        whose adapter is in no slot (after ``write`` it is in none until the next ``page``)
        keeps ``y``, as a row without one does.
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
