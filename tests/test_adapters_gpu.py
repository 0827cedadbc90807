"""Low-rank adapters against a 64-bit restatement.

Bound of an output: half a step of its type, and the fp32 work before it.  A sum of
H products in 32 bits is off by at most H steps of 2^-23 of the sum of magnitudes
(tensor cores may cut instead of rounding); the low-rank value may be carried as two
16-bit parts, which keeps 2^-16 of it; the second product adds rank steps, the scale
and the final addition two more.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
STEP = 2.0 ** -23
HALF = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}
TYPES = [torch.bfloat16, torch.float16]


def make(M, H, N, r, S, dtype, seed=0, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def n(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    o = dict(x=n(M, H) * size, y=n(M, N), a=n(S, r, H) / math.sqrt(H), b=n(S, N, r) / math.sqrt(r))
    o = {k: v.to(dtype) for k, v in o.items()}
    o["scale"] = torch.rand((S,), generator=g, device=DEV) + 0.5
    return o, g


def reference(y, x, a, b, slots, scale):
    """The rows' results and their bounds, for slots (-1: no adapter) on the host."""
    M, N = y.shape
    S, r, H = a.shape
    want, bound = y.double().clone(), torch.zeros((M, N), dtype=torch.float64, device=DEV)
    half, tiny = HALF[y.dtype]
    for s in sorted(set(slots.tolist()) - {-1}):
        m = (slots == s).nonzero().reshape(-1)
        f = 1.0 if scale is None else scale[s].double()
        xs, A, B = x[m].double(), a[s].double(), b[s].double()
        v, size = xs @ A.T, xs.abs() @ A.abs().T
        low = f * (v @ B.T)
        off = f * (((H + 2) * STEP * size + 2.0 ** -16 * v.abs()) @ B.abs().T
                   + (r + 4) * STEP * (v.abs() @ B.abs().T))
        want[m] += low
        bound[m] = half * 1.01 * want[m].abs() + tiny + off * 1.01 + 2 * STEP * (y[m].double().abs()
                                                                                + low.abs())
    return want, bound


def check(o, ids, slots, scale="own", out=None, **more):
    from vllm_expert_pager import adapters

    scale = o["scale"] if isinstance(scale, str) else scale
    y, x = o["y"], o["x"]
    want, bound = reference(y, x, o["a"], o["b"], slots, scale)
    got = adapters.add_low_rank(y, x, o["a"], o["b"], ids, scale=scale, out=out, **more)
    torch.cuda.synchronize()
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, first at " \
        f"{bad.nonzero()[0].tolist()}, rows {sorted(set(bad.nonzero()[:, 0].tolist()))[:9]}"
    return got


def fresh(o):
    return torch.full_like(o["y"], math.nan)


def patterns(M, S, g):
    """Row -> slot of the batches that a server sees."""
    i = torch.arange(M, device=DEV)
    yield "one adapter", torch.full((M,), S - 1, device=DEV)
    yield "each its own", i % S
    yield "prompts", (i * 5 // max(M, 1)) % S
    yield "any order", torch.randint(-1, S, (M,), generator=g, device=DEV)
    yield "none", torch.full((M,), -1, device=DEV)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H, N, r", [(2048, 1024, 16), (64, 64, 8), (512, 2048, 64), (96, 40, 128),
                                     (1000, 72, 24), (8, 8, 1)])
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 33, 64, 65, 130])
def test_add_low_rank_matches_the_definition(dtype, H, N, r, M):
    S = 6
    o, g = make(M, H, N, r, S, dtype, seed=M + r)
    for _, slots in patterns(M, S, g):
        check(o, slots.to(torch.int32), slots, out=fresh(o))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H, N, r", [(1, 1, 1), (3, 5, 2), (1021, 2047, 13), (65, 129, 3),
                                     (63, 1000, 17), (2047, 31, 127), (8, 24, 65), (24, 7, 16),
                                     (130, 66, 33)])
@pytest.mark.parametrize("M", [1, 5, 64, 300])
def test_sizes_that_no_vector_divides(dtype, H, N, r, M):
    S = 5
    o, g = make(M, H, N, r, S, dtype, seed=M + r)
    for _, slots in patterns(M, S, g):
        check(o, slots.to(torch.int64), slots, out=fresh(o))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M, H, N, r, S", [
    (255, 256, 512, 16, 200), (256, 128, 256, 64, 3), (257, 256, 128, 8, 64),
    (1023, 64, 192, 32, 7), (1024, 128, 128, 16, 1), (1025, 128, 128, 16, 300),
    (2048, 512, 2048, 16, 8), (4099, 250, 130, 13, 11), (5000, 512, 256, 64, 4096),
    (9001, 64, 64, 128, 2)])
def test_long_batches(dtype, M, H, N, r, S):
    o, g = make(M, H, N, r, S, dtype, seed=M)
    for name, slots in patterns(M, S, g):
        if name == "each its own" and S > 300:
            slots = slots % 50 * 7
        elif name == "any order" and S > 300:
            slots = torch.where(slots >= 0, slots % 40 * 100, -1)
        check(o, slots.to(torch.int32), slots, out=fresh(o))
    # A long prompt between single tokens.
    slots = torch.arange(M, device=DEV) % min(S, 40)
    slots[20 : M - 30] = S - 1
    check(o, slots.to(torch.int32), slots, out=fresh(o))


@pytest.mark.parametrize("M", [4, 300, 3000])
def test_in_place_and_ids_out_of_range(M):
    S = 4
    o, g = make(M, 128, 96, 16, S, torch.bfloat16, seed=M)
    slots = torch.randint(-1, S, (M,), generator=g, device=DEV)
    odd = torch.tensor([-1, -7, S, 1 << 40, -(1 << 62), (1 << 32) + 1], device=DEV)
    ids = torch.where(slots >= 0, slots, odd[torch.arange(M, device=DEV) % 6])
    before = o["y"].clone()
    want, bound = reference(before, o["x"], o["a"], o["b"], slots, o["scale"])
    from vllm_expert_pager import adapters

    got = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, scale=o["scale"])
    assert got is o["y"]
    assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(got[slots < 0], before[slots < 0])


@pytest.mark.parametrize("M", [9, 200, 2500])
def test_slot_map(M):
    """Adapter ids through an expert_map: entries of -1, slots and ids out of range."""
    S, num = 5, 64
    o, g = make(M, 256, 64, 8, S, torch.float16, seed=M)
    slot_map = torch.full((num,), -1, dtype=torch.int32, device=DEV)
    slot_map[torch.arange(S, device=DEV) * 11] = torch.arange(S, dtype=torch.int32, device=DEV)
    slot_map[63] = S        # a slot that the slab does not have
    slot_map[62] = 1 << 30
    ids = torch.randint(-2, num + 3, (M,), generator=g, device=DEV)
    slots = torch.where((ids >= 0) & (ids < num), slot_map[ids.clamp(0, num - 1)].long(), -1)
    slots[slots >= S] = -1
    for t in (torch.int32, torch.int64):
        check(o, ids.to(t), slots, slot_map=slot_map, out=fresh(o))
    wide = slot_map.long()
    wide[62] = -(1 << 40)
    check(o, ids.to(torch.int32), slots, slot_map=wide, out=fresh(o))
    check(o, slots.to(torch.int32), slots, scale=None, out=fresh(o))


@pytest.mark.parametrize("M", [3, 70, 1500])
def test_what_no_row_uses_is_not_read(M):
    """NaN and inf in free slots, in rows without an adapter's x, and around strided rows."""
    S = 6
    H, N, r = 192, 136, 24
    o, g = make(M, H, N, r, S, torch.bfloat16, seed=M)
    o["a"][4:], o["b"][4:], o["scale"][4:] = math.nan, math.inf, math.nan
    slots = torch.randint(-1, 4, (M,), generator=g, device=DEV)
    o["x"][slots < 0] = math.nan
    for offset in (0, 8, 3):  # rows at any distance and alignment
        wide = {k: torch.full((M, 400), math.nan, dtype=torch.bfloat16, device=DEV)
                for k in ("x", "y", "out")}
        x = wide["x"][:, offset : offset + H]
        y = wide["y"][:, offset : offset + N]
        out = wide["out"][:, offset : offset + N]
        x.copy_(o["x"])
        y.copy_(o["y"])
        check({**o, "x": x, "y": y}, slots.to(torch.int32), slots, out=out)
        rest = torch.ones((400,), dtype=torch.bool, device=DEV)
        rest[offset : offset + N] = False
        assert wide["out"][:, rest].isnan().all()  # the columns around out stay as they were
    # y and x may be columns of one buffer, and out y itself.
    both = torch.zeros((M, H + N), dtype=torch.bfloat16, device=DEV)
    both[:, :H], both[:, H:] = o["x"], o["y"]
    ref, bound = reference(o["y"], o["x"], o["a"], o["b"], slots, o["scale"])
    from vllm_expert_pager import adapters

    got = adapters.add_low_rank(both[:, H:], both[:, :H], o["a"], o["b"], slots,
                                scale=o["scale"])
    assert ((got.double() - ref).abs() <= bound).all()
    keep = both[:, :H]
    assert torch.equal(keep.isnan(), o["x"].isnan())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M", [3, 70, 1500])
def test_aligned_rows_that_end_inside_a_vector(dtype, M):
    """Rows on 16-byte boundaries whose widths are no multiple of 8: the values behind a row's
    end are neither used nor written."""
    S = 5
    for H, N, r in ((192, 131, 24), (512, 1999, 64), (189, 136, 16), (77, 65, 5)):
        o, g = make(M, H, N, r, S, dtype, seed=M + N)
        slots = torch.randint(-1, S, (M,), generator=g, device=DEV)
        pitch = (max(H, N) + 23) // 8 * 8
        wide = {k: torch.full((M, pitch), math.nan, dtype=dtype, device=DEV)
                for k in ("x", "y", "out")}
        x, y, out = wide["x"][:, :H], wide["y"][:, 8 : 8 + N], wide["out"][:, :N]
        x.copy_(o["x"])
        y.copy_(o["y"])
        check({**o, "x": x, "y": y}, slots, slots, out=out)
        assert wide["out"][:, N:].isnan().all()
        want = wide["out"][:, :N].clone()
        from vllm_expert_pager import adapters

        adapters.add_low_rank(y, x, o["a"], o["b"], slots, scale=o["scale"])  # in place
        assert torch.equal(y, want)
        assert wide["y"][:, :8].isnan().all() and wide["y"][:, 8 + N :].isnan().all()


@pytest.mark.parametrize("M", [2, 40, 1200])
def test_rows_are_apart(M):
    """A row's result is the same bits whatever rows it shares the batch with, in any order."""
    S = 7
    from vllm_expert_pager import adapters

    o, g = make(M, 320, 200, 16, S, torch.bfloat16, seed=M)
    slots = torch.randint(-1, S, (M,), generator=g, device=DEV).to(torch.int32)
    first = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], slots, out=fresh(o))
    for _ in range(2):
        again = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], slots, out=fresh(o))
        assert torch.equal(first, again)
    perm = torch.randperm(M, generator=g, device=DEV)
    moved = adapters.add_low_rank(o["y"][perm], o["x"][perm], o["a"], o["b"], slots[perm])
    assert torch.equal(moved, first[perm])


def test_large_and_small_values():
    """Low-rank values beyond float16's range and deep below it keep their precision; an
    infinity or NaN stays in its row."""
    for M in (6, 400):
        for size in (1e4, 1e-4):
            o, g = make(M, 64, 32, 8, 3, torch.float16, seed=M, size=size)
            slots = torch.arange(M, device=DEV) % 3
            if size > 1:  # v around 3e5, scaled back into range
                o["a"] = (o["a"].float() * 30).to(torch.float16)
                o["scale"] = torch.full((3,), 2.0 ** -12, device=DEV)
            check(o, slots, slots, out=fresh(o))
        o, g = make(M, 64, 32, 8, 3, torch.float16, seed=M)
        slots = torch.arange(M, device=DEV) % 3
        clean = check(o, slots, slots, out=fresh(o))
        o["x"][2, 5] = math.nan
        o["x"][3, 7] = math.inf
        from vllm_expert_pager import adapters

        got = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], slots, scale=o["scale"],
                                    out=fresh(o))
        assert got[2].isnan().all() and not got[3].isfinite().any()
        rest = [i for i in range(M) if i not in (2, 3)]
        assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("big", ["x", "y"])
def test_offsets_past_32_bits(big):
    H, N, r, S, pitch = 128, 96, 16, 2, (1 << 30) + 8
    for M, step in ((3, pitch), (1100, (1 << 21) + 8)):
        o, _ = make(M, H, N, r, S, torch.bfloat16, seed=M)
        slots = torch.arange(M, device=DEV) % S
        width = H if big == "x" else N
        buf = torch.empty(((M - 1) * step + width,), dtype=torch.bfloat16, device=DEV)
        rows = buf.as_strided((M, width), (step, 1))
        rows.copy_(o[big])
        o[big] = rows
        if big == "x":
            check(o, slots, slots, out=fresh(o))
        else:
            want, bound = reference(o["y"].clone(), o["x"], o["a"], o["b"], slots, o["scale"])
            from vllm_expert_pager import adapters

            got = adapters.add_low_rank(rows, o["x"], o["a"], o["b"], slots, scale=o["scale"])
            assert ((got.double() - want).abs() <= bound).all()
        del buf, rows, o


@pytest.mark.parametrize("M", [5, 1300])
def test_replays_in_graphs_and_on_streams(M):
    from vllm_expert_pager import adapters

    S = 4
    o, g = make(M, 256, 128, 16, S, torch.bfloat16, seed=M)
    ids = torch.zeros((M,), dtype=torch.int32, device=DEV)

    def step(out=None):
        return adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, scale=o["scale"],
                                     out=torch.empty_like(o["y"]) if out is None else out)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(3):
        ids.copy_(torch.randint(-1, S, (M,), generator=g, device=DEV))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        slots = ids.long()
        check(o, ids, slots, out=fresh(o))
        assert all(torch.equal(out, want) for _, out in graphs)
    sides = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)


# ---- the pager ----

def adapter(num, r, H, N, dtype, g):
    a = (torch.randn((r, H), generator=g) / math.sqrt(H)).to(dtype)
    b = (torch.randn((N, r), generator=g) / math.sqrt(r)).to(dtype)
    return a, b, 0.5 + float(torch.rand((), generator=g))


def pager_of(num, slots, rank, H, N, dtype, seed=0):
    from vllm_expert_pager.adapters import AdapterPager

    g = torch.Generator().manual_seed(seed)
    pager = AdapterPager(num, slots, rank, H, N, dtype, DEV)
    all_ = [adapter(i, 1 + i % rank, H, N, dtype, g) for i in range(num)]
    for i, (a, b, f) in enumerate(all_):
        pager.write(i, a, b, f)
    return pager, all_, g


def slabs(all_, rank, H, N, dtype):
    """All adapters as slabs padded to one rank."""
    a = torch.zeros((len(all_), rank, H), dtype=dtype, device=DEV)
    b = torch.zeros((len(all_), N, rank), dtype=dtype, device=DEV)
    for i, (u, w, _) in enumerate(all_):
        a[i, : u.shape[0]] = u.to(DEV)
        b[i, :, : u.shape[0]] = w.to(DEV)
    return a, b, torch.tensor([f for *_, f in all_], device=DEV)


@pytest.mark.parametrize("rank, H, N", [(12, 96, 72), (16, 257, 131)])
def test_pager_serves_more_adapters_than_slots(rank, H, N):
    num, S, dtype = 40, 6, torch.bfloat16
    pager, all_, g = pager_of(num, S, rank, H, N, dtype)
    try:
        for step in range(30):
            M = (1, 9, 700)[step % 3]
            requests = torch.randint(-1, num, (S,), generator=g)
            ids = requests[torch.randint(0, S, (M,), generator=g)]
            y = torch.randn((M, N), generator=g).to(dtype).to(DEV)
            x = torch.randn((M, H), generator=g).to(dtype).to(DEV)
            if step == 11:  # an adapter that is in a slot gets new weights
                i = int(requests.clamp(min=0)[0])
                all_[i] = adapter(i, rank, H, N, dtype, g)
                pager.write(i, *all_[i])
            slot = pager.page(requests.to(DEV))
            got = pager.add(y, x, ids.to(DEV), out=torch.empty_like(y))
            a, b, f = slabs(all_, rank, H, N, dtype)
            want, bound = reference(y, x, a, b, ids.to(DEV), f)
            assert ((got.double() - want).abs() <= bound).all(), step
            live = requests[requests >= 0].unique()
            assert (slot[live.to(DEV)] >= 0).all()
            assert int((slot >= 0).sum()) <= S
        assert int(pager.table.misses) > S and int(pager.table.hits) > 0
        with pytest.raises(ValueError, match="at most 6 adapters"):
            pager.page(torch.zeros((7,), dtype=torch.int32, device=DEV))
        # A row whose adapter is in host memory only keeps y.
        out_of = int((pager.slot_map < 0).nonzero()[0])
        got = pager.add(y, x, torch.full((M,), out_of, device=DEV), out=torch.empty_like(y))
        assert torch.equal(got, y)
    finally:
        pager.release()
    with pytest.raises(RuntimeError, match="released"):
        pager.page(torch.zeros((1,), dtype=torch.int32, device=DEV))


def test_pager_step_replays_in_a_graph():
    num, S, rank, H, N, M, dtype = 24, 5, 8, 128, 64, 33, torch.float16
    pager, all_, g = pager_of(num, S, rank, H, N, dtype, seed=3)
    try:
        requests = torch.zeros((S,), dtype=torch.int32, device=DEV)
        rows = torch.zeros((M,), dtype=torch.int64, device=DEV)
        x = torch.zeros((M, H), dtype=dtype, device=DEV)
        y = torch.zeros((M, N), dtype=dtype, device=DEV)
        out = torch.empty_like(y)
        pager.page(requests)
        pager.add(y, x, rows, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pager.page(requests)
            pager.add(y, x, rows, out=out)
            with pytest.raises(RuntimeError, match="during a capture"):
                pager.write(0, *all_[0])
        a, b, f = slabs(all_, rank, H, N, dtype)
        for _ in range(12):
            new = torch.randint(-1, num, (S,), generator=g)
            ids = new[torch.randint(0, S, (M,), generator=g)]
            requests.copy_(new)
            rows.copy_(ids)
            x.copy_(torch.randn((M, H), generator=g))
            y.copy_(torch.randn((M, N), generator=g))
            graph.replay()
            torch.cuda.synchronize()
            want, bound = reference(y, x, a, b, ids.to(DEV), f)
            assert ((out.double() - want).abs() <= bound).all()
        del graph
    finally:
        pager.release()


def test_pager_refusals():
    from vllm_expert_pager.adapters import AdapterPager

    t = torch.bfloat16
    pager = AdapterPager(4, 2, 5, 16, 8, t, DEV)
    try:
        assert pager.rank == 8
        y, x = torch.ones((3, 8), dtype=t, device=DEV), torch.ones((3, 16), dtype=t, device=DEV)
        with pytest.raises(RuntimeError, match="page the step"):
            pager.add(y, x, torch.zeros((3,), dtype=torch.int32, device=DEV))
        for i in (-1, 4):
            with pytest.raises(ValueError, match="adapter must be in"):
                pager.write(i, torch.zeros((2, 16), dtype=t), torch.zeros((8, 2), dtype=t))
        for a, b in ((torch.zeros((9, 16)), torch.zeros((8, 9))),
                     (torch.zeros((2, 15)), torch.zeros((8, 2))),
                     (torch.zeros((2, 16)), torch.zeros((8, 3))),
                     (torch.zeros((16,)), torch.zeros((8, 1)))):
            with pytest.raises(ValueError, match="expected a"):
                pager.write(0, a.to(t), b.to(t))
        with pytest.raises(ValueError, match="of this pager are"):
            pager.write(0, torch.zeros((2, 16)), torch.zeros((8, 2)))
        with pytest.raises(ValueError, match="CUDA tensor"):
            pager.page(torch.zeros((1,), dtype=torch.int32))
        # Never written: zero.  An empty step pages nothing.
        pager.page(torch.tensor([1, 2], dtype=torch.int32, device=DEV))
        assert torch.equal(pager.add(y, x, torch.tensor([1, 2, 1], device=DEV),
                                     out=torch.empty_like(y)), y)
        pager.page(torch.zeros((0,), dtype=torch.int64, device=DEV))
    finally:
        pager.release()
        pager.release()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M, H, N, r", [
    (1, 2048, 1024, 16), (5, 3, 7, 2), (40, 200, 40, 33), (300, 1021, 131, 128),
    (1100, 512, 72, 16), (1100, 835, 65, 40), (2000, 1024, 128, 64), (1500, 96, 31, 100),
    (3000, 512, 256, 64), (9000, 1024, 192, 48), (20000, 832, 128, 64), (20000, 832, 64, 128)])
def test_low_rank_values_are_whole(dtype, M, H, N, r):
    """Two low-rank values that agree in all but their last bits, subtracted: what is left is
    exact only if they enter the second product with the 24 bits of their sums."""
    from vllm_expert_pager import adapters

    S = 3
    most, least = {torch.bfloat16: (2.0 ** -9, 2.0 ** -19),
                   torch.float16: (2.0 ** -12, 2.0 ** -23)}[dtype]
    x = torch.zeros((M, H), dtype=dtype, device=DEV)
    a = torch.zeros((S, r, H), dtype=dtype, device=DEV)
    b = torch.zeros((S, N, r), dtype=dtype, device=DEV)
    at = [0, H // 2, H - 1]
    x[:, at] = 1.0
    a[:, 0, at] = torch.tensor([1.0, most, least], dtype=dtype, device=DEV)
    a[:, r - 1, at] = torch.tensor([1.0, most, 0.0], dtype=dtype, device=DEV)
    b[:, :, 0], b[:, :, r - 1] = 1.0, -1.0
    ids = torch.arange(M, dtype=torch.int32, device=DEV) % S
    got = adapters.add_low_rank(torch.zeros((M, N), dtype=dtype, device=DEV), x, a, b, ids)
    assert torch.equal(got, torch.full_like(got, least))


def classes(t):
    """Of every value: 0 finite, 1 and -1 the infinities, 2 NaN."""
    return torch.where(t.isnan(), 2, torch.where(t.isinf(), t.sign(), 0.0)).to(torch.int8)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M, H, N", [(6, 64, 40), (50, 61, 37), (1100, 64, 72), (1100, 835, 65),
                                     (1100, 1024, 128)])
@pytest.mark.parametrize("r", [1, 2, 8, 13, 16, 24, 65, 128])
def test_infinities_are_those_of_the_definition(dtype, M, H, N, r):
    """Infinite values of x, a and b give the infinity or the NaN that the sums of the
    definition give, in the rows and columns that they reach, and nothing elsewhere."""
    from vllm_expert_pager import adapters

    S = 2
    o, g = make(M, H, N, r, S, dtype, seed=M + r)
    slots = torch.arange(M, device=DEV) % S

    def run():
        return adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], slots, scale=o["scale"],
                                     out=fresh(o))

    def want():
        out = o["y"].double()
        for s in range(S):
            m = slots == s
            v = (o["x"][m].double()[:, None, :] * o["a"][s].double()).sum(2)
            out[m] += o["scale"][s].double() * (v[:, None, :] * o["b"][s].double()).sum(2)
        return out

    for positive in (False, True):
        if positive:
            o = {k: t.abs() for k, t in o.items()}
        clean = run()
        o["x"][2, 5] = math.inf
        o["x"][3, 7] = -math.inf
        keep = o["b"][1, 11 % N].clone()
        o["b"][1, 11 % N, r // 2] = -math.inf
        got, ref = run(), want()
        assert torch.equal(classes(got), classes(ref.to(dtype)))
        same = torch.ones_like(got, dtype=torch.bool)
        same[2], same[3] = False, False
        same[slots == 1, 11 % N] = False
        assert torch.equal(got[same], clean[same])
        if positive:  # sums of one sign: nothing cancels
            assert (got[2] == math.inf).sum() == N and (got[3] == -math.inf).sum() >= N - 1
        o["x"][2, 5] = o["x"][3, 7] = 1.0
        o["b"][1, 11 % N] = keep


@pytest.mark.parametrize("M", [4, 1100])
def test_values_beside_an_infinity_and_at_the_range_end(M):
    """An infinite low-rank value beside a finite one beyond float16's range, which b gives the
    other sign; and in bfloat16 a finite one above bfloat16's largest."""
    from vllm_expert_pager import adapters

    H, N = 16, 24
    ids = torch.zeros((M,), dtype=torch.int32, device=DEV)

    def zeros(dtype, r):
        return (torch.zeros((M, N), dtype=dtype, device=DEV),
                torch.zeros((M, H), dtype=dtype, device=DEV),
                torch.zeros((1, r, H), dtype=dtype, device=DEV),
                torch.zeros((1, N, r), dtype=dtype, device=DEV))

    y, x, a, b = zeros(torch.float16, 2)
    x[:], a[:] = 1.0, 1.0
    x[:, 1], a[0, 0, 0], a[0, 1, 1] = 6e4, math.inf, 6e4
    b[0, :, 0], b[0, :, 1] = 1.0, -1.0
    assert (adapters.add_low_rank(y, x, a, b, ids) == math.inf).all()
    y, x, a, b = zeros(torch.bfloat16, 1)
    x[:, 0], x[:, 1] = torch.finfo(torch.bfloat16).max, 2.0 ** 119 + 2.0 ** 118
    a[0, 0, :2], b[:] = 1.0, 2.0 ** -100
    v = x[0, 0].double() + x[0, 1].double()
    got = adapters.add_low_rank(y, x, a, b, ids)
    assert torch.equal(got, (v * 2.0 ** -100).to(torch.bfloat16).expand(M, N))
    # Low-rank values of one bit, of none, and far below the row's largest, times infinity.
    for dtype in TYPES:
        for value, want in ((1.0, math.inf), (-2.0 ** -14, -math.inf), (0.0, math.nan)):
            for beside in (0.0, 2.0 ** 15):
                y, x, a, b = zeros(dtype, 3)
                x[:, 0], x[:, 1] = 1.0, beside
                a[0, 1, 0], a[0, 0, 1], b[0, :, 1] = value, 2.0 ** 10, math.inf
                got = adapters.add_low_rank(y, x, a, b, ids)
                assert torch.equal(classes(got), classes(torch.full_like(got, want)))


@pytest.mark.parametrize("M", [3, 1100])
def test_autograd_sees_the_update_in_place(M):
    """A value that autograd has saved may not change unseen, as with torch's own updates."""
    from vllm_expert_pager import adapters

    o, _ = make(M, 64, 32, 8, 2, torch.bfloat16)
    ids = torch.zeros((M,), dtype=torch.int32, device=DEV)
    gate = torch.ones((M, 32), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    for out in (None, "out"):
        t = o["y"] if out is None else torch.zeros_like(o["y"])
        z = t * gate
        before = t._version
        adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, out=None if out is None else t)
        assert t._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
    h = gate.exp()  # saves its result
    with torch.no_grad():
        adapters.add_low_rank(h, o["x"], o["a"], o["b"], ids)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    # What is only read stays as it was, and tensors without a version are taken as before.
    versions = [o[k]._version for k in ("x", "a", "b", "y")]
    adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, out=torch.empty_like(o["y"]))
    assert versions == [o[k]._version for k in ("x", "a", "b", "y")]
    with torch.inference_mode():
        y = o["y"].clone()
    want = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, out=torch.empty_like(o["y"]))
    assert torch.equal(adapters.add_low_rank(y, o["x"], o["a"], o["b"], ids), want)


def test_add_follows_a_replayed_page():
    """A captured page that is replayed after an eager one moves adapters: the add behind it
    reads the slots that are current, eagerly and in a graph of its own."""
    num, S, rank, H, N, dtype = 12, 3, 8, 64, 48, torch.bfloat16
    pager, all_, g = pager_of(num, S, rank, H, N, dtype, seed=5)
    try:
        a, b, f = slabs(all_, rank, H, N, dtype)
        requests = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
        pager.page(requests)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pager.page(requests)
        M = 9
        y = torch.randn((M, N), generator=g).to(dtype).to(DEV)
        x = torch.randn((M, H), generator=g).to(dtype).to(DEV)
        rows = torch.zeros((M,), dtype=torch.int32, device=DEV)
        out = torch.empty_like(y)
        pager.add(y, x, rows, out=out)
        torch.cuda.synchronize()
        adds = torch.cuda.CUDAGraph()
        with torch.cuda.graph(adds):
            pager.add(y, x, rows, out=out)
        for step in range(6):
            pager.page(torch.randperm(num, generator=g)[:S].to(DEV))
            new = torch.randperm(num, generator=g)[:S]
            requests.copy_(new)
            graph.replay()
            ids = new[torch.randint(0, S, (M,), generator=g)].to(DEV)
            rows.copy_(ids)
            want, bound = reference(y, x, a, b, ids, f)
            got = pager.add(y, x, ids, out=torch.empty_like(y))
            assert ((got.double() - want).abs() <= bound).all(), step
            adds.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, got)
        # New weights: the rows of the adapter keep y until it is paged again.
        i = int(new[0])
        rows.fill_(i)
        all_[i] = adapter(i, rank, H, N, dtype, g)
        pager.write(i, *all_[i])
        assert torch.equal(pager.add(y, x, rows, out=torch.empty_like(y)), y)
        pager.page(rows[:1])
        a, b, f = slabs(all_, rank, H, N, dtype)
        want, bound = reference(y, x, a, b, rows.long(), f)
        got = pager.add(y, x, rows, out=torch.empty_like(y))
        assert ((got.double() - want).abs() <= bound).all()
        # The number behind the last adapter is no adapter.
        last = torch.full((M,), num, dtype=torch.int32, device=DEV)
        assert torch.equal(pager.add(y, x, last, out=torch.empty_like(y)), y)
        del graph, adds
    finally:
        pager.release()


@pytest.mark.parametrize("M", [3, 1100])
def test_an_empty_slot_map_has_no_adapter(M):
    from vllm_expert_pager import adapters

    o, _ = make(M, 64, 32, 8, 2, torch.bfloat16)
    ids = torch.zeros((M,), dtype=torch.int32, device=DEV)
    for t in (torch.int32, torch.int64):
        got = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, out=fresh(o),
                                    slot_map=torch.empty((0,), dtype=t, device=DEV))
        assert torch.equal(got, o["y"])


def test_one_row_in_place_at_another_stride():
    from vllm_expert_pager import adapters

    o, _ = make(1, 64, 48, 8, 2, torch.bfloat16)
    for slot in (1, -1):
        ids = torch.full((1,), slot, dtype=torch.int32, device=DEV)
        want = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, out=fresh(o))
        for offset in (0, 3):
            buf = torch.full((200,), 7.0, dtype=torch.bfloat16, device=DEV)
            y = buf.as_strided((1, 48), (100, 1), offset)
            y.copy_(o["y"])
            out = buf.as_strided((1, 48), (48, 1), offset)
            assert adapters.add_low_rank(y, o["x"], o["a"], o["b"], ids, out=out) is out
            assert torch.equal(out, want)
            assert (buf[offset + 48 :] == 7.0).all() and (buf[:offset] == 7.0).all()


def test_calls_of_several_threads():
    """Launches of one kernel with other amounts of shared memory, from threads that do not
    hold the interpreter's lock: none takes away what another has asked for."""
    import threading

    from vllm_expert_pager import native

    lib = native.lib()
    M, H, N, r = 1100, 8, 8, 1
    statuses = {}

    def calls(S, stream, x, y, a, b, ids, scratch):
        need = lib.xp_low_rank_scratch_bytes(M, S)
        statuses[S] = {lib.xp_add_low_rank(
            x.data_ptr(), H, y.data_ptr(), N, y.data_ptr(), N, 1, M, H, N, r, a.data_ptr(),
            b.data_ptr(), S, None, ids.data_ptr(), 4, None, 0, 0, scratch.data_ptr(), need,
            stream.cuda_stream) for _ in range(4000)}

    threads = []
    for S in (4200, 8192):
        o, _ = make(M, H, N, r, S, torch.bfloat16)
        ids = torch.full((M,), -1, dtype=torch.int32, device=DEV)
        scratch = torch.empty((lib.xp_low_rank_scratch_bytes(M, S),), dtype=torch.uint8, device=DEV)
        threads.append(threading.Thread(target=calls, args=(
            S, torch.cuda.Stream(), o["x"], o["y"], o["a"], o["b"], ids, scratch)))
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert statuses == {4200: {native.XP_OK}, 8192: {native.XP_OK}}


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M, H, N, r", [(1100, 512, 256, 16), (1100, 1024, 256, 64),
                                        (5000, 1021, 131, 13), (1100, 61, 95, 100),
                                        (4000, 2048, 512, 128)])
def test_waits_that_give_up_are_counted(dtype, M, H, N, r):
    """With no time to wait, blocks give up: their columns are NaN, the others right, the host
    can read how many did, and the next call finds everything as before."""
    from vllm_expert_pager import adapters, native

    S = 4
    o, g = make(M, H, N, r, S, dtype, seed=M)
    slots = torch.randint(-1, S, (M,), generator=g, device=DEV)
    ids = slots.to(torch.int32)
    want, bound = reference(o["y"], o["x"], o["a"], o["b"], slots, o["scale"])
    clean = check(o, ids, slots, out=fresh(o))
    before = adapters.wait_errors()
    limit = native.lib().xp_low_rank_wait_limit(0)
    try:
        got = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, scale=o["scale"],
                                    out=torch.zeros_like(o["y"]))
        gave_up = adapters.wait_errors() - before
    finally:
        assert native.lib().xp_low_rank_wait_limit(limit) == 0
    assert gave_up > 0 and got.isnan().any()
    assert (got.isnan() | ((got.double() - want).abs() <= bound)).all()
    assert torch.equal(got[slots < 0], o["y"][slots < 0])
    assert torch.equal(check(o, ids, slots, out=fresh(o)), clean)
    assert adapters.wait_errors() - before == gave_up


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M, H, N, r, S", [
    # Clusters of four: aligned and not, columns for some CTAs only, H just split and not.
    (1100, 2048, 192, 8, 8), (1100, 2048, 100, 128, 4), (1100, 1021, 2047, 13, 8),
    (1025, 769, 64, 32, 2), (1300, 768, 136, 64, 8), (1300, 832, 136, 64, 8),
    # Of two.
    (5000, 1024, 192, 64, 8), (5000, 1021, 131, 16, 8), (5000, 832, 64, 128, 8),
    # One CTA a tile, one and two of them on an SM, ranks of every kind.
    (16384, 1024, 128, 64, 8), (16384, 1024, 72, 16, 8), (16384, 832, 128, 128, 8),
    (16384, 1021, 131, 40, 8), (24000, 1024, 128, 64, 8), (24000, 896, 64, 32, 8),
    # More slots than tiles.
    (1600, 1024, 72, 16, 600)])
def test_long_batches_of_wide_rows(dtype, M, H, N, r, S):
    """Rows so wide that the CTAs of a tile share their sums."""
    from vllm_expert_pager import adapters

    o, g = make(M, H, N, r, S, dtype, seed=M + r)
    i = torch.arange(M, device=DEV)
    for slots in (torch.randint(-1, S, (M,), generator=g, device=DEV), i * 5 // M % S,
                  torch.full((M,), S - 1, device=DEV)):
        ids = slots.to(torch.int32)
        first = check(o, ids, slots, out=fresh(o))
        for _ in range(3):
            again = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, scale=o["scale"],
                                          out=fresh(o))
            assert torch.equal(again, first)
        y = o["y"].clone()
        adapters.add_low_rank(y, o["x"], o["a"], o["b"], ids, scale=o["scale"])
        assert torch.equal(y, first)


def test_wait_errors_leave_a_capture_alone():
    from vllm_expert_pager import adapters

    o, _ = make(1100, 64, 32, 8, 2, torch.bfloat16)
    ids = torch.zeros((1100,), dtype=torch.int32, device=DEV)
    want = adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, out=fresh(o))
    out = fresh(o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adapters.add_low_rank(o["y"], o["x"], o["a"], o["b"], ids, out=out)
        with pytest.raises(ValueError, match="wait_errors failed"):
            adapters.wait_errors()
    before = adapters.wait_errors()
    graph.replay()
    assert adapters.wait_errors(DEV) == before and torch.equal(out, want)
