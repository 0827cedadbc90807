"""The token-side operators together, as a MoE layer outside a vLLM model uses them.

Router logits -> ``route`` -> ``LayerPager`` (decode steps, and prefills through the
working slab) -> ``moe.contributions`` -> ``moe.moe_sum``, beside a projection that all
tokens share with every request's low-rank adapter on it, paged by ``AdapterPager``.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
E, S, W, TOPK, H = 64, 16, 16, 8, 2048


@pytest.fixture
def layer():
    from vllm_expert_pager import synthetic
    from vllm_expert_pager.pager import PARAMS, LayerPager, WorkingSlab
    from vllm_expert_pager.store import Store

    experts = synthetic.fp8_experts_device(E, DEV, seed=5)
    row_bytes = {n: r * c for n, (r, c) in synthetic.SHAPES.items()}
    store = Store(1, E, E, 2 * W, row_bytes, False, 0.89, None, DEV)
    for n in PARAMS:
        q = experts[n][0].cpu()
        for e in range(E):
            store.write(0, e, n, q[e])
    scales = {f"{n[:-7]}_weight_scale": experts[n][1] for n in PARAMS}
    shapes = {n: (synthetic.SHAPES[n], torch.float8_e4m3fn) for n in PARAMS}
    all_shapes = dict(shapes)
    all_shapes.update({k: (tuple(v.shape[1:]), v.dtype) for k, v in scales.items()})
    pager = LayerPager(store, 0, S, scales, shapes, WorkingSlab(W, all_shapes, store, DEV))
    yield pager, experts
    store.release()


def moe_of(pager, experts, x, r):
    """The layer's MoE on the pager (as the vLLM hook chooses the path), and unpaged."""
    from vllm_expert_pager import moe

    (w13, s13), (w2, s2) = experts["w13_weight"], experts["w2_weight"]
    config = moe.moe_config(w13.shape, w2.shape, TOPK, 64)
    ref, out = torch.empty_like(x), torch.empty_like(x)
    moe.moe_sum(moe.contributions(x, w13, w2, s13, s2, r.weights, r.ids, None, E, config), ref)

    def run(slabs, expert_map):
        return moe.contributions(x, slabs["w13_weight"], slabs["w2_weight"],
                                 slabs["w13_weight_scale"], slabs["w2_weight_scale"], r.weights,
                                 r.ids, expert_map, E, config)

    if r.ids.numel() <= S:
        res = pager.decode(r.ids)
        moe.moe_sum(run(res.slabs, res.expert_map), out)
    else:
        acc = []
        pager.working_chunks(r.ids, lambda k, n, slabs, m: acc.append(run(slabs, m)))
        total = acc[0]
        for c in acc[1:]:
            total.add_(c)
        moe.moe_sum(total, out)
    return out, ref


def test_layer_steps(layer):
    from vllm_expert_pager import routing
    from vllm_expert_pager.adapters import AdapterPager

    pager, experts = layer
    g = torch.Generator(device=DEV).manual_seed(1)
    gate = torch.randn((E, H), generator=g, device=DEV) / math.sqrt(H)
    shared = (torch.randn((H, H), generator=g, device=DEV) / math.sqrt(H)).to(torch.bfloat16)
    num, rank = 12, 16
    lora = AdapterPager(num, 4, rank, H, H, torch.bfloat16, DEV)
    a = (torch.randn((num, rank, H), generator=g, device=DEV) / math.sqrt(H)).to(torch.bfloat16)
    b = (torch.randn((num, H, rank), generator=g, device=DEV) / 4).to(torch.bfloat16)
    for i in range(num):
        lora.write(i, a[i].cpu(), b[i].cpu(), 0.25 + i)
    usage = torch.zeros((E,), dtype=torch.int64, device=DEV)
    try:
        for step, T in enumerate((1, 2, 64, 1, 640, 2)):
            x = (torch.randn((T, H), generator=g, device=DEV) * 0.5).to(torch.bfloat16)
            logits = x.float() @ gate.t()
            r = routing.route(logits, TOPK)
            assert torch.equal(r.ids.long(), logits.topk(TOPK).indices)  # no equal logits here
            usage += r.counts
            out, ref = moe_of(pager, experts, x, r)
            requests = torch.randint(-1, num, (4,), generator=g, device=DEV)
            rows = requests[torch.arange(T, device=DEV) * 4 // T]
            y = x @ shared.t()
            lora.page(requests)
            got = lora.add(y, x, rows, out=torch.empty_like(y))
            torch.cuda.synchronize()
            assert torch.equal(out, ref), step  # paged as unpaged, bit for bit
            for i in set(rows.tolist()):
                m = rows == i
                if i < 0:
                    assert torch.equal(got[m], y[m])
                    continue
                low = (0.25 + i) * (x[m].double() @ a[i].double().t() @ b[i].double().t())
                want = y[m].double() + low
                # Half a step of bfloat16, and 2^-14 of the update's scale for the sums.
                size = (0.25 + i) * (x[m].double().abs() @ a[i].double().abs().t()
                                     @ b[i].double().abs().t())
                assert ((got[m].double() - want).abs() <= 2.0 ** -8 * want.abs()
                        + 2.0 ** -14 * size).all(), (step, i)
        assert int(usage.sum()) == TOPK * (1 + 2 + 64 + 1 + 640 + 2)
    finally:
        lora.release()


def test_layer_decode_step_in_a_graph(layer):
    """Routing, paging, adapters and the MoE's inputs of a decode step, captured once."""
    from vllm_expert_pager import routing
    from vllm_expert_pager.adapters import AdapterPager

    pager, experts = layer
    g = torch.Generator(device=DEV).manual_seed(2)
    T, num = 2, 6
    lora = AdapterPager(num, 3, 8, H, 256, torch.bfloat16, DEV)
    for i in range(num):
        lora.write(i, torch.full((8, H), 2.0 ** -11, dtype=torch.bfloat16),
                   torch.full((256, 8), float(i), dtype=torch.bfloat16))
    logits = torch.zeros((T, E), device=DEV)
    rows = torch.zeros((T,), dtype=torch.int32, device=DEV)
    x = torch.ones((T, H), dtype=torch.bfloat16, device=DEV)
    y = torch.zeros((T, 256), dtype=torch.bfloat16, device=DEV)

    def step():
        r = routing.route(logits, TOPK)
        res = pager.decode(r.ids)
        lora.page(rows)
        return r, res, lora.add(y, x, rows, out=torch.empty_like(y))

    try:
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r, res, out = step()
        for _ in range(8):
            logits.copy_(torch.randn((T, E), generator=g, device=DEV))
            rows.copy_(torch.randint(0, num, (T,), generator=g, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(r.ids.long(), logits.topk(TOPK).indices)
            for e in set(r.ids.view(-1).tolist()):
                slot = int(res.expert_map[e])
                for n in ("w13_weight", "w2_weight"):
                    assert torch.equal(res.slabs[n][slot].view(torch.uint8),
                                       experts[n][0][e].view(torch.uint8))
            # 2048 ones by 2^-11 is 1 for each of 8 ranks, by i: 8 i, exact.
            assert torch.equal(out, (8.0 * rows[:, None]).expand(T, 256).to(torch.bfloat16))
        assert pager.step_errors() == 0
        del graph
    finally:
        lora.release()


def test_router_tuning_over_paged_experts(layer):
    """A router's step with its balance loss: the gradients reach the gate through the logits,
    and agree with differences of the loss along a direction."""
    from vllm_expert_pager import routing

    g = torch.Generator(device=DEV).manual_seed(3)
    T = 128
    x = torch.randn((T, H), generator=g, device=DEV) * 0.5
    gate = (torch.randn((E, H), generator=g, device=DEV) / math.sqrt(H)).requires_grad_()
    back = torch.randn((T, TOPK), generator=g, device=DEV)  # of the weights, as a MoE gives it
    r = routing.route(x @ gate.t(), TOPK, balance=True)
    ((r.weights * back).sum() + 10.0 * r.loss).backward()
    way = torch.randn((E, H), generator=g, device=DEV) / math.sqrt(H)
    h = 1e-4

    def value(w):
        p = torch.softmax(x.double() @ w.t(), 1)
        top = p.gather(1, r.ids.long())
        top = top / top.sum(1, keepdim=True)
        share = r.counts.double() / (T * TOPK)
        return (top * back).sum() + 10.0 * E * (share * p.mean(0)).sum()

    w = gate.detach().double()
    slope = float((value(w + h * way) - value(w - h * way)) / (2 * h))
    got = float((gate.grad.double() * way).sum())
    # Differences: h^2; the logits' 32-bit products of 2048 terms: 2048 steps of 2^-23.
    assert abs(got - slope) <= 4e-4 * float((gate.grad * way).abs().sum())


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_tensors_of_another_device_than_the_current_one():
    from vllm_expert_pager import adapters, routing

    def run(dev):
        g = torch.Generator().manual_seed(3)
        logits = torch.randn((3000, 256), generator=g).to(dev).requires_grad_()
        r = routing.route(logits, 8, balance=True)
        grad, = torch.autograd.grad(r.loss + r.weights[:, 0].sum(), logits)
        outs = [r.weights.detach(), r.ids, r.counts, r.loss.detach(), grad]
        for M in (5, 1500):
            y, x, a, b = (torch.randn(s, generator=g).to(dev, torch.bfloat16) for s in
                          ((M, 96), (M, 1024), (4, 16, 1024), (4, 96, 16)))
            ids = (torch.arange(M) % 5 - 1).to(dev)
            outs.append(adapters.add_low_rank(y, x, a, b, ids))
        assert adapters.wait_errors(dev) == 0
        return [t.cpu() for t in outs]

    with torch.cuda.device(0):
        here, there = run(torch.device("cuda", 0)), run(torch.device("cuda", 1))
    assert all(torch.equal(u, v) for u, v in zip(here, there))
