"""Routing kernels against a 64-bit restatement of their definition.

Tolerances, in steps of 2^-23 relative (an fp32 rounding is half a step): with
x = l - m, the fast exponential is off by at most 2 + 1.173 |x| steps and the
subtraction by |x| / 2; a softmax sum's error is the p-weighted mean of its terms'
(sum p |x| <= ln E) plus half a step for each of its (values per lane + 5)
additions; the division adds one.  ``steps`` adds these up, rounded up.  Outputs in
16 bits add half a step of their type.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
STEP = 2.0 ** -23
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# Half a step relative, and half the smallest subnormal.
HALF = {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
        torch.float16: (2.0 ** -11, 2.0 ** -25)}


def per_lane(E):
    return 2 if E <= 64 else 8 if E <= 256 else 16 if E <= 512 else 32 if E <= 1024 else 128


def steps(x, E):
    """Relative error bound of exp(x) / sum, in units of STEP."""
    return 2 * x.abs() + 2 * math.log(E + 1) + per_lane(E) / 2 + 10


def make(T, E, dtype, seed=0, ties=False, closed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((T, E), generator=g, device=DEV) * 2
    if ties:
        x = x.round()
    if closed:
        x[:, torch.randperm(E, generator=g, device=DEV)[:closed]] = -math.inf
    return x.to(dtype), g


def softmax64(z, live):
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.where(live[:, None], torch.exp(z - m), 0.0)
    s = e.sum(1, keepdim=True)
    return e / torch.where(s > 0, s, 1.0), z - m


def reference(logits, K, renormalize, valid=None):
    """ids, weights, p, x = l - m, counts, loss, tokens in 64 bits."""
    z = logits.double()
    T, E = z.shape
    live = torch.ones((T,), dtype=torch.bool, device=DEV) if valid is None else valid.bool()
    z = torch.where(live[:, None], z, 0.0)  # what a padded row holds does not count
    p, x = softmax64(z, live)
    v, i = torch.sort(z, dim=1, descending=True, stable=True)
    open_ = (v[:, :K] > -math.inf) & live[:, None]
    ids = torch.where(open_, i[:, :K], -1)
    w = torch.where(open_, p.gather(1, i[:, :K]), 0.0)
    if renormalize:
        s = w.sum(1, keepdim=True)
        w = w / torch.where(s > 0, s, 1.0)
    counts = torch.bincount(ids[ids >= 0], minlength=E)
    n = int(live.sum())
    f = counts.double() / max(n * K, 1)
    loss = E * (f * p.sum(0) / max(n, 1)).sum()
    return ids, w, p, x, counts, loss, n


def reference_grad(ids, w, p, counts, n, K, renormalize, gw=None, gl=None):
    """The gradient by its formula, and the magnitudes that its rounding errors go by."""
    T, E = p.shape
    row = torch.arange(T, device=DEV)[:, None].expand(T, K)
    ok = ids >= 0
    grad, size = torch.zeros_like(p), torch.zeros_like(p)
    h = torch.zeros_like(p)
    if gl is not None:
        h = h + gl.double() * E * (counts.double() / max(n * K, 1)) / max(n, 1)
    if gw is not None:
        g = torch.where(ok, gw.double(), 0.0)
        if renormalize:
            d = w * (g - (w * g).sum(1, keepdim=True))
            grad[row[ok], ids[ok]] = d[ok]
            size[row[ok], ids[ok]] = (w * (g.abs() + (w * g.abs()).sum(1, keepdim=True)))[ok]
        else:
            h = h.clone()
            h[row[ok], ids[ok]] += g[ok]
    inner = (p * h).sum(1, keepdim=True)
    grad = grad + p * (h - inner)
    size = size + p * (h.abs() + (p * h.abs()).sum(1, keepdim=True))
    return grad, size


def close(got, want, bound):
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst " \
        f"{float(((got.double() - want).abs() / bound.clamp(min=1e-300)).max())} bounds"


def check_route(logits, K, renormalize, valid=None, train=True, seed=1):
    from vllm_expert_pager import routing

    T, E = logits.shape
    ids, w, p, x, counts, loss, n = reference(logits, K, renormalize, valid)
    leaf = logits.detach().requires_grad_(train)
    r = routing.route(leaf, K, renormalize=renormalize, valid=valid, balance=train)
    torch.cuda.synchronize()
    assert r.weights.dtype == torch.float32 and r.ids.dtype == torch.int32
    assert r.counts.dtype == torch.int64
    assert torch.equal(r.ids.long(), ids)
    assert torch.equal(r.counts, counts)
    xs = torch.where(ids >= 0, x.gather(1, ids.clamp(min=0)), 0.0)
    close(r.weights.detach(), w, (steps(xs, E) * w * STEP).clamp(min=1e-37))
    if not train:
        assert r.loss is None
        return r
    # P adds up a warp's tokens, the CTA's 16 warps and 444 CTAs at most.
    adds = T / (148 * 8) + 16 + 444
    finite = torch.where(p > 1e-38, x.abs(), 0.0)  # smaller ones are below every bound
    rel = (steps(finite.max() if T else torch.zeros(()), E) + adds) * STEP
    close(r.loss.detach(), loss, float(rel) * loss + 1e-300)
    g = torch.Generator(device=DEV).manual_seed(seed)
    gw = torch.randn((T, K), generator=g, device=DEV)
    gl = torch.rand((), generator=g, device=DEV) * 100 * max(n, 1)
    half, tiny = HALF[logits.dtype]
    for use_w, use_l in ((True, True), (True, False), (False, True)):
        outs = [o for o, u in ((r.weights, use_w), (r.loss, use_l)) if u]
        ups = [o for o, u in ((gw, use_w), (gl, use_l)) if u]
        grad, = torch.autograd.grad(outs, leaf, ups, retain_graph=True)
        want, size = reference_grad(ids, w, p, counts, n, K, renormalize,
                                    gw if use_w else None, gl if use_l else None)
        assert grad.dtype == logits.dtype and grad.shape == logits.shape
        rows = steps(finite.amax(1, keepdim=True) if E and T else finite, E)
        close(grad, want, 4 * rows * STEP * size + half * want.abs() * 1.01 + tiny + 1e-36)
    return r


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T, E, K", [
    (1, 256, 8), (3, 1, 1), (17, 2, 2), (64, 60, 4), (33, 64, 32), (16, 65, 7), (40, 257, 8),
    (300, 512, 16), (129, 777, 3), (70, 1024, 8), (21, 1025, 8), (9, 4095, 5), (40, 4096, 32),
    (5003, 96, 6), (6001, 256, 8)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_matches_the_definition(dtype, T, E, K, renormalize):
    logits, _ = make(T, E, dtype, seed=T + E)
    check_route(logits, K, renormalize)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_route_without_gradient(dtype):
    for T, E, K in ((1, 256, 8), (2048, 256, 8), (77, 300, 12)):
        logits, _ = make(T, E, dtype, seed=T)
        for renormalize in (True, False):
            check_route(logits, K, renormalize, train=False)


@pytest.mark.parametrize("E", [48, 256, 1000, 4096])
def test_equal_logits_go_to_the_lower_expert(E):
    logits, _ = make(200, E, torch.float32, seed=3, ties=True)
    logits[5] = 1.0
    logits[6, ::2] = 0.0
    logits[6, 1::2] = -0.0  # equal to 0
    check_route(logits, 8, True)
    check_route(logits.to(torch.bfloat16), 8, False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("renormalize", [True, False])
def test_closed_experts_and_empty_rows(dtype, renormalize):
    logits, _ = make(120, 100, dtype, seed=5, closed=30)
    logits[7] = -math.inf                    # no expert is open
    logits[8] = -math.inf
    logits[8, 41] = -3.0                     # one is
    logits[9, :] = torch.finfo(dtype).min    # all at the lowest value: even
    logits[10, ::3] = torch.finfo(dtype).min
    logits[11] = -math.inf
    logits[11, 90:] = torch.finfo(dtype).min
    r = check_route(logits, 8, renormalize)
    assert (r.ids[7] == -1).all() and (r.weights[7] == 0).all()
    assert r.ids[8].tolist() == [41] + [-1] * 7 and float(r.weights.detach()[8, 0]) == 1.0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_padded_rows_are_not_read(dtype):
    logits, g = make(333, 128, dtype, seed=7)
    valid = torch.rand((333,), generator=g, device=DEV) < 0.6
    logits[~valid] = math.nan
    logits[int((~valid).nonzero()[0]), 0] = math.inf
    for v in (valid, valid.to(torch.uint8)):
        r = check_route(logits, 8, True, valid=v)
        assert (r.ids[~valid] == -1).all() and (r.weights[~valid] == 0).all()
    none = torch.zeros_like(valid)
    r = check_route(logits, 8, False, valid=none)
    assert float(r.loss.detach()) == 0.0 and int(r.counts.sum()) == 0


def test_nan_and_inf_logits_show_in_their_rows_only():
    from vllm_expert_pager import routing

    logits, _ = make(64, 200, torch.float32, seed=9)
    clean = routing.route(logits, 6)
    logits[3, 150] = math.nan
    logits[3, 10] = -math.nan
    logits[4, 17] = math.inf
    r = routing.route(logits, 6, balance=True)
    assert r.ids[3, :2].tolist() == [10, 150] and r.weights[3].isnan().all()
    assert int(r.ids[4, 0]) == 17 and r.weights[4, 0].isnan()
    rest = [i for i in range(64) if i not in (3, 4)]
    assert torch.equal(r.ids[rest], clean.ids[rest])
    assert torch.equal(r.weights[rest], clean.weights[rest])
    assert r.loss.isnan()
    assert ((r.ids >= 0) & (r.ids < 200)).all()


def test_no_tokens():
    from vllm_expert_pager import routing

    leaf = torch.zeros((0, 32), device=DEV, requires_grad=True)
    r = routing.route(leaf, 4, balance=True)
    assert r.weights.shape == (0, 4) and r.ids.shape == (0, 4)
    assert r.counts.tolist() == [0] * 32 and float(r.loss.detach()) == 0.0
    grad, = torch.autograd.grad(r.loss + r.weights.sum(), leaf)
    assert grad.shape == (0, 32)
    loss, counts = routing.balance_loss(leaf, torch.zeros((0, 4), dtype=torch.int64, device=DEV))
    assert float(loss.detach()) == 0.0 and int(counts.sum()) == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_of_a_wider_buffer(dtype):
    """Rows apart from one another, at offsets that no vector load may start at, columns apart,
    and one row for all tokens."""
    wide, _ = make(90, 300, dtype, seed=11)
    for view in (wide[:, 8:264], wide[:, 3:259], wide[:, 1:61], wide[::3, :256],
                 wide[:, ::2], wide.t()[:64], wide[:1, :256].expand(50, 256)):
        check_route(view, 8, True)


def test_offsets_past_32_bits():
    pitch = (1 << 30) + 264
    buf = torch.empty((2 * pitch + 256,), dtype=torch.bfloat16, device=DEV)
    logits, _ = make(3, 256, torch.bfloat16, seed=13)
    rows = buf.as_strided((3, 256), (pitch, 1))
    rows.copy_(logits)
    check_route(rows, 8, True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T, E, K, ids_dtype", [
    (1, 256, 8, torch.int32), (509, 256, 8, torch.int64), (4099, 60, 4, torch.int32),
    (50, 33, 40, torch.int16), (700, 2000, 8, torch.int32)])
def test_balance_loss_matches_the_definition(dtype, T, E, K, ids_dtype):
    from vllm_expert_pager import routing

    logits, g = make(T, E, dtype, seed=T + 1)
    ids = torch.randint(-1, E + 1, (T, K), generator=g, device=DEV)  # some out of range, repeats
    valid = torch.rand((T,), generator=g, device=DEV) < 0.8 if T > 1 else None
    live = torch.ones((T,), dtype=torch.bool, device=DEV) if valid is None else valid
    z = logits.double()
    p, x = softmax64(z, live)
    used = ids[live].reshape(-1)
    counts = torch.bincount(used[(used >= 0) & (used < E)], minlength=E)
    n = int(live.sum())
    want = E * (counts.double() / max(n * K, 1) * p.sum(0) / max(n, 1)).sum()
    leaf = logits.detach().requires_grad_()
    loss, got = routing.balance_loss(leaf, ids.to(ids_dtype), valid=valid)
    assert torch.equal(got, counts)
    bound = (steps(x.abs().max(), E) + T / (148 * 8) + 460) * STEP
    close(loss.detach(), want, float(bound) * want + 1e-300)
    with torch.no_grad():
        again, _ = routing.balance_loss(leaf, ids.to(ids_dtype), valid=valid)
    assert torch.equal(again, loss.detach())
    gl = torch.tensor(17.0 * max(n, 1), device=DEV)
    grad, = torch.autograd.grad(loss, leaf, gl)
    ref, size = reference_grad(ids, None, p, counts, n, K, True, None, gl)
    half, tiny = HALF[dtype]
    close(grad, ref, 4 * steps(x.abs().amax(1, keepdim=True), E) * STEP * size
          + half * ref.abs() * 1.01 + tiny + 1e-36)


def test_gradients_agree_with_differences():
    """The kernels' gradient along a direction against central differences of the 64-bit
    definition, whose own error is O(h^2) = 1e-8 of the value's scale."""
    from vllm_expert_pager import routing

    T, E, K, h = 37, 24, 4, 1e-4
    logits, g = make(T, E, torch.float32, seed=17)
    gw = torch.randn((T, K), generator=g, device=DEV)
    way = torch.randn((T, E), generator=g, device=DEV)
    for renormalize in (True, False):
        ids, *_ = reference(logits, K, renormalize)

        def value(z):
            p, _ = softmax64(z, torch.ones((T,), dtype=torch.bool, device=DEV))
            w = p.gather(1, ids)
            if renormalize:
                w = w / w.sum(1, keepdim=True)
            counts = torch.bincount(ids.reshape(-1), minlength=E).double()
            return (w * gw).sum() + 3.0 * E * (counts / (T * K) * p.mean(0)).sum()

        z = logits.double()
        slope = (value(z + h * way.double()) - value(z - h * way.double())) / (2 * h)
        leaf = logits.detach().requires_grad_()
        r = routing.route(leaf, K, renormalize=renormalize, balance=True)
        ((r.weights * gw).sum() + 3.0 * r.loss).backward()
        got = (leaf.grad.double() * way.double()).sum()
        assert abs(float(got - slope)) < 1e-5 * float((leaf.grad * way).abs().sum())


def test_results_do_not_depend_on_the_run():
    from vllm_expert_pager import routing

    logits, g = make(30000, 256, torch.bfloat16, seed=19)
    first = None
    for _ in range(3):
        leaf = logits.detach().requires_grad_()
        r = routing.route(leaf, 8, balance=True)
        grad, = torch.autograd.grad(r.loss * 1000 + r.weights.square().sum(), leaf)
        got = [r.weights.detach(), r.ids, r.counts, r.loss.detach(), grad]
        first = first or got
        assert all(torch.equal(u, v) for u, v in zip(first, got))


def test_forward_and_backward_replay_in_a_graph():
    from vllm_expert_pager import routing

    T, E, K = 700, 128, 6
    logits, _ = make(T, E, torch.bfloat16, seed=23)
    static = logits.clone().requires_grad_()
    gw = torch.ones((T, K), device=DEV)

    def step():
        r = routing.route(static, K, balance=True)
        grad, = torch.autograd.grad((r.weights, r.loss), static, (gw, torch.ones_like(r.loss)))
        return r.weights.detach(), r.ids, r.counts, r.loss.detach(), grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs: each holds scratch of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for seed in (29, 31):
        new, _ = make(T, E, torch.bfloat16, seed=seed)
        with torch.no_grad():
            static.copy_(new)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, outs in graphs:
            assert all(torch.equal(u, v) for u, v in zip(outs, want))


def test_streams_and_gradient_forms():
    """Calls on a side stream, one of them while another runs; expanded and missing
    upstream gradients; a leaf used twice."""
    from vllm_expert_pager import routing

    logits, _ = make(5000, 256, torch.float32, seed=37)
    want = routing.route(logits, 8, balance=True)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(routing.route(logits, 8, balance=True))
    torch.cuda.synchronize()
    for r in got:
        assert torch.equal(r.ids, want.ids) and torch.equal(r.weights, want.weights)
        assert torch.equal(r.loss, want.loss) and torch.equal(r.counts, want.counts)
    leaf = logits.detach().requires_grad_()
    r = routing.route(leaf, 8, renormalize=False)
    r.weights.sum().backward()  # an expanded gradient
    want1, _ = torch.autograd.grad(
        routing.route(leaf, 8, renormalize=False).weights, leaf,
        torch.ones((5000, 8), device=DEV)), None
    assert torch.equal(leaf.grad, want1[0])
    leaf.grad = None
    (routing.route(leaf, 8, balance=True).loss + routing.route(leaf, 8, balance=True).loss).backward()
    one = torch.autograd.grad(routing.route(leaf, 8, balance=True).loss, leaf)[0]
    assert torch.equal(leaf.grad, one + one)
    ids = torch.zeros((5000, 2), dtype=torch.int32, device=DEV)
    for value in (routing.route(leaf, 8).weights.sum(), routing.balance_loss(leaf, ids)[0]):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(value, leaf, create_graph=True)


def test_refusals_on_the_device():
    from vllm_expert_pager import routing

    logits, _ = make(4, 16, torch.float32)
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        routing.route(logits, 2, valid=torch.ones((4,), dtype=torch.bool))
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        routing.balance_loss(logits, torch.zeros((4, 2), dtype=torch.int32))


@pytest.mark.parametrize("T, E", [(1 << 26, 5), (1 << 25, 50), (1 << 24, 200), (1 << 23, 300),
                                  (1 << 22, 800), (1 << 21, 1100), (1 << 20, 4096)])
def test_mean_probabilities_of_long_batches(T, E):
    """P adds up 2^26 tokens as exactly as a few: one row for all tokens, so that every
    addition rounds the same way.  32 tokens are summed in 32 bits, those sums in 64."""
    from vllm_expert_pager import routing

    row, _ = make(1, E, torch.float32, seed=E)
    logits = row.expand(T, E)
    p, x = softmax64(row.double(), torch.ones((1,), dtype=torch.bool, device=DEV))
    rel = (float(steps(x.abs().max(), E)) + 40) * STEP
    if E <= 200:
        top = int(row.argmax())
        r = routing.route(logits, 1, balance=True)
        assert int(r.counts[top]) == T and int(r.counts.sum()) == T
        want = E * float(p[0, top])
        assert abs(float(r.loss) - want) <= rel * want
        del r
    ids = torch.full((T, 1), E // 2, dtype=torch.int32, device=DEV)
    loss, counts = routing.balance_loss(logits, ids)
    assert int(counts[E // 2]) == T
    want = E * float(p[0, E // 2])
    assert abs(float(loss) - want) <= rel * want


@pytest.mark.parametrize("E", [50, 256, 1100])
def test_rows_without_an_open_expert_in_a_long_batch(E):
    """Rows that add nothing to P, and rows that hold no token, wherever a warp's sum moves on
    to 64 bits."""
    T = 200000
    logits, g = make(T, E, torch.bfloat16, seed=E)
    logits[torch.rand((T,), generator=g, device=DEV) < 0.3] = -math.inf
    valid = torch.rand((T,), generator=g, device=DEV) < 0.7
    for v in (None, valid):
        check_route(logits, 3, False, valid=v)


@pytest.mark.parametrize("E", [7, 200, 1030])
def test_gradient_where_neighbouring_tokens_choose_the_same_experts(E):
    """Each token's choices, in another order than those of the tokens that its warp has
    before and after it: other lanes set the same places."""
    T, K = 40000, min(E, 32)
    g = torch.Generator(device=DEV).manual_seed(E)
    logits = torch.randn((T, E), generator=g, device=DEV) * 0.01
    logits[:, :K] += 4.0
    for renormalize in (True, False):
        check_route(logits, K, renormalize)
