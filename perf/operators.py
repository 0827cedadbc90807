"""Workloads of the token-side operators of a paged mixture-of-experts layer.

Three operators, each as a user's program calls it and in a plain form:

* ``route``: router logits to the top-k experts of every token, their weights and the
  number of tokens per expert; in training also the balance loss and the gradient of
  the logits.
* ``balance``: the balance loss and the per-expert counts of a routing chosen elsewhere,
  with the gradient of the logits.
* ``adapters``: the low-rank updates of many requests' adapters added to the output of
  a projection that all requests share.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "vllm-expert-pager_b200")
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases ----

def _route(name, tokens, experts, topk, dtype, *, renormalize=True, train=False, balance=False,
           closed=0, padded=0.0):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "topk": topk,
            "dtype": dtype, "renormalize": renormalize, "train": train, "balance": balance,
            "closed": closed, "padded": padded}


def _balance(name, tokens, experts, topk, dtype, *, padded=0.0):
    return {"name": name, "op": "balance", "tokens": tokens, "experts": experts, "topk": topk,
            "dtype": dtype, "padded": padded}


def _adapters(name, rows, requests, active, slots, rank, inputs, outputs, dtype):
    return {"name": name, "op": "adapters", "rows": rows, "requests": requests,
            "active": active, "slots": slots, "rank": rank, "inputs": inputs,
            "outputs": outputs, "dtype": dtype}


def listed():
    return [
        # One token of a batch-1 decode: 256 experts, 8 per token.
        _route("route token", 1, 256, 8, "fp32"),
        # A 2048-token prompt of the same model.
        _route("route prompt", 2048, 256, 8, "bf16"),
        # Fine-tuning without a balance term: few experts, some of them closed to routing,
        # weights left as probabilities, padded rows.
        _route("route tune odd", 5003, 60, 4, "fp16", renormalize=False, train=True, closed=7,
               padded=0.1),
        # A training step of the router with its balance loss.
        _route("route train", 16384, 256, 8, "bf16", train=True, balance=True),
        # The loss of a short batch whose routing an engine's own router chose.
        _balance("balance short", 509, 256, 8, "bf16", padded=0.2),
        # A packed training batch, many experts, logits in 32 bits.
        _balance("balance large", 65536, 512, 8, "fp32", padded=0.03),
        # One request's token beside the expert layer's up projection (2048 -> 1024).
        _adapters("adapter token", 1, 1, 1, 8, 16, 2048, 1024, "bf16"),
        # A decode batch, 32 adapters in 32 slots, square projection.
        _adapters("adapter decode", 64, 64, 32, 32, 16, 2048, 2048, "bf16"),
        # A wide decode batch with large ranks.
        _adapters("adapter decode wide", 256, 256, 100, 128, 64, 2048, 1024, "fp16"),
        # A few prompts together, small ranks, beside the down projection (512 -> 2048).
        _adapters("adapter prompts", 2048, 5, 4, 8, 16, 512, 2048, "bf16"),
        # Ragged prompts and sizes that no vector width divides.
        _adapters("adapter odd", 4099, 23, 11, 16, 13, 1021, 2047, "fp16"),
        # A long prefill batch of several adapters.
        _adapters("adapter prefill", 16384, 12, 6, 8, 64, 2048, 2048, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(("route", "balance", "adapters"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if op == "route":
        experts = _log(rng, 8, 1024)
        case = _route("", _log(rng, 1, 16384), experts, rng.randint(1, min(16, experts // 2)),
                      dtype, renormalize=rng.random() < 0.5, train=rng.random() < 0.6,
                      closed=rng.choice((0, 0, rng.randint(0, experts // 4))),
                      padded=rng.choice((0.0, 0.0, round(rng.uniform(0.01, 0.5), 3))))
        case["balance"] = case["train"] and rng.random() < 0.5
    elif op == "balance":
        experts = _log(rng, 8, 1024)
        tokens = min(_log(rng, 1, 65536), (1 << 25) // experts)
        case = _balance("", tokens, experts, rng.randint(1, min(16, experts // 2)), dtype,
                        padded=rng.choice((0.0, round(rng.uniform(0.01, 0.5), 3))))
    else:
        rows = _log(rng, 1, 16384)
        slots = _log(rng, 1, 64 if rows <= 1024 else 16)
        requests = _log(rng, 1, min(rows, 256))
        inputs, outputs = _log(rng, 64, 4096), _log(rng, 64, 4096)
        rank = _log(rng, 1, 128)
        if rng.random() < 0.7:
            inputs, outputs = inputs // 8 * 8, outputs // 8 * 8
            rank = max(8, rank // 8 * 8)
        while rows * (inputs + 2 * outputs) > 16384 * 6144 or rows * rank > 16384 * 64:
            rows = rows // 2
        case = _adapters("", max(rows, 1), min(requests, max(rows, 1)), 0, slots, rank, inputs,
                         outputs, rng.choice(("bf16", "fp16")))
        case["active"] = min(slots, case["requests"], _log(rng, 1, slots))
    case.pop("name")
    return case


# ---- inputs ----

def _logits(case, gen):
    """Router logits whose expert popularity follows a Zipf law, as decode traces do."""
    T, E = case["tokens"], case["experts"]
    rank = torch.randperm(E, generator=gen, device="cuda").float()
    x = torch.randn((T, E), generator=gen, device="cuda") * 1.5 - 0.5 * torch.log1p(rank)
    return x.to(_TYPES[case["dtype"]])


def _valid(case, gen):
    """Rows of the batch that hold a token (padding is false); None where nothing is padded."""
    if not case["padded"]:
        return None
    return torch.rand((case["tokens"],), generator=gen, device="cuda") >= case["padded"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "adapters":
        return _prepare_adapters(case, gen)
    T, E, K = case["tokens"], case["experts"], case["topk"]
    state = dict(case, logits=_logits(case, gen), valid=_valid(case, gen))
    # Upstream gradients: of the weights, and of the loss (a loss scale, as training in
    # 16 bits uses one).
    state["grad_weights"] = torch.randn((T, K), generator=gen, device="cuda")
    state["grad_loss"] = torch.rand((), generator=gen, device="cuda") * 512.0 + 512.0
    if case["op"] == "route":
        if case["closed"]:
            closed = torch.randperm(E, generator=gen, device="cuda")[: case["closed"]]
            state["logits"][:, closed] = -math.inf
    else:
        # A routing with some noise, as an engine's own router would choose it.
        noisy = state["logits"].float() + torch.randn((T, E), generator=gen, device="cuda")
        state["ids"] = noisy.topk(K).indices.to(torch.int32)
    return state


def _prepare_adapters(case, gen):
    """Requests' rows lie together, in the order of the requests; every eighth request has no
    adapter.  One request per row is a decode batch."""
    M, R, S = case["rows"], case["requests"], case["slots"]
    r, H, N, t = case["rank"], case["inputs"], case["outputs"], _TYPES[case["dtype"]]
    new = dict(generator=gen, device="cuda")
    slots = torch.randperm(S, **new)[: case["active"]]
    request = slots[torch.randperm(R, **new) % case["active"]]
    request[7::8] = -1
    if R < M:
        start = torch.randperm(M - 1, **new)[: R - 1].sort().values + 1
        first = torch.zeros((M,), dtype=torch.int64, device="cuda")
        first[start] = 1
        ids = request[first.cumsum(0)]
    else:
        ids = request
    x = torch.randn((M, H), **new)
    return dict(case, ids=ids.to(torch.int32), x=x.to(t),
                y=torch.randn((M, N), **new).to(t),
                a=(torch.randn((S, r, H), **new) / math.sqrt(H)).to(t),
                b=(torch.randn((S, N, r), **new) / math.sqrt(r)).to(t),
                scale=torch.rand((S,), **new) + 0.5,
                out=torch.empty((M, N), dtype=t, device="cuda"))


# ---- one pass ----

def run(state):
    if own:
        return {"route": _own_route, "balance": _own_balance, "adapters": _own_adapters}[
            state["op"]](state)
    return {"route": _plain_route, "balance": _plain_balance, "adapters": _plain_adapters}[
        state["op"]](state)


def _modules():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from vllm_expert_pager import adapters, routing

    return routing, adapters


def _own_route(state):
    routing, _ = _modules()
    logits = state["logits"].detach()
    if state["train"]:
        logits.requires_grad_()
    r = routing.route(logits, state["topk"], renormalize=state["renormalize"],
                      valid=state["valid"], balance=state["balance"])
    out = {"weights": r.weights.detach(), "ids": r.ids, "counts": r.counts}
    if state["balance"]:
        out["loss"] = r.loss.detach()
        out["grad"], = torch.autograd.grad(
            (r.weights, r.loss), logits, (state["grad_weights"], state["grad_loss"]))
    elif state["train"]:
        out["grad"], = torch.autograd.grad(r.weights, logits, state["grad_weights"])
    return out


def _own_balance(state):
    routing, _ = _modules()
    logits = state["logits"].detach().requires_grad_()
    loss, counts = routing.balance_loss(logits, state["ids"], valid=state["valid"])
    grad, = torch.autograd.grad(loss, logits, state["grad_loss"])
    return {"loss": loss.detach(), "counts": counts, "grad": grad}


def _own_adapters(state):
    _, adapters = _modules()
    return adapters.add_low_rank(state["y"], state["x"], state["a"], state["b"], state["ids"],
                                 scale=state["scale"], out=state["out"])


# ---- plain forms ----

def _softmax(z, valid):
    """Row softmax of 32-bit logits; rows without a token or a finite logit are zero."""
    top = z.amax(1, keepdim=True)
    live = top > -math.inf
    if valid is not None:
        live = live & valid[:, None]
    e = torch.where(live, torch.exp(z - torch.where(live, top, 0.0)), 0.0)
    return e / torch.where(live, e.sum(1, keepdim=True), 1.0)


def _counts(ids, valid, experts):
    use = ids >= 0
    if valid is not None:
        use = use & valid[:, None]
    at = torch.where(use, ids, experts).long().reshape(-1)
    one = torch.ones_like(at)
    return torch.zeros((experts + 1,), dtype=torch.int64, device=ids.device).scatter_add_(
        0, at, one)[:experts]


def _balance_terms(p, counts, valid, topk):
    """The loss, and its derivative by every probability."""
    T, E = p.shape
    n = torch.full((), T, device=p.device) if valid is None else valid.sum()
    n = n.clamp(min=1).to(torch.float32)
    share = counts.to(torch.float32) / (n * topk)
    mean = (p.sum(0, dtype=torch.float64) / n).to(torch.float32)
    return E * (share * mean).sum(), E * share / n


def _plain_route(state):
    z, K, valid = state["logits"].float(), state["topk"], state["valid"]
    T, E = z.shape
    order = torch.sort(z, dim=1, descending=True, stable=True)
    open_ = order.values[:, :K] > -math.inf
    if valid is not None:
        open_ = open_ & valid[:, None]
    picked = order.indices[:, :K]
    p = _softmax(z, valid)
    w = torch.where(open_, p.gather(1, picked), 0.0)
    total = w.sum(1, keepdim=True)
    if state["renormalize"]:
        w = w / torch.where(total > 0, total, 1.0)
    ids = torch.where(open_, picked, -1).to(torch.int32)
    counts = _counts(ids, valid, E)
    out = {"weights": w, "ids": ids, "counts": counts}
    if not state["train"]:
        return out
    g = torch.where(open_, state["grad_weights"], 0.0)
    if state["renormalize"]:
        inner = w * (g - (w * g).sum(1, keepdim=True))
        grad = torch.zeros_like(z).scatter_add_(1, picked, inner)
        by_p = torch.zeros_like(z)
    else:
        grad = torch.zeros_like(z)
        by_p = torch.zeros_like(z).scatter_add_(1, picked, g)
    if state["balance"]:
        out["loss"], slope = _balance_terms(p, counts, valid, K)
        by_p = by_p + state["grad_loss"] * slope
    grad = grad + p * (by_p - (p * by_p).sum(1, keepdim=True))
    out["grad"] = grad.to(state["logits"].dtype)
    return out


def _plain_balance(state):
    z, valid = state["logits"].float(), state["valid"]
    p = _softmax(z, valid)
    counts = _counts(state["ids"], valid, z.shape[1])
    loss, slope = _balance_terms(p, counts, valid, state["topk"])
    by_p = state["grad_loss"] * slope
    grad = p * (by_p - (p * by_p).sum(1, keepdim=True))
    return {"loss": loss, "counts": counts, "grad": grad.to(state["logits"].dtype)}


def _plain_adapters(state):
    """All slots at once: every row against every adapter, the other adapters' products
    replaced by zeros."""
    x, a, b, ids = state["x"].float(), state["a"].float(), state["b"].float(), state["ids"]
    S, r, H = a.shape
    mine = ids[:, None] == torch.arange(S, device=ids.device, dtype=ids.dtype)
    v = (x @ a.reshape(S * r, H).t()).view(-1, S, r)
    v = torch.where(mine[:, :, None], v * state["scale"][:, None], 0.0).reshape(-1, S * r)
    update = v @ b.permute(0, 2, 1).reshape(S * r, -1)
    return (state["y"].float() + update).to(state["y"].dtype)


# ---- what a pass cannot do without ----

def work(case):
    size = torch.empty((), dtype=_TYPES[case["dtype"]]).element_size()
    if case["op"] == "adapters":
        M, r, H, N = case["rows"], case["rank"], case["inputs"], case["outputs"]
        with_adapter = M * (1 - case["requests"] // 8 / case["requests"])
        return {"bytes": M * (H + 2 * N) * size + case["active"] * r * (H + N) * size + 4 * M,
                "flops": 2 * with_adapter * r * (H + N)}
    T, E, K = case["tokens"], case["experts"], case["topk"]
    read = T * E * size + (T if case["padded"] else 0)
    if case["op"] == "route":
        b = read + T * K * 8 + E * 8
        if case["train"]:
            b += T * E * size + T * K * 4
        # A comparison of each logit; where all probabilities are needed, an exponential
        # and a product, in training the gradient's two products too.
        f = T * E * (6 if case["train"] else 3)
    else:
        b, f = read + T * K * 4 + E * 8 + T * E * size, T * E * 6
    return {"bytes": b, "flops": f}


# ---- the definition in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adapters":
        out = s["y"].double()
        for slot in range(case["slots"]):
            mine = (s["ids"] == slot).nonzero().reshape(-1)
            if mine.numel():
                low = s["x"][mine].double() @ s["a"][slot].double().T
                out[mine] += s["scale"][slot].double() * (low @ s["b"][slot].double().T)
        return out
    z = s["logits"].double()
    T, E = z.shape
    K = case["topk"]
    live = torch.isfinite(z).any(1)
    if s["valid"] is not None:
        live &= s["valid"]
    n = T if s["valid"] is None else int(s["valid"].sum())
    p = torch.zeros_like(z)
    p[live] = torch.softmax(z[live], 1)
    by_p, grad = torch.zeros_like(z), torch.zeros_like(z)
    out = {}
    if case["op"] == "route":
        value, index = torch.sort(z, dim=1, descending=True, stable=True)
        value, index = value[:, :K], index[:, :K].clone()
        index[~(torch.isfinite(value) & live[:, None])] = -1
        row, col = (index >= 0).nonzero(as_tuple=True)
        expert = index[row, col]
        w = torch.zeros((T, K), dtype=torch.float64, device=z.device)
        w[row, col] = p[row, expert]
        if case["renormalize"]:
            w[live] /= w[live].sum(1, keepdim=True)
        out["weights"], out["ids"] = w, index.to(torch.int32)
        g = torch.zeros_like(w)
        g[row, col] = s["grad_weights"].double()[row, col]
        if case["renormalize"]:
            grad[row, expert] = (w * (g - (w * g).sum(1, keepdim=True)))[row, col]
        else:
            by_p[row, expert] = g[row, col]
    else:
        expert = s["ids"].long()[live].reshape(-1) if s["valid"] is None else \
            s["ids"].long()[s["valid"]].reshape(-1)
    counts = torch.bincount(expert, minlength=E)
    out["counts"] = counts
    if case["op"] == "balance" or case["balance"]:
        share = counts.double() / (max(n, 1) * K)
        out["loss"] = E * (share * p.sum(0) / max(n, 1)).sum()
        by_p += s["grad_loss"].double() * E * share / max(n, 1)
    if case["op"] == "balance" or case["train"]:
        out["grad"] = grad + p * (by_p - (p * by_p).sum(1, keepdim=True))
    return out
