"""Timed cases of the operators around the experts' products: routing, its balance loss, 4-bit weights.

Four kinds of case, each with a plain form in elementary torch operations (float32 throughout) and the
call that a user makes of the library:

  route    moe_route(logits, top_k): the choice of experts, its weights, the counts and the order of the
           slots by expert that the grouped product takes; no gradient
  balance  the same with the balance loss, and the gradient of weights and loss with respect to the logits
  w4       w4_matmul(x, q, scales, zeros): a few rows times one matrix of 4-bit weights
  moe_w4   moe_w4_matmul(x, q, scales, counts, order, zeros): the same for expert matrices, rows by expert

A case is a dict of plain values; inputs come from the seed given to prepare().  4-bit weights are bytes
of two values along k (low half: even k), value (q - zero) * scale with one scale (and zero) per matrix
row and group of k; without zeros the zero is 8.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False  # set from outside: False computes the plain forms, True calls the library

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BALANCE_FACTOR = 0.01  # the balance loss's share of a training loss


def _route(name, kind, tokens, experts, top_k, dtype, normalize=True, padded=False, groups=False):
    return {"name": name, "kind": kind, "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "normalize": normalize, "padded": padded, "groups": groups}


def _w4(name, rows, k, n, group, zeros=False):
    return {"name": name, "kind": "w4", "rows": rows, "k": k, "n": n, "group": group, "zeros": zeros}


def _moe_w4(name, experts, tokens, top_k, k, n, group, zeros=False):
    return {"name": name, "kind": "moe_w4", "experts": experts, "tokens": tokens, "top_k": top_k, "k": k, "n": n,
            "group": group, "zeros": zeros}


def listed():
    return [
        # One token of one sequence being served: bound by the launch.
        _route("route_token", "route", 1, 64, 2, "float16"),
        # A ragged batch of served tokens, some rows padding, weights of the whole softmax.
        _route("route_batch", "route", 173, 48, 6, "bfloat16", normalize=False, padded=True),
        # The prefill of a 64-expert layer: 16384 tokens.
        _route("route_prefill", "route", 16384, 64, 2, "float32"),
        # A training step of a small expert layer: 512 tokens over 16 experts.
        _route("balance_small", "balance", 512, 16, 2, "float32"),
        # A training step of the 64-expert layer, padded batch, mixed precision logits.
        _route("balance_train", "balance", 16384, 64, 4, "bfloat16", padded=True),
        # The largest router: many fine experts, half of the expert groups closed to each token, odd token count.
        _route("balance_wide", "balance", 65521, 256, 8, "float32", normalize=False, groups=True),
        # One token through a square layer: bound by the launch.
        _w4("w4_token", 1, 2048, 2048, 128),
        # One token through the expert-sized layer: bound by the weights' bytes.
        _w4("w4_decode", 1, 4096, 14336, 128),
        # A served batch of odd size, small groups with zero points, odd n.
        _w4("w4_batch", 13, 4096, 14335, 32, zeros=True),
        # A larger batch: each weight is used 64 times.
        _w4("w4_rows", 64, 8192, 8192, 64),
        # The small expert layer of 16 experts, 512 tokens with one expert each.
        _moe_w4("moe_w4_small", 16, 512, 1, 1024, 2048, 128),
        # The 64-expert layer in decode: 256 rows (128 tokens, two experts each), nearly every expert is read.
        _moe_w4("moe_w4_decode", 64, 128, 2, 4096, 14336, 128, zeros=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("route", "balance", "w4", "moe_w4"))
    if kind in ("route", "balance"):
        experts = _log_int(rng, 4, 512)
        tokens = _log_int(rng, 1 if kind == "route" else 64, min(65536, 65521 * 256 // experts))
        top_k = rng.randint(1, min(16, experts // 2))
        case = _route("", kind, tokens, experts, top_k, rng.choice(("float32", "float16", "bfloat16")),
                      top_k > 1 and rng.random() < 0.6, tokens > 16 and rng.random() < 0.4, rng.random() < 0.3)
    elif kind == "w4":
        group = rng.choice((32, 64, 128))
        k = group * _log_int(rng, 512 // group, 8192 // group)
        case = _w4("", _log_int(rng, 1, 64), k, min(_log_int(rng, 500, 14336), 8192 * 8192 // k), group,
                   rng.random() < 0.5)
    else:
        group = rng.choice((32, 64, 128))
        experts = _log_int(rng, 4, 128)
        k = group * _log_int(rng, 512 // group, 4096 // group)
        n = min(_log_int(rng, 500, 14336), 64 * 4096 * 14336 // (experts * k))
        top_k = rng.randint(1, min(4, experts))
        case = _moe_w4("", experts, _log_int(rng, 1, 256 // top_k), top_k, k, n, group, rng.random() < 0.5)
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs

def _popularity(experts):
    """Log of a Zipf(1.2) share of tokens per expert, as the library's expert workload has."""
    return -1.2 * np.log(np.arange(1, experts + 1))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _draw_experts(tokens, experts, top_k, gen):
    """top_k distinct experts per token, popular ones more often; int64 [tokens, top_k]."""
    shift = torch.from_numpy(_popularity(experts)).float().cuda()
    shift = shift[torch.randperm(experts, generator=gen, device="cuda")]
    noise = torch.rand(tokens, experts, generator=gen, device="cuda").clamp_(1e-7, 1 - 1e-7)
    return (shift - torch.log(-torch.log(noise))).topk(top_k, dim=1).indices


def _weights(lead, n, k, group, zeros, gen):
    q = torch.randint(0, 256, (*lead, n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(*lead, n, k // group, generator=gen, device="cuda") * 0.004 + 0.001).half()
    z = None
    if zeros:
        z = torch.randint(4, 12, (*lead, n, k // group), generator=gen, device="cuda", dtype=torch.uint8)
    return {"q": q, "scales": scales, "zeros": z}


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": case}
    if case["kind"] in ("route", "balance"):
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        shift = torch.from_numpy(_popularity(experts)).float().cuda()
        logits = torch.randn(tokens, experts, generator=gen, device="cuda") * 1.5 + 0.5 * shift
        if case["groups"]:  # eight groups of experts (fewer with few experts), half of them closed to each token
            groups = min(8, max(1, experts // max(1, 2 * top_k)) * 2)
            open_ = torch.rand(tokens, groups, generator=gen, device="cuda").argsort(dim=1) < (groups + 1) // 2
            of_expert = torch.arange(experts, device="cuda") * groups // experts
            logits = logits.masked_fill(~open_[:, of_expert], -math.inf)
        state["logits"] = logits.to(TYPES[case["dtype"]])
        state["mask"] = None
        if case["padded"]:
            state["mask"] = torch.rand(tokens, generator=gen, device="cuda") < 0.9
        if case["kind"] == "balance":
            state["logits"].requires_grad_(True)
            state["d_weights"] = torch.randn(tokens, top_k, generator=gen, device="cuda") * 0.01
            state["d_loss"] = torch.full((), BALANCE_FACTOR, device="cuda")
    elif case["kind"] == "w4":
        state["x"] = torch.randn(case["rows"], case["k"], generator=gen, device="cuda").half()
        state.update(_weights((), case["n"], case["k"], case["group"], case["zeros"], gen))
    else:
        tokens, experts = case["tokens"], case["experts"]
        ids = _draw_experts(tokens, experts, case["top_k"], gen).flatten()
        state["x"] = torch.randn(tokens, case["k"], generator=gen, device="cuda").half()
        state["counts"] = torch.zeros(experts, dtype=torch.int32, device="cuda")
        state["counts"].index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
        state["order"] = ids.sort(stable=True).indices.int()
        state.update(_weights((experts,), case["n"], case["k"], case["group"], case["zeros"], gen))
    return state


# ---------------------------------------------------------------- plain forms

def _plain_choice(logits, mask, top_k):
    """float32 logits with padded rows closed, ids and their logits (-inf where there is no expert)."""
    z = logits.detach().float()
    if mask is not None:
        z = z.masked_fill(~mask[:, None], -math.inf)
    value, index = z.sort(dim=1, descending=True, stable=True)
    value, index = value[:, :top_k], index[:, :top_k]
    return z, value, index


def _plain_route(state):
    case = state["case"]
    z, value, index = _plain_choice(state["logits"], state["mask"], case["top_k"])
    experts = case["experts"]
    routed = value[:, :1] > -math.inf
    top = torch.where(routed, value[:, :1], 0.0)
    e = torch.exp(value - top)
    p = None
    if not case["normalize"] or case["kind"] == "balance":
        p = torch.exp(z - top)
        total = p.sum(1, keepdim=True)
        p = p / torch.where(routed, total, 1.0)
    if case["normalize"]:
        weights = e / torch.where(routed, e.sum(1, keepdim=True), 1.0)
    else:
        weights = e / torch.where(routed, total, 1.0)
    chosen = value > -math.inf
    ids = torch.where(chosen, index, -1).int()
    slot = torch.where(chosen, index, experts).flatten()
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=z.device)
    counts.index_add_(0, slot, torch.ones_like(slot, dtype=torch.int32))
    order = slot.sort(stable=True).indices.int()
    return weights, ids, counts[:experts], order, p, index, routed


def _plain_balance(state):
    case = state["case"]
    weights, ids, counts, order, p, index, routed = _plain_route(state)
    experts = case["experts"]
    tokens = routed.sum().clamp(min=1).float()
    share = counts.float() / counts.sum().clamp(min=1).float()
    loss = experts * (share * (p.sum(0) / tokens)).sum()
    c = (state["d_loss"] * experts / tokens) * share
    d = p * (c - (p * c).sum(1, keepdim=True))
    part = weights * state["d_weights"]
    if case["normalize"]:
        part = part - weights * part.sum(1, keepdim=True)
    else:
        d = d - p * part.sum(1, keepdim=True)
    d.scatter_add_(1, index, part)
    return weights, ids, counts, order, loss, d.to(state["logits"].dtype)


def _plain_values(state, group):
    """The weights in float32, [..., n, k]."""
    q = state["q"]
    w = torch.stack((q & 15, q >> 4), dim=-1).float()
    grouped = w.view(*q.shape[:-1], -1, group)
    grouped.sub_(8.0 if state["zeros"] is None else state["zeros"].float().unsqueeze(-1))
    grouped.mul_(state["scales"].float().unsqueeze(-1))
    return w.view(*q.shape[:-1], 2 * q.shape[-1])


def _plain_w4(state):
    return state["x"].float() @ _plain_values(state, state["case"]["group"]).t()


def _plain_moe_w4(state):
    """Each expert's rows in a batch of equal height (an expert has at most one row of each token), one product."""
    case = state["case"]
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    order, ends = state["order"].long(), state["counts"].long().cumsum(0)
    row = torch.arange(tokens * top_k, device=order.device)
    expert = torch.searchsorted(ends, row, right=True)
    place = row - (ends - state["counts"])[expert]
    x = torch.zeros(experts, case["k"], tokens, device=order.device)
    x[expert, :, place] = state["x"].float()[order // top_k]
    y = torch.bmm(_plain_values(state, case["group"]), x)
    out = torch.empty(tokens * top_k, case["n"], device=order.device)
    out[order] = y[expert, :, place]
    return out


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from grouped_gemm_gpu_kernel_amd import torch_ops

        if kind in ("route", "balance"):
            r = torch_ops.moe_route(state["logits"], case["top_k"], token_mask=state["mask"],
                                    normalize=case["normalize"], balance=kind == "balance")
            if kind == "route":
                return r.weights, r.ids, r.counts, r.order
            d_logits, = torch.autograd.grad((r.weights, r.balance_loss), (state["logits"],),
                                            (state["d_weights"], state["d_loss"]))
            return r.weights.detach(), r.ids, r.counts, r.order, r.balance_loss.detach(), d_logits
        if kind == "w4":
            return torch_ops.w4_matmul(state["x"], state["q"], state["scales"], state["zeros"])
        return torch_ops.moe_w4_matmul(state["x"], state["q"], state["scales"], state["counts"], state["order"],
                                       state["zeros"])
    if kind == "route":
        return _plain_route(state)[:4]
    if kind == "balance":
        return _plain_balance(state)
    return _plain_w4(state) if kind == "w4" else _plain_moe_w4(state)


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_route(state):
    case = state["case"]
    experts, top_k = case["experts"], case["top_k"]
    z = state["logits"].detach().double().cpu().numpy()
    live = np.ones(len(z), bool) if state["mask"] is None else state["mask"].cpu().numpy()
    chosen = np.argsort(-z, axis=1, kind="stable")[:, :top_k]
    ids = np.where(live[:, None], chosen, -1)
    flat = np.where(ids < 0, experts, ids).reshape(-1)
    counts = np.bincount(flat, minlength=experts + 1)[:experts]
    order = np.argsort(flat, kind="stable")
    leaf = torch.from_numpy(z).cuda().requires_grad_(True)
    rows = torch.from_numpy(np.flatnonzero(live)).cuda()
    picked = torch.from_numpy(chosen).cuda()[rows]
    mine = leaf[rows]
    p = torch.softmax(mine, dim=1)
    w = torch.gather(p, 1, picked)
    if case["normalize"]:
        w = torch.softmax(torch.gather(mine, 1, picked), dim=1)
    weights = torch.zeros(len(z), top_k, dtype=torch.float64, device="cuda").index_copy(0, rows, w)
    out = [weights.detach(), torch.from_numpy(ids).int(), torch.from_numpy(counts).int(), torch.from_numpy(order).int()]
    if case["kind"] == "balance":
        share = torch.from_numpy(counts / max(1, counts.sum())).cuda()
        loss = experts * (share * p.sum(0) / max(1, len(rows))).sum()
        total = (weights * state["d_weights"].double()).sum() + state["d_loss"].double() * loss
        out += [loss.detach(), torch.autograd.grad(total, leaf)[0]]
    return tuple(out)


def _exact_values(q, scales, zeros, group):
    n, half = q.shape
    w = torch.empty(n, 2 * half, dtype=torch.float64, device=q.device)
    w[:, 0::2] = (q % 16).double()
    w[:, 1::2] = torch.div(q, 16, rounding_mode="floor").double()
    zero = torch.full_like(scales, 8.0).double() if zeros is None else zeros.double()
    return (w - zero.repeat_interleave(group, 1)) * scales.double().repeat_interleave(group, 1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("route", "balance"):
        return _exact_route(state)
    if case["kind"] == "w4":
        return state["x"].double() @ _exact_values(state["q"], state["scales"], state["zeros"], case["group"]).t()
    order = state["order"].long()
    y = torch.empty(len(order), case["n"], dtype=torch.float64, device=order.device)
    start = 0
    for e, count in enumerate(state["counts"].tolist()):
        if count:
            rows = order[start:start + count]
            zeros = None if state["zeros"] is None else state["zeros"][e]
            y[rows] = state["x"][rows // case["top_k"]].double() @ _exact_values(
                state["q"][e], state["scales"][e], zeros, case["group"]).t()
            start += count
    return y


# ---------------------------------------------------------------- work

def work(case):
    if case["kind"] in ("route", "balance"):
        tokens, experts, slots = case["tokens"], case["experts"], case["tokens"] * case["top_k"]
        logits = tokens * experts * (4 if case["dtype"] == "float32" else 2)
        moved = logits + slots * (4 + 4 + 4) + experts * 4 + (tokens if case["padded"] else 0)
        flops = 4 * tokens * experts
        if case["kind"] == "balance":  # the logits again, their gradient, the weights' gradient and the ids
            moved += 2 * logits + slots * (4 + 4) + 4
            flops += 12 * tokens * experts
        return {"bytes": moved, "flops": flops}
    k, n, groups = case["k"], case["n"], case["k"] // case["group"]
    matrix = n * k // 2 + n * groups * (3 if case["zeros"] else 2)
    if case["kind"] == "w4":
        return {"bytes": matrix + case["rows"] * (2 * k + 4 * n), "flops": 2 * case["rows"] * k * n}
    rows = case["tokens"] * case["top_k"]
    share = np.exp(_popularity(case["experts"]))
    read = float((1.0 - (1.0 - share / share.sum()) ** rows).sum())  # experts with a row, expected
    return {"bytes": read * matrix + case["tokens"] * 2 * k + rows * (4 * n + 4) + 4 * case["experts"],
            "flops": 2 * rows * k * n}
