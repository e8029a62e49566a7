"""Timed cases of the 8-bit path of a feed-forward layer: the norm that writes 8-bit rows, and the products that read them.

Values are float8_e4m3fn with float32 scales: one for each 128 values of a row of activations (ceil(K / 128) a row), one
for each block of 128 x 128 of a weight matrix; the last block of a row or column may be cut.  Four kinds of case, each
with a plain form in elementary torch operations (float32 throughout) and the call that a user makes of the library:

  norm     rms_norm_fp8(x, weight, residual): x + residual, its root-mean-square norm as 8-bit rows (and in x's type)
  matmul   fp8_matmul(x, x_scales, w, w_scales): rows times one matrix
  gated    fp8_gated(x, x_scales, gate, gate_scales, up, up_scales): silu(x gate^T) * (x up^T) as 8-bit rows
  moe      moe_fp8_matmul and moe_fp8_gated (gated=True): the same for expert matrices, rows by expert

A case is a dict of plain values; inputs come from the seed given to prepare().  Quantised rows come back as the 8-bit
numbers and their scales, both whole.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False  # set from outside: False computes the plain forms, True calls the library

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
FP8 = torch.float8_e4m3fn
BLOCK = 128
LARGEST = 448.0  # of float8_e4m3fn
SMALLEST_SCALE = 2.0 ** -126
EPS = 1e-6


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _norm(name, tokens, hidden, dtype, residual=True, plain=False):
    return {"name": name, "kind": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "residual": residual,
            "plain": plain}


def _dense(name, rows, k, n, gated=False, dtype="bfloat16"):
    return {"name": name, "kind": "gated" if gated else "matmul", "rows": rows, "k": k, "n": n, "dtype": dtype}


def _moe(name, experts, tokens, top_k, k, n, gated=False, dtype="bfloat16", padded=False):
    return {"name": name, "kind": "moe", "gated": gated, "experts": experts, "tokens": tokens, "top_k": top_k, "k": k,
            "n": n, "dtype": dtype, "padded": padded}


def listed():
    return [
        # One token of one sequence being served: bound by the launch.
        _norm("norm_token", 1, 4096, "bfloat16"),
        # A served batch of odd size without a residual, the router's 16-bit rows beside the experts' 8-bit ones.
        _norm("norm_batch", 173, 8192, "float16", residual=False, plain=True),
        # The prefill of 16384 tokens: bound by the bytes of x and the residual.
        _norm("norm_prefill", 16384, 8192, "bfloat16", plain=True),
        # One token through the expert-sized layer: bound by the weights' bytes.
        _dense("matmul_token", 1, 4096, 14336),
        # A served batch of odd size and an odd number of columns, as float32 rows.
        _dense("matmul_batch", 61, 4096, 14335, dtype="float32"),
        # A short prompt: too many rows for the weights' bytes to count alone, too few to fill the card's tiles.
        _dense("matmul_prompt", 777, 8192, 8192, dtype="float16"),
        # The largest square problem: bound by the matrix instructions.
        _dense("matmul_square", 8192, 8192, 8192),
        # One token through both projections of the expert-sized layer.
        _dense("gated_token", 1, 4096, 14336, gated=True),
        # The small expert layer of 16 experts, 512 tokens with one expert each, some of them padding.
        _moe("gated_moe_small", 16, 512, 1, 1024, 2048, gated=True, padded=True),
        # The prefill of an expert layer's projections: 4096 tokens, two of 32 experts each.
        _moe("gated_moe_prefill", 32, 4096, 2, 4096, 14336, gated=True),
        # The 64-expert layer in decode: 256 rows (128 tokens, two experts each), nearly every expert is read.
        _moe("moe_decode", 64, 128, 2, 4096, 14336),
        # The 64-expert layer's prefill: 16384 rows, expert sizes far apart.
        _moe("moe_prefill", 64, 8192, 2, 4096, 14336),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("norm", "matmul", "gated", "moe"))
    dtype = rng.choice(("float32", "float16", "bfloat16"))
    if kind == "norm":
        hidden = _log_int(rng, 300, 16384)
        tokens = _log_int(rng, 1, min(32768, 16384 * 8192 // hidden))
        case = _norm("", tokens, hidden, dtype, rng.random() < 0.6, rng.random() < 0.5)
    elif kind in ("matmul", "gated"):
        k = 16 * _log_int(rng, 16, 896)
        n = _log_int(rng, 200, 14336)
        rows = _log_int(rng, 1, min(8192, 4096 * 8192 * 8192 // (n * k)))
        case = _dense("", rows, k, n, kind == "gated", dtype)
    else:
        experts = _log_int(rng, 4, 128)
        k = 16 * _log_int(rng, 16, 256)
        n = min(_log_int(rng, 200, 14336), 32 * 4096 * 14336 // (experts * k))
        top_k = rng.randint(1, min(4, experts))
        tokens = _log_int(rng, 1, 4096 * 2 // top_k)
        case = _moe("", experts, tokens, top_k, k, n, rng.random() < 0.5, dtype, tokens > 16 and rng.random() < 0.4)
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs

def _popularity(experts):
    """Log of a Zipf(1.2) share of tokens per expert, as the library's expert workload has."""
    return -1.2 * np.log(np.arange(1, experts + 1))


def _draw_experts(tokens, experts, top_k, gen):
    """top_k distinct experts per token, popular ones more often; int64 [tokens, top_k]."""
    shift = torch.from_numpy(_popularity(experts)).float().cuda()
    shift = shift[torch.randperm(experts, generator=gen, device="cuda")]
    noise = torch.rand(tokens, experts, generator=gen, device="cuda").clamp_(1e-7, 1 - 1e-7)
    return (shift - torch.log(-torch.log(noise))).topk(top_k, dim=1).indices


def _eight_bits(shape, gen):
    """Normal values of which a block's largest is near the type's, as quantised blocks have them."""
    return (torch.randn(*shape, generator=gen, device="cuda") * 112).clamp_(-LARGEST, LARGEST).to(FP8)


def _rows(rows, k, gen):
    """Activations: a block's largest value lies between 1 and 12."""
    scales = torch.exp2(torch.rand(rows, _blocks(k), generator=gen, device="cuda") * 3.5) / LARGEST
    return _eight_bits((rows, k), gen), scales


def _matrix(lead, n, k, gen):
    """Weights of the size 1 / sqrt(k), one matrix at a time, so that the normal numbers take little room."""
    scales = (torch.rand(*lead, _blocks(n), _blocks(k), generator=gen, device="cuda") + 0.5) / (112 * math.sqrt(k))
    if not lead:
        return _eight_bits((n, k), gen), scales
    q = torch.empty(*lead, n, k, dtype=FP8, device="cuda")
    for e in range(lead[0]):
        q[e] = _eight_bits((n, k), gen)
    return q, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["kind"] == "norm":
        shape, dtype = (case["tokens"], case["hidden"]), TYPES[case["dtype"]]
        state["x"] = torch.randn(*shape, generator=gen, device="cuda").to(dtype)
        state["weight"] = (1 + 0.2 * torch.randn(case["hidden"], generator=gen, device="cuda")).to(dtype)
        state["residual"] = None
        if case["residual"]:  # the stream grows along the layers, in some features far more than in others
            grown = torch.exp2(torch.randn(case["hidden"], generator=gen, device="cuda"))
            state["residual"] = (torch.randn(*shape, generator=gen, device="cuda") * grown).to(dtype)
        return state
    k, n = case["k"], case["n"]
    gated = case["kind"] == "gated" or (case["kind"] == "moe" and case["gated"])
    lead = (case["experts"],) if case["kind"] == "moe" else ()
    state["x"], state["x_scales"] = _rows(case["tokens"] if lead else case["rows"], k, gen)
    state["w"], state["w_scales"] = _matrix(lead, n, k, gen)
    if gated:
        state["up"], state["up_scales"] = _matrix(lead, n, k, gen)
    if lead:
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        ids = _draw_experts(tokens, experts, top_k, gen)
        if case["padded"]:  # a padding token's slots have no expert and stand last in the order
            live = torch.rand(tokens, 1, generator=gen, device="cuda") < 0.9
            ids = torch.where(live, ids, experts)
        ids = ids.flatten()
        counts = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        counts.index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
        state["counts"] = counts[:experts].contiguous()
        state["order"] = ids.sort(stable=True).indices.int()
        state["row_weights"] = None if gated else torch.rand(tokens * top_k, generator=gen, device="cuda")
    return state


# ---------------------------------------------------------------- plain forms

def _quantised(y):
    """8-bit rows of float32 rows: the numbers and a scale for each block of 128, zeros in what a cut block lacks."""
    rows, n = y.shape
    full = torch.nn.functional.pad(y, (0, _blocks(n) * BLOCK - n)).unflatten(1, (-1, BLOCK))
    scales = (full.abs().amax(2) / LARGEST).clamp_(min=SMALLEST_SCALE)
    q = (full / scales.unsqueeze(2)).to(FP8).flatten(1)
    return (q if q.shape[1] == n else q[:, :n].contiguous()), scales


def _values(q, scales):
    """A weight matrix in float32."""
    w = q.float()
    n, k = w.shape
    s = scales.repeat_interleave(BLOCK, 1)[:, :k]
    whole = n // BLOCK
    w[:whole * BLOCK].unflatten(0, (-1, BLOCK)).mul_(s[:whole, None])
    if whole < len(s):
        w[whole * BLOCK:].mul_(s[whole])
    return w


def _row_values(q, scales):
    return q.float() * scales.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _plain_norm(state):
    case = state["case"]
    h = state["x"].float()
    if case["residual"]:
        h = h + state["residual"].float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * state["weight"].float()
    out = list(_quantised(y))
    if case["plain"]:
        out.append(y.to(state["x"].dtype))
    if case["residual"]:
        out.append(h.to(state["x"].dtype))
    return out


def _plain_gated(x, gate, up):
    g = x @ gate.t()
    return g / (1 + torch.exp(-g)) * (x @ up.t())


def _plain_moe(state):
    """Expert by expert, on its rows alone: in a batch of equal heights most rows would be empty."""
    case = state["case"]
    rows, top_k, n = case["tokens"] * case["top_k"], case["top_k"], case["n"]
    order = state["order"].long()
    x = _row_values(state["x"], state["x_scales"])
    y = torch.zeros(rows, n, device=x.device)
    start = 0
    for e, count in enumerate(state["counts"].tolist()):
        if count == 0:
            continue
        slots = order[start:start + count]
        mine = x[slots // top_k]
        w = _values(state["w"][e], state["w_scales"][e])
        if case["gated"]:
            y[slots] = _plain_gated(mine, w, _values(state["up"][e], state["up_scales"][e]))
        else:
            y[slots] = (mine @ w.t()) * state["row_weights"][slots, None]
        start += count
    return _quantised(y) if case["gated"] else y.to(TYPES[case["dtype"]])


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from grouped_gemm_gpu_kernel_amd import torch_ops

        if kind == "norm":
            r = torch_ops.rms_norm_fp8(state["x"], state["weight"], state["residual"], eps=EPS, plain=case["plain"])
            return [t for t in (r.q, r.scales, r.y, r.residual) if t is not None]
        if kind == "matmul":
            return torch_ops.fp8_matmul(state["x"], state["x_scales"], state["w"], state["w_scales"],
                                        out_dtype=TYPES[case["dtype"]])
        if kind == "gated":
            return tuple(torch_ops.fp8_gated(state["x"], state["x_scales"], state["w"], state["w_scales"], state["up"],
                                             state["up_scales"]))
        if case["gated"]:
            return tuple(torch_ops.moe_fp8_gated(state["x"], state["x_scales"], state["w"], state["w_scales"],
                                                 state["up"], state["up_scales"], state["counts"], state["order"]))
        return torch_ops.moe_fp8_matmul(state["x"], state["x_scales"], state["w"], state["w_scales"], state["counts"],
                                        state["order"], row_weights=state["row_weights"],
                                        out_dtype=TYPES[case["dtype"]])
    if kind == "norm":
        return _plain_norm(state)
    if kind == "moe":
        return _plain_moe(state)
    x, w = _row_values(state["x"], state["x_scales"]), _values(state["w"], state["w_scales"])
    if kind == "matmul":
        return (x @ w.t()).to(TYPES[case["dtype"]])
    return _quantised(_plain_gated(x, w, _values(state["up"], state["up_scales"])))


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_quantised(y):
    rows, n = y.shape
    q = torch.empty(rows, n, dtype=FP8, device=y.device)
    scales = torch.empty(rows, _blocks(n), dtype=torch.float64, device=y.device)
    for b in range(_blocks(n)):
        part = y[:, b * BLOCK:(b + 1) * BLOCK]
        s = torch.clamp(part.abs().max(1).values / LARGEST, min=SMALLEST_SCALE)
        scales[:, b] = s
        q[:, b * BLOCK:(b + 1) * BLOCK] = (part / s[:, None]).to(FP8)
    return [q, scales]


def _exact_values(q, scales, rows_a_block):
    i = torch.arange(q.shape[0], device=q.device) // rows_a_block
    j = torch.arange(q.shape[1], device=q.device) // BLOCK
    return q.double() * scales.double()[i][:, j]


def _exact_product(state, x, e=None):
    def of(name):
        q, s = state[name], state[name + "_scales"]
        return _exact_values(q if e is None else q[e], s if e is None else s[e], BLOCK)

    y = torch.mm(x, of("w").t())
    if "up" in state:
        y = y * torch.sigmoid(y) * torch.mm(x, of("up").t())
    return y


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        h = state["x"].double()
        if case["residual"]:
            h += state["residual"].double()
        y = h / torch.sqrt(torch.mean(h * h, dim=1) + EPS)[:, None] * state["weight"].double()
        return _exact_quantised(y) + [y] * case["plain"] + [h] * case["residual"]
    x = _exact_values(state["x"], state["x_scales"], 1)
    if case["kind"] != "moe":
        y = _exact_product(state, x)
        return tuple(_exact_quantised(y)) if case["kind"] == "gated" else y
    order = state["order"].long()
    y = torch.zeros(len(order), case["n"], dtype=torch.float64, device=order.device)
    start = 0
    for e, count in enumerate(state["counts"].tolist()):
        slots = order[start:start + count]
        part = _exact_product(state, x[slots // case["top_k"]], e)
        y[slots] = part if case["gated"] else part * state["row_weights"].double()[slots, None]
        start += count
    return tuple(_exact_quantised(y)) if case["gated"] else y


# ---------------------------------------------------------------- work

def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
    if case["kind"] == "norm":
        values = case["tokens"] * case["hidden"]
        moved = values * (size * (1 + case["plain"] + 2 * case["residual"]) + 1)
        return {"bytes": moved + 4 * case["tokens"] * _blocks(case["hidden"]) + size * case["hidden"],
                "flops": 6 * values}
    k, n = case["k"], case["n"]
    gated = case["kind"] == "gated" or (case["kind"] == "moe" and case["gated"])
    matrices = 2 if gated else 1
    matrix = matrices * (n * k + 4 * _blocks(n) * _blocks(k))
    row_in = k + 4 * _blocks(k)
    row_out = n + 4 * _blocks(n) if gated else n * size
    if case["kind"] != "moe":
        return {"bytes": matrix + case["rows"] * (row_in + row_out), "flops": 2 * matrices * case["rows"] * k * n}
    rows = case["tokens"] * case["top_k"]
    live = rows * (0.9 if case["padded"] else 1.0)
    share = np.exp(_popularity(case["experts"]))
    read = float((1.0 - (1.0 - share / share.sum()) ** live).sum())  # experts with a row, expected
    return {"bytes": read * matrix + case["tokens"] * row_in + rows * (row_out + 4 + (0 if gated else 4))
            + 4 * case["experts"], "flops": 2 * matrices * live * k * n}
