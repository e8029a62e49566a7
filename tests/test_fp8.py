"""The 8-bit path of a feed-forward layer (csrc/gg_norm.hip, csrc/gg_fp8*.hip; torch_ops.rms_norm_fp8, fp8_matmul,
fp8_gated and their expert forms) against the formulas in 64 bits, and the path as a layer uses it.

Bounds, with u = 2^-24.

Products: S = sum |x w| over an output's terms (values: numbers times scales).  In binary16 (float32 outputs, 8-bit rows, few
rows) numbers and products are exact; sums are made in lanes, instructions of 32 terms and blocks of 128 scaled by a product
of two scales (one rounding) with one multiply-add each: no chain is longer than K / 32 + 64 additions and an
instruction may round its 32 terms by a few u, (K / 32 + 128) u S in all.  The 8-bit instructions align 8 products at a
time to the largest one's power of two and drop what is 2^-13 of it or less: each of 8 terms loses up to 2^-13 of the largest
of its 8, at most 2^-10 S in all.  Both, and half a step of y's type.

8-bit rows of values h that are off by at most d from the 64-bit ones: a scale is off by max d / 448 and 2 u of its own;
a number is a value's nearest after at most 3 u of it (the scale, its reciprocal, the product), half a step of e4m3:
2^-4 of the value, or half the subnormals' step, 2^-10 scales.  A float32 scale's error is within the first bound.

Norm: mean(h^2) of H terms, chains of at most 64 + 16 additions, (H / 512 + 80) u relative, half of it on the root; h one
rounding of its terms' sizes, the factor, its product and the weight's 4 u."""
import ctypes
import math
import re
import subprocess
import threading
from pathlib import Path

import pytest
import torch

from grouped_gemm_gpu_kernel_amd import _lib, build, torch_ops
from test_kernel_resources import _scratch
from test_moe_route import _c_layout

U = 2.0 ** -24
FP8 = torch.float8_e4m3fn
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def blocks(n):
    return (n + 127) // 128


def row_values(q, s):
    return q.double() * s.double().repeat_interleave(128, -1)[..., :q.shape[-1]]


def matrix_values(q, s):
    wide = s.double().repeat_interleave(128, -1)[..., :q.shape[-1]]
    return q.double() * wide.repeat_interleave(128, -2)[..., :q.shape[-2], :]


def check_rows(q, s, h, d):
    """8-bit rows against float64 values h that the kernel's may be off from by d."""
    assert q.dtype == FP8 and s.dtype == torch.float32 and q.shape == h.shape and s.shape == (h.shape[0], blocks(h.shape[1]))
    pad = blocks(h.shape[1]) * 128 - h.shape[1]
    most = torch.nn.functional.pad(h, (0, pad)).abs().unflatten(1, (-1, 128)).amax(2)
    most_d = torch.nn.functional.pad(d, (0, pad)).unflatten(1, (-1, 128)).amax(2)
    want = (most / 448).clamp(min=2.0 ** -126)
    off = (s.double() - want).abs()
    bound = most_d / 448 + 2 * U * want
    assert (off <= bound).all(), float((off / bound).max())
    off = (row_values(q, s) - h).abs()
    wide = s.double().repeat_interleave(128, 1)[:, :h.shape[1]]
    bound = torch.maximum(2.0 ** -4 * (h.abs() + d), 2.0 ** -10 * wide) * (1 + 8 * U) + 3 * U * h.abs() + d
    assert (off <= bound).all(), float((off / bound).max())


def check_product(y, x, w, exact, row_weights=None):
    """y against x @ w.T; x [R, K], w [N, K] float64."""
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    bound = product_bound(size, x.shape[1], exact)
    if row_weights is not None:
        want, bound = want * row_weights[:, None], bound * row_weights.abs()[:, None] + want.abs() * row_weights.abs()[:, None] * U
    bound = bound + want.abs() * torch.finfo(y.dtype).eps / 2 * 1.01 + (2.0 ** -25 if y.dtype == torch.float16 else 2.0 ** -126)
    off = (y.double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


def product_bound(size, k, exact):
    return size * ((k / 32 + 128) * U + (0.0 if exact else 2.0 ** -10))


def gate_values(p, u, activation):
    if activation == "silu":
        return p * torch.sigmoid(p) * u
    return p * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3)) * u


def check_gated(rows, x, gate, up, activation="silu"):
    """Gated rows against 64 bits: the activation's slope is at most 1.13 in size, its own error 8 u of its value and,
    where exp of an argument is off by that argument's rounding, 2 u |p| more of it."""
    p, u = x @ gate.t(), x @ up.t()
    dp = product_bound(x.abs() @ gate.abs().t(), x.shape[1], True)
    du = product_bound(x.abs() @ up.abs().t(), x.shape[1], True)
    act = gate_values(p, torch.ones_like(p), activation)
    d = 1.13 * dp * (u.abs() + du) + act.abs() * du + (10 + 8 * p.abs()) * U * (act * u).abs()
    check_rows(rows.q, rows.scales, act * u, d)


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def numbers(shape, seed, spread=112.0):
    return (torch.randn(*shape, generator=_gen(seed), device="cuda") * spread).clamp(-448, 448).to(FP8)


def rows_of(m, k, seed):
    s = torch.exp2(torch.rand(m, blocks(k), generator=_gen(seed + 1), device="cuda") * 4) / 448
    return numbers((m, k), seed), s


def matrix_of(lead, n, k, seed):
    s = (torch.rand(*lead, blocks(n), blocks(k), generator=_gen(seed + 1), device="cuda") + 0.5) / (112 * math.sqrt(k))
    return numbers((*lead, n, k), seed), s


def routing(tokens, experts, top_k, seed, drop=0.0):
    """ids [T, k] (-1: none), counts and order as moe_route writes them."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(experts, generator=g)[:top_k] for _ in range(tokens)])
    ids[torch.rand(tokens, top_k, generator=g) < drop] = -1
    flat = torch.where(ids < 0, experts, ids).flatten()
    counts = torch.bincount(flat, minlength=experts + 1)[:experts].int()
    return ids.cuda(), counts.cuda(), flat.sort(stable=True).indices.int().cuda()


def check_moe(y, x, x_scales, w, w_scales, ids, exact, row_weights=None):
    xv, flat = row_values(x, x_scales), ids.flatten()
    fan = len(flat) // len(xv)
    assert (y[flat < 0] == 0).all()
    for e in range(len(w)):
        at = (flat == e).nonzero()[:, 0]
        if len(at):
            check_product(y[at], xv[at // fan], matrix_values(w[e], w_scales[e]), exact,
                          None if row_weights is None else row_weights.double().flatten()[at])


def check_moe_gated(rows, x, x_scales, gate, up, ids, activation="silu"):
    xv, flat = row_values(x, x_scales), ids.flatten()
    fan = len(flat) // len(xv)
    assert (rows.q[flat < 0].float() == 0).all() and (rows.scales[flat < 0] == 2.0 ** -126).all()
    for e in range(len(gate[0])):
        at = (flat == e).nonzero()[:, 0]
        if len(at):
            check_gated(torch_ops.Fp8Rows(rows.q.view(torch.uint8)[at].view(FP8), rows.scales[at]), xv[at // fan],
                        matrix_values(gate[0][e], gate[1][e]), matrix_values(up[0][e], up[1][e]), activation)


# ---------------------------------------------------------------- CPU

@pytest.mark.parametrize("struct,mirror", [("ggk_norm_fp8_args", _lib.GGKNormFp8Args), ("ggk_fp8_args", _lib.GGKFp8Args)])
def test_structs_mirror_the_header(tmp_path, struct, mirror):
    got, want = _c_layout(tmp_path, struct, mirror)
    assert got == want


NORM = dict(rows=3, columns=300, type=_lib.GGK_TYPE_BF16, weight_type=_lib.GGK_TYPE_BF16, x=0x1000, ldx=300, q=0x1000,
            ldq=300, scales=0x1000, lds=3, eps=1e-6)


@pytest.mark.parametrize("over,status", [
    ({}, 0), ({"rows": -1}, 1), ({"rows": (1 << 30) + 1}, 1), ({"columns": 0}, 1), ({"columns": 32769}, 1), ({"type": 3}, 1),
    ({"weight": 0x1000}, 0), ({"weight": 0x1000, "weight_type": _lib.GGK_TYPE_F32}, 0),
    ({"weight": 0x1000, "weight_type": _lib.GGK_TYPE_F16}, 1), ({"weight_type": 7}, 0), ({"weight": 0x1000, "weight_type": 7}, 1),
    ({"ldx": 299}, 1), ({"ldq": 299}, 1), ({"lds": 2}, 1), ({"residual": 0x1000, "ldr": 299}, 1),
    ({"residual": 0x1000, "ldr": 300}, 0), ({"y": 0x1000, "ldy": 299}, 1), ({"y": 0x1000, "ldy": 300}, 0),
    ({"sum": 0x1000, "ldsum": 299}, 1), ({"sum": 0x1000, "ldsum": 300}, 0), ({"x": None}, 17), ({"q": None}, 17),
    ({"scales": None}, 17), ({"rows": 0, "x": None, "q": None, "scales": None}, 0),
    ({"rows": 1, "ldx": 0, "ldq": 0, "lds": 0}, 0)])
def test_norm_arguments_are_checked_on_the_host(over, status):
    args = _lib.GGKNormFp8Args(**{**NORM, **over})
    assert _lib.lib().ggk_norm_fp8_check(ctypes.byref(args)) == status
    if status:  # refused before anything is launched
        assert _lib.lib().ggk_norm_fp8(ctypes.byref(args), None) == status
    assert _lib.lib().ggk_norm_fp8_check(None) == 1 and _lib.lib().ggk_norm_fp8(None, None) == 1


BASE = dict(rows=4, x_rows=4, n=200, k=272, experts=0, gate=0, x=0x1000, ldx=272, x_scales=0x1000, ldxs=3, w=0x1000, ldw=272,
            w_scales=0x1000, ldws=3, y=0x1000, ldy=200, y_type=_lib.GGK_TYPE_BF16)
GATE = dict(gate=1, up=0x1000, ldu=272, up_scales=0x1000, ldus=3, y_scales=0x1000, ldys=2)
MOE = dict(experts=3, counts=0x1000, order=0x1000, stride_w=200 * 272, stride_ws=6)


@pytest.mark.parametrize("over,status", [
    ({}, 0), ({"rows": -1}, 1), ({"rows": 5}, 1), ({"n": -1}, 1), ({"n": (1 << 28) + 1}, 1), ({"k": 0}, 1), ({"k": 264}, 1),
    ({"k": 288}, 1), ({"k": (1 << 22) + 16, "ldx": 1 << 23, "ldw": 1 << 23, "ldxs": 1 << 16, "ldws": 1 << 16}, 1),
    ({"ldx": 256}, 1), ({"ldx": 280}, 1), ({"ldx": 288}, 0), ({"x": 0x1008}, 1), ({"w": 0x1008}, 1), ({"ldw": 256}, 1),
    ({"ldw": 280}, 1), ({"ldw": (1 << 22) + 16}, 1), ({"ldw": 1 << 22}, 0), ({"ldxs": 2}, 1), ({"ldws": 2}, 1), ({"ldy": 199}, 1),
    ({"y_type": 3}, 1), ({"gate": 3}, 1), ({"gate": -1}, 1), ({"x": None}, 17), ({"x_scales": None}, 17), ({"w": None}, 17),
    ({"w_scales": None}, 17), ({"y": None}, 17), ({"rows": 0, "x_rows": 0, "x": None, "y": None}, 0),
    ({"n": 0, "w": None, "w_scales": None, "y": None}, 0), ({"n": 1, "ldw": 0, "ldws": 0}, 0),
    (GATE, 0), ({**GATE, "gate": 2}, 0), ({**GATE, "up": None}, 17), ({**GATE, "up": 0x1008}, 1), ({**GATE, "up_scales": None}, 17),
    ({**GATE, "y_scales": None}, 17), ({**GATE, "ldu": 256}, 1), ({**GATE, "ldus": 2}, 1), ({**GATE, "ldys": 1}, 1),
    ({**GATE, "row_weights": 0x1000}, 1), (MOE, 0), ({**MOE, **GATE, "stride_u": 200 * 272, "stride_us": 6}, 0),
    ({**MOE, **GATE, "stride_u": 8}, 1), ({**MOE, "rows": 8}, 0), ({**MOE, "rows": 7}, 1), ({**MOE, "x_rows": 0}, 1),
    ({**MOE, "counts": None}, 17), ({**MOE, "order": None}, 17), ({**MOE, "stride_w": 8}, 1), ({**MOE, "stride_w": -16}, 1),
    ({**MOE, "stride_ws": -1}, 1), ({**MOE, "experts": 1025}, 1), ({**MOE, "experts": -1}, 1),
    ({**MOE, "row_weights": 0x1000}, 0)])
def test_product_arguments_are_checked_on_the_host(over, status):
    args = _lib.GGKFp8Args(**{**BASE, **over})
    assert _lib.lib().ggk_fp8_check(ctypes.byref(args)) == status
    if status:
        assert _lib.lib().ggk_fp8_multiply(ctypes.byref(args), None) == status
    assert _lib.lib().ggk_fp8_check(None) == 1 and _lib.lib().ggk_fp8_multiply(None, None) == 1


@pytest.mark.parametrize("over,floats", [
    ({}, 0), (MOE, 0), ({**MOE, **GATE, "stride_u": 200 * 272, "stride_us": 6}, 0), ({**GATE, "up": None}, 0), (GATE, 0),
    ({**GATE, "k": 4096, "ldx": 4096, "ldw": 4096, "ldu": 4096, "ldxs": 32, "ldws": 32, "ldus": 32}, 2 * 4 * 200),
    ({**GATE, "rows": 1 << 24, "x_rows": 1 << 24, "n": 1, "k": 4096, "ldx": 4096, "ldxs": 32, "ldws": 32, "ldus": 32, "ldw": 4096,
      "ldu": 4096}, 0), ({**GATE, "rows": 1 << 22, "x_rows": 1 << 22, "n": 1, "k": 4096, "ldx": 4096, "ldxs": 32, "ldws": 32, "ldus": 32,
                         "ldw": 4096, "ldu": 4096}, 1 << 25),
    ({**GATE, "n": 199, "k": 4096, "ldx": 4096, "ldw": 4096, "ldu": 4096, "ldxs": 32, "ldws": 32, "ldus": 32}, 2 * 4 * 200)])
def test_workspace_of_gated_calls(over, floats):
    args, got = _lib.GGKFp8Args(**{**BASE, **over}), ctypes.c_longlong(-1)
    status = _lib.lib().ggk_fp8_check(ctypes.byref(args))
    assert _lib.lib().ggk_fp8_workspace(ctypes.byref(args), ctypes.byref(got)) == status
    assert got.value == (-1 if status else floats)
    assert _lib.lib().ggk_fp8_workspace(None, ctypes.byref(got)) == 1 and _lib.lib().ggk_fp8_workspace(ctypes.byref(args), None) == 1
    args.workspace = 0x1008
    assert _lib.lib().ggk_fp8_check(ctypes.byref(args)) == 1


def _fake(*shape, dtype=torch.float32, device="cuda:0"):
    return torch.empty(*shape, dtype=dtype, device=device)


def test_refusals_of_the_norm():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad

    with pytest.raises(ValueError, match="on a GPU"):
        torch_ops.rms_norm_fp8(torch.zeros(1, 64))
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        torch_ops.rms_norm_fp8([1.0])
    with FakeTensorMode():
        x, half = _fake(3, 64), _fake(3, 64, dtype=torch.float16)
        for args, error, text in [
                ((_fake(3, 64, dtype=torch.float64),), TypeError, "float32, float16 or bfloat16"), ((_fake(64),), ValueError, "2-D"),
                ((_fake(64, 3).t(),), ValueError, "contiguous rows"), ((_fake(1, 64).expand(3, 64),), ValueError, "overlap"),
                ((_fake(3, 0),), ValueError, "columns"), ((_fake(3, 32769),), ValueError, "columns"),
                ((x, _fake(63)), ValueError, "entries"), ((x, _fake(1, 64)), ValueError, "1-D"),
                ((x, _fake(64, dtype=torch.float16)), TypeError, "weight"), ((half, _fake(64, dtype=torch.bfloat16)), TypeError, "weight"),
                ((x, _fake(128)[::2]), ValueError, "contiguous"), ((x, _fake(64, device="cpu")), ValueError, "weight is on"),
                ((x, 1.0), TypeError, "weight must be a torch.Tensor"), ((x, None, half), TypeError, "residual must be torch.float32"),
                ((x, None, _fake(4, 64)), ValueError, "residual has shape"),
                ((x, None, _fake(64, 3).t()), ValueError, "contiguous rows"),
                ((x.clone().requires_grad_(True),), RuntimeError, "no gradient: detach x"),
                ((x, _fake(64).requires_grad_(True)), RuntimeError, "detach weight"),
                ((x, None, x.clone().requires_grad_(True)), RuntimeError, "detach residual"),
                ((torch._neg_view(x),), ValueError, "resolve_neg")]:
            with pytest.raises(error, match=text):
                torch_ops.rms_norm_fp8(*args)
        with forward_ad.dual_level(), torch.no_grad():
            for name, args in [("x", (forward_ad.make_dual(x, x),)), ("weight", (x, forward_ad.make_dual(_fake(64), _fake(64)))),
                               ("residual", (x, None, forward_ad.make_dual(x, x)))]:
                with pytest.raises(RuntimeError, match=f"forward-mode derivative: {name}"):
                    torch_ops.rms_norm_fp8(*args)
        with pytest.raises(Exception):  # a tensor without data is not taken for one left out
            torch_ops.rms_norm_fp8(x, _fake(64))


def test_refusals_of_the_products():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad

    def q(*shape, **k):
        return _fake(*shape, dtype=FP8, **k)

    with pytest.raises(ValueError, match="on a GPU"):
        torch_ops.fp8_matmul(torch.zeros(1, 64).to(FP8), torch.zeros(1, 1), torch.zeros(4, 64).to(FP8), torch.zeros(1, 1))
    with pytest.raises(TypeError, match="torch.Tensors"):
        torch_ops.fp8_matmul(1, 2, 3, 4)
    with FakeTensorMode():
        x, xs, w, ws = q(3, 272), _fake(3, 3), q(200, 272), _fake(2, 3)
        dense = [
            ((_fake(3, 272), xs, w, ws), TypeError, "x must be"), ((q(272), xs, w, ws), ValueError, "2-D"),
            ((q(3, 256), xs, w, ws), ValueError, "columns"), ((q(272, 3).t(), xs, w, ws), ValueError, "contiguous rows"),
            ((q(3, 280)[:, :272], xs, w, ws), ValueError, "16 bytes"), ((q(1, 272).expand(3, 272), xs, w, ws), ValueError, "overlap"),
            ((q(3, 264), xs, q(200, 264), ws), ValueError, "multiple of 16"), ((q(3, 0), _fake(3, 0), q(200, 0), _fake(2, 0)), ValueError, "multiple of 16"),
            ((x, _fake(3, 2), w, ws), ValueError, "x_scales has shape"), ((x, _fake(3, 3).half(), w, ws), TypeError, "x_scales"),
            ((x, _fake(3, 3).t().contiguous().t(), w, ws), ValueError, "contiguous rows"), ((x, _fake(3, 3, device="cpu"), w, ws), ValueError, "x_scales is on"),
            ((x, xs, _fake(200, 272), ws), TypeError, "w must be"), ((x, xs, w, _fake(1, 3)), ValueError, "128 x 128"),
            ((x, xs, w, _fake(2, 4)), ValueError, "128 x 128"), ((x, xs, w, ws.half()), TypeError, "w_scales"),
            ((x, xs, q(200, 280)[:, :272], ws), ValueError, "16 bytes"), ((x, xs, q(272, 200).t(), ws), ValueError, "contiguous rows"),
            ((x, xs, q(1, 272).expand(200, 272), ws), ValueError, "overlap"), ((x, xs, q(2, 200, 272), ws), ValueError, "dimensions"),
            ((x, xs, w, _fake(1, 3).expand(2, 3)), ValueError, "overlap"),
            ((x, xs, q(2, (1 << 22) + 16)[:, :272], _fake(1, 3)), ValueError, "2\\^22"),
            ((q(3, 272, device="cpu"), xs, w, ws), ValueError, "on a GPU"), ((x, xs, q(200, 272, device="cpu"), ws), ValueError, "w is on"),
            ((x, xs.clone().requires_grad_(True), w, ws), RuntimeError, "detach x_scales"),
            ((x, xs, w, ws.clone().requires_grad_(True)), RuntimeError, "detach w_scales"),
            ((x, torch._neg_view(xs), w, ws), ValueError, "resolve_neg")]
        for args, error, text in dense:
            with pytest.raises(error, match=text):
                torch_ops.fp8_matmul(*args)
        with pytest.raises(TypeError, match="out_dtype"):
            torch_ops.fp8_matmul(x, xs, w, ws, out_dtype=torch.float64)
        for up, us, error, text in [(q(201, 272), ws, ValueError, "up has shape"), (w, _fake(1, 3), ValueError, "128 x 128"),
                                    (w, None, TypeError, "up_scales must be"), (None, ws, TypeError, "up must be")]:
            with pytest.raises(error, match=text):
                torch_ops.fp8_gated(x, xs, w, ws, up, us)
        for activation in ("tanh", None, 1, ["silu"]):
            with pytest.raises(ValueError, match="activation"):
                torch_ops.fp8_gated(x, xs, w, ws, w, ws, activation=activation)
        with pytest.raises(ValueError, match="gate has shape|gate_scales has shape"):
            torch_ops.fp8_gated(x, xs, w, _fake(1, 3), w, ws)
        w3, ws3, counts, order = q(4, 200, 272), _fake(4, 2, 3), _fake(4, dtype=torch.int32), _fake(6, dtype=torch.int32)
        for args, error, text in [
                ((x, xs, w, ws, counts, order), ValueError, "dimensions"), ((x, xs, w3, ws, counts, order), ValueError, "dimensions"),
                ((x, xs, w3, _fake(3, 2, 3), counts, order), ValueError, "128 x 128"), ((x, xs, w3, ws3, counts[:3], order), ValueError, "entries"),
                ((x, xs, w3, ws3, counts.long(), order), TypeError, "int32"), ((x, xs, w3, ws3, counts, order.long()), TypeError, "int32"),
                ((x, xs, w3, ws3, counts, order[:5]), ValueError, "multiple"), ((x, xs, w3, ws3, counts, 6), TypeError, "order must be"),
                ((x, xs, w3, ws3, None, order), TypeError, "counts and order"), ((x, xs, w3, ws3, counts, None), TypeError, "counts and order"),
                ((x, xs, q(1025, 200, 272), _fake(1025, 2, 3), _fake(1025, dtype=torch.int32), order), ValueError, "experts"),
                ((q(0, 272), _fake(0, 3), w3, ws3, counts, order), ValueError, "multiple")]:
            with pytest.raises(error, match=text):
                torch_ops.moe_fp8_matmul(*args)
        for weights, error, text in [(_fake(5), ValueError, "entries"), (_fake(6).half(), TypeError, "float32"),
                                     (_fake(6).requires_grad_(True), RuntimeError, "detach row_weights")]:
            with pytest.raises(error, match=text):
                torch_ops.moe_fp8_matmul(x, xs, w3, ws3, counts, order, row_weights=weights)
        with pytest.raises(TypeError, match="counts and order"):
            torch_ops.moe_fp8_gated(x, xs, w3, ws3, w3, ws3, None, order)
        with forward_ad.dual_level(), torch.no_grad():
            with pytest.raises(RuntimeError, match="forward-mode derivative: x_scales"):
                torch_ops.fp8_matmul(x, forward_ad.make_dual(xs, xs), w, ws)
            with pytest.raises(RuntimeError, match="forward-mode derivative: up_scales"):
                torch_ops.fp8_gated(x, xs, w, ws, w, forward_ad.make_dual(ws, ws))
        with pytest.raises(Exception):  # a tensor without data is not taken for one left out
            torch_ops.fp8_matmul(x, xs, w, ws)


@pytest.mark.parametrize("name", ["gg_norm.o", "gg_fp8.o", "gg_fp8_tiles.o"])
def test_kernels_spill_nothing(name, tmp_path):
    assert not {k: v for k, v in _scratch(name, tmp_path).items() if v}


@pytest.mark.parametrize("name", ["gg_fp8.o", "gg_fp8_tiles.o"])
def test_matrix_results_and_lds_loads_have_their_wait_states(name, tmp_path):
    """In the built kernels no result of a matrix instruction is read by another kind, and no branch taken, before its wait states
    (8 for 16 x 16 x 32, 12 for 16 x 16 x 128), and every load into LDS directly follows the 5 of its statement."""
    built = build.BUILD / name
    if not built.exists():
        pytest.skip("no regular build in the tree (build first)")
    llvm = Path("/opt/rocm/llvm/bin")
    subprocess.run([str(llvm / "llvm-objcopy"), f"--dump-section=.hip_fatbin={tmp_path / 'fat'}", str(built),
                    str(tmp_path / "copy.o")], check=True)
    subprocess.run([str(llvm / "clang-offload-bundler"), "--unbundle", "--type=o",
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={tmp_path / 'fat'}",
                    f"--output={tmp_path / 'gfx950.o'}"], check=True)
    text = subprocess.run([str(llvm / "llvm-objdump"), "-d", "--mcpu=gfx950", str(tmp_path / "gfx950.o")], check=True,
                          capture_output=True, text=True).stdout
    code = [line.split("//")[0].strip() for line in text.splitlines() if line.startswith("\t")]
    needed = {"v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x128_f8f6f4": 12}

    def registers(operands):
        found = set()
        for first, last, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", operands):
            found |= {int(one)} if one else set(range(int(first), int(last) + 1))
        return found

    def states_of(line):
        return int(line.split()[1], 0) + 1 if line.startswith("s_nop") else 1

    bad, products, loads = [], 0, 0
    for i, line in enumerate(code):
        kind = line.split()[0] if line else ""
        if kind.startswith("global_load_lds") or (kind.startswith("buffer_load") and line.endswith(" lds")):
            loads += 1
            if not code[i - 1].startswith("s_nop") or states_of(code[i - 1]) < 5:
                bad.append((code[i - 1], line))
        if not kind.startswith("v_mfma"):
            continue
        products += 1
        result, states = registers(line.split(",")[0]), 0
        for after in code[i + 1:]:
            if states >= needed[kind]:
                break
            if after.startswith("v_mfma"):
                if result & registers(",".join(after.split(",")[1:3])):
                    bad.append((line, after, states))
                if result & registers(after):  # the next of a chain: checked as the one before
                    break
            elif result & registers(after) or after.startswith(("s_cbranch", "s_branch", "s_setpc")):
                bad.append((line, after, states))
                break
            states += states_of(after)
    assert products > 100 and loads > 50 and not bad, bad[:3]


# ---------------------------------------------------------------- the norm

def check_norm(out, x, weight, residual, eps=1e-6):
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    columns = h.shape[1]
    w = torch.ones(columns, dtype=torch.float64, device=h.device) if weight is None else weight.double()
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w
    d = y.abs() * ((columns / 512 + 80) / 2 + 6) * U
    if residual is not None:  # the rounding of h, and what it changes in the root
        slip = (x.double().abs() + residual.double().abs()) * U
        d = d + slip * (y / h).abs().nan_to_num() + y.abs() * (slip * h.abs()).mean(1, keepdim=True) / (
            h.square().mean(1, keepdim=True) + eps)
    check_rows(out.q, out.scales, y, d)
    half = torch.finfo(x.dtype).eps / 2 * 1.01
    least = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126}[x.dtype]
    if out.y is not None:
        assert out.y.dtype == x.dtype and ((out.y.double() - y).abs() <= (y.abs() + d) * half + d + least).all()
    if residual is not None:
        assert out.residual.dtype == x.dtype and ((out.residual.double() - h).abs() <= h.abs() * half + least).all()
    else:
        assert out.residual is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [
    (1, 1), (3, 7), (5, 8), (2, 127), (7, 128), (4, 129), (6, 500), (5, 512), (9, 520), (3, 1000), (2, 2048), (3, 2056), (2, 2049),
    (4, 4096), (3, 4104), (2, 5000), (3, 8192), (2, 8200), (1, 16384), (2, 16392), (1, 16385), (2, 32768), (1, 32767)])
def test_norm(torch_cuda, dtype, rows, columns):
    g = _gen(rows * 40000 + columns)
    x = (torch.randn(rows, columns, generator=g, device="cuda") * torch.exp2(torch.randn(columns, generator=g, device="cuda"))).to(dtype)
    r = (torch.randn(rows, columns, generator=g, device="cuda") * 3).to(dtype)
    w = 1 + 0.3 * torch.randn(columns, generator=g, device="cuda")
    check_norm(torch_ops.rms_norm_fp8(x), x, None, None)
    check_norm(torch_ops.rms_norm_fp8(x, w.to(dtype), r, plain=True), x, w.to(dtype), r)
    check_norm(torch_ops.rms_norm_fp8(x, w, plain=True, eps=0.5), x, w, None, 0.5)
    check_norm(torch_ops.rms_norm_fp8(x, None, r, eps=0.0), x, None, r, 0.0)


@pytest.mark.gpu
def test_norm_of_padded_rows_and_odd_starts(torch_cuda):
    for dtype in TYPES:
        wide = torch.randn(6, 777, generator=_gen(1), device="cuda").to(dtype)
        for at, columns in [(0, 512), (1, 512), (3, 513), (8, 256)]:
            x, r = wide[:, at:at + columns], wide.flip(0)[:, 200:200 + columns]
            w = wide.flatten()[at:at + columns]
            check_norm(torch_ops.rms_norm_fp8(x, w, r, plain=True), x, w, r)
        assert torch_ops.rms_norm_fp8(wide[:0]).q.shape == (0, 777)
        one = wide[2:3, 5:405]
        check_norm(torch_ops.rms_norm_fp8(one, plain=True), one, None, None)


@pytest.mark.gpu
def test_norm_of_odd_values(torch_cuda):
    x = torch.randn(9, 512, generator=_gen(2), device="cuda")
    clean = torch_ops.rms_norm_fp8(x, plain=True)
    x[0] = 0.0
    x[1, 5] = math.nan
    x[2, 300] = math.inf
    x[3] = 1e-30
    x[4] = 1e17
    x[5, 128:256] = 0.0
    x[6] *= 1e-12
    out = torch_ops.rms_norm_fp8(x, plain=True)
    assert (out.q[0].float() == 0).all() and (out.scales[0] == 2.0 ** -126).all() and (out.y[0] == 0).all()
    assert out.q[1].float().isnan().all() and out.scales[1].isnan().all()  # the row's factor is NaN
    # An infinite mean: the factor is 0, what it multiplies 0 but for the infinity itself.
    assert (out.q[2].float()[:256] == 0).all() and out.q[2].float()[256:384].isnan().all() and out.scales[2, 2].isnan()
    check_norm(torch_ops.Fp8Norm(*(None if t is None else t[3:7] for t in out)), x[3:7], None, None)
    assert (out.scales[5, 1] == 2.0 ** -126).all()
    for a, b in zip(out[:3], clean[:3]):
        assert torch.equal(a[7:].float(), b[7:].float())
    # A weight's infinity and NaN stay in their blocks.
    w = torch.ones(512, device="cuda")
    w[130], w[400] = math.inf, math.nan
    x = torch.randn(2, 512, generator=_gen(3), device="cuda")
    out = torch_ops.rms_norm_fp8(x, w)
    assert out.scales[:, 1].isinf().all() and out.q[:, 130].float().isnan().all() and (out.q[:, 131:256].float() == 0).all()
    assert out.scales[:, 3].isnan().all() and out.q[:, 384:].float().isnan().all()
    y = (x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-6))[:, :128]
    check_rows(out.q.view(torch.uint8)[:, :128].contiguous().view(FP8), out.scales[:, :1], y, y.abs() * 60 * U)


@pytest.mark.gpu
def test_norm_of_more_than_4_gb(torch_cuda):
    rows, columns = 2 ** 32 // 2 // 16384 + 50, 16384
    x = torch.zeros(rows, columns, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(30, columns, generator=_gen(4), device="cuda").bfloat16()
    x[-30:] = tail
    out = torch_ops.rms_norm_fp8(x)
    check_norm(torch_ops.Fp8Norm(out.q.view(torch.uint8)[-30:].view(FP8), out.scales[-30:], None, None), tail, None, None)
    assert not out.q.view(torch.uint8)[:-30].any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,columns", [(700, 4096), (64, 333), (3, 32768)])
def test_norm_numbers_are_the_nearest(torch_cuda, rows, columns):
    """Values x w of bfloat16 terms are whole numbers of 16 bits times powers of two, and the factor cancels in a number, 448 x w
    over the block's largest |x w|: a quotient a / b with b below 2^16, which lies on a tie of e4m3 (five bits) or is off it by
    2^-21 of itself at least, and the kernel's is off by 2^-23 at most.  So every number is the nearest, ties to even."""
    x = torch.randn(rows, columns, generator=_gen(rows), device="cuda").bfloat16()
    weight = torch.randn(columns, generator=_gen(columns), device="cuda").bfloat16()
    v = torch.nn.functional.pad(x.double() * weight.double(), (0, blocks(columns) * 128 - columns)).unflatten(1, (-1, 128))
    want = (v * 448 / v.abs().amax(2, keepdim=True)).flatten(1)[:, :columns].float().to(FP8)
    assert torch.equal(torch_ops.rms_norm_fp8(x, weight).q.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.gpu
def test_norm_in_place(torch_cuda):
    """In the C-ABI the sum may be the residual's own memory, and y x's."""
    x = torch.randn(5, 3000, generator=_gen(5), device="cuda").half()
    r = torch.randn(5, 3000, generator=_gen(6), device="cuda").half()
    want = torch_ops.rms_norm_fp8(x, None, r, plain=True)
    q, s = torch.empty_like(want.q), torch.empty_like(want.scales)
    args = _lib.GGKNormFp8Args(rows=5, columns=3000, type=_lib.GGK_TYPE_F16, x=x.data_ptr(), ldx=3000, residual=r.data_ptr(),
                               ldr=3000, eps=1e-6, q=q.data_ptr(), ldq=3000, scales=s.data_ptr(), lds=24, y=x.data_ptr(),
                               ldy=3000, sum=r.data_ptr(), ldsum=3000)
    assert _lib.lib().ggk_norm_fp8(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(q.float(), want.q.float()) and torch.equal(s, want.scales)
    assert torch.equal(x, want.y) and torch.equal(r, want.residual)


# ---------------------------------------------------------------- products

SHAPES = [(1, 16, 1), (1, 128, 128), (2, 144, 130), (5, 272, 17), (8, 256, 96), (9, 400, 257), (16, 1040, 48), (17, 128, 300),
          (31, 640, 129), (33, 1024, 200), (64, 16, 64), (65, 384, 255), (100, 2064, 140), (129, 256, 513), (200, 528, 260),
          (256, 128, 256), (257, 400, 300), (300, 1168, 520), (515, 272, 257),
          # many rows: tiles of 256 rows (y's rows by way of LDS, then not) and of 128
          (40000, 272, 257), (40000, 16, 300), (30011, 144, 516), (33000, 272, 136), (6000, 400, 1000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product(torch_cuda, dtype, m, k, n):
    x, w = rows_of(m, k, m + n), matrix_of((), n, k, 7 * k + n)
    y = torch_ops.fp8_matmul(*x, *w, out_dtype=dtype)
    assert y.dtype == dtype and y.shape == (m, n)
    check_product(y, row_values(*x), matrix_values(*w), dtype == torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_gated(torch_cuda, activation, m, k, n):
    x, gate, up = rows_of(m, k, m + n), matrix_of((), n, k, 7 * k + n), matrix_of((), n, k, 9 * k + n)
    out = torch_ops.fp8_gated(*x, *gate, *up, activation=activation)
    check_gated(out, row_values(*x), matrix_values(*gate), matrix_values(*up), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(1, 4096, 520), (7, 8192, 129), (13, 2080, 300), (50, 4096, 257), (64, 2064, 7171), (200, 2064, 389)])
def test_gated_with_and_without_a_workspace(torch_cuda, m, k, n, activation):
    """One launch, or both products into a workspace and their rows in a second; nothing past the workspace is written, nor to
    one that the call does not want (64 rows of many columns)."""
    x, gate, up = rows_of(m, k, m + n), matrix_of((), n, k, 7 * k + n), matrix_of((), n, k, 9 * k + n)
    values = row_values(*x), matrix_values(*gate), matrix_values(*up)
    check_gated(torch_ops.fp8_gated(*x, *gate, *up, activation=activation), *values, activation)
    for with_it in (False, True):
        y = torch.zeros(m, n, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(m, blocks(n), device="cuda")
        args = _lib.GGKFp8Args(
            rows=m, x_rows=m, n=n, k=k, gate=1 if activation == "silu" else 2, x=x[0].data_ptr(), ldx=k, x_scales=x[1].data_ptr(),
            ldxs=blocks(k), w=gate[0].data_ptr(), ldw=k, w_scales=gate[1].data_ptr(), ldws=blocks(k), up=up[0].data_ptr(), ldu=k,
            up_scales=up[1].data_ptr(), ldus=blocks(k), y=y.data_ptr(), ldy=n, y_scales=scales.data_ptr(), ldys=blocks(n))
        wanted = ctypes.c_longlong(-1)
        assert _lib.lib().ggk_fp8_workspace(ctypes.byref(args), ctypes.byref(wanted)) == 0
        floats = wanted.value
        assert floats == (0 if m == 64 else 2 * m * ((n + 3) // 4 * 4))
        workspace = torch.full((floats + 64,), 77.0, device="cuda")
        if with_it:
            args.workspace = workspace.data_ptr()
        assert _lib.lib().ggk_fp8_multiply(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
        check_gated(torch_ops.Fp8Rows(y.view(FP8), scales), *values, activation)
        assert (workspace[floats if with_it else 0:] == 77).all()


@pytest.mark.gpu
def test_gated_on_streams_and_in_a_graph(torch_cuda):
    """Calls that use a workspace, several at a time."""
    m, k, n = 5, 4096, 700
    gate, up = matrix_of((), n, k, 1), matrix_of((), n, k, 2)
    inputs = [rows_of(m, k, 10 + i) for i in range(4)]

    def call(x):
        out = torch_ops.fp8_gated(*x, *gate, *up)
        return out.q.view(torch.uint8), out.scales

    eager = [call(x) for x in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(5):
        got = []
        for x, stream in zip(inputs, streams):
            with torch.cuda.stream(stream):
                got.append(call(x))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for a, b in zip(got, eager) for p, q in zip(a, b))
    x = tuple(t.clone() for t in inputs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, again = call(x), call(x)
    for i in (2, 0, 3, 1):
        x[0].copy_(inputs[i][0])
        x[1].copy_(inputs[i][1])
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, eager[i])) and all(torch.equal(p, q) for p, q in zip(again, eager[i]))
        call(inputs[3 - i])
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 6, 13, 30, 60, 200, 700, 9000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sums_of_integers_are_exact(torch_cuda, m, dtype):
    """Numbers of a few units and scales of powers of two: every sum is a whole number below 2^8 scales' worth, so that any
    term that is left out or counted twice shows."""
    k, n = 1168, 393
    g = _gen(m)
    x = (torch.rand(m, k, generator=g, device="cuda") < 0.02).float() * torch.randint(-2, 3, (m, k), generator=g, device="cuda")
    w = torch.randint(-3, 4, (n, k), generator=g, device="cuda").float()
    xs = torch.exp2(torch.randint(0, 2, (m, blocks(k)), generator=g, device="cuda").float())
    ws = torch.exp2(torch.randint(-1, 1, (blocks(n), blocks(k)), generator=g, device="cuda").float())
    want = row_values(x.to(FP8), xs) @ matrix_values(w.to(FP8), ws).t()
    keep = want.abs() <= 128  # bfloat16 has 8 bits: whole numbers and halves up to here
    y = torch_ops.fp8_matmul(x.to(FP8), xs, w.to(FP8), ws, out_dtype=dtype)
    got, want = (y.double(), want) if dtype == torch.float32 else (y.double()[keep], want.to(dtype).double()[keep])
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 14336, 4096), (61, 4096, 14336), (777, 2048, 4096), (2048, 2048, 2048)])
def test_larger(torch_cuda, m, n, k):
    x, w, up = rows_of(m, k, 1), matrix_of((), n, k, 2), matrix_of((), n, k, 3)
    xv, wv = row_values(*x), matrix_values(*w)
    check_product(torch_ops.fp8_matmul(*x, *w), xv, wv, False)
    check_product(torch_ops.fp8_matmul(*x, *w, out_dtype=torch.float32), xv, wv, True)
    check_gated(torch_ops.fp8_gated(*x, *w, *up), xv, wv, matrix_values(*up))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40, 300, 40000])
def test_strides_and_alignment(torch_cuda, m):
    k, n = 272, 200
    x, xs = rows_of(m, k, 1)
    w, ws = matrix_of((), n, k, 2)
    u, us = matrix_of((), n, k, 3)

    def wide(t, before, after):
        out = torch.full((t.shape[0] + 2, before + t.shape[1] + after), 0x7F if t.dtype == FP8 else 0, dtype=torch.uint8,
                         device="cuda").view(FP8) if t.dtype == FP8 else torch.full(
                             (t.shape[0] + 2, before + t.shape[1] + after), math.nan, device="cuda")
        out.view(torch.uint8 if t.dtype == FP8 else torch.float32)[1:-1, before:before + t.shape[1]] = (
            t.view(torch.uint8) if t.dtype == FP8 else t)
        return out[1:-1, before:before + t.shape[1]]

    want = torch_ops.fp8_matmul(x, xs, w, ws)
    rows = torch_ops.fp8_gated(x, xs, w, ws, u, us)
    # What stands around the rows is NaN: none of it may be read into a sum.
    for before in (16, 48):
        args = (wide(x, before, 16), wide(xs, 1, 2), wide(w, 16, before), wide(ws, 3, 1))
        assert torch.equal(torch_ops.fp8_matmul(*args), want)
        got = torch_ops.fp8_gated(*args, wide(u, 32, before), wide(us, 1, 0))
        assert torch.equal(got.q.view(torch.uint8), rows.q.view(torch.uint8)) and torch.equal(got.scales, rows.scales)
    both, scales = torch.cat((w[:128], u[:128])), torch.cat((ws[:1], us[:1]))  # the halves of one matrix
    got = torch_ops.fp8_gated(x, xs, both[:128], scales[:1], both[128:], scales[1:])
    want = torch_ops.fp8_gated(x, xs, w[:128].contiguous(), ws[:1], u[:128].contiguous(), us[:1])
    assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.scales, want.scales)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 20, 70, 300, 20000])
def test_odd_values(torch_cuda, m):
    """NaN numbers and scales, infinite scales: they reach the outputs that they are terms of and no others."""
    k, n = 400, 300
    x, xs = rows_of(m, k, 1)
    w, ws = matrix_of((), n, k, 2)
    clean = torch_ops.fp8_matmul(x, xs, w, ws)
    clean_rows = torch_ops.fp8_gated(x, xs, w, ws, w, ws)
    bad = x.clone()
    bad.view(torch.uint8)[1, 399] = 0x7F
    y = torch_ops.fp8_matmul(bad, xs, w, ws)
    keep = torch.arange(m, device="cuda") != 1
    assert y[1].isnan().all() and torch.equal(y[keep], clean[keep])
    rows = torch_ops.fp8_gated(bad, xs, w, ws, w, ws)
    assert rows.scales[1].isnan().all() and rows.q[1].float().isnan().all()
    assert torch.equal(rows.scales[keep], clean_rows.scales[keep])
    bad = w.clone()
    bad.view(torch.uint8)[299, 0] = 0xFF
    y = torch_ops.fp8_matmul(x, xs, bad, ws)
    assert y[:, 299].isnan().all() and torch.equal(y[:, :299], clean[:, :299])
    bad = ws.clone()
    bad[0, 3] = math.inf
    y = torch_ops.fp8_matmul(x, xs, w, bad)
    assert (~y[:, :128].isfinite()).all() and torch.equal(y[:, 128:], clean[:, 128:])
    bad = xs.clone()
    bad[0, 0] = math.nan
    y = torch_ops.fp8_matmul(x, bad, w, ws)
    assert y[0].isnan().all() and torch.equal(y[1:], clean[1:])
    zero = torch_ops.fp8_gated(torch.zeros_like(x), xs, w, ws, w, ws)
    assert (zero.q.float() == 0).all() and (zero.scales == 2.0 ** -126).all()
    big = torch_ops.fp8_matmul(x, xs * 1e5, w, ws, out_dtype=torch.float16)  # past the type's range
    assert big.isinf().any() and not big.isnan().any()


@pytest.mark.gpu
def test_empty(torch_cuda):
    x, w, up = rows_of(4, 128, 1), matrix_of((), 96, 128, 2), matrix_of((), 96, 128, 3)
    assert torch_ops.fp8_matmul(x[0][:0], x[1][:0], *w).shape == (0, 96)
    assert torch_ops.fp8_matmul(*x, w[0][:0], w[1][:0]).shape == (4, 0)
    rows = torch_ops.fp8_gated(x[0][:0], x[1][:0], *w, *up)
    assert rows.q.shape == (0, 96) and rows.scales.shape == (0, 1)
    rows = torch_ops.fp8_gated(*x, w[0][:0], w[1][:0], up[0][:0], up[1][:0])
    assert rows.q.shape == (4, 0) and rows.scales.shape == (4, 0)
    w3, none = matrix_of((3,), 96, 128, 4), torch.zeros(0, dtype=torch.int32, device="cuda")
    counts = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert torch_ops.moe_fp8_matmul(*x, *w3, counts, none).shape == (0, 96)
    order = torch.arange(8, dtype=torch.int32, device="cuda")  # no slot has an expert
    assert not torch_ops.moe_fp8_matmul(*x, *w3, counts, order).any()
    rows = torch_ops.moe_fp8_gated(*x, *w3, *w3, counts, order)
    assert (rows.q.float() == 0).all() and (rows.scales == 2.0 ** -126).all()


MOE_CASES = [(1, 4, 2, 130, 144, 0.0), (7, 8, 2, 64, 272, 0.3), (40, 3, 1, 257, 128, 0.1), (200, 16, 3, 200, 400, 0.2),
             (600, 5, 2, 300, 256, 0.1), (1500, 4, 2, 140, 400, 0.05), (300, 200, 4, 96, 128, 0.0), (90, 1024, 2, 33, 16, 0.1),
             (2500, 2, 1, 520, 528, 0.0), (9000, 5, 2, 520, 1040, 0.1), (9000, 7, 2, 519, 1040, 0.0), (1500, 4, 2, 1000, 1040, 0.2),
             (6000, 600, 1, 130, 528, 0.0),
             # gated by way of a workspace, with few slots and with many an expert
             (1, 8, 2, 1792, 4096, 0.0), (3, 4, 2, 301, 4096, 0.2), (16, 2, 2, 200, 4096, 0.0), (174, 5, 4, 396, 3008, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top_k,n,k,drop", MOE_CASES)
def test_experts(torch_cuda, tokens, experts, top_k, n, k, drop):
    x, w, up = rows_of(tokens, k, 1), matrix_of((experts,), n, k, 2), matrix_of((experts,), n, k, 3)
    ids, counts, order = routing(tokens, experts, top_k, 4, drop)
    weights = torch.randn(tokens * top_k, generator=_gen(5), device="cuda")
    for dtype in TYPES:
        check_moe(torch_ops.moe_fp8_matmul(*x, *w, counts, order, out_dtype=dtype), *x, *w, ids, dtype == torch.float32)
    check_moe(torch_ops.moe_fp8_matmul(*x, *w, counts, order, row_weights=weights), *x, *w, ids, False, weights)
    rows = torch_ops.moe_fp8_gated(*x, *w, *up, counts, order, activation="gelu")
    check_moe_gated(rows, *x, w, up, ids, "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,n,k", [(37, 140, 144), (700, 140, 144), (9000, 520, 1040), (5, 139, 4096), (60, 139, 4096)])
def test_counts_and_order_are_not_trusted(torch_cuda, tokens, n, k):
    """Negative counts are 0, counts past the rows are cut, entries outside [0, R) are dropped, rows that the order does not
    name stay as they were; in a slot named twice each value is one of its products."""
    experts, top_k = 4, 2
    rows, in_n, in_k = tokens * top_k, blocks(n), blocks(k)
    x, w = rows_of(tokens, k, 1), matrix_of((experts,), n, k, 2)
    up = matrix_of((experts,), n, k, 3)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(3)).int().cuda()
    order[5], order[9] = -3, rows + 7  # two slots that nothing names
    lost = sorted(set(range(rows)) - set(order.tolist()))
    counts = torch.tensor([rows // 2, -5, 1 << 30, 1 << 30], dtype=torch.int32, device="cuda")
    expert = torch.where(torch.arange(rows) < rows // 2, 0, 2)
    for gate, with_workspace in ((0, False), (1, False), (1, True)):
        y = torch.full((rows, n), 0x55, dtype=torch.uint8, device="cuda") if gate else torch.full((rows, n), 77.0, device="cuda")
        scales = torch.full((rows, in_n), 77.0, device="cuda")
        args = _lib.GGKFp8Args(
            rows=rows, x_rows=tokens, n=n, k=k, experts=experts, gate=gate, x=x[0].data_ptr(), ldx=k, x_scales=x[1].data_ptr(), ldxs=in_k,
            w=w[0].data_ptr(), ldw=k, stride_w=n * k, w_scales=w[1].data_ptr(), ldws=in_k, stride_ws=in_n * in_k, counts=counts.data_ptr(),
            order=order.data_ptr(), y=y.data_ptr(), ldy=n, y_type=_lib.GGK_TYPE_F32)
        if gate:
            args.up, args.ldu, args.stride_u = up[0].data_ptr(), k, n * k
            args.up_scales, args.ldus, args.stride_us = up[1].data_ptr(), in_k, in_n * in_k
            args.y_scales, args.ldys = scales.data_ptr(), in_n
        if with_workspace:
            wanted = ctypes.c_longlong(-1)
            assert _lib.lib().ggk_fp8_workspace(ctypes.byref(args), ctypes.byref(wanted)) == 0
            assert wanted.value == (2 * rows * ((n + 3) // 4 * 4) if k == 4096 else 0)
            workspace = torch.full((wanted.value + 4,), math.nan, device="cuda")
            args.workspace = workspace.data_ptr()
        assert _lib.lib().ggk_fp8_multiply(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
        ids = torch.full((rows,), -2)
        for place, slot in enumerate(order.tolist()):
            if 0 <= slot < rows:
                ids[slot] = expert[place]
        ids = ids.cuda()
        if gate:
            named = (ids >= 0).nonzero()[:, 0]
            assert (y[lost] == 0x55).all() and (scales[lost] == 77).all()
            xv = row_values(*x)
            for e in (0, 2):
                at = named[ids[named] == e]
                check_gated(torch_ops.Fp8Rows(y[at].view(FP8), scales[at]), xv[at // top_k], matrix_values(w[0][e], w[1][e]),
                            matrix_values(up[0][e], up[1][e]))
        else:
            assert (y[lost] == 77).all()
            y[lost] = 0
            check_moe(y, *x, *w, torch.where(ids < 0, -1, ids), True)
    twice = torch.zeros(rows, dtype=torch.int32, device="cuda")
    y = torch_ops.moe_fp8_matmul(*x, *w, counts, twice, out_dtype=torch.float32)
    xv = row_values(*x)[:1]
    both = torch.cat([xv @ matrix_values(w[0][e], w[1][e]).t() for e in (0, 2)])
    # Its columns are made by many workgroups: each value is one or the other's.
    assert bool(((y[0].double() - both).abs() <= 1e-4 * both.abs().max()).any(0).all())


@pytest.mark.gpu
def test_expert_strides_and_offsets_past_32_bits(torch_cuda):
    """Matrices of a wider tensor, matrices more than 4 GB apart, one for all experts, and x of more than 4 GB."""
    n, k, experts = 140, 144, 3
    x, w, up = rows_of(50, k, 1), matrix_of((experts,), n, k, 2), matrix_of((experts,), n, k, 3)
    ids, counts, order = routing(50, experts, 2, 4)
    wide = torch.full((experts, n + 5, 176), 0x7F, dtype=torch.uint8, device="cuda")
    wide[:, :n, 16:160] = w[0].view(torch.uint8)
    check_moe(torch_ops.moe_fp8_matmul(*x, wide.view(FP8)[:, :n, 16:160], w[1], counts, order), *x, *w, ids, False)
    far = torch.empty(experts, 3 << 29, dtype=torch.uint8, device="cuda")[:, :n * k].view(experts, n, k)
    far.copy_(w[0].view(torch.uint8))
    check_moe(torch_ops.moe_fp8_matmul(*x, far.view(FP8), w[1], counts, order), *x, *w, ids, False)
    check_moe_gated(torch_ops.moe_fp8_gated(*x, far.view(FP8), w[1], *up, counts, order), *x, w, up, ids)
    shared, scales = w[0].view(torch.uint8)[:1].expand(experts, n, k).view(FP8), w[1][:1].expand(experts, 2, 2)
    check_moe(torch_ops.moe_fp8_matmul(*x, shared, scales, counts, order), *x, shared, scales, ids, False)
    del far
    rows = 2 ** 32 // 4096 + 700
    big = torch.zeros(rows, 4096, dtype=torch.uint8, device="cuda").view(FP8)[:, :k]
    big.view(torch.uint8)[-50:] = x[0].view(torch.uint8)
    big_scales = torch.ones(rows, 2, device="cuda")
    big_scales[-50:] = x[1]
    check_product(torch_ops.fp8_matmul(big, big_scales, w[0][0], w[1][0])[-50:], row_values(*x), matrix_values(w[0][0], w[1][0]), False)
    last = torch.arange(rows - 50, rows, device="cuda")
    slots = torch.cat([last, torch.arange(rows - 50, device="cuda")]).int()  # the last rows first
    counts = torch.tensor([20, 600, rows - 620], dtype=torch.int32, device="cuda")
    y = torch_ops.moe_fp8_matmul(big, big_scales, *w, counts, slots)
    got = torch.full((50,), 1, device="cuda")
    got[:20] = 0
    check_moe(y[last], *x, *w, got, False)
    assert not y[:rows - 50].any()


@pytest.mark.gpu
def test_long_matrix_past_32_bits(torch_cuda):
    n, k = 2 ** 32 // 4096 + 100, 4096
    w = torch.zeros(n, k, dtype=torch.uint8, device="cuda").view(FP8)
    ws = torch.ones(blocks(n), blocks(k), device="cuda")
    tail = numbers((100, k), 5)
    w.view(torch.uint8)[-100:] = tail.view(torch.uint8)
    for m in (2, 300):
        x = rows_of(m, k, 6)
        y = torch_ops.fp8_matmul(*x, w, ws)
        check_product(y[:, -100:], row_values(*x), tail.double(), False)
        assert not y[:, :-100].any()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,n,k", [(90, 140, 272), (9000, 520, 1040)])
def test_streams_graphs_and_threads(torch_cuda, tokens, n, k):
    experts = 6
    w, up = matrix_of((experts,), n, k, 1), matrix_of((experts,), n, k, 2)
    inputs = [torch.randn(tokens, k, generator=_gen(i), device="cuda").bfloat16() for i in range(5)]
    routes = [routing(tokens, experts, 2, i, 0.1)[1:] for i in range(5)]
    dense = matrix_of((), 400, k, 4)

    def layer(x, counts, order):
        h = torch_ops.rms_norm_fp8(x, None, x, plain=True)
        a = torch_ops.moe_fp8_gated(h.q, h.scales, *w, *up, counts, order)
        b = torch_ops.moe_fp8_matmul(h.q, h.scales, *w, counts, order)
        return h.y, h.residual, a.q.view(torch.uint8), a.scales, b, torch_ops.fp8_matmul(h.q, h.scales, *dense)

    def same(a, b):
        return all(torch.equal(p, q) for p, q in zip(a, b))

    eager = [layer(x, *r) for x, r in zip(inputs, routes)]
    assert all(same(layer(x, *r), e) for x, r, e in zip(inputs, routes, eager))  # the same call gives the same bits
    torch.cuda.synchronize()
    got = []
    for x, r in zip(inputs, routes):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(layer(x, *r))
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(got, eager))
    results = [None] * 5

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                results[i] = layer(inputs[i], *routes[i])
        torch.cuda.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(5)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(same(a, b) for a, b in zip(results, eager))
    x, counts, order = inputs[0].clone(), routes[0][0].clone(), routes[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, counts, order)
    for i in (3, 1, 4, 2):
        x.copy_(inputs[i])
        counts.copy_(routes[i][0])
        order.copy_(routes[i][1])
        graph.replay()
        assert same(out, eager[i])
        layer(inputs[i], *routes[i])
        torch.cuda.synchronize()


# ---------------------------------------------------------------- the layer

@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 8, 2), (50, 16, 4), (700, 6, 2)])
def test_layer(torch_cuda, tokens, experts, top_k):
    """A mixture-of-experts layer in 8 bits: norm with the residual, routing from its 16-bit rows, gated projections, down
    projection with the routing's weights, their sum onto the residual, the next norm; every step against 64 bits on that
    step's own inputs.  Padding tokens end as their residual."""
    width, inner = 256, 208
    gate, up, down = (matrix_of((experts,), *shape, seed) for shape, seed in
                      (((inner, width), 1), ((inner, width), 2), ((width, inner), 3)))
    g = _gen(9)
    x = torch.randn(tokens, width, generator=g, device="cuda").bfloat16()
    stream = torch.randn(tokens, width, generator=g, device="cuda").bfloat16()
    weight = (1 + 0.1 * torch.randn(width, generator=g, device="cuda")).bfloat16()
    router = torch.randn(width, experts, generator=g, device="cuda").bfloat16()
    mask = torch.ones(tokens, dtype=torch.bool, device="cuda")
    mask[1::7] = False
    h = torch_ops.rms_norm_fp8(x, weight, stream, plain=True)
    check_norm(h, x, weight, stream)
    r = torch_ops.moe_route(h.y @ router, top_k, token_mask=mask)
    a = torch_ops.moe_fp8_gated(h.q, h.scales, *gate, *up, r.counts, r.order)
    check_moe_gated(a, h.q, h.scales, gate, up, r.ids)
    y = torch_ops.moe_fp8_matmul(a.q, a.scales, *down, r.counts, r.order, row_weights=r.weights)
    check_moe(y, a.q, a.scales, *down, r.ids.view(-1, 1), False, r.weights)
    total = y.view(tokens, top_k, width).sum(1)
    after = torch_ops.rms_norm_fp8(total, weight, h.residual)
    check_norm(after, total, weight, h.residual)
    assert torch.equal(after.residual[~mask], h.residual[~mask])
