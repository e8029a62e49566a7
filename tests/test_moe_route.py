"""Routing of a mixture-of-experts layer (csrc/gg_route.hip, torch_ops.moe_route) against a plain numpy
statement of it in 64 bits: ids, counts and order equal; weights, loss and gradient within bounds that
count the float32 roundings on the way.

With u = 2^-24 and d the spread of a row's finite logits, expf's argument z - max is off by at most u d,
the function by 2 u, so exp is off by (d + 2) u relative; sums of at most 1024 such terms, held in
lanes and added in a tree or in runs of at most 1024 (partial sums over tokens likewise), add at most
32 u for every chain of additions here; a division and a product 2 u.  A weight is off by at most
2 (d + 32) u relative, the loss, two such sums deep, by 4 (d + 32) u, and a gradient by 4 (d + 32) u of
the sum of the magnitudes that it is a difference of, and half a step of its type."""
import ctypes
import math
import subprocess
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

from grouped_gemm_gpu_kernel_amd import _lib, torch_ops

U = 2.0 ** -24
TINY = 2.0 ** -120  # exp of arguments below -88 is flushed to 0 or loses bits


# ---------------------------------------------------------------- the definition

def plain_route(z, top_k=None, ids=None, mask=None, normalize=True, scale=1.0):
    """float64 logits -> dict of weights, ids, counts, order, loss, p (softmax), routed, f."""
    z = np.asarray(z, np.float64)
    tokens, experts = z.shape
    live = np.ones(tokens, bool) if mask is None else np.asarray(mask, bool)
    if ids is None:
        out = np.full((tokens, top_k), -1, np.int64)
        for t in range(tokens):
            if live[t]:
                best = sorted(range(experts), key=lambda e: (not np.isnan(z[t, e]), -z[t, e] if z[t, e] == z[t, e] else 0, e))
                best = [e for e in best if not z[t, e] == -np.inf][:top_k]
                out[t, :len(best)] = best
    else:
        out = np.asarray(ids, np.int64).copy()
        for t in range(tokens):
            for s in range(out.shape[1]):
                e = out[t, s]
                if not live[t] or e < 0 or e >= experts or z[t, e] == -np.inf:
                    out[t, s] = -1
    has = out >= 0
    routed = has.any(axis=1)
    flat = np.where(has, out, experts).reshape(-1)
    counts = np.bincount(flat, minlength=experts + 1)[:experts]
    order = np.argsort(flat, kind="stable")
    p = np.zeros_like(z)
    a = np.zeros(out.shape)
    with np.errstate(all="ignore"):
        for t in np.flatnonzero(routed):
            e = np.exp(z[t] - np.fmax.reduce(z[t]))
            p[t] = e / e.sum()
            zs = z[t, out[t][has[t]]]
            if normalize:
                e = np.exp(zs - np.fmax.reduce(zs))
                a[t, has[t]] = e / e.sum()
            else:
                a[t, has[t]] = p[t, out[t][has[t]]]
    n, total = int(routed.sum()), int(counts.sum())
    f = counts / max(1, total)
    loss = experts * float((f * (p.sum(axis=0) / max(1, n))).sum())
    return {"weights": scale * a, "a": a, "ids": out, "counts": counts, "order": order, "loss": loss, "p": p,
            "routed": routed, "has": has, "f": f, "n": n}


def plain_gradient(r, normalize, scale, d_weights=None, d_loss=None):
    """The gradient with respect to the logits, and the sum of the magnitudes of its terms."""
    p, a, ids, has = r["p"], r["a"], r["ids"], r["has"]
    tokens, experts = p.shape
    d, size = np.zeros_like(p), np.zeros_like(p)
    for t in np.flatnonzero(r["routed"]):
        if d_loss is not None:
            c = d_loss * experts * r["f"] / r["n"]
            d[t] += p[t] * (c - (p[t] * c).sum())
            size[t] += p[t] * (np.abs(c) + (p[t] * np.abs(c)).sum())
        if d_weights is not None:
            g = np.where(has[t], scale * d_weights[t], 0.0)
            mean, spread = (a[t] * g).sum(), (a[t] * np.abs(g)).sum()
            for s in np.flatnonzero(has[t]):
                e = ids[t, s]
                d[t, e] += a[t, s] * (g[s] - mean) if normalize else a[t, s] * g[s]
                size[t, e] += a[t, s] * (abs(g[s]) + spread)
            if not normalize:
                d[t] -= p[t] * mean
                size[t] += p[t] * spread
    return d, size


def spread_of(z):
    fine = np.where(np.isfinite(z), z, np.nan)
    with np.errstate(all="ignore"):
        d = np.nanmax(fine, axis=1) - np.nanmin(fine, axis=1) if z.size else np.zeros(len(z))
    return np.minimum(np.nan_to_num(d), 200.0)[:, None]


# ---------------------------------------------------------------- CPU

def _c_layout(tmp_path, struct, mirror):
    fields = [f for f, _ in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "grouped_gemm_amd_kernels.h"\n'
                   f'int main(void) {{\n  printf("%zu\\n", sizeof({struct}));\n' +
                   "".join(f'  printf("%zu\\n", offsetof({struct}, {f}));\n' for f in fields) + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    root = Path(__file__).resolve().parents[1]
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{root / 'include'}", str(src),
                    "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    return got, [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


@pytest.mark.parametrize("struct,mirror", [("ggk_route_args", _lib.GGKRouteArgs),
                                           ("ggk_route_gradient_args", _lib.GGKRouteGradientArgs)])
def test_structs_mirror_the_header(tmp_path, struct, mirror):
    got, want = _c_layout(tmp_path, struct, mirror)
    assert got == want


def _route_args(**over):
    size = _lib.lib().ggk_route_workspace(over.get("tokens", 10), 8)
    args = dict(tokens=10, experts=8, slots=2, type=_lib.GGK_TYPE_F32, logits=0x1000, ld=8, normalize=1, scale=1.0,
                weights=0x1000, ids=0x1000, counts=0x1000, order=0x1000, workspace=0x1000, workspace_bytes=size)
    args.update(over)
    return _lib.GGKRouteArgs(**args)


@pytest.mark.parametrize("over,status", [
    ({}, 0), ({"tokens": -1}, 1), ({"experts": 0}, 1), ({"experts": 1025, "ld": 1025}, 1), ({"slots": 0}, 1),
    ({"slots": 9}, 1), ({"slots": 9, "given_ids": 0x1000}, 0), ({"slots": 65, "given_ids": 0x1000}, 1),
    ({"type": 3}, 1), ({"ld": 7}, 1), ({"tokens": 1, "ld": 0}, 0), ({"workspace": None, "workspace_bytes": 0}, 0), ({"logits": None}, 17),
    ({"counts": None}, 17), ({"order": None}, 17), ({"loss": 0x1000}, 17), ({"slope": 0x1000}, 17),
    ({"loss": 0x1000, "slope": 0x1000}, 0), ({"tokens": (1 << 29) + 1}, 1), ({"tokens": 1 << 29}, 0),
    ({"tokens": 1000, "workspace_bytes": 0}, 1), ({"tokens": 1000, "workspace": None}, 17),
    ({"tokens": 1000, "workspace": 0x1008}, 1),
    ({"tokens": 0, "logits": None, "weights": None, "ids": None, "order": None}, 0)])
def test_route_arguments_are_checked_on_the_host(over, status):
    assert _lib.lib().ggk_route_check(ctypes.byref(_route_args(**over))) == status
    assert _lib.lib().ggk_route_check(None) == 1
    assert _lib.lib().ggk_route(None, None) == 1 and _lib.lib().ggk_route_gradient(None, None) == 1
    if status:  # refused before anything is launched
        assert _lib.lib().ggk_route(ctypes.byref(_route_args(**over)), None) == status


def test_route_gradient_arguments_are_checked_on_the_host():
    def status(**over):
        args = dict(tokens=10, experts=8, slots=2, type=_lib.GGK_TYPE_F16, logits=0x1000, ld=8, ids=0x1000,
                    d_logits=0x1000)
        args.update(over)
        return _lib.lib().ggk_route_gradient_check(ctypes.byref(_lib.GGKRouteGradientArgs(**args)))

    assert status() == 0 and status(d_loss=0x1000, slope=0x1000) == 0
    assert status(d_loss=0x1000) == 17 and status(logits=None) == 17 and status(d_logits=None) == 17
    assert status(type=-1) == 1 and status(ld=3) == 1 and status(experts=0) == 1 and status(slots=65) == 1


def test_few_tokens_take_no_workspace():
    """One workgroup routes 128 tokens of up to 256 experts, and 32 above, where each takes a wave."""
    size = _lib.lib().ggk_route_workspace
    for experts, most in ((1, 128), (64, 128), (256, 128), (257, 32), (512, 32), (768, 32), (769, 0), (1024, 0)):
        assert size(most, experts) == 0 or most == 0
        assert size(most + 1, experts) > 0


def test_refusals_of_the_torch_call():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with pytest.raises(ValueError, match="on a GPU"):
        torch_ops.moe_route(torch.zeros(3, 4), 2)
    with pytest.raises(TypeError, match="torch.Tensor"):
        torch_ops.moe_route([[1.0]], 1)
    with FakeTensorMode():
        def logits(*shape, dtype=torch.float32):
            return torch.empty(*shape, dtype=dtype, device="cuda:0")

        z = logits(6, 8)
        for bad, error, text in [
                ((logits(6, 8, dtype=torch.float64), 2), TypeError, "float32, float16 or bfloat16"),
                ((logits(6), 2), ValueError, "2-D"), ((logits(6, 8).t(), 2), ValueError, "contiguous rows"),
                ((logits(1, 8).expand(6, 8), 2), ValueError, "rows overlap"), ((logits(6, 0), 1), ValueError, "experts"),
                ((logits(6, 1025), 1), ValueError, "experts"), ((z, 0), ValueError, "top_k"),
                ((z, 9), ValueError, "top_k"), ((logits(6, 100), 65), ValueError, "top_k"), ((z,), ValueError, "one of"),
                ((z, 2.0), TypeError, "integer")]:
            with pytest.raises(error, match=text):
                torch_ops.moe_route(*bad)
        ids = torch.empty(6, 2, dtype=torch.int32, device="cuda:0")
        mask = torch.empty(6, dtype=torch.bool, device="cuda:0")
        for bad, error, text in [
                ({"ids": ids, "top_k": 2}, ValueError, "one of"), ({"ids": ids.long()}, TypeError, "int32"),
                ({"ids": ids[:5]}, ValueError, "ids must be"), ({"ids": ids.t().contiguous().t()}, ValueError, "contiguous"),
                ({"ids": ids.cpu()}, ValueError, "expected cuda"), ({"ids": ids[:, :0]}, ValueError, "slots"),
                ({"top_k": 2, "token_mask": mask.int()}, TypeError, "bool"),
                ({"top_k": 2, "token_mask": mask[:5]}, ValueError, "entries"),
                ({"top_k": 2, "token_mask": torch.empty(12, dtype=torch.bool, device="cuda:0")[::2]}, ValueError,
                 "contiguous")]:
            with pytest.raises(error, match=text):
                torch_ops.moe_route(z, **bad)
        with pytest.raises(ValueError, match="2\\^30"):
            torch_ops.moe_route(logits((1 << 27) + 1, 8), 8)


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_derivatives_are_refused(requires_grad):
    """A dual tensor does not require a gradient by itself; its tangent would be lost without a word."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad

    with FakeTensorMode(), forward_ad.dual_level():
        z = torch.empty(6, 8, device="cuda:0")
        dual = forward_ad.make_dual(z.requires_grad_(requires_grad), torch.empty(6, 8, device="cuda:0"))
        ids = torch.empty(6, 2, dtype=torch.int32, device="cuda:0")
        for arguments in ({"top_k": 2}, {"top_k": 2, "balance": True}, {"ids": ids}):
            with pytest.raises(RuntimeError, match="forward-mode derivative: logits"):
                torch_ops.moe_route(dual, **arguments)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode derivative: logits"):
                torch_ops.moe_route(dual, **arguments)


# ---------------------------------------------------------------- GPU

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _check(z, top_k=None, ids=None, mask=None, normalize=True, scale=1.0, d_weights=None, d_loss=None):
    """moe_route with its gradient, against the definition; z is a GPU tensor."""
    leaf = z.detach().requires_grad_(True) if z.is_contiguous() else z.detach()
    leaf.requires_grad_(True)
    r = torch_ops.moe_route(leaf, top_k, ids=ids, token_mask=mask, normalize=normalize, scale=scale, balance=True)
    z64 = z.detach().double().cpu().numpy()
    want = plain_route(z64, top_k, None if ids is None else ids.cpu().numpy(),
                       None if mask is None else mask.cpu().numpy(), normalize, scale)
    assert r.ids.dtype == r.counts.dtype == r.order.dtype == torch.int32
    np.testing.assert_array_equal(r.ids.cpu().numpy(), want["ids"])
    np.testing.assert_array_equal(r.counts.cpu().numpy(), want["counts"])
    np.testing.assert_array_equal(r.order.cpu().numpy(), want["order"])
    d = spread_of(z64)
    w = r.weights.detach().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(w), np.isnan(want["weights"]))
    fine = ~np.isnan(w)
    off = np.abs(w - want["weights"])
    assert (off[fine] <= (np.abs(want["weights"]) * 2 * (d + 32) * U + TINY)[fine]).all()
    assert (w[~want["has"]] == 0).all()
    loss = float(r.balance_loss)
    if math.isnan(want["loss"]):
        assert math.isnan(loss)
    else:
        assert abs(loss - want["loss"]) <= want["loss"] * 4 * (float(d.max(initial=0)) + 32) * U + TINY
    # without a gradient, the same call gives the same bits
    with torch.no_grad():
        again = torch_ops.moe_route(leaf, top_k, ids=ids, token_mask=mask, normalize=normalize, scale=scale)
    assert again.balance_loss is None and not again.weights.requires_grad
    for x, y in zip(again[:4], r[:4]):
        assert torch.equal(x.view(torch.int32), y.detach().view(torch.int32))
    outs, grads = [], []
    if d_weights is not None:
        outs.append(r.weights)
        grads.append(d_weights)
    if d_loss is not None:
        outs.append(r.balance_loss)
        grads.append(torch.full((), d_loss, device="cuda"))
    got, = torch.autograd.grad(outs, leaf, grads)
    assert got.dtype == z.dtype and got.shape == z.shape
    grad, size = plain_gradient(want, normalize, scale,
                                None if d_weights is None else d_weights.double().cpu().numpy(), d_loss)
    got = got.double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(grad))
    step = torch.finfo(z.dtype).eps / 2
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: TINY, torch.float32: TINY}[z.dtype]
    bound = size * 4 * (d + 32) * U + np.abs(grad) * step * 1.01 + least
    fine = ~np.isnan(grad)
    assert (np.abs(got - grad)[fine] <= bound[fine]).all(), np.nanmax(np.abs(got - grad) / bound)
    return r


def _logits(tokens, experts, dtype, seed, ties=False):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(tokens, experts, generator=g) * 2
    if ties:
        z = z.round()
    return z.to(TYPES[dtype]).cuda()


SHAPES = [(1, 1, 1), (1, 64, 2), (2, 2, 2), (3, 5, 1), (17, 16, 4), (63, 17, 3), (64, 32, 32), (65, 33, 5), (130, 48, 6),
          (100, 64, 64), (257, 65, 8), (70, 128, 2), (33, 129, 7), (40, 200, 16), (90, 256, 8), (31, 257, 17), (20, 511, 10),
          (35, 512, 64), (19, 777, 1), (66, 1000, 33), (23, 1024, 64), (1025, 40, 4), (4097, 12, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,experts,top_k", SHAPES)
def test_shapes_and_types(torch_cuda, tokens, experts, top_k, dtype):
    z = _logits(tokens, experts, dtype, tokens * 7 + experts)
    dw = torch.randn(tokens, top_k, generator=torch.Generator().manual_seed(1)).cuda()
    for normalize, scale in ((True, 1.0), (False, 2.5)):
        _check(z, top_k, normalize=normalize, scale=scale, d_weights=dw, d_loss=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [32, 33, 100, 128, 129])
@pytest.mark.parametrize("experts,top_k", [(256, 8), (257, 8), (700, 20)])
def test_few_tokens_of_many_experts(torch_cuda, tokens, experts, top_k):
    """Both sides of what one workgroup routes."""
    z = _logits(tokens, experts, "bf16", tokens + experts)
    dw = torch.randn(tokens, top_k, generator=torch.Generator().manual_seed(1)).cuda()
    mask = (torch.rand(tokens, generator=torch.Generator().manual_seed(2)) < 0.8).cuda()
    _check(z, top_k, mask=mask, d_weights=dw, d_loss=0.4)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [511, 16385, 40000])
def test_many_tokens(torch_cuda, tokens):
    """More blocks of tokens than one, ragged ends; popular experts."""
    z = _logits(tokens, 24, "f32", tokens) + torch.linspace(3, 0, 24, device="cuda")
    dw = torch.randn(tokens, 3, generator=torch.Generator().manual_seed(1)).cuda()
    mask = (torch.rand(tokens, generator=torch.Generator().manual_seed(2)) < 0.8).cuda()
    _check(z, 3, mask=mask, d_weights=dw, d_loss=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("experts,top_k", [(9, 4), (64, 8), (100, 12), (256, 16), (600, 20), (1024, 64)])
@pytest.mark.parametrize("normalize", [True, False])
def test_ties_masks_and_odd_values(torch_cuda, experts, top_k, normalize):
    """Ties (signed zeros too), rows with every expert closed, rows with fewer open ones than slots, padding,
    the type's lowest value, wide rows."""
    z = _logits(120, experts, "f32", experts, ties=True)
    z[0] = -math.inf
    z[1] = 0.0
    z[2] = torch.where(torch.arange(experts, device="cuda") % 2 == 0, 0.0, -0.0)
    z[3, 1:] = -math.inf
    z[4, : experts - 2] = -math.inf
    z[5] = torch.finfo(torch.float32).min
    z[6, ::2] = torch.finfo(torch.float32).min
    z[7] *= 40
    z[8, : experts // 2] = -math.inf
    mask = torch.ones(120, dtype=torch.bool, device="cuda")
    mask[20:30] = False
    mask[-1] = False
    z[25] = math.nan  # padding may hold anything
    z[26] = math.inf
    dw = torch.randn(120, top_k, generator=torch.Generator().manual_seed(1)).cuda()
    _check(z, top_k, mask=mask, normalize=normalize, scale=0.7, d_weights=dw, d_loss=0.5)
    _check(z, top_k, mask=torch.zeros_like(mask), normalize=normalize, d_weights=dw, d_loss=0.5)  # nothing routed


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [10, 64, 300])
@pytest.mark.parametrize("normalize", [True, False])
def test_nan_and_infinity_show(torch_cuda, experts, normalize):
    """A NaN or +inf logit of an unmasked token is chosen first and makes that row NaN, and no other."""
    z = _logits(30, experts, "f32", experts)
    z[3, 7] = math.nan
    z[4, 2] = z[4, 5] = math.nan
    z[5, 1] = math.inf
    z[6, 0] = math.inf
    z[6, 9] = math.nan
    dw = torch.randn(30, 2, generator=torch.Generator().manual_seed(1)).cuda()
    r = _check(z, 2, normalize=normalize, d_weights=dw, d_loss=0.5)
    assert r.ids[3, 0] == 7 and r.ids[4].tolist() == [2, 5] and r.ids[5, 0] == 1 and r.ids[6].tolist() == [9, 0]
    assert not torch.isnan(r.weights[7:]).any() and math.isnan(float(r.balance_loss))
    mask = torch.ones(30, dtype=torch.bool, device="cuda")
    mask[3:7] = False
    assert math.isfinite(float(_check(z, 2, mask=mask, normalize=normalize, d_weights=dw, d_loss=0.5).balance_loss))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("experts", [100, 128, 255, 256, 300, 512, 1000, 1024])
def test_choices_held_by_few_lanes(torch_cuda, experts, dtype):
    """The best logits next to each other or in steps that put them all in one lane, sorted both ways, equal in runs,
    and with NaN at the first and last expert."""
    z = torch.zeros(12, experts)
    step = torch.arange(experts, dtype=torch.float32)
    z[0], z[1] = step / 64, -step / 64
    z[2, :20] = 4 + torch.arange(20) / 16
    z[3, -20:] = 4 - torch.arange(20) / 16
    for row, stride in ((4, 4), (5, 16), (6, 64)):
        z[row, ::stride] = 3 + torch.arange(len(z[row, ::stride])) / 64
    z[7] = (step / 7).floor()
    z[8] = -(step / 50).floor()
    z[9, 0] = z[9, -1] = math.nan
    z[10, 1::64] = 5
    z[11, 4:8] = torch.tensor([7.0, 6, 7, 6])
    z = z.repeat(13, 1).to(TYPES[dtype]).cuda()
    for top_k in (1, 3, 4, 9, 16, 17, 40):
        dw = torch.randn(len(z), top_k, generator=torch.Generator().manual_seed(1)).cuda()
        _check(z, top_k, d_weights=dw, d_loss=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("experts,slots", [(5, 3), (64, 4), (70, 64), (500, 6)])
@pytest.mark.parametrize("normalize", [True, False])
def test_given_experts(torch_cuda, experts, slots, normalize):
    """ids given: any order, the same expert twice, none, out of range, closed ones; rows with none left."""
    z = _logits(90, experts, "bf16", experts)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-2, experts + 2, (90, slots), generator=g).int()
    ids[0] = -1
    ids[1] = experts
    ids[2] = 3
    ids[3] = torch.iinfo(torch.int32).max
    ids[4] = torch.iinfo(torch.int32).min
    z[5, 2] = -math.inf
    ids[5] = 2
    z[6] = -math.inf
    dw = torch.randn(90, slots, generator=g).cuda()
    mask = torch.ones(90, dtype=torch.bool, device="cuda")
    mask[40:45] = False
    _check(z, ids=ids.cuda(), mask=mask, normalize=normalize, scale=1.5, d_weights=dw, d_loss=0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("experts", [8, 31, 64, 256])
def test_padded_and_unaligned_rows(torch_cuda, experts, dtype):
    wide = _logits(50, experts + 13, dtype, 5)
    dw = torch.randn(50, 2, generator=torch.Generator().manual_seed(1)).cuda()
    for off in (0, 1, 4, 8):
        _check(wide[:, off:off + experts], 2, d_weights=dw, d_loss=0.5)
    flat = _logits(1, 50 * experts + 1, dtype, 6).flatten()
    _check(flat[1:].view(50, experts), 2, d_weights=dw, d_loss=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [True, False])
def test_one_gradient_at_a_time(torch_cuda, normalize):
    z = _logits(300, 40, "f32", 9)
    dw = torch.randn(300, 4, generator=torch.Generator().manual_seed(1)).cuda()
    _check(z, 4, normalize=normalize, d_weights=dw)
    _check(z, 4, normalize=normalize, d_loss=2.0)
    leaf = z.clone().requires_grad_(True)
    r = torch_ops.moe_route(leaf, 4, normalize=normalize)  # no balance loss; an expanded incoming gradient
    r.weights.sum().backward()
    want, size = plain_gradient(plain_route(z.double().cpu().numpy(), 4, normalize=normalize), normalize, 1.0,
                                np.ones((300, 4)))
    assert (np.abs(leaf.grad.double().cpu().numpy() - want) <= size * 4 * (20 + 32) * U + 2 * U * np.abs(want) + TINY).all()
    assert not r.ids.requires_grad and not r.counts.requires_grad and not r.order.requires_grad


@pytest.mark.gpu
def test_gradient_against_differences(torch_cuda):
    """The definition's own gradient against central differences in 64 bits (step 1e-5: truncation 1e-10,
    rounding 1e-16 / 1e-5), and the kernel's against the definition's in _check."""
    z = _logits(12, 10, "f32", 4)
    dw = torch.randn(12, 3, generator=torch.Generator().manual_seed(1)).cuda()
    for normalize in (True, False):
        _check(z, 3, normalize=normalize, scale=1.3, d_weights=dw, d_loss=0.5)
        z64, dw64 = z.double().cpu().numpy(), dw.double().cpu().numpy()
        base = plain_route(z64, 3, normalize=normalize, scale=1.3)
        grad, _ = plain_gradient(base, normalize, 1.3, dw64, 0.5)

        def value(x):
            r = plain_route(x, ids=base["ids"], normalize=normalize, scale=1.3)
            return (r["weights"] * dw64).sum() + 0.5 * r["loss"]

        for t, e in [(0, 0), (3, 7), (5, int(base["ids"][5, 0])), (11, int(base["ids"][11, 2]))]:
            up, down = z64.copy(), z64.copy()
            up[t, e] += 1e-5
            down[t, e] -= 1e-5
            assert abs((value(up) - value(down)) / 2e-5 - grad[t, e]) < 1e-8


@pytest.mark.gpu
def test_a_second_derivative_is_refused(torch_cuda):
    z = _logits(20, 8, "f32", 2).requires_grad_(True)
    r = torch_ops.moe_route(z, 2, balance=True)
    d, = torch.autograd.grad((r.weights.square().sum() + r.balance_loss,), z, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()


@pytest.mark.gpu
def test_a_gradient_of_dual_tensors_is_refused(torch_cuda):
    """Forward mode over the backward pass: the tangents of the incoming gradients would be lost."""
    from torch.autograd import forward_ad

    z = _logits(20, 8, "f32", 2).requires_grad_(True)
    r = torch_ops.moe_route(z, 2, balance=True)
    dw, dl = torch.ones(20, 2, device="cuda"), torch.ones((), device="cuda")
    with forward_ad.dual_level():
        for grads in ((forward_ad.make_dual(dw, dw), dl), (dw, forward_ad.make_dual(dl, dl))):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad((r.weights, r.balance_loss), z, grads, retain_graph=True)
        torch.autograd.grad((r.weights, r.balance_loss), z, (dw, dl))


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [True, False])
def test_incoming_gradients_held_as_negatives_or_not_at_all(torch_cuda, normalize):
    """A lazily conjugated complex value's imaginary part holds its values' negatives, and a zero tensor nothing: the
    gradient of what they stand for."""
    z = _logits(40, 8, "f32", 2).requires_grad_(True)
    dw = torch.randn(40, 2, generator=torch.Generator().manual_seed(1)).cuda()
    dl = torch.full((), 0.3, device="cuda")

    def gradient(d_weights, d_loss):
        r = torch_ops.moe_route(z, 2, normalize=normalize, balance=True)
        return torch.autograd.grad((r.weights, r.balance_loss), z, (d_weights, d_loss))[0]

    def negative(t):
        t = torch.imag(torch.complex(t, -t).conj())
        assert t.is_neg()
        return t

    want = gradient(dw, dl)
    assert torch.equal(gradient(negative(dw), dl), want)
    assert torch.equal(gradient(dw, negative(dl)), want)
    none = torch._efficientzerotensor((40, 2), device="cuda")
    assert torch.equal(gradient(none, dl), gradient(torch.zeros_like(dw), dl))
    assert torch.equal(gradient(none, torch._efficientzerotensor((), device="cuda")), torch.zeros_like(z))
    # through torch's own operators
    r = torch_ops.moe_route(z, 2, normalize=normalize, balance=True)
    back, = torch.autograd.grad(torch.imag(torch.complex(dl, r.balance_loss).conj()), z)
    r = torch_ops.moe_route(z, 2, normalize=normalize, balance=True)
    assert torch.equal(back, torch.autograd.grad(-r.balance_loss, z)[0])


@pytest.mark.gpu
def test_saved_tensors_changed_in_place_are_noticed(torch_cuda):
    """ids changed before the backward pass raise; counts and order, which it does not read, may be."""
    z = _logits(200, 8, "f32", 2).requires_grad_(True)
    r = torch_ops.moe_route(z, 2, balance=True)
    r.counts.add_(1)
    r.order.zero_()
    r.weights.sum().backward()
    r = torch_ops.moe_route(z, 2, balance=True)
    r.ids.zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        r.weights.sum().backward()


@pytest.mark.gpu
def test_no_tokens(torch_cuda):
    z = torch.empty(0, 12, device="cuda", requires_grad=True)
    r = torch_ops.moe_route(z, 3, balance=True)
    assert r.weights.shape == r.ids.shape == (0, 3) and r.order.numel() == 0
    assert (r.counts == 0).all() and float(r.balance_loss) == 0.0
    got, = torch.autograd.grad((r.weights, r.balance_loss), z, (torch.empty(0, 3, device="cuda"), torch.ones((), device="cuda")))
    assert got.shape == (0, 12)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top_k", [(2 ** 25 + 7, 2, 1), (2 ** 21 + 3, 32, 17), (2 ** 20 + 5, 300, 4)])
@pytest.mark.parametrize("step", [0.25, 0.6, 0.9])
def test_loss_over_many_tokens(torch_cuda, tokens, experts, top_k, step):
    """The same logits for every token, so that the roundings of a running sum of p all go the same way.

    Sums of p make chains of at most 64 additions in a lane and 64 of such runs (2^25 tokens by 512 blocks of 32 groups
    are 2048 a lane), 10 over a block's groups and waves, 512 / 8 + 8 over the blocks: 210 u, and 16 u for p and what
    follows the sums."""
    row = (-torch.arange(experts) * step).bfloat16()
    row[experts // 2:] -= 1
    z = row.cuda().repeat(tokens, 1)
    r = torch_ops.moe_route(z, top_k, balance=True)
    p = np.exp(row.double().numpy())
    p /= p.sum()
    want = experts / top_k * p[:top_k].sum()
    assert r.counts.tolist() == [tokens] * top_k + [0] * (experts - top_k)
    assert abs(float(r.balance_loss) - want) <= 226 * U * want, (float(r.balance_loss) / want - 1) / U
    z.requires_grad_(True)
    r = torch_ops.moe_route(z, top_k, balance=True)
    got, = torch.autograd.grad(r.balance_loss, z, torch.full((), float(tokens), device="cuda"))
    c = np.where(np.arange(experts) < top_k, experts / top_k, 0.0)
    grad = p * (c - (p * c).sum())
    size = p * (c + (p * c).sum())
    bound = size * 4 * (20 + 32) * U + np.abs(grad) * 2.0 ** -8 * 1.01 + TINY
    assert (got == got[0]).all()  # equal rows, wherever they stand
    assert (np.abs(got[-1].double().cpu().numpy() - grad) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,slots,dtype", [(2 ** 21 + 11, 8, 2, "f32"), (1200007, 256, 4, "bf16"),
                                                        (1100003, 100, 3, "f16"), (400009, 520, 2, "f32")])
def test_loss_of_many_padded_tokens_and_given_experts(torch_cuda, tokens, experts, slots, dtype):
    """Random logits with sums of p in runs, padding, closed experts and experts given; against float64 of the same logits.

    The sums' chains as in test_loss_over_many_tokens (226 u in all), p off by (d + 32) u as for the weights."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    z = (torch.randn(tokens, experts, generator=g, device="cuda") * 2).to(TYPES[dtype])
    z[:, 3].masked_fill_(torch.rand(tokens, generator=g, device="cuda") < 0.3, -math.inf)
    mask = torch.rand(tokens, generator=g, device="cuda") < 0.9
    for ids in (None, torch.randint(-1, experts, (tokens, slots), generator=g, device="cuda", dtype=torch.int32)):
        r = torch_ops.moe_route(z, slots if ids is None else None, ids=ids, token_mask=mask, balance=True)
        routed = (r.ids >= 0).any(1)
        if ids is None:
            assert torch.equal(routed, mask)
        p, spread = torch.zeros(experts, dtype=torch.float64, device="cuda"), 0.0
        for part, on in zip(z.split(1 << 17), routed.split(1 << 17)):
            part = part[on].double()
            p += torch.softmax(part, 1).sum(0)
            spread = max(spread, float(part.amax() - part.masked_fill(part == -math.inf, math.inf).amin()))
        chosen = r.ids[r.ids >= 0].long()
        counts = torch.bincount(chosen, minlength=experts)
        assert torch.equal(r.counts.long(), counts)
        want = experts * float((counts / len(chosen) * p).sum() / routed.sum())
        assert abs(float(r.balance_loss) - want) <= (226 + spread + 32) * U * want
        flat = torch.where(r.ids < 0, experts, r.ids).flatten()
        assert torch.equal(r.order.long(), flat.sort(stable=True).indices)


@pytest.mark.gpu
def test_rows_past_32_bits(torch_cuda):
    """Logits whose last rows lie past 2^31 elements: 9 GB of bfloat16, of which a few rows are looked at."""
    experts, tokens = 1024, 2 ** 31 // 1024 + 1000
    z = torch.zeros(tokens, experts, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 5, tokens - 900, tokens - 1], device="cuda")
    z[at, at % experts] = 3.0
    z.requires_grad_(True)
    r = torch_ops.moe_route(z, 1, normalize=False, balance=True)
    want = math.exp(3.0) / (math.exp(3.0) + experts - 1)
    assert r.ids[at, 0].tolist() == (at % experts).tolist()
    assert (r.weights[at, 0] - want).abs().max() <= want * 2 * (3 + 32) * U
    expected = torch.bincount(at % experts, minlength=experts)
    expected[0] = tokens - 3  # every other row ties, and takes expert 0 (as row 0 does)
    assert torch.equal(r.counts.long(), expected)
    assert torch.equal(r.order.sort().values, torch.arange(tokens, dtype=torch.int32, device="cuda"))
    d_w = torch.zeros(tokens, 1, device="cuda")
    d_w[-1] = 1.0
    got, = torch.autograd.grad(r.weights, z, d_w)
    last = got[-1].double()
    e = (tokens - 1) % experts
    assert abs(float(last[e]) - want * (1 - want)) <= want * 2.0 ** -8
    assert not got[:-1].any()


@pytest.mark.gpu
def test_loss_and_its_gradient_past_32_bits(torch_cuda):
    """The loss over rows that end past 2^31 elements, and its gradient there.  Chains of additions as in
    test_loss_over_many_tokens, shorter ones (514 tokens a lane)."""
    experts, tokens = 1024, 2 ** 31 // 1024 + 1000
    z = torch.zeros(tokens, experts, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([5, tokens - 900, tokens - 1], device="cuda")
    z[at, at % experts] = 3.0
    z.requires_grad_(True)
    r = torch_ops.moe_route(z, 1, balance=True)
    chosen = (at % experts).tolist()
    counts = np.zeros(experts)
    counts[0] = tokens - len(chosen)
    p_sum = np.full(experts, (tokens - len(chosen)) / experts)
    total = math.exp(3.0) + experts - 1
    for e in chosen:
        counts[e] += 1
        p_sum += 1.0 / total
        p_sum[e] += (math.exp(3.0) - 1.0) / total
    f = counts / tokens
    want = experts * (f * p_sum / tokens).sum()
    assert abs(float(r.balance_loss) - want) <= 226 * U * want
    got, = torch.autograd.grad(r.balance_loss, z, torch.full((), float(tokens), device="cuda"))
    for row, e in ((3, None), (tokens - 2, None), (5, 5), (tokens - 1, chosen[-1])):
        p = np.full(experts, 1.0 / experts)
        if e is not None:
            p = np.full(experts, 1.0 / total)
            p[e] = math.exp(3.0) / total
        c = experts * f
        grad, size = p * (c - (p * c).sum()), p * (c + (p * c).sum())
        off = np.abs(got[row].double().cpu().numpy() - grad)
        assert (off <= size * 4 * (3 + 32) * U + np.abs(grad) * 2.0 ** -8 * 1.01 + TINY).all(), row


@pytest.mark.gpu
def test_streams_and_two_calls_at_once(torch_cuda):
    zs = [_logits(3000, 64, "f32", s) for s in range(4)]
    want = [torch_ops.moe_route(z, 4, balance=True) for z in zs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in zs]
    got = []
    for z, stream in zip(zs, streams):
        with torch.cuda.stream(stream):
            got.append(torch_ops.moe_route(z, 4, balance=True))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_calls_and_gradients_from_several_threads(torch_cuda):
    out = [None] * 6

    def work(i):
        z = _logits(3000, 64, "f32", i).requires_grad_(True)
        for _ in range(10):
            r = torch_ops.moe_route(z, 4, balance=True)
            out[i], = torch.autograd.grad(r.weights.square().sum() + r.balance_loss, z)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    together = list(out)
    for i in range(6):
        work(i)
    assert all(torch.equal(a, b) for a, b in zip(together, out))


@pytest.mark.gpu
def test_saved_on_the_host_and_computed_again(torch_cuda):
    """Saved logits that come back in other strides (padded rows, dense again from the host), and a checkpointed call."""
    from torch.utils.checkpoint import checkpoint

    z = _logits(300, 40, "bf16", 1)[:, 3:36].detach().requires_grad_(True)

    def value(z):
        r = torch_ops.moe_route(z, 4, balance=True)
        return r.weights.square().sum() + r.balance_loss

    want, = torch.autograd.grad(value(z), z)
    with torch.autograd.graph.save_on_cpu():
        assert torch.equal(torch.autograd.grad(value(z), z)[0], want)
    assert torch.equal(torch.autograd.grad(checkpoint(value, z, use_reentrant=False), z)[0], want)
    loss = value(z)
    for _ in range(2):  # the same graph twice
        assert torch.equal(torch.autograd.grad(loss, z, retain_graph=True)[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize("leaf", [True, False])
def test_capture_with_an_eager_graph_alive_is_refused(torch_cuda, leaf):
    """The leaf's gradient belongs to the default stream while an eager graph made there lives."""
    z = _logits(300, 16, "f32", 0).requires_grad_(True)

    def forward():
        return torch_ops.moe_route(z if leaf else z * 2.0, 2, balance=True)

    alive = forward()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(forward().balance_loss, z)
    torch.cuda.synchronize()
    del graph
    want, = torch.autograd.grad(alive.balance_loss, z)  # eager calls go on as before
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(forward().balance_loss, z)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_capture_that_reaches_an_eager_operator_is_refused(torch_cuda):
    """The leaf's gradient belongs to a side stream, but the logits were made by an operator on the default stream."""
    w = _logits(300, 16, "f32", 0).requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = w * 1.0
    torch.cuda.current_stream().wait_stream(side)
    z = w * 2.0
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(torch_ops.moe_route(z, 2, balance=True).balance_loss, z)
    torch.cuda.synchronize()
    del alive, graph
    # eager calls go on as before
    got, = torch.autograd.grad(torch_ops.moe_route(z, 2, balance=True).balance_loss, w)
    leaf = z.detach().requires_grad_(True)
    assert torch.equal(got, 2.0 * torch.autograd.grad(torch_ops.moe_route(leaf, 2, balance=True).balance_loss, leaf)[0])


@pytest.mark.gpu
def test_captured_with_an_eager_graph_of_a_side_stream_alive(torch_cuda):
    static = _logits(300, 16, "f32", 0).requires_grad_(True)

    def step(z):
        return torch.autograd.grad(torch_ops.moe_route(z, 2, balance=True).balance_loss, z)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = torch_ops.moe_route(static, 2, balance=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in range(1, 4):
        fresh = _logits(300, 16, "f32", seed)
        with torch.no_grad():
            static.copy_(fresh)
        graph.replay()
        assert torch.equal(out, step(fresh.requires_grad_(True)))
        torch.cuda.synchronize()
    del alive


@pytest.mark.gpu
def test_captured_and_replayed(torch_cuda):
    """Forward and backward in a graph, replayed with new logits between the program's own calls."""
    static = _logits(700, 48, "f32", 0).requires_grad_(True)
    dw = torch.randn(700, 3, generator=torch.Generator().manual_seed(1)).cuda()
    dl = torch.full((), 0.1, device="cuda")

    def step(z):
        r = torch_ops.moe_route(z, 3, balance=True)
        return (*[x.detach() for x in r], torch.autograd.grad((r.weights, r.balance_loss), z, (dw, dl))[0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in range(1, 5):
        fresh = _logits(700, 48, "f32", seed)
        with torch.no_grad():
            static.copy_(fresh)
        graph.replay()
        want = step(fresh.requires_grad_(True))
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)
