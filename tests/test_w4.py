"""Products with 4-bit weights (csrc/gg_w4.hip, torch_ops.w4_matmul and moe_w4_matmul) against the sum in 64
bits, and the chain of a mixture-of-experts layer: routing, products, combination.

Bound: with S = sum_k |x| |q - z| |s| the sum of the magnitudes of one output's terms and u = 2^-24, the
products x (q - z) are exact in float32 (11 and at most 9 bits), each addition rounds by u of a partial sum
no larger than S: at most n u S for a chain of n additions.  Sums here are made in lanes, instructions of
32 terms and groups, so no chain is longer than K / 32 + 64 terms, and an instruction may round its 32
terms by a few u: (K / 32 + 128) u S in all, and half a step of the output's type."""
import ctypes
import math
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from grouped_gemm_gpu_kernel_amd import _lib, torch_ops
from test_moe_route import _c_layout

U = 2.0 ** -24


def values(q, scales, zeros=None):
    """The weights in float64, [..., N, K]."""
    w = torch.stack((q & 15, q >> 4), dim=-1).flatten(-2).double()
    group = w.shape[-1] // scales.shape[-1]
    z = torch.full_like(scales, 8.0) if zeros is None else zeros
    return (w - z.double().repeat_interleave(group, -1)) * scales.double().repeat_interleave(group, -1)


def check(y, x, w, row_weights=None):
    """y against x @ w.T, row by row; x [R, K] float64, w [N, K] float64."""
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    k = x.shape[1]
    if row_weights is not None:
        want, size = want * row_weights[:, None], size * row_weights.abs()[:, None]
    bound = size * (k / 32 + 128) * U + want.abs() * torch.finfo(y.dtype).eps / 2 * 1.01 + (
        2.0 ** -25 if y.dtype == torch.float16 else 2.0 ** -126)
    off = (y.double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


# ---------------------------------------------------------------- CPU

def test_struct_mirrors_the_header(tmp_path):
    got, want = _c_layout(tmp_path, "ggk_w4_args", _lib.GGKW4Args)
    assert got == want


BASE = dict(rows=4, x_rows=4, n=8, k=128, group=64, experts=0, x=0x1000, ldx=128, q=0x1000, ldq=64, scales=0x1000, lds=2,
            y=0x1000, ldy=8, y_type=_lib.GGK_TYPE_F32)
MOE = dict(experts=3, counts=0x1000, order=0x1000, stride_q=512, stride_s=16)


@pytest.mark.parametrize("over,status", [
    ({}, 0), ({"rows": -1}, 1), ({"rows": 5}, 1), ({"n": -1}, 1), ({"group": 16}, 1), ({"group": 48}, 1),
    ({"group": 96}, 1), ({"group": 0}, 1), ({"k": 96}, 1), ({"k": 0}, 1), ({"ldx": 127}, 1), ({"ldq": 48}, 1), ({"ldq": 72}, 1),
    ({"q": 0x1008}, 1), ({"lds": 1}, 1), ({"zeros": 0x1000, "ldz": 1}, 1), ({"zeros": 0x1000, "ldz": 2}, 0),
    ({"ldy": 7}, 1), ({"y_type": _lib.GGK_TYPE_BF16}, 1), ({"x": None}, 17), ({"q": None}, 17), ({"scales": None}, 17),
    ({"y": None}, 17), ({"rows": 0, "x_rows": 0, "x": None, "y": None}, 0), ({"n": 0, "q": None}, 0), (MOE, 0),
    ({**MOE, "rows": 8}, 0), ({**MOE, "rows": 7}, 1), ({**MOE, "x_rows": 0}, 1), ({**MOE, "counts": None}, 17),
    ({**MOE, "order": None}, 17), ({**MOE, "stride_q": 520}, 1), ({**MOE, "stride_q": -512}, 1),
    ({**MOE, "experts": 1025}, 1), ({**MOE, "experts": -1}, 1),
    ({"n": (1 << 28) + 1}, 1), ({"k": (1 << 28) + 64, "ldx": 1 << 29, "ldq": 1 << 28, "lds": 1 << 23}, 1),
    ({"n": 1 << 28, "k": 1 << 28, "ldx": 1 << 28, "ldq": 1 << 27, "lds": 1 << 22, "ldy": 1 << 28}, 0)])
def test_arguments_are_checked_on_the_host(over, status):
    args = _lib.GGKW4Args(**{**BASE, **over})
    assert _lib.lib().ggk_w4_check(ctypes.byref(args)) == status
    if status:  # refused before anything is launched
        assert _lib.lib().ggk_w4_multiply(ctypes.byref(args), None) == status
    assert _lib.lib().ggk_w4_check(None) == 1 and _lib.lib().ggk_w4_multiply(None, None) == 1


def test_refusals_of_the_torch_calls():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with pytest.raises(ValueError, match="on a GPU"):
        torch_ops.w4_matmul(torch.zeros(1, 64).half(), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2).half())
    with FakeTensorMode():
        def t(*shape, dtype=torch.float16, device="cuda:0"):
            return torch.empty(*shape, dtype=dtype, device=device)

        x, q, s = t(3, 128), t(6, 64, dtype=torch.uint8), t(6, 2)
        z = t(6, 2, dtype=torch.uint8)
        for bad, error, text in [
                ((x.float(), q, s), TypeError, "x must be torch.float16"), ((t(128), q, s), ValueError, "2-D"),
                ((t(128, 3).t(), q, s), ValueError, "contiguous rows"), ((t(3, 126), q, s), ValueError, "columns"),
                ((x, q.char(), s), TypeError, "q must be torch.uint8"), ((x, q, s.float()), TypeError, "scales"),
                ((x, q, s, z.char()), TypeError, "zeros"), ((x, q, s, z[:, :1]), ValueError, "zeros has shape"),
                ((x, q, s[:5]), ValueError, "scales has shape"), ((x, q, t(6, 3)), ValueError, "group"),
                ((x, q, t(6, 8)), ValueError, "group"), ((x, q, t(6, 0)), ValueError, "group"),
                ((x, q.cpu(), s), ValueError, "q is on"), ((x, t(64, 6, dtype=torch.uint8).t(), s), ValueError, "contiguous"),
                ((x, t(6, 72, dtype=torch.uint8)[:, :64], s), ValueError, "16 bytes"),
                ((x, t(1, 64, dtype=torch.uint8).expand(6, 64), s), ValueError, "overlap"),
                ((x, t(2, 6, 64, dtype=torch.uint8), s), ValueError, "dimensions"),
                ((x, t((1 << 28) + 1, 64, dtype=torch.uint8), t((1 << 28) + 1, 2)), ValueError, "at most"),
                ((t(1, (1 << 28) + 64), t(1, (1 << 27) + 32, dtype=torch.uint8), t(1, 1)), ValueError, "at most")]:
            with pytest.raises(error, match=text):
                torch_ops.w4_matmul(*bad)
        with pytest.raises(TypeError, match="out_dtype"):
            torch_ops.w4_matmul(x, q, s, out_dtype=torch.bfloat16)
        with pytest.raises(RuntimeError, match="no gradient"):
            torch_ops.w4_matmul(x.clone().requires_grad_(True), q, s)
        q3, s3 = t(2, 6, 64, dtype=torch.uint8), t(2, 6, 2)
        counts, order = t(2, dtype=torch.int32), t(6, dtype=torch.int32)
        for bad, error, text in [
                ((x, q, s, counts, order), ValueError, "experts"), ((x, q3, s, counts, order), ValueError, "dimensions"),
                ((x, q3, s3, counts[:1], order), ValueError, "entries"), ((x, q3, s3, counts.long(), order), TypeError, "int32"),
                ((x, q3, s3, counts, order.long()), TypeError, "int32"),
                ((x, q3, s3, counts, t(7, dtype=torch.int32)), ValueError, "multiple"),
                ((t(0, 128), q3, s3, counts, order), ValueError, "multiple"),
                ((x, q3, s3, counts, t(12, dtype=torch.int32)[::2]), ValueError, "contiguous"),
                ((x, t(1025, 6, 64, dtype=torch.uint8), t(1025, 6, 2), counts, order), ValueError, "experts")]:
            with pytest.raises(error, match=text):
                torch_ops.moe_w4_matmul(*bad)
        for w, error, text in [(t(6), TypeError, "float32"), (t(5, dtype=torch.float32), ValueError, "entries"),
                               (t(6, dtype=torch.float32).requires_grad_(True), RuntimeError, "no gradient")]:
            with pytest.raises(error, match=text):
                torch_ops.moe_w4_matmul(x, q3, s3, counts, order, row_weights=w)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor does not require a gradient by itself; its tangent would be lost without a word."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad

    with FakeTensorMode(), forward_ad.dual_level():
        def t(*shape, dtype=torch.float16):
            return torch.empty(*shape, dtype=dtype, device="cuda:0")

        def dual(a):
            return forward_ad.make_dual(a, torch.empty_like(a))

        x, q, s = t(3, 128), t(6, 64, dtype=torch.uint8), t(6, 2)
        q3, s3, w = t(2, 6, 64, dtype=torch.uint8), t(2, 6, 2), t(6, dtype=torch.float32)
        counts, order = t(2, dtype=torch.int32), t(6, dtype=torch.int32)
        for name, call in [
                ("x", lambda: torch_ops.w4_matmul(dual(x), q, s)), ("scales", lambda: torch_ops.w4_matmul(x, q, dual(s))),
                ("x", lambda: torch_ops.moe_w4_matmul(dual(x), q3, s3, counts, order)),
                ("scales", lambda: torch_ops.moe_w4_matmul(x, q3, dual(s3), counts, order)),
                ("row_weights", lambda: torch_ops.moe_w4_matmul(x, q3, s3, counts, order, row_weights=dual(w)))]:
            with pytest.raises(RuntimeError, match=f"forward-mode derivative: {name}"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match=f"forward-mode derivative: {name}"):
                call()


def test_tensors_without_data_are_refused():
    """Fake tensors never come to a launch, where their null addresses would stand for zero points and masks left out."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def t(*shape, dtype=torch.float16):
            return torch.empty(*shape, dtype=dtype, device="cuda:0")

        x, q, s, z = t(3, 128), t(6, 64, dtype=torch.uint8), t(6, 2), t(6, 2, dtype=torch.uint8)
        q3, s3, counts, order = t(2, 6, 64, dtype=torch.uint8), t(2, 6, 2), t(2, dtype=torch.int32), t(6, dtype=torch.int32)
        for call in (lambda: torch_ops.w4_matmul(x, q, s), lambda: torch_ops.w4_matmul(x, q, s, z),
                     lambda: torch_ops.moe_w4_matmul(x, q3, s3, counts, order),
                     lambda: torch_ops.moe_route(t(600, 8), 2),
                     lambda: torch_ops.moe_route(t(600, 8), 2, token_mask=t(600, dtype=torch.bool))):
            with pytest.raises(RuntimeError, match="data is not allocated"):
                call()


def test_views_whose_memory_holds_other_values_are_refused():
    """Views with the negative bit (the imaginary part of a conjugate): memory holds the values' negatives."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def t(*shape, dtype=torch.float16):
            return torch.empty(*shape, dtype=dtype, device="cuda:0")

        x, q, s = t(1, 128), t(6, 64, dtype=torch.uint8), t(6, 2)
        q3, s3, counts, order = t(2, 6, 64, dtype=torch.uint8), t(2, 6, 2), t(2, dtype=torch.int32), t(1, dtype=torch.int32)
        w = torch.imag(t(1, dtype=torch.complex64).conj())
        assert w.is_neg() and w.is_contiguous()
        with pytest.raises(ValueError, match="row_weights is a view"):
            torch_ops.moe_w4_matmul(x, q3, s3, counts, order, row_weights=w)
        with pytest.raises(ValueError, match="x is a view"):
            torch_ops.w4_matmul(torch._neg_view(x), q, s)
        with pytest.raises(ValueError, match="scales is a view"):
            torch_ops.w4_matmul(x, q, torch._neg_view(s))
        with pytest.raises(ValueError, match="logits is a view"):
            torch_ops.moe_route(torch._neg_view(t(600, 8)), 2)
        with pytest.raises(ValueError, match="logits is a view"):
            torch_ops.moe_route(torch._efficientzerotensor((600, 8), device="cuda:0"), 2)


def test_matrix_results_are_read_behind_their_wait_states(tmp_path):
    """A matrix instruction's result may be read by another kind of instruction 8 wait states later at the earliest.  The
    compiler sees to it inside a basic block, but was seen to leave it out where a branch lies between (row tiles skipped
    inside the loop over K gave wrong sums): in the built kernels no result is read, and no branch taken, before
    that."""
    root = Path(__file__).resolve().parents[1]
    built = root / "grouped_gemm_gpu_kernel_amd" / "_build" / "gg_w4.o"
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

    def registers(operands):
        found = set()
        for first, last, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", operands):
            found |= {int(one)} if one else set(range(int(first), int(last) + 1))
        return found

    bad, seen = [], 0
    for i, line in enumerate(code):
        if not line.startswith("v_mfma"):
            continue
        seen += 1
        result, states = registers(line.split(",")[0]), 0
        for after in code[i + 1:]:
            if states >= 8:
                break
            kind = after.split()[0]
            operands = after.split(",")
            if kind.startswith("v_mfma"):
                if result & registers(",".join(operands[1:3])):
                    bad.append((line, after, states))
                if result & registers(after):  # the next of a chain: checked as the one before
                    break
            elif result & registers(after) or kind.startswith(("s_cbranch", "s_branch", "s_setpc")):
                bad.append((line, after, states))
                break
            states += int(after.split()[1], 0) + 1 if kind == "s_nop" else 1
    assert seen > 100 and not bad, bad[:3]


# ---------------------------------------------------------------- GPU

def _weights(lead, n, k, group, zeros, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (*lead, n, k // 2), generator=g, dtype=torch.uint8).cuda()
    s = ((torch.rand(*lead, n, k // group, generator=g) - 0.3) * 0.05).half().cuda()
    z = torch.randint(0, 16, (*lead, n, k // group), generator=g, dtype=torch.uint8).cuda() if zeros else None
    return q, s, z


def _x(rows, k, seed):
    return torch.randn(rows, k, generator=torch.Generator().manual_seed(seed)).half().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256, 0])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 16, 2), (1, 17, 5), (2, 40, 8), (3, 129, 3), (5, 64, 16), (8, 33, 7),
                                      (15, 100, 4), (16, 16, 9), (17, 31, 6), (33, 200, 4), (64, 80, 10), (65, 48, 3),
                                      (130, 20, 2), (1, 2000, 33)])
def test_shapes_and_groups(torch_cuda, rows, n, k, group, zeros):
    """k counts groups (of 128 where one group is the whole row: group 0)."""
    group, k = (128 * k, 128 * k) if group == 0 else (group, group * k)
    q, s, z = _weights((), n, k, group, zeros, rows + n + k)
    x = _x(rows, k, 1)
    w = values(q, s, z)
    check(torch_ops.w4_matmul(x, q, s, z), x.double(), w)
    check(torch_ops.w4_matmul(x, q, s, z, out_dtype=torch.float16), x.double(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(1, 4096, 8192), (7, 1003, 14336), (40, 2050, 4096), (200, 512, 2048)])
def test_larger(torch_cuda, rows, n, k):
    q, s, z = _weights((), n, k, 128, True, 3)
    x = _x(rows, k, 2)
    first = torch_ops.w4_matmul(x, q, s, z)
    check(first, x.double(), values(q, s, z))
    for _ in range(3):  # the same call gives the same bits
        assert torch.equal(torch_ops.w4_matmul(x, q, s, z), first)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [128, 640, 64])
@pytest.mark.parametrize("rows,n", [(3, 4200), (12, 2064), (9, 8500), (4, 24000), (40, 4100), (35, 24000), (50, 14300)])
def test_each_start_along_k(torch_cuda, rows, n, group):
    """Columns enough that workgroups begin with every part of K, the last part not a whole one."""
    k = 128 * 85
    q, s, z = _weights((), n, k, group, rows % 2 == 0, n + group)
    x = _x(rows, k, n)
    check(torch_ops.w4_matmul(x, q, s, z), x.double(), values(q, s, z))


@pytest.mark.gpu
def test_strides_and_alignment(torch_cuda):
    """Column slices of wider x, scales and zeros at any offset, q by 16 bytes."""
    q, s, z = _weights((), 50, 512, 64, True, 4)
    wide_q = torch.zeros(50, 256 + 48, dtype=torch.uint8, device="cuda")
    wide_q[:, 16:272] = q
    wide_s = torch.full((50, 8 + 5), math.nan, dtype=torch.float16, device="cuda")
    wide_s[:, 3:11] = s
    wide_z = torch.full((50, 8 + 3), 99, dtype=torch.uint8, device="cuda")
    wide_z[:, 1:9] = z
    for rows in (1, 3, 20):
        for off in (0, 1, 3, 8):
            x = torch.full((rows, 512 + 11), math.nan, dtype=torch.float16, device="cuda")
            x[:, off:off + 512] = _x(rows, 512, rows)
            x = x[:, off:off + 512]
            y = torch_ops.w4_matmul(x, wide_q[:, 16:272], wide_s[:, 3:11], wide_z[:, 1:9])
            check(y, x.double(), values(q, s, z))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 16, 40])
def test_odd_values(torch_cuda, rows):
    """Subnormal and large x, zero and subnormal scales, every weight and zero point; NaN and infinity reach the
    outputs of their own row (x) or column (scales) and no other."""
    q, s, z = _weights((), 70, 384, 32, True, 5)
    s[3] = 0
    s[4] = 2.0 ** -24  # the least subnormal
    x = _x(rows, 384, 6)
    x[0, ::2] = 2.0 ** -24
    x[0, 1::4] = 60000.0
    x[0, 3::4] = -60000.0
    w = values(q, s, z)
    check(torch_ops.w4_matmul(x, q, s, z), x.double(), w)
    s[10, 2] = math.nan
    s[11, 3] = math.inf
    x[rows - 1, 5] = math.inf
    y = torch_ops.w4_matmul(x, q, s, z)
    fine = torch.ones_like(y, dtype=torch.bool)
    fine[rows - 1] = False
    fine[:, 10:12] = False
    assert torch.isfinite(y[fine]).all()
    # an infinite scale gives infinity or NaN, by whether it multiplies a group's sum or each weight of it
    assert torch.isnan(y[:, 10]).all() and not torch.isfinite(y[:, 11]).any()
    assert not torch.isfinite(y[rows - 1]).any()
    if rows > 1:
        keep = [j for j in range(70) if j not in (10, 11)]
        check(y[: rows - 1, keep], x[: rows - 1].double(), w[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 16, 33])
@pytest.mark.parametrize("group", [32, 128])
def test_sums_of_integers_are_exact(torch_cuda, rows, group):
    """Whole x and scales of 1: every partial sum is a whole number below 2^24, which float32 holds, in any order.  One
    term a row of x is 2^11 times the others, so that bits lost in an instruction's alignment show."""
    q, s, z = _weights((), 333, 4096, group, True, 17)
    s.fill_(1.0)
    g = torch.Generator().manual_seed(18)
    x = torch.randint(-1, 2, (rows, 4096), generator=g).half().cuda()
    x[:, 7::512] = 2048.0  # 8 terms of at most 15 * 2048, 4088 of at most 15: below 2^19
    want = x.double() @ values(q, s, z).t()
    assert torch.equal(torch_ops.w4_matmul(x, q, s, z).double(), want)
    want = x.double() @ values(q, s).t()
    assert torch.equal(torch_ops.w4_matmul(x, q, s).double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(2, 2000), (2, 8000), (2, 14300), (9, 2000), (9, 6400), (9, 14300), (33, 2000),
                                    (40, 4100), (50, 14300)])
@pytest.mark.parametrize("group", [64, 128])
def test_each_width_is_exact(torch_cuda, rows, n, group):
    """The same for narrow and wide matrices, whose workgroups take other numbers of columns."""
    q, s, _ = _weights((), n, 1408, group, False, 19)
    s.fill_(1.0)
    x = torch.randint(-1, 2, (rows, 1408), generator=torch.Generator().manual_seed(20)).half().cuda()
    x[:, 7::512] = 2048.0
    assert torch.equal(torch_ops.w4_matmul(x, q, s).double(), x.double() @ values(q, s).t())


@pytest.mark.gpu
def test_half_output_overflows_to_infinity(torch_cuda):
    q = torch.full((2, 64), 255, dtype=torch.uint8, device="cuda")
    s = torch.ones(2, 1, dtype=torch.float16, device="cuda")
    x = torch.full((1, 128), 1000.0, dtype=torch.float16, device="cuda")
    assert torch_ops.w4_matmul(x, q, s).tolist() == [[7 * 128 * 1000.0] * 2]
    assert torch.isinf(torch_ops.w4_matmul(x, q, s, out_dtype=torch.float16)).all()


@pytest.mark.gpu
def test_empty(torch_cuda):
    q, s, _ = _weights((), 5, 64, 32, False, 1)
    assert torch_ops.w4_matmul(_x(0, 64, 1), q, s).shape == (0, 5)
    assert torch_ops.w4_matmul(_x(3, 64, 1), q[:0], s[:0]).shape == (3, 0)
    q, s, _ = _weights((2,), 5, 64, 32, False, 1)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    counts = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert torch_ops.moe_w4_matmul(_x(0, 64, 1), q, s, counts, none).shape == (0, 5)


def _routing(tokens, experts, top_k, seed, drop=0.0):
    """ids [tokens, top_k] with some -1, their counts and order."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(experts, generator=g)[:top_k] for _ in range(tokens)])
    ids[torch.rand(tokens, top_k, generator=g) < drop] = -1
    flat = torch.where(ids < 0, experts, ids).flatten()
    counts = torch.bincount(flat, minlength=experts + 1)[:experts].int().cuda()
    return ids.cuda(), counts, flat.sort(stable=True).indices.int().cuda()


def _check_moe(y, x, q, s, z, ids, row_weights=None):
    fan = ids.shape[1]
    flat = ids.flatten().tolist()
    for e in sorted(set(flat) - {-1}):
        rows = torch.tensor([o for o, f in enumerate(flat) if f == e], device="cuda")
        rw = None if row_weights is None else row_weights.flatten()[rows].double()
        check(y[rows], x[rows // fan if len(x) * fan == len(flat) else rows].double(),
              values(q[e], s[e], None if z is None else z[e]), rw)
    gone = torch.tensor([o for o, f in enumerate(flat) if f == -1], dtype=torch.long, device="cuda")
    assert (y[gone] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top_k,n,k,group,drop", [
    (1, 4, 1, 16, 64, 32, 0.0), (1, 8, 8, 40, 128, 64, 0.0), (3, 64, 2, 33, 256, 128, 0.0), (7, 5, 3, 100, 96, 96, 0.3),
    (40, 3, 2, 64, 128, 128, 0.1), (200, 4, 1, 50, 320, 64, 0.0), (33, 1, 1, 20, 64, 64, 0.5), (64, 130, 6, 17, 64, 32, 0.2),
    (9, 1024, 16, 16, 64, 64, 0.0), (300, 2, 2, 48, 1024, 128, 0.05), (5, 16, 4, 2000, 512, 128, 1.0)])
@pytest.mark.parametrize("zeros", [False, True])
def test_experts(torch_cuda, tokens, experts, top_k, n, k, group, drop, zeros):
    q, s, z = _weights((experts,), n, k, group, zeros, tokens + experts)
    ids, counts, order = _routing(tokens, experts, top_k, tokens, drop)
    x = _x(tokens, k, 3)
    _check_moe(torch_ops.moe_w4_matmul(x, q, s, counts, order, z), x, q, s, z, ids)
    rw = torch.randn(tokens, top_k, generator=torch.Generator().manual_seed(5)).cuda()
    y = torch_ops.moe_w4_matmul(x, q, s, counts, order, z, row_weights=rw, out_dtype=torch.float16)
    _check_moe(y, x, q, s, z, ids, rw)
    slots = _x(tokens * top_k, k, 4)  # one row a slot
    y = torch_ops.moe_w4_matmul(slots, q, s, counts, order, z)
    _check_moe(y, slots.view(tokens * top_k, k), q, s, z, ids.view(-1, 1))


# Cases of every form of the experts' kernel: rows an item, waves that split K; the experts' slots (with items of up to 4, 16
# and 32 rows and of more than one item), slots without an expert, N.
FORM_CASES = [
    ((32, 1), [1, 4, 5, 16, 17, 32, 33, 70, 0, 2, 3, 9, 1, 0, 31, 6], 5, 1100),
    ((32, 1), [3, 0, 20, 64, 16], 0, 3300),
    ((32, 1), [2, 1, 40, 0, 8, 1, 1, 19, 1, 4, 1, 1, 1, 1, 1, 17], 40, 8011),  # more items than workgroups
    ((32, 1), [1] * 200 + [7] * 56, 3, 81),
    ((16, 1), [1, 0, 2] * 99 + [5, 16, 17, 40], 9, 100),
    ((16, 1), [0] * 700 + [3, 33, 4] * 100, 0, 33),
    ((16, 2), [1, 4, 5, 16, 17, 32, 33, 70, 0, 2, 3, 9, 1, 0, 31, 6], 5, 600),
    ((16, 2), [30, 60, 16, 47], 2, 3999),  # more items than workgroups
    ((16, 2), [2, 1, 0] * 100 + [20], 0, 40),
    ((16, 4), [1, 4, 5, 16, 17, 33, 0, 2], 4, 500)]


def _form(n, slots, experts):
    """The kernel's form, by the launch's rule."""
    waves = (n + 15) // 16 * min(slots, experts)
    if waves >= 1024 and experts <= 256:
        return 32, 1
    return (16, 1) if waves >= 1024 else (16, 2) if waves >= 512 else (16, 4)


def _slots_of(takes, without, seed):
    """Each slot's expert in a random order, counts and order."""
    flat = torch.cat([torch.full((c,), e) for e, c in enumerate(takes)] + [torch.full((without,), -1)])
    flat = flat[torch.randperm(len(flat), generator=torch.Generator().manual_seed(seed))]
    order = torch.where(flat < 0, len(takes), flat).sort(stable=True).indices.int().cuda()
    return flat.cuda(), torch.tensor(takes, dtype=torch.int32, device="cuda"), order


def _check_slots(y, x, q, s, z, flat, row_weights=None):
    """y[o] against x[o] by flat[o]'s matrix, the experts one after the other; rows without one are zeros."""
    assert (y[flat < 0] == 0).all()
    for e in flat[flat >= 0].unique().tolist():
        rows = (flat == e).nonzero()[:, 0]
        check(y[rows], x[rows].double(), values(q[e], s[e], None if z is None else z[e]),
              None if row_weights is None else row_weights[rows].double())


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,k", [(128, 128), (128, 128 * 5), (256, 256 * 5), (32, 32 * 33), (64, 64 * 17), (96, 96 * 7)])
@pytest.mark.parametrize("form,takes,without,n", FORM_CASES)
def test_each_form_of_the_experts(torch_cuda, form, takes, without, n, group, k, zeros):
    flat, counts, order = _slots_of(takes, without, n + k)
    slots = len(flat)
    assert _form(n, slots, len(takes)) == form
    q, s, z = _weights((len(takes),), n, k, group, zeros, n)
    x = _x(slots, k, slots)
    first = torch_ops.moe_w4_matmul(x, q, s, counts, order, z)
    _check_slots(first, x, q, s, z, flat)
    rw = torch.randn(slots, generator=torch.Generator().manual_seed(5)).cuda()
    y = torch_ops.moe_w4_matmul(x, q, s, counts, order, z, row_weights=rw, out_dtype=torch.float16)
    _check_slots(y, x, q, s, z, flat, rw)
    assert torch.equal(torch_ops.moe_w4_matmul(x, q, s, counts, order, z), first)


@pytest.mark.gpu
@pytest.mark.parametrize("group,k", [(128, 1408), (64, 1408), (96, 96 * 15)])
@pytest.mark.parametrize("form,takes,without,n", FORM_CASES)
def test_each_form_of_the_experts_is_exact(torch_cuda, form, takes, without, n, group, k):
    """Whole numbers, as in test_sums_of_integers_are_exact."""
    flat, counts, order = _slots_of(takes, without, n + k)
    q, s, _ = _weights((len(takes),), n, k, group, False, n)
    s.fill_(1.0)
    x = torch.randint(-1, 2, (len(flat), k), generator=torch.Generator().manual_seed(20)).half().cuda()
    x[:, 7::512] = 2048.0
    y = torch_ops.moe_w4_matmul(x, q, s, counts, order)
    assert (y[flat < 0] == 0).all()
    for e in flat[flat >= 0].unique().tolist():
        rows = (flat == e).nonzero()[:, 0]
        assert torch.equal(y[rows].double(), x[rows].double() @ values(q[e], s[e]).t()), e


@pytest.mark.gpu
@pytest.mark.parametrize("experts,n,form", [(8, 2048, (32, 1)), (300, 300, (16, 1)), (8, 1300, (16, 2))])
def test_tokens_of_several_slots_in_each_form(torch_cuda, experts, n, form):
    """x one row a token, three slots each."""
    tokens, top_k, k = 70, 3, 640
    assert _form(n, tokens * top_k, experts) == form
    q, s, z = _weights((experts,), n, k, 64, True, n)
    ids, counts, order = _routing(tokens, experts, top_k, n, 0.2)
    x = _x(tokens, k, n)
    y = torch_ops.moe_w4_matmul(x, q, s, counts, order, z)
    _check_slots(y, x.repeat_interleave(top_k, 0), q, s, z, ids.flatten())


@pytest.mark.gpu
def test_one_expert_takes_all(torch_cuda):
    q, s, _ = _weights((12,), 100, 256, 128, False, 1)
    for tokens in (1, 15, 17, 129):
        for e in (0, 5, 11):
            ids = torch.full((tokens, 1), e, device="cuda")
            counts = torch.zeros(12, dtype=torch.int32, device="cuda")
            counts[e] = tokens
            x = _x(tokens, 256, tokens)
            y = torch_ops.moe_w4_matmul(x, q, s, counts, torch.arange(tokens, dtype=torch.int32, device="cuda"))
            _check_moe(y, x, q, s, None, ids)


@pytest.mark.gpu
def test_counts_and_order_are_not_trusted(torch_cuda):
    """Negative counts are 0, what goes past the order's end is dropped, entries outside it are passed over: the rows
    that remain are right, and nothing around y is written."""
    q, s, _ = _weights((4,), 24, 64, 32, False, 2)
    x = _x(10, 64, 7)
    order = torch.arange(10, dtype=torch.int32, device="cuda")

    def run(counts, order):
        c = torch.tensor(counts, dtype=torch.int32, device="cuda")
        return torch_ops.moe_w4_matmul(x, q, s, c, order)

    big = torch.iinfo(torch.int32).max
    _check_moe(run([3, -5, 4, 2], order), x, q, s, None, torch.tensor([0] * 3 + [2] * 4 + [3] * 2 + [-1])[:, None])
    _check_moe(run([3, 4, 400, 50], order), x, q, s, None, torch.tensor([0] * 3 + [1] * 4 + [2] * 3)[:, None])
    _check_moe(run([1, big, big, big], order), x, q, s, None, torch.tensor([0] + [1] * 9)[:, None])
    _check_moe(run([-big - 1] * 4, order), x, q, s, None, torch.full((10, 1), -1))
    bad = order.clone()
    bad[2], bad[6], bad[9] = -1, 10, big
    y = run([5, 0, 5, 0], bad)
    good = [0, 1, 3, 4, 5, 7, 8]
    expert = torch.tensor([0] * 5 + [2] * 5)[:, None]
    _check_moe(y[good], x[good], q, s, None, expert[good])


@pytest.mark.gpu
def test_expert_strides_and_offsets_past_32_bits(torch_cuda):
    """Expert matrices in a wider tensor, and one whose matrices lie 1.5 GB apart: the last starts past 4 GB."""
    q, s, z = _weights((3,), 20, 128, 32, True, 8)
    wide = torch.zeros(3, 25, 96, dtype=torch.uint8, device="cuda")
    wide[:, :20, 16:80] = q
    ids, counts, order = _routing(30, 3, 2, 9)
    x = _x(30, 128, 9)
    _check_moe(torch_ops.moe_w4_matmul(x, wide[:, :20, 16:80], s, counts, order, z), x, q, s, z, ids)
    far = torch.empty(4, 3 << 29, dtype=torch.uint8, device="cuda")[:3, : 20 * 64].view(3, 20, 64)
    far.copy_(q)
    _check_moe(torch_ops.moe_w4_matmul(x, far, s, counts, order, z), x, q, s, z, ids)
    shared = q[:1].expand(3, 20, 64)  # one matrix for all experts
    _check_moe(torch_ops.moe_w4_matmul(x, shared, s, counts, order, z), x, shared, s, z, ids)


@pytest.mark.gpu
def test_long_rows_past_32_bits(torch_cuda):
    """A matrix of more than 2^32 bytes: its last rows."""
    n, k = (2 ** 32 // 4096) + 100, 8192
    q = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    s = torch.zeros(n, 1, dtype=torch.float16, device="cuda")
    tail_q, tail_s, _ = _weights((), 60, k, k, False, 10)
    q[-60:], s[-60:] = tail_q, tail_s
    x = _x(2, k, 10)
    y = torch_ops.w4_matmul(x, q, s)
    check(y[:, -60:], x.double(), values(tail_q, tail_s))
    assert (y[:, :-60] == 0).all()


@pytest.mark.gpu
def test_more_row_tiles_than_a_grid_has(torch_cuda):
    """Over 65535 tiles of 32 rows of one matrix, and as many slots that a workgroup of the experts' kernel makes hundreds of
    items; whole numbers, exact."""
    rows = 65536 * 32 + 77
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-3, 4, (rows, 32), generator=g, device="cuda").half()
    q, s, _ = _weights((6,), 9, 32, 32, False, 2)
    s.fill_(1.0)
    assert torch.equal(torch_ops.w4_matmul(x, q[0], s[0]).double(), x.double() @ values(q[0], s[0]).t())
    x = x[:300000].contiguous()
    ids = torch.randint(-1, 6, (300000, 2), generator=g, device="cuda")
    flat = ids.flatten()
    slot = torch.where(flat < 0, 6, flat)
    counts, order = torch.bincount(slot, minlength=7)[:6].int(), slot.sort(stable=True).indices.int()
    y = torch_ops.moe_w4_matmul(x, q, s, counts, order)
    assert (y[flat < 0] == 0).all()
    for e in range(6):
        at = (flat == e).nonzero()[:, 0]
        assert torch.equal(y[at].double(), x[at // 2].double() @ values(q[e], s[e]).t())


@pytest.mark.gpu
def test_streams_and_graphs(torch_cuda):
    q, s, z = _weights((6,), 70, 256, 64, True, 11)
    xs = [_x(24, 256, i) for i in range(5)]
    routes = [_routing(24, 6, 2, i, 0.1) for i in range(5)]
    eager = [torch_ops.moe_w4_matmul(x, q, s, c, o, z) for x, (_, c, o) in zip(xs, routes)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, (_, c, o), stream in zip(xs, routes, streams):
        with torch.cuda.stream(stream):
            got.append(torch_ops.moe_w4_matmul(x, q, s, c, o, z))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, eager))
    x, counts, order = xs[0].clone(), routes[0][1].clone(), routes[0][2].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = torch_ops.moe_w4_matmul(x, q, s, counts, order, z)
        d = torch_ops.w4_matmul(x, q[0], s[0], z[0])
    for i in (3, 1, 4, 2):
        x.copy_(xs[i])
        counts.copy_(routes[i][1])
        order.copy_(routes[i][2])
        graph.replay()
        assert torch.equal(y, eager[i])
        assert torch.equal(d, torch_ops.w4_matmul(xs[i], q[0], s[0], z[0]))
        torch.cuda.synchronize()


# ---------------------------------------------------------------- the layer

@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 8, 2), (50, 16, 4), (300, 12, 2)])
def test_layer_in_decode(torch_cuda, tokens, experts, top_k):
    """Routing, both products of each expert in 4 bits with an activation between, the weighted sum per token; every
    step against 64 bits on that step's own inputs, padding tokens end as zeros."""
    width, inner = 256, 192
    up = _weights((experts,), inner, width, 64, True, 12)
    down = _weights((experts,), width, inner, 96, False, 13)
    x = _x(tokens, width, 14)
    logits = torch.randn(tokens, experts, generator=torch.Generator().manual_seed(15)).half().cuda()
    mask = torch.ones(tokens, dtype=torch.bool, device="cuda")
    mask[1::7] = False
    r = torch_ops.moe_route(logits, top_k, token_mask=mask)
    h = torch_ops.moe_w4_matmul(x, up[0], up[1], r.counts, r.order, up[2])
    _check_moe(h, x, *up, r.ids)
    h = torch.nn.functional.silu(h).half()
    y = torch_ops.moe_w4_matmul(h, down[0], down[1], r.counts, r.order, row_weights=r.weights)
    _check_moe(y, h, *down, r.ids.view(-1, 1), r.weights)
    out = y.view(tokens, top_k, width).sum(1)
    assert torch.isfinite(out).all() and (out[~mask] == 0).all() and out[mask].abs().sum() > 0


@pytest.mark.gpu
def test_layer_in_training(torch_cuda):
    """Routing with its loss, the grouped float16 product on the routing's counts and order, the weighted sum, and
    the gradients of both back to the logits."""
    from test_moe_route import plain_gradient, plain_route

    tokens, experts, top_k, k, n = 400, 9, 2, 96, 80
    g = torch.Generator().manual_seed(16)
    x = torch.randn(tokens, k, generator=g).half().cuda()
    w = torch.randn(experts, k, n, generator=g).half().cuda()
    logits = torch.randn(tokens, experts, generator=g).cuda().requires_grad_(True)
    r = torch_ops.moe_route(logits, top_k, balance=True)
    rows = torch.empty(tokens * top_k, n, device="cuda")
    plan = torch_ops.MoeGroupedGemmPlan(x[(r.order // top_k).long()].contiguous(), w, rows)
    plan.run(r.counts)
    slots = torch.empty_like(rows)
    slots[r.order.long()] = rows
    slots = slots.view(tokens, top_k, n)
    want = (x.double()[:, None, None] @ w.double()[r.ids.long()]).squeeze(2)
    assert (slots - want).abs().max() <= 1e-3 * math.sqrt(k) * float(x.abs().max() * w.abs().max())
    out = (r.weights[..., None] * slots).sum(1)
    up = torch.randn(tokens, n, generator=g).cuda()
    ((out * up).sum() + 0.01 * r.balance_loss).backward()
    d_weights = (slots * up[:, None]).sum(2)  # float32, as autograd makes it: n terms, off by at most n u of their sizes
    ref = plain_route(logits.detach().double().cpu().numpy(), top_k)
    grad, size = plain_gradient(ref, True, 1.0, d_weights.double().cpu().numpy(), 0.01)
    _, most = plain_gradient(ref, True, 1.0, (slots * up[:, None]).abs().sum(2).double().cpu().numpy(), 0.01)
    off = np.abs(logits.grad.double().cpu().numpy() - grad)
    assert (off <= size * 4 * (20 + 32) * U + 2 * n * U * most + 1e-30).all()
