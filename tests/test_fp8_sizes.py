"""The 8-bit path at sizes where one launch ends: threads of a launch are counted in 32 bits."""
import ctypes
import math

import pytest
import torch

from grouped_gemm_gpu_kernel_amd import _lib, torch_ops
from test_fp8 import (BASE, FP8, GATE, MOE, _gen, blocks, check_gated, check_norm, check_product, matrix_of, matrix_values, numbers,
                      row_values, rows_of)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,columns", [(2 ** 26 + 2 ** 25 + 7, 16), (2 ** 24 + 5, 2049)])
def test_norm_of_more_rows_than_a_launch_has(torch_cuda, rows, columns):
    """Rows of a wave each (four a workgroup of 256 threads) and of a workgroup each."""
    torch.cuda.empty_cache()
    x = torch.zeros(rows, columns, dtype=torch.bfloat16, device="cuda")
    marked = torch.tensor([0, 1, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 1, rows // 2, rows - 6, rows - 2, rows - 1], device="cuda")
    if rows > 2 ** 25:
        marked = torch.cat((marked, torch.tensor([2 ** 25 - 1, 2 ** 25, 2 ** 26 - 1, 2 ** 26, 2 ** 26 + 1], device="cuda")))
    some = torch.randn(len(marked), columns, generator=_gen(1), device="cuda").bfloat16()
    x[marked] = some
    out = torch_ops.rms_norm_fp8(x)
    del x
    q = out.q.view(torch.uint8)
    check_norm(torch_ops.Fp8Norm(q[marked].view(FP8), out.scales[marked], None, None), some, None, None)
    q[marked] = 0
    out.scales[marked] = 2.0 ** -126
    for first in range(0, rows, 2 ** 22):  # a part at a time: reductions of many values take room
        assert not q[first:first + 2 ** 22].any() and (out.scales[first:first + 2 ** 22] == 2.0 ** -126).all()
    del out, q
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_norm_of_several_launches_has_every_output(torch_cuda):
    """With residual, weight and y, rows padded."""
    rows, columns = 2 ** 25 + 3, 8
    torch.cuda.empty_cache()
    wide = torch.zeros(rows, 9, dtype=torch.float16, device="cuda")
    last = torch.randn(40, columns, generator=_gen(2), device="cuda").half()
    wide[-40:, :columns] = last
    x, weight = wide[:, :columns], torch.randn(columns, generator=_gen(3), device="cuda").half()
    out = torch_ops.rms_norm_fp8(x, weight, x, plain=True)
    tail = torch_ops.Fp8Norm(out.q.view(torch.uint8)[-40:].view(FP8), out.scales[-40:], out.y[-40:], out.residual[-40:])
    check_norm(tail, last, weight, last)
    assert not out.q.view(torch.uint8)[:-40].any() and not out.y[:-40].any() and not out.residual[:-40].any()


def marks(count, n):
    """Places near both ends, near powers of two and in between."""
    at = {0, 1, n - 1, n - 2, n // 2, n // 3}
    for p in range(20, 30):
        at |= {2 ** p - 1, 2 ** p, 2 ** p + 1}
    return torch.tensor(sorted(a for a in at if a < n)[-count:], device="cuda")


@pytest.mark.gpu
def test_product_of_more_rows_than_a_launch_has(torch_cuda):
    """Streams of 32 rows by 32 columns, 256 threads each: 2^24 of them are 2^32 threads."""
    torch.cuda.empty_cache()
    rows, k = 2 ** 29 + 2 ** 20 + 11, 16
    x = torch.zeros(rows, k, dtype=torch.uint8, device="cuda")
    at = marks(24, rows)
    some = numbers((len(at), k), 1)
    x[at] = some.view(torch.uint8)
    xs = torch.ones(rows, 1, device="cuda")
    w = matrix_of((), 1, k, 2)
    y = torch_ops.fp8_matmul(x.view(FP8), xs, *w, out_dtype=torch.float32)
    del x, xs
    check_product(y[at], some.double(), matrix_values(*w), True)
    y[at] = 0
    for first in range(0, rows, 2 ** 26):
        assert not y[first:first + 2 ** 26].any()
    del y
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(1, 2 ** 27 + 2 ** 20 + 5), (12, 2 ** 28), (20, 2 ** 27 + 33)])
def test_product_of_more_columns_than_a_launch_has(torch_cuda, rows, n):
    """Up to 8 rows by 16 columns, up to 16 by 32, of 512 threads each: 2^23 of them are 2^32 threads; n up to its limit."""
    torch.cuda.empty_cache()
    k = 16
    w = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    at = marks(24, n)
    some = numbers((len(at), k), 1)
    w[at] = some.view(torch.uint8)
    ws = torch.ones(blocks(n), 1, device="cuda")
    x = rows_of(rows, k, 2)
    y = torch_ops.fp8_matmul(*x, w.view(FP8), ws)
    del w, ws
    check_product(y[:, at], row_values(*x), some.double(), True)
    y[:, at] = 0
    for first in range(0, n, 2 ** 24):
        assert not y[:, first:first + 2 ** 24].any()
    del y
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(3, 20), (40, 70), (130, 260)])
def test_longest_rows(torch_cuda, rows, n):
    """K and the distance of rows at their limit.  Sums of whole numbers are exact: terms of one, of which a float holds 2^24."""
    torch.cuda.empty_cache()
    k = _lib.GGK_FP8_MAX_K
    x, w = (torch.randint(-1, 2, shape, generator=_gen(shape[0]), device="cuda", dtype=torch.int8).to(FP8)
            for shape in ((rows, k), (n, k)))
    xs, ws = torch.ones(rows, blocks(k), device="cuda"), torch.ones(blocks(n), blocks(k), device="cuda")
    want = torch.zeros(rows, n, dtype=torch.float64, device="cuda")
    for at in range(0, k, 2 ** 18):
        want += x[:, at:at + 2 ** 18].double() @ w[:, at:at + 2 ** 18].double().t()
    for fast, dtype in ((False, torch.float32), (False, torch.bfloat16), (True, torch.float16)):
        assert torch.equal(torch_ops.fp8_matmul(x, xs, w, ws, out_dtype=dtype, fast=fast), want.to(dtype))
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(1)).int().cuda()
    counts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    y = torch_ops.moe_fp8_matmul(x, xs, w.expand(2, n, k), ws.expand(2, *ws.shape), counts, order, out_dtype=torch.float32)
    assert torch.equal(y.double(), want)
    gated = torch_ops.fp8_gated(x, xs * 2.0 ** -8, w, ws, w, ws)
    p = want * 2.0 ** -8
    h = p * torch.sigmoid(p) * p
    off = (gated.q.double() * gated.scales.double().repeat_interleave(128, 1)[:, :n] - h).abs()
    most = h.abs().amax(1, keepdim=True)  # a number is off by half a step, 2^-4 of the value or 2^-10 of the scale
    assert (off <= torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 / 448 * most) * 1.001).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 40, 300])
def test_rows_of_x_far_apart(torch_cuda, rows):
    """Offsets of x past 32 bits inside a tile, and rows of scales that are padded."""
    torch.cuda.empty_cache()
    k, n, apart = 272, 150, 2 ** 25 + 16
    far = torch.empty(rows, apart, dtype=torch.uint8, device="cuda")[:, 16:16 + k].view(FP8)
    x, xs = rows_of(rows, k, 1)
    far.view(torch.uint8).copy_(x.view(torch.uint8))
    wide = torch.full((rows, 1000), math.nan, device="cuda")
    wide[:, 7:10] = xs
    w, up = matrix_of((), n, k, 2), matrix_of((), n, k, 3)
    for dtype in (torch.float32, torch.bfloat16):
        check_product(torch_ops.fp8_matmul(far, wide[:, 7:10], *w, out_dtype=dtype), row_values(x, xs), matrix_values(*w), True)
    check_gated(torch_ops.fp8_gated(far, wide[:, 7:10], *w, *up), row_values(x, xs), matrix_values(*w), matrix_values(*up))
    counts, order = torch.tensor([rows], dtype=torch.int32, device="cuda"), torch.arange(rows, dtype=torch.int32, device="cuda")
    y = torch_ops.moe_fp8_matmul(far, wide[:, 7:10], w[0][None], w[1][None], counts, order, out_dtype=torch.float32)
    check_product(y, row_values(x, xs), matrix_values(*w), True)
    del far
    torch.cuda.empty_cache()
