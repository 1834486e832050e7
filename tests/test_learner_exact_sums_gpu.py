"""Sums over many rows and many gradients, of whole numbers that float32 adds
without rounding: a row or a value that is left out or taken twice shows,
whatever the size, where a bound on roundings would hide it."""

import pytest
import torch

import per_b200
from test_grad_norm_gpu import params
from test_layer_norm_gpu import BF16, F16, F32

pytestmark = pytest.mark.gpu


def signs(n, seed, dtype=F32):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randint(0, 2, (n,), generator=g, device="cuda", dtype=torch.int8) * 2 - 1).to(dtype)


def alternating(rows, dim, stride, offset, dtype, seed):
    """Rows of +1 and -1 by turns, each row beginning with either: mean 0 and variance 1 without
    rounding, since every power-of-two part of a row that begins at an even place sums to 0."""
    x = torch.zeros(rows, stride, device="cuda", dtype=dtype)[:, offset:offset + dim]
    x[:, ::2] = signs(rows, seed, dtype)[:, None]
    x[:, 1::2] = -x[:, ::2]
    return x


@pytest.mark.parametrize("rows,dim", [(3_000_001, 8), (200_003, 256), (100_003, 1024), (20_011, 4096),
                                      (5003, 16384), (1013, 131072)])
@pytest.mark.parametrize("stride,offset", [(0, 0), (5, 3)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_column_sums_take_every_row_once(dtype, stride, offset, rows, dim):
    x = alternating(rows, dim, dim + stride, offset, dtype, seed=rows)
    w = torch.ones(dim, device="cuda", requires_grad=True)
    b = torch.zeros(dim, device="cuda", requires_grad=True)
    dy = signs(rows * dim, rows + 1, dtype).view(rows, dim)
    y = per_b200.layer_norm(x, dim, w, b, eps=0.0)
    assert torch.equal(y, x)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    # sums of +-1 below 2^24 in size, so in any order and grouping without rounding
    want_w, want_b = torch.zeros(dim, device="cuda"), torch.zeros(dim, device="cuda")
    for a in range(0, rows, 1 + (1 << 27) // dim):
        part = slice(a, a + 1 + (1 << 27) // dim)
        want_w += (dy[part] * x[part]).sum(0, dtype=torch.float32)
        want_b += dy[part].sum(0, dtype=torch.float32)
    assert torch.equal(db, want_b)
    assert torch.equal(dw, want_w)


LISTS = [[1], [7, 9, 8], [4095, 1, 4097], [1_000_003], [300_000] * 20, [65_536] * 63 + [5], [99_999, 1, 2, 3] * 40,
         [5001] * 2500, [16_000_000]]


@pytest.mark.parametrize("dtype", [F32, BF16, F16, None])
@pytest.mark.parametrize("start", [0, 1, 3])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norms_take_every_value_once(sizes, start, dtype):
    """dtype None: the types by turns."""
    flats, grads = {}, []
    total = sum(sizes)
    for k, n in enumerate(sizes):
        t = dtype or (F32, BF16, F16)[k % 3]
        if t not in flats:
            flats[t] = [signs(total + start, 5, t), start]
        flat, at = flats[t]
        grads.append(flat[at:at + n])
        flats[t][1] = at + n
    assert total < 1 << 24
    # |+-1| summed in any order: a whole number below 2^24
    assert float(per_b200.grad_norm(grads, 1.0)) == total
    # the squares too; only the root is rounded (float64, then float32)
    got = float(per_b200.grad_norm(grads, 2.0))
    assert abs(got - total ** 0.5) <= total ** 0.5 * (2.0 ** -24 + 2.0 ** -50)
    p = params(grads)
    assert float(per_b200.clip_grad_norm_(p, float("inf"), 1.0)) == total


def test_rows_whose_squares_leave_float32():
    """Their inverse standard deviation is 0: the result is the bias, the input's gradient 0."""
    for dtype in (F32, BF16):
        for dim in (40, 256, 1000, 1001, 4096, 4099, 9000, 20000, 70001):
            for size in (3e19, 1e25, 1e30):
                x = torch.full((3, dim), -size, device="cuda", dtype=dtype)
                x[:, :dim // 4] = size
                x[1] = torch.linspace(-1, 1, dim, device="cuda")
                w, b = torch.full((dim,), 2.0, device="cuda"), torch.linspace(-1, 1, dim, device="cuda")
                x.requires_grad_()
                y = per_b200.layer_norm(x, dim, w, b)
                assert torch.equal(y[::2], b.to(dtype).expand(2, dim))
                dx, = torch.autograd.grad(y, x, torch.ones_like(y))
                assert float(dx[::2].abs().max()) == 0.0
                alone = per_b200.layer_norm(x.detach()[1:2].clone(), dim, w, b)
                assert bool((y[1].float() - alone[0].float()).abs().max() <= 2.0 ** -7 * alone.float().abs().max())
