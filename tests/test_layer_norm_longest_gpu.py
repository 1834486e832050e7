"""Layer norm of rows beyond what a cluster of CTAs holds, and sums of so many
terms that float32 alone would lose them. Where values are regular the results
are known in closed form: a term is rounded to the step of the sum it goes to,
always the same way, so that nothing averages out."""

import pytest
import torch

import per_b200
from oracle import learner as ref
from test_layer_norm_gpu import BF16, EPS, F16, F32, check_forward, check_train, normal, params_like, \
    rows_like_activations

pytestmark = pytest.mark.gpu

# Additions in float32 that a term passes through, and the handful of operations around them: runs
# of 32 in a thread, float64 beyond, the partial rows' joins.
DEPTH = 64


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [131072, 131080, 140001])
def test_sixteen_bit_rows_beyond_a_cluster(dim, dtype):
    x = rows_like_activations(6, dim, dtype, seed=dim)
    for ptype in (F32, dtype):
        w, b = params_like(dim, ptype, "both")
        check_forward(x, w, b)
        check_train(x, w, b, normal(6, dim, seed=3).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_columns_beyond_the_row_splits(dtype):
    dim = 303_201
    x = rows_like_activations(9, dim, dtype)
    w, b = params_like(dim, F32, "both")
    check_train(x, w, b, normal(9, dim, seed=3).to(dtype))


def test_a_row_of_many_million_values():
    dim, c = 1 << 27, 1 + 1 / 128
    x = torch.full((1, dim), c, device="cuda")
    x[:, 1::2] = -c
    x.requires_grad_()
    y = per_b200.layer_norm(x, dim)
    r = 1 / (c * c + EPS) ** 0.5
    h = c * r  # mean 0, so y is h and -h by turns
    e = DEPTH * ref.U32
    sign = torch.ones(1, dim, device="cuda")
    sign[:, 1::2] = -1
    # |h| below 1: the bound of oracle.learner.layer_norm_bound with this depth
    assert float((y.detach().double() * sign - h).abs().max()) <= 2 * e + 2 * ref.U32
    # dy = sign (1 + t): g h averages to (1 + t) h, and what is left of dx is r (1 + t) (1 - h^2)
    t = 1 / 128
    dx, = torch.autograd.grad(y, x, sign * (1 + t))
    want = r * (1 + t) * (1 - h * h)
    # r e (g + 2 avg g + |h| (b + c2) + (1 + |h|) c2) with |h|, c2 / (1 + t) <= 1, b <= 3 (1 + t)
    assert float((dx.double() * sign - want).abs().max()) <= r * (1 + t) * 9 * e


def test_column_sums_of_many_rows():
    rows, dim, c, t = 3000, 303_201, 1 + 1 / 128, 2.0 ** -14
    x = torch.full((rows, dim), c, device="cuda")
    x[:, 1::2] = -c
    mean = c / dim  # one value more than -c balances
    w, b = torch.ones(dim, device="cuda", requires_grad=True), torch.zeros(dim, device="cuda", requires_grad=True)
    y = per_b200.layer_norm(x, dim, w, b)
    dw, db = torch.autograd.grad(y, (w, b), torch.full((rows, dim), 1 + t, device="cuda"))
    r = 1 / (c * c - mean * mean + EPS) ** 0.5
    want = torch.full((dim,), (c - mean) * r, device="cuda", dtype=torch.float64)
    want[1::2] = (-c - mean) * r
    want *= rows * (1 + t)
    e = DEPTH * ref.U32
    assert float((db.double() - rows * (1 + t)).abs().max()) <= (e + ref.U32) * rows * (1 + t)
    # h is off by 2 e, the sum of its products by e more
    assert float((dw.double() - want).abs().max()) <= 3.1 * e * rows * (1 + t)
