"""Layer norm over many rows of the lengths that take a cluster of CTAs, so that
each cluster goes through a number of rows: every row, and the sums over them,
against float64."""

import pytest
import torch

import per_b200
from oracle import learner as ref
from test_layer_norm_gpu import BF16, EPS, F16, F32, check_forward, check_train, close, normal, params_like, \
    rows_like_activations

pytestmark = pytest.mark.gpu

ROWS = 1009  # the GPU holds 18 to 74 such clusters at once: more than ten rows each


def only_parameters(x, w, b, dy):
    """The gradients of weight and bias where the input's is not wanted."""
    w, b = (t.detach().requires_grad_() for t in (w, b))
    return torch.autograd.grad(per_b200.layer_norm(x, x.shape[-1], w, b), (w, b), dy)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [9000, 9001, 20000, 20001])
def test_clusters_over_many_rows(dim, dtype):
    x = rows_like_activations(ROWS, dim, dtype, seed=dim)
    w, b = params_like(dim, F32, "both")
    dy = normal(ROWS, dim, seed=3).to(dtype)
    full = check_train(x, w, b, dy)
    alone = only_parameters(x, w, b, dy)
    assert torch.equal(alone[0], full[1]) and torch.equal(alone[1], full[2])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [9000, 20000])
def test_clusters_over_many_rows_inside_packed_rows(dim, dtype):
    """Rows that start anywhere between two 16-byte boundaries, each in its turn."""
    x = rows_like_activations(ROWS, dim + 5, dtype, seed=dim)[:, 3:3 + dim]
    w, b = params_like(dim, dtype, "both")
    check_forward(x, w, b)
    full = check_train(x, w, b, normal(ROWS, dim + 7, seed=4).to(dtype)[:, 7:])
    assert full[0].shape == x.shape


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("dim", [9000, 9001, 20001])
def test_one_gradient_row_between_boundaries(dim, dtype):
    """An upstream gradient of one row for all that no 16-byte copy can take: it is fetched value by
    value for every row, with the input's gradient wanted and without."""
    x = rows_like_activations(ROWS, dim, dtype, seed=dim)
    w, b = params_like(dim, F32, "both")
    row = normal(dim + 1, seed=8).to(dtype)[1:]
    assert row.data_ptr() % 16
    dy = row.expand(ROWS, dim)
    full = check_train(x, w, b, dy)
    bounds = ref.layer_norm_backward_bound(dy, x, w, EPS, dtype, F32)
    for _ in range(3):
        alone = only_parameters(x, w, b, dy)
        for got, again, bound, what in zip(alone, full[1:], bounds[1:], ("dw", "db")):
            close(got, *bound, what)
            assert torch.equal(got, again)
