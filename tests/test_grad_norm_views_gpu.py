"""Gradients and a known norm that are lazily negated views: what lies in memory
has the other sign."""

import pytest
import torch

import per_b200

pytestmark = pytest.mark.gpu


def negated(t):
    """The values of t, held in memory with the other sign."""
    v = torch._neg_view(t.neg())
    assert v.is_neg() and torch.equal(v, t)
    return v


def param(grad):
    p = torch.nn.Parameter(torch.zeros_like(grad))
    p.grad = grad
    return p


def test_known_norm_that_is_a_negated_view():
    norm = torch.tensor([8.0], device="cuda")
    want, got = param(torch.ones(5, device="cuda")), param(torch.ones(5, device="cuda"))
    per_b200.clip_grads_with_norm_([want], 2.0, norm)
    per_b200.clip_grads_with_norm_([got], 2.0, negated(norm))
    assert torch.equal(got.grad, want.grad) and float(got.grad[0]) > 0
    # the imaginary part of a conjugated number is such a view
    z = torch.complex(torch.zeros(1, device="cuda"), torch.full((1,), -8.0, device="cuda")).conj().imag
    assert z.is_neg() and float(z) == 8.0
    got = param(torch.ones(5, device="cuda"))
    per_b200.clip_grads_with_norm_([got], 2.0, z)
    assert torch.equal(got.grad, want.grad)


@pytest.mark.parametrize("kind", [1.0, 2.0, float("inf")])
def test_gradients_that_are_negated_views(kind):
    g = torch.randn(3001, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    want, got = param(g.clone()), param(negated(g))
    a = per_b200.clip_grad_norm_([want], 0.5, kind)
    b = per_b200.clip_grad_norm_([got], 0.5, kind)
    assert torch.equal(a, b) and torch.equal(got.grad, want.grad)
    assert torch.equal(per_b200.grad_norm(negated(g), kind), per_b200.grad_norm(g, kind))
