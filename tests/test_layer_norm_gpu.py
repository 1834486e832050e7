"""Layer norm, forward and backward, against float64 evaluations of its
formulas, within bounds derived from the roundings of the float32 evaluation
(oracle/learner.py)."""

import pytest
import torch

import per_b200
from oracle import learner as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)]
EPS = 1e-5


def normal(*shape, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def rows_like_activations(rows, dim, dtype, seed=0):
    x = normal(rows, dim, seed=seed) * (0.5 + normal(rows, 1, seed=seed + 1).abs())
    return (x + normal(rows, 1, seed=seed + 2)).to(dtype)


def params_like(dim, dtype, affine, seed=7):
    w = (1 + 0.2 * normal(dim, seed=seed)).to(dtype) if affine in ("both", "weight") else None
    b = (0.2 * normal(dim, seed=seed + 1)).to(dtype) if affine in ("both", "bias") else None
    return w, b


def close(got, want, bound, what):
    assert got.shape == want.shape, what
    far = (got.double() - want).abs() - bound
    assert bool((far <= 0).all()), f"{what}: over the bound by {float(far.max()):.3g}"


def check_forward(x, w, b, eps=EPS):
    y = per_b200.layer_norm(x, (x.shape[-1],), w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    x2 = x.reshape(-1, x.shape[-1])
    want, bound = ref.layer_norm_bound(x2, w, b, eps, x.dtype)
    close(y.reshape(x2.shape), want, bound, "y")
    return y


def check_train(x, w, b, dy, eps=EPS):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = per_b200.layer_norm(leaves[0], (x.shape[-1],), leaves[1], leaves[2], eps)
    x2, dy2 = x.reshape(-1, x.shape[-1]), dy.reshape(-1, x.shape[-1])
    want, bound = ref.layer_norm_bound(x2, w, b, eps, x.dtype)
    close(y.detach().reshape(x2.shape), want, bound, "y")
    y.backward(dy)
    ptype = w.dtype if w is not None else b.dtype if b is not None else F32
    dx, dw, db = ref.layer_norm_backward_bound(dy2, x2, w, eps, x.dtype, ptype)
    assert leaves[0].grad.dtype == x.dtype and leaves[0].grad.shape == x.shape
    close(leaves[0].grad.reshape(x2.shape), *dx, "dx")
    if w is not None:
        assert leaves[1].grad.dtype == w.dtype
        close(leaves[1].grad, *dw, "dw")
    if b is not None:
        close(leaves[2].grad, *db, "db")
    return [leaves[0].grad] + [t.grad for t in leaves[1:] if t is not None]


# dimensions around each of the kernels' tile widths, odd ones, and rows beyond
# the registers of a CTA
DIMS = [1, 2, 3, 5, 8, 16, 31, 32, 33, 63, 64, 100, 127, 128, 129, 255, 256, 257, 384, 511, 512,
        513, 520, 777, 1000, 1023, 1024, 1025, 1536, 2000, 2047, 2048, 2049, 2056, 4096, 4097,
        5000, 8191, 8192, 8193, 8200, 12288, 16384, 16392, 20000, 32768, 32776, 40001]


@pytest.mark.parametrize("dim", DIMS)
def test_every_width_in_every_type(dim):
    rows = 37 if dim < 10000 else 5
    for k, (dtype, ptype) in enumerate(TYPES):
        x = rows_like_activations(rows, dim, dtype, seed=dim + k)
        w, b = params_like(dim, ptype, "both")
        check_forward(x, w, b)
        check_train(x, w, b, normal(rows, dim, seed=3).to(dtype))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 7, 8, 9, 31, 33, 147, 148, 149, 295, 297, 1000, 4737,
                                  20011])
@pytest.mark.parametrize("dim", [32, 40, 256, 1001, 2048])
def test_every_number_of_rows(rows, dim):
    for dtype, ptype in ((F32, F32), (BF16, BF16)):
        x = rows_like_activations(rows, dim, dtype, seed=rows)
        w, b = params_like(dim, ptype, "both")
        check_train(x, w, b, normal(rows, dim, seed=5).to(dtype))


@pytest.mark.parametrize("affine", ["none", "weight", "bias", "both"])
@pytest.mark.parametrize("dim", [1, 30, 256, 1000, 20000])
def test_with_and_without_weight_and_bias(affine, dim):
    for dtype, ptype in TYPES:
        x = rows_like_activations(19, dim, dtype)
        w, b = params_like(dim, ptype, affine)
        check_forward(x, w, b)
        check_train(x, w, b, normal(19, dim, seed=9).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim,stride,offset", [(32, 74, 41), (32, 74, 0), (8, 74, 32), (1, 74, 40),
                                               (256, 522, 257), (1000, 1008, 8), (1000, 1001, 1),
                                               (2048, 2049, 0), (9000, 9100, 50), (9000, 9100, 48)])
def test_rows_inside_packed_rows(dtype, dim, stride, offset):
    """Views as a buffer's sample() returns them, read where they lie."""
    packed = rows_like_activations(67, stride, dtype)
    x = packed[:, offset:offset + dim]
    w, b = params_like(dim, F32, "both")
    check_forward(x, w, b)
    check_forward(x.contiguous(), w, b)
    dy = normal(67, stride + 3, seed=4).to(dtype)[:, 3:3 + dim]
    got = check_train(x, w, b, dy)
    assert got[0].is_contiguous()


def test_unaligned_parameters():
    for dtype, ptype in TYPES:
        for dim in (24, 264, 1000, 2048, 9000):
            flat = normal(2 * dim + 7).to(ptype)
            w, b = flat[1:1 + dim], flat[dim + 4:2 * dim + 4]
            x = rows_like_activations(11, dim, dtype)
            check_forward(x, w, b)
            check_train(x, w, b, normal(11, dim).to(dtype))


def test_leading_dimensions_and_orders():
    w, b = params_like(48, F32, "both")
    x = normal(6, 5, 7, 48)
    check_train(x, w, b, normal(6, 5, 7, 48, seed=2))
    check_forward(normal(48), w, b)                             # one row, no leading dimension
    check_forward(x.transpose(0, 2), w, b)                      # rows in another order
    check_train(x.transpose(1, 2), w, b, normal(6, 7, 5, 48, seed=2))
    check_forward(normal(48, 9).t(), w, b)                      # columns apart
    check_forward(normal(1, 48).expand(4, 48), w, b)            # one row four times
    check_forward(normal(9, 2, 48)[:, 0], w, b)
    check_forward(normal(3, 9, 80)[:, ::2, 16:64], w, b)
    check_forward(normal(5, 1, 48).as_strided((5, 1, 48), (48, 1, 1)), w, b)
    overlapping = normal(100).as_strided((40, 48), (1, 1))      # rows one value apart
    check_forward(overlapping, w, b)


def test_several_normalized_dimensions():
    x = normal(4, 3, 5, 6).requires_grad_()
    w, b = normal(5, 6, seed=1).requires_grad_(), normal(5, 6, seed=2).requires_grad_()
    dy = normal(4, 3, 5, 6, seed=3)
    y = per_b200.layer_norm(x, (5, 6), w, b, EPS)
    y.backward(dy)
    flat = lambda t: t.detach().reshape(-1, 30)  # noqa: E731
    want, bound = ref.layer_norm_bound(flat(x), flat(w)[0], flat(b)[0], EPS, F32)
    close(flat(y), want, bound, "y")
    dx, dw, db = ref.layer_norm_backward_bound(flat(dy), flat(x), flat(w)[0], EPS, F32, F32)
    close(flat(x.grad), *dx, "dx")
    close(flat(w.grad)[0], *dw, "dw")
    close(flat(b.grad)[0], *db, "db")
    assert w.grad.shape == (5, 6)


@pytest.mark.parametrize("dim", [16, 300, 2048, 20000])
def test_rows_far_from_zero(dim):
    """A mean of 10,000 standard deviations: the row's spread survives."""
    for dtype in (F32, BF16):
        x = (10000 + normal(9, dim)).to(dtype)
        x[0] = x[0, 0]  # and a constant row
        w, b = params_like(dim, F32, "both")
        check_forward(x, w, b)
        check_train(x, w, b, normal(9, dim, seed=1).to(dtype))


def test_extreme_values_stay_in_their_row():
    for dtype in (F32, BF16, F16):
        for dim in (20, 256, 1000, 9000):
            x = rows_like_activations(12, dim, dtype)
            w, b = params_like(dim, F32, "both")
            clean = per_b200.layer_norm(x, dim, w, b)
            for row, value in ((0, float("nan")), (5, float("inf")), (11, -float("inf"))):
                bad = x.clone()
                bad[row, dim // 2] = value
                y = per_b200.layer_norm(bad, dim, w, b)
                keep = torch.arange(12, device="cuda") != row
                assert torch.equal(y[keep], clean[keep])
                assert bool(y[row].isnan().all())
            # rows of equal values give the bias: their sum (a multiple of 1/2 below 2^23) and mean
            # are exact, so is the difference
            flat = torch.full((3, dim), 0.5, device="cuda", dtype=dtype)
            assert torch.equal(per_b200.layer_norm(flat, dim, None, b), b.to(dtype).expand(3, dim))


def test_epsilon():
    x = normal(6, 128) * 1e-3
    for eps in (0.0, 1e-12, 1e-6, 0.5):
        check_forward(x, None, None, eps)
        check_train(x, None, None, normal(6, 128, seed=1), eps)


def test_empty_inputs():
    w, b = (t.requires_grad_() for t in params_like(12, F32, "both"))
    x = torch.empty(0, 12, device="cuda", requires_grad=True)
    y = per_b200.layer_norm(x, 12, w, b)
    assert y.shape == (0, 12)
    y.sum().backward()
    assert x.grad.shape == (0, 12)
    assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b))
    assert per_b200.layer_norm(torch.empty(3, 0, device="cuda"), 0).shape == (3, 0)
    assert per_b200.layer_norm(torch.empty(0, 5, 12, device="cuda"), 12, w.detach()).shape == (0, 5, 12)


def test_gradient_of_a_broadcast_sum():
    """y.sum() hands back one expanded value, y[0] + ... one row for all."""
    w, b = params_like(200, F32, "both")
    x = normal(33, 200)
    check_train(x, w, b, torch.ones((), device="cuda").expand(33, 200))
    check_train(x, w, b, normal(1, 200, seed=8).expand(33, 200))
    check_train(x, w, b, normal(33, 1, seed=8).expand(33, 200))


def test_only_some_gradients_wanted():
    x, dy = normal(70, 300), normal(70, 300, seed=1)
    w, b = params_like(300, F32, "both")
    full = check_train(x, w, b, dy)
    for want in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(want >> k & 1)) for k, t in enumerate((x, w, b))]
        per_b200.layer_norm(leaves[0], 300, leaves[1], leaves[2]).backward(dy)
        for k, t in enumerate(leaves):
            if want >> k & 1:
                assert torch.equal(t.grad, full[k])
            else:
                assert t.grad is None
    xs = [t.clone().requires_grad_() for t in (x, w, b)]
    y = per_b200.layer_norm(xs[0], 300, xs[1], xs[2])
    gw, = torch.autograd.grad(y, [xs[1]], dy)  # one of three, though all require it
    assert torch.equal(gw, full[1])


def test_gradient_against_differences():
    """Central differences of a float64 evaluation, at the kernel's own inputs."""
    rows, dim = 3, 24
    x, w, b = normal(rows, dim), *params_like(dim, F32, "both")
    dy = normal(rows, dim, seed=6)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    per_b200.layer_norm(leaves[0], dim, leaves[1], leaves[2]).backward(dy)

    def loss(x, w, b):
        return float((ref.layer_norm(x, w, b, EPS)[0] * dy.double()).sum())

    h = 1e-5
    bounds = ref.layer_norm_backward_bound(dy, x, w, EPS, F32, F32)
    for k in range(3):
        base = [t.double() for t in (x, w, b)]
        for at in range(0, base[k].numel(), 5):
            ends = []
            for s in (h, -h):
                moved = [t.clone() for t in base]
                moved[k].view(-1)[at] += s
                ends.append(loss(*moved))
            slope = (ends[0] - ends[1]) / (2 * h)
            # third derivatives here are below 1e4 in size, differences of float64 losses of
            # about 100 are good to 1e-12: 1e-6 covers h^2 / 6 of the one and the other over h
            assert abs(slope - float(leaves[k].grad.view(-1)[at])) <= \
                1e-6 + float(bounds[k][1].view(-1)[at])


def test_same_bits_every_time():
    x, dy = normal(5003, 512), normal(5003, 512, seed=1)
    w, b = params_like(512, F32, "both")
    first = check_train(x, w, b, dy)
    for _ in range(5):
        for a, c in zip(first, check_train(x, w, b, dy)):
            assert torch.equal(a, c)


def test_weights_with_gaps_and_in_another_order():
    for dim in (24, 300, 2048):
        x, dy = normal(17, dim), normal(17, dim, seed=1)
        spread = normal(dim, 3, seed=2)
        w, b = spread[:, 1], spread[:, 2]
        check_forward(x, w, b)
        check_train(x, w, b, dy)
    x, dy = normal(9, 5, 6), normal(9, 5, 6, seed=1)
    w = normal(6, 5, seed=2).t()  # [5, 6], columns first
    leaves = [x.clone().requires_grad_(), w.detach().requires_grad_()]
    y = per_b200.layer_norm(leaves[0], (5, 6), leaves[1])
    y.backward(dy)
    flat = lambda t: t.detach().reshape(-1, 30)  # noqa: E731
    want, bound = ref.layer_norm_bound(flat(x), flat(w)[0], None, EPS, F32)
    close(flat(y), want, bound, "y")
    dx, dw, _ = ref.layer_norm_backward_bound(flat(dy), flat(x), flat(w)[0], EPS, F32, F32)
    close(flat(leaves[0].grad), *dx, "dx")
    close(flat(leaves[1].grad)[0], *dw, "dw")


@pytest.mark.parametrize("dim", [40, 1001, 1024, 5001, 20001, 70001])
def test_one_gradient_row_for_all(dim):
    """An upstream gradient of stride 0 over the rows, read where it lies."""
    for dtype in (F32, BF16):
        x = rows_like_activations(7, dim, dtype)
        w, b = params_like(dim, F32, "both")
        check_train(x, w, b, normal(1, dim, seed=8).to(dtype).expand(7, dim))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("dim", [40, 77, 1000, 1001, 9000, 9001, 20000, 20001, 70001])
def test_each_gradient_alone(dtype, dim):
    x, dy = rows_like_activations(23, dim, dtype), normal(23, dim, seed=1).to(dtype)
    w, b = params_like(dim, F32, "both")
    full = check_train(x, w, b, dy)
    for k in range(3):
        leaves = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        per_b200.layer_norm(leaves[0], dim, leaves[1], leaves[2]).backward(dy)
        assert torch.equal(leaves[k].grad, full[k])


@pytest.mark.parametrize("dim", [3, 20, 70, 600, 3000])
def test_output_beside_the_input_in_one_buffer(dim):
    """The C entry point writes columns between the ones it reads, and nothing else."""
    from per_b200 import _lib

    for dtype, code in ((F32, 0), (BF16, 1)):
        for gap in (0, 1, 5):
            width = 2 * dim + 3 * gap + 1
            buf = normal(50, width).to(dtype)
            old = buf.clone()
            eb = buf.element_size()
            n = _lib.Norm(50, dim, code, code, EPS)
            rc = _lib.lib.per_layer_norm(n, buf.data_ptr() + gap * eb, width, None, None,
                                         buf.data_ptr() + (2 * gap + dim) * eb, width, None,
                                         torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            torch.cuda.synchronize()
            want, bound = ref.layer_norm_bound(old[:, gap:gap + dim], None, None, EPS, dtype)
            got = buf[:, 2 * gap + dim:2 * gap + 2 * dim]
            close(got, want, bound, "y")
            buf[:, 2 * gap + dim:2 * gap + 2 * dim] = old[:, 2 * gap + dim:2 * gap + 2 * dim]
            assert torch.equal(buf, old)


def test_rows_beyond_the_workspace_of_a_wave():
    """Millions of short rows: each thread's row walks far."""
    x = normal(3_000_000, 8)
    w, b = params_like(8, F32, "both")
    check_train(x, w, b, normal(3_000_000, 8, seed=1))


def test_recomputed_activations():
    from torch.utils.checkpoint import checkpoint

    m = torch.nn.Sequential(torch.nn.Linear(64, 64), per_b200.LayerNorm(64), torch.nn.ReLU()).cuda()
    x = normal(30, 64).requires_grad_()
    want = torch.autograd.grad(m(x).square().sum(), [x, *m.parameters()])
    got = torch.autograd.grad(checkpoint(m, x, use_reentrant=False).square().sum(), [x, *m.parameters()])
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_calls_from_several_threads():
    import threading

    x, w = normal(2000, 777), torch.ones(777, device="cuda")
    want = per_b200.layer_norm(x, 777, w)
    leaf = x.clone().requires_grad_()
    wantg, = torch.autograd.grad(per_b200.layer_norm(leaf, 777, w).square().sum(), [leaf])
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                leaf = x.clone().requires_grad_()
                y = per_b200.layer_norm(leaf, 777, w)
                g, = torch.autograd.grad(y.square().sum(), [leaf])
                n = per_b200.grad_norm([g])
                s.synchronize()
                if not torch.equal(y, want) or not torch.equal(g, wantg) or not float(n) > 0:
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


FIRST_CALL = """
import sys
sys.path.insert(0, {path!r})
import torch, per_b200
x = torch.randn(300, {dim}, device="cuda", requires_grad=True)
w = torch.ones({dim}, device="cuda", requires_grad=True)
b = torch.zeros({dim}, device="cuda", requires_grad=True)
p = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in {sizes}]
for q in p:
    q.grad = torch.randn_like(q)
start = [q.grad.clone() for q in p]
dy = torch.randn(300, {dim}, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = per_b200.layer_norm(x, {dim}, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    norm = per_b200.clip_grad_norm_(p, 0.5)
g.replay()
torch.cuda.synchronize()
y2 = per_b200.layer_norm(x, {dim}, w, b)
for a, c in zip(grads, torch.autograd.grad(y2, (x, w, b), dy)):
    assert torch.equal(a, c)
assert torch.equal(y, y2)
clipped = [q.grad.clone() for q in p]
for q, s in zip(p, start):
    q.grad.copy_(s)
assert torch.equal(per_b200.clip_grad_norm_(p, 0.5), norm)
for q, c in zip(p, clipped):
    assert torch.equal(q.grad, c)
print("fine")
"""


@pytest.mark.parametrize("dim,sizes", [(256, [1000, 7]), (1001, [3_000_000, 5]), (20000, [100] * 300)])
def test_first_call_of_a_process_is_captured(dim, sizes):
    import os
    import subprocess
    import sys

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-per_b200")
    out = subprocess.run([sys.executable, "-c", FIRST_CALL.format(path=path, dim=dim, sizes=sizes)],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "fine" in out.stdout, out.stderr[-2000:]


def test_second_derivative_is_refused():
    x = normal(4, 8).requires_grad_()
    y = per_b200.layer_norm(x, 8)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(y.square().sum(), x, create_graph=True)


def test_forward_mode_is_refused():
    x, w = normal(4, 8), torch.ones(8, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            per_b200.layer_norm(dual, 8)
        dual = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            per_b200.layer_norm(x, 8, dual, w)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            per_b200.layer_norm(x, 8, w, dual)


def test_lazily_negated_views():
    x, w, b, dy = normal(6, 40), normal(40), normal(40), normal(6, 40)
    neg = [torch._neg_view(t.neg()) for t in (x, w, b, dy)]  # the same values, negated when read
    assert all(t.is_neg() for t in neg)
    check_forward(neg[0], neg[1], neg[2])
    leaves = [t.detach().requires_grad_() for t in neg[:3]]
    got = torch.autograd.grad(per_b200.layer_norm(leaves[0], 40, *leaves[1:]), leaves, neg[3])
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(per_b200.layer_norm(leaves[0], 40, *leaves[1:]), leaves, dy)
    assert all(torch.equal(g, h) for g, h in zip(got, want))  # the same calls on copies


def test_second_backward_and_changed_inputs_are_refused():
    x = normal(4, 8).requires_grad_()
    y = per_b200.layer_norm(x, 8)
    y.sum().backward(retain_graph=True)
    y.sum().backward()
    with pytest.raises(RuntimeError):
        y.sum().backward()
    h = x * 2
    y = per_b200.layer_norm(h, 8)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_bad_arguments():
    x = normal(4, 8)
    w = torch.ones(8, device="cuda")
    with pytest.raises(ValueError, match="normalized_shape"):
        per_b200.layer_norm(x, 7)
    with pytest.raises(ValueError, match="normalized_shape"):
        per_b200.layer_norm(x, ())
    with pytest.raises(ValueError, match="normalized_shape"):
        per_b200.layer_norm(x, (2, 4, 8))
    with pytest.raises(ValueError, match="shape"):
        per_b200.layer_norm(x, 8, w[:7])
    with pytest.raises(ValueError, match="eps"):
        per_b200.layer_norm(x, 8, w, eps=-1.0)
    with pytest.raises(ValueError, match="device"):
        per_b200.layer_norm(x, 8, w.cpu())
    with pytest.raises(TypeError):
        per_b200.layer_norm(x.double(), 8)
    with pytest.raises(TypeError):
        per_b200.layer_norm(x.to(torch.int32), 8)
    with pytest.raises(TypeError):
        per_b200.layer_norm(x, 8, w.bfloat16())
    with pytest.raises(TypeError):
        per_b200.layer_norm(x.half(), 8, w.bfloat16())
    with pytest.raises(TypeError):
        per_b200.layer_norm(x.half(), 8, w.half(), w)
    with pytest.raises(RuntimeError, match="CUDA"):
        per_b200.layer_norm(x.cpu(), 8)


def test_row_offsets_beyond_32_bits():
    rows, dim = 70000, 32768  # 2.3e9 values
    x = torch.empty(rows, dim, device="cuda", dtype=BF16)
    x[:] = normal(dim).to(BF16)
    picked = [0, 1, 65535, 65536, 65537, rows - 1]
    for r in picked:
        x[r] = rows_like_activations(1, dim, BF16, seed=r)[0]
    w, b = params_like(dim, BF16, "both")
    x.requires_grad_()
    y = per_b200.layer_norm(x, dim, w, b)
    rows_x = x.detach()[picked]
    want, bound = ref.layer_norm_bound(rows_x, w, b, EPS, BF16)
    close(y.detach()[picked], want, bound, "y")
    dy = torch.zeros_like(y)
    dy[picked] = normal(len(picked), dim, seed=1).to(BF16)
    dx, = torch.autograd.grad(y, [x], dy)
    want = ref.layer_norm_backward_bound(dy[picked], rows_x, w, EPS, BF16, BF16)[0]
    close(dx[picked], *want, "dx")
    assert float(dx[2:60000].abs().max()) == 0.0


def test_other_stream():
    x = normal(4000, 1024)
    w, b = params_like(1024, F32, "both")
    want = check_train(x, w, b, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000)
        late = x * 1.0  # written on the side stream, after the sleep
        got = check_train(late, w, b, late)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(want, got):
        assert torch.equal(a, c)


def train_step(x, w, b, dy, out):
    y = per_b200.layer_norm(x, x.shape[-1], w, b)
    out["y"] = y.detach()
    out["grads"] = torch.autograd.grad(y, (x, w, b), dy)


def test_captured_training_steps():
    """Two graphs with workspaces of their own, replayed by turns and at once."""
    made = []
    for seed, dim in ((1, 512), (2, 1001)):
        x, dy = normal(3000, dim, seed=seed), normal(3000, dim, seed=seed + 10)
        w, b = params_like(dim, F32, "both", seed=seed)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        out = {}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            train_step(*leaves, dy, out)
        torch.cuda.current_stream().wait_stream(side)
        eager = [out["y"].clone(), *(g.clone() for g in out["grads"])]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            train_step(*leaves, dy, out)
        made.append((g, leaves, dy, out, eager))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for together in (False, True):
        for _ in range(3):
            for (g, _, _, out, _), s in zip(made, streams):
                if together:
                    s.wait_stream(torch.cuda.current_stream())
                    with torch.cuda.stream(s):
                        g.replay()
                else:
                    g.replay()
            torch.cuda.synchronize()
            for _, _, _, out, eager in made:
                for a, c in zip(eager, [out["y"], *out["grads"]]):
                    assert torch.equal(a, c)
    # new inputs in the same places
    g, leaves, dy, out, _ = made[0]
    with torch.no_grad():
        leaves[0].copy_(normal(3000, 512, seed=77))
    g.replay()
    torch.cuda.synchronize()
    want = check_train(leaves[0].detach(), leaves[1].detach(), leaves[2].detach(), dy)
    for a, c in zip(want, out["grads"]):
        assert torch.equal(a, c)


def test_capture_beside_a_living_eager_graph_is_refused():
    x, w = normal(8, 16).requires_grad_(), torch.ones(16, device="cuda", requires_grad=True)
    eager = per_b200.layer_norm(x, 16, w).sum()  # on the default stream, kept alive
    z = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="eager graph"):
            per_b200.layer_norm(x, 16, w)
        with torch.no_grad():  # without gradients nothing stands against it
            y = per_b200.layer_norm(x, 16, w)
        z += 1
    g.replay()
    torch.cuda.synchronize()
    assert float(z.sum()) == 4.0 and torch.equal(y, per_b200.layer_norm(x, 16, w))
    del eager
    g2 = torch.cuda.CUDAGraph()
    out = {}
    with torch.cuda.graph(g2):
        y = per_b200.layer_norm(x, 16, w)
        out["g"], = torch.autograd.grad(y, (x,), torch.ones_like(y))
    g2.replay()
    torch.cuda.synchronize()
    want = ref.layer_norm_backward_bound(torch.ones_like(x), x.detach(), w.detach(), EPS, F32, F32)[0]
    close(out["g"], *want, "dx")


def test_module_matches_the_function():
    m = per_b200.LayerNorm(64, eps=1e-3, device="cuda")
    with torch.no_grad():
        m.weight.copy_(normal(64))
        m.bias.copy_(normal(64, seed=1))
    x = normal(10, 64, seed=2)
    assert torch.equal(m(x), per_b200.layer_norm(x, 64, m.weight, m.bias, 1e-3))
    m(x).sum().backward()
    assert m.weight.grad is not None and m.bias.grad is not None
