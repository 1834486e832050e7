"""Tracers do not see the learner's calls, so a trace would hold their results as
constants: every call refuses to be traced, on any device and before any other
check, and what merely watches operators is served as before."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import per_b200


def clip(t):
    p = torch.nn.Parameter(torch.ones_like(t))
    p.grad = t * 1.0
    per_b200.clip_grad_norm_([p], 1.0)
    return p.grad


def clip_known(t):
    p = torch.nn.Parameter(torch.ones_like(t))
    p.grad = t * 1.0
    per_b200.clip_grads_with_norm_([p], 1.0, t.sum())
    return p.grad


CALLS = {"layer_norm": lambda t: per_b200.layer_norm(t, (8,)), "grad_norm": lambda t: per_b200.grad_norm([t]),
         "clip_grad_norm_": clip, "clip_grads_with_norm_": clip_known}


def in_fake_mode(f, x):
    with FakeTensorMode() as mode:
        f(mode.from_tensor(x))


TRACERS = {
    "jit": lambda f, x: torch.jit.trace(f, (x,), check_trace=False),
    "fx": lambda f, x: make_fx(f)(x),
    "fx_before_autograd": lambda f, x: make_fx(f, pre_dispatch=True)(x),
    "fx_fake": lambda f, x: make_fx(f, tracing_mode="fake")(x),
    "fake": in_fake_mode,
}


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("tracer", TRACERS)
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused(call, tracer, device):
    x = torch.ones(4, 8, device=device)
    with pytest.raises(RuntimeError, match="traced"), torch.set_grad_enabled(call != "layer_norm"):
        TRACERS[tracer](CALLS[call], x)


@pytest.mark.filterwarnings("ignore")
def test_a_module_cannot_be_traced():
    net = torch.nn.Sequential(torch.nn.Linear(4, 8), per_b200.LayerNorm(8), torch.nn.Linear(8, 1))
    with torch.no_grad(), pytest.raises(RuntimeError, match="layer_norm cannot be traced"):
        torch.jit.trace(net, torch.ones(3, 4))


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_tracing_a_backward_pass_is_refused():
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    y = per_b200.layer_norm(x, 8)  # before the trace
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda dy: torch.autograd.grad(y, x, dy)[0])(torch.ones(4, 8, device="cuda"))


@pytest.mark.gpu
def test_transforms_are_refused():
    x, w = torch.randn(5, 4, 8, device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="layer_norm takes plain tensors"):
        torch.vmap(lambda t: per_b200.layer_norm(t, 8))(x)
    with pytest.raises(RuntimeError, match="layer_norm takes plain tensors"):
        torch.func.grad(lambda t: per_b200.layer_norm(x, 8, t).sum())(w)
    with pytest.raises(RuntimeError, match="layer_norm takes plain tensors"):
        torch.func.grad(lambda t: per_b200.layer_norm(x, 8, None, t).sum())(w)
    with pytest.raises(RuntimeError, match="grad_norm takes plain tensors"):
        torch.vmap(lambda t: per_b200.grad_norm([t]))(x)


@pytest.mark.gpu
def test_what_watches_operators_is_served():
    from torch.utils.flop_counter import FlopCounterMode

    lin = torch.nn.Linear(8, 8).cuda()
    x = torch.randn(4, 8, device="cuda")
    want = per_b200.layer_norm(lin(x), 8)
    with FlopCounterMode(display=False) as count:
        got = per_b200.layer_norm(lin(x), 8)
        got.sum().backward()
    assert torch.equal(got, want) and count.get_total_flops() > 0


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_compiled_code_breaks_its_graph_and_runs():
    norm = per_b200.LayerNorm(8, device="cuda")
    net = torch.nn.Sequential(torch.nn.Linear(8, 8).cuda(), norm, torch.nn.ReLU())
    compiled = torch.compile(net, backend="eager")
    for seed in range(3):
        x = torch.randn(4, 8, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))
        with torch.no_grad():
            assert torch.equal(compiled(x), net(x))
        compiled(x).sum().backward()
        got, norm.weight.grad = norm.weight.grad, None
        net(x).sum().backward()
        assert torch.equal(got, norm.weight.grad)
        norm.weight.grad = None
