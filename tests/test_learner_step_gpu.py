"""Layer norm and gradient clipping together, as a learner's step runs them
between sample and update_priorities: the gradients against a float64 network,
a whole captured update, and the profiler command's learner."""

import subprocess
import sys

import pytest
import torch
import torch.nn as nn

from oracle import learner as ref

OBS, ACT, BATCH, MAX_NORM = 32, 8, 64, 0.05


def data(seed=3):
    g = torch.Generator().manual_seed(seed)
    batch = {"obs": torch.randn(BATCH, OBS, generator=g), "action": torch.randn(BATCH, ACT, generator=g),
             "reward": torch.randn(BATCH, 1, generator=g)}
    return batch, torch.rand(BATCH, generator=g) * 0.9 + 0.1


def weights_of(seed=21):
    """The learner's parameters, drawn on the CPU so that both networks get the same."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for net, i, o in (("actor", OBS, ACT), ("q0", OBS + ACT, 1), ("q1", OBS + ACT, 1)):
        layers = []
        for a, b, norm in ((i, 256, True), (256, 256, True), (256, o, False)):
            layers += [torch.randn(b, a, generator=g) * (2 / a) ** 0.5, torch.randn(b, generator=g) * 0.1]
            if norm:
                layers += [1 + 0.2 * torch.randn(b, generator=g), 0.2 * torch.randn(b, generator=g)]
        out[net] = layers
    return out


class Relu(torch.autograd.Function):
    nearest = float("inf")  # smallest |input| seen

    @staticmethod
    def forward(ctx, x):
        Relu.nearest = min(Relu.nearest, float(x.abs().min()))
        ctx.save_for_backward(x)
        return x.clamp(min=0)

    @staticmethod
    def backward(ctx, g):
        return g * (ctx.saved_tensors[0] > 0)


def exact_gradients():
    """The clipped gradients, the norm and |TD| in float64 on the CPU, from the formulas."""
    batch, w = data()
    params = {k: [t.double().requires_grad_() for t in v] for k, v in weights_of().items()}
    batch, w = {k: v.double() for k, v in batch.items()}, w.double()

    def net(p, x):
        for k in (0, 4):
            x = x @ p[k].T + p[k + 1]
            x = Relu.apply(ref.layer_norm(x, p[k + 2], p[k + 3], 1e-5)[0])
        return x @ p[8].T + p[9]

    qin = torch.cat([batch["obs"], batch["action"]], 1)
    tds = [net(params[q], qin).squeeze(1) - batch["reward"].squeeze(1) for q in ("q0", "q1")]
    loss = sum((w * td.pow(2)).mean() for td in tds) + 1e-3 * net(params["actor"], batch["obs"]).pow(2).mean()
    flat = [t for v in params.values() for t in v]
    grads = torch.autograd.grad(loss, flat)
    norm = ref.grad_norm(grads)
    k = ref.scale_of(norm, MAX_NORM)
    return [g * k for g in grads], norm, tds[0].abs().detach()


def test_no_unit_sits_on_the_kink():
    """The premise of the comparison below: no activation is so near to zero that float32's error
    (about 1e-6 here) could switch it."""
    Relu.nearest = float("inf")
    _, norm, _ = exact_gradients()
    assert Relu.nearest > 2e-5
    assert norm > 2 * MAX_NORM


@pytest.mark.gpu
def test_gradients_of_a_step():
    from per_b200 import profile_utd

    want, norm, td = exact_gradients()
    learner = profile_utd.Learner(OBS, ACT, 2, "cuda", layer_norm=True, max_grad_norm=MAX_NORM)
    with torch.no_grad():
        for p, t in zip(learner.params, [t for v in weights_of().values() for t in v]):
            assert p.shape == t.shape
            p.copy_(t)
    batch, w = data()
    got_td = learner.step({k: v.cuda() for k, v in batch.items()}, w.cuda())
    # A product of 256 terms is off by at most 256 u of the product of the norms, a layer norm by
    # about 70 u; three layers forward and three back, each passing errors on without
    # amplifying them by more than about 2: 6 * 326 u * 2^3 = 9.3e-4 in the worst case.
    bound = 6 * 326 * ref.U32 * 8
    assert float((got_td.double().cpu() - td).norm()) <= bound * float(td.norm() + data()[0]["reward"].norm())
    total = sum(float(g.square().sum()) for g in want) ** 0.5
    for p, g in zip(learner.params, want):
        assert float((p.grad.double().cpu() - g).norm()) <= bound * total
    got = sum(float(p.grad.double().square().sum()) for p in learner.params) ** 0.5
    assert abs(got - MAX_NORM) <= 1e-5 * MAX_NORM  # 1e-6 over a norm above 0.1, and rounding


@pytest.mark.gpu
def test_captured_update_from_sample_to_priorities():
    """One update (sample, critic with layer norms, backward, clip, weight step, priorities) captured
    into a graph and replayed gives the bits of the same update run eagerly."""
    import per_b200

    fields = {"obs": OBS, "action": ACT, "reward": 1, "next_obs": OBS, "done": 1}

    def make():
        torch.manual_seed(0)
        buf = per_b200.PERBuffer(10_000, fields)
        buf.add({k: torch.randn(5000, d, device="cuda") for k, d in fields.items()})
        net = nn.Sequential(nn.Linear(OBS + ACT, 200), per_b200.LayerNorm(200), nn.ReLU(),
                            nn.Linear(200, 1)).cuda()
        return buf, net, buf.sample_out(256)

    def update(buf, net, slot):
        batch, idx, w = buf.sample(256, out=slot)
        obs = per_b200.layer_norm(batch["obs"], OBS)  # a field view, normalised where it lies
        td = net(torch.cat([obs, batch["action"]], 1)).squeeze(1) - batch["reward"].squeeze(1)
        grads = torch.autograd.grad((w * td.square()).mean(), list(net.parameters()))
        for p, g in zip(net.parameters(), grads):
            p.grad = g
        norm = per_b200.clip_grad_norm_(net.parameters(), 0.1)
        with torch.no_grad():
            for p in net.parameters():
                p.sub_(p.grad, alpha=0.1)
        buf.update_priorities(idx, td.detach().abs())
        return norm

    state = []
    for captured in (False, True):
        buf, net, slot = make()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            norms = [update(buf, net, slot).clone() for _ in range(2)]
        torch.cuda.current_stream().wait_stream(side)
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                norm = update(buf, net, slot)
            for _ in range(6):
                g.replay()
                norms.append(norm.clone())
        else:
            norms += [update(buf, net, slot).clone() for _ in range(6)]
        torch.cuda.synchronize()
        assert buf.status()["errors"] == 0
        state.append((torch.stack(norms), [p.detach().clone() for p in net.parameters()],
                      buf.priorities.clone()))
    assert torch.equal(state[0][0], state[1][0])
    for a, b in zip(state[0][1], state[1][1]):
        assert torch.equal(a, b)
    assert torch.equal(state[0][2], state[1][2])
    assert bool((state[0][0] > 0).all())


@pytest.mark.gpu
def test_profiler_command_runs_the_learner():
    import json
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run(
        [sys.executable, "-m", "per_b200.profile_utd", "--utd", "4", "--batch-size", "64", "--capacity",
         "20000", "--steps", "3", "--warmup", "1", "--num-q", "3", "--layer-norm", "--max-grad-norm", "1.5"],
        cwd=os.path.join(root, "triton-per_b200"), capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    r = json.loads(out.stdout.strip().splitlines()[-1])
    assert r["layer_norm"] is True and r["max_grad_norm"] == 1.5
    assert 0 < r["replay_share"] < 1 and r["status"]["errors"] == 0
