"""The global gradient norm and its clipping against float64, within bounds
derived from the roundings of the float32 evaluation (oracle/learner.py)."""

import math

import pytest
import torch

import per_b200
from oracle import learner as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def normal(*shape, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def bucket(sizes, dtype, seed=0, scale=1.0, start=0):
    """Gradients one behind the other in one buffer, at any alignment."""
    flat = (normal(start + sum(sizes), seed=seed) * scale).to(dtype)
    at, out = start, []
    for n in sizes:
        out.append(flat[at:at + n])
        at += n
    return out, flat


def check_norm(got, grads, norm_type=2.0):
    want = ref.grad_norm(grads, norm_type)
    assert got.dtype == F32 and got.shape == () and got.is_cuda
    n = sum(g.numel() for g in grads)
    bound = 0.0 if norm_type == math.inf else ref.norm_bound(n)
    assert abs(float(got) - want) <= want * (bound + 2 * ref.U32), (float(got), want)
    return want


def check_clip(grads, max_norm, norm_type=2.0):
    before = [g.clone() for g in grads]
    got = per_b200.clip_grad_norm_(params(grads), max_norm, norm_type)
    want = check_norm(got, before, norm_type)
    k = ref.scale_of(want, max_norm)
    rel = ref.norm_bound(sum(g.numel() for g in grads)) + 6 * ref.U32
    for g, old in zip(grads, before):
        exact = old.double() * k
        off = (g.double() - exact).abs()
        bound = exact.abs() * rel + ref.half_step(g.dtype) * exact.abs() * (1 + rel) + ref.tiny(g.dtype)
        assert bool((off <= bound).all())
    return got


SIZES = [[1], [7], [8], [9], [256], [1000003], [1, 2, 3, 4, 5, 6, 7, 8, 9], [10240, 256, 65536, 256, 256, 1],
         [8192], [8191], [8193], [16384 * 3 + 5, 1, 1, 70000], [3, 100000, 2, 0, 5, 0], [300000] * 20]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clipping(dtype, sizes):
    for start in (0, 1, 3):
        grads, _ = bucket(sizes, dtype, seed=start, start=start)
        for kind in (2.0, 1.0, math.inf):
            check_norm(per_b200.grad_norm(grads, kind), grads, kind)
        check_clip(grads, 0.25)


@pytest.mark.parametrize("kind", [1.0, 2, math.inf])
def test_other_norms_clip(kind):
    grads, _ = bucket([1000, 3, 50000], F32)
    check_clip(grads, 0.5, kind)


@pytest.mark.parametrize("count", [63, 64, 65, 300, 1023, 1024, 1025, 2500])
def test_many_tensors_of_mixed_types(count):
    grads = []
    for i in range(count):
        dtype = (F32, BF16, F16)[i % 3]
        grads.append(normal(1 + (i * 37) % 500, seed=i).to(dtype))
    check_norm(per_b200.grad_norm(grads), grads)
    check_clip(grads, 3.0)


def test_neighbours_are_left_alone():
    """What lies between and around the gradients of a buffer keeps its bits."""
    for dtype in (F32, BF16, F16):
        flat = normal(5000).to(dtype)
        old = flat.clone()
        grads = [flat[3:10], flat[17:1000], flat[1001:1002], flat[1003:4993]]
        check_clip(grads, 0.1)
        inside = torch.zeros(5000, dtype=torch.bool, device="cuda")
        for a, b in ((3, 10), (17, 1000), (1001, 1002), (1003, 4993)):
            inside[a:b] = True
        assert torch.equal(flat[~inside], old[~inside])


def test_below_the_threshold_nothing_changes():
    grads, flat = bucket([100000, 33], F32)
    old = flat.clone()
    got = per_b200.clip_grad_norm_(params(grads), 1e6)
    check_norm(got, [old])
    assert torch.equal(flat, old)
    assert float(per_b200.clip_grad_norm_(params(grads), math.inf)) == float(got)
    assert torch.equal(flat, old)


def test_zero_threshold_and_zero_gradients():
    grads, flat = bucket([5000], F32)
    per_b200.clip_grad_norm_(params(grads), 0.0)
    assert float(flat.abs().max()) == 0.0
    assert float(per_b200.clip_grad_norm_(params(grads), 1.0)) == 0.0
    assert float(flat.abs().max()) == 0.0


def test_values_whose_squares_leave_float32():
    for scale in (1e25, 1e-25, 1e-38):
        grads, _ = bucket([70001, 5], F32, scale=scale)
        check_norm(per_b200.grad_norm(grads), grads)
    grads, _ = bucket([70001, 5], F32, scale=1e25)
    check_clip(grads, 1.0)
    grads, _ = bucket([70001, 5], BF16, scale=1e30)
    check_norm(per_b200.grad_norm(grads), grads)
    mixed = [torch.full((10,), 1e-30, device="cuda"), torch.full((10,), 1e20, device="cuda")]
    check_norm(per_b200.grad_norm(mixed), mixed)


def test_not_a_number_and_infinity():
    for dtype in (F32, BF16, F16):
        for kind in (2.0, 1.0, math.inf):
            grads, flat = bucket([9000, 100], dtype)
            flat[4321] = math.nan
            assert math.isnan(float(per_b200.clip_grad_norm_(params(grads), 1.0, kind)))
            assert bool(flat.isnan().all())
            grads, flat = bucket([9000, 100], dtype)
            flat[77] = -math.inf
            assert float(per_b200.clip_grad_norm_(params(grads), 1.0, kind)) == math.inf
            assert bool(flat[77].isnan())  # inf times 0
            flat[77] = 0
            assert float(flat.abs().max()) == 0.0


def test_error_if_nonfinite_leaves_the_gradients():
    grads, flat = bucket([500], F32)
    old = flat.clone()
    want = per_b200.grad_norm(grads)
    got = per_b200.clip_grad_norm_(params(grads), 0.5, error_if_nonfinite=True)
    assert torch.equal(got, want) and not torch.equal(flat, old)
    for bad in (math.nan, math.inf):
        flat.copy_(old)
        flat[3] = bad
        before = flat.clone()
        with pytest.raises(RuntimeError, match="not finite"):
            per_b200.clip_grad_norm_(params(grads), 0.5, error_if_nonfinite=True)
        assert torch.equal(flat.nan_to_num(1.0), before.nan_to_num(1.0))


def test_known_norm():
    grads, flat = bucket([5000, 70], F32)
    old = flat.clone()
    p = params(grads)
    per_b200.clip_grads_with_norm_(p, 2.0, torch.tensor(8.0, device="cuda"))
    # the factor 2 / (8 + 1e-6) in float32, three roundings
    assert bool(((flat.double() - old.double() * (2 / (8 + 1e-6))).abs() <= 4 * ref.U32 * old.abs()).all())
    once = flat.clone()
    per_b200.clip_grads_with_norm_(p, 2.0, torch.tensor([1.0], device="cuda"))
    assert torch.equal(flat, once)
    for bad in (torch.tensor(8.0), torch.tensor(8.0, device="cuda", dtype=torch.float64),
                torch.ones(2, device="cuda"), grads[0][:1]):
        with pytest.raises(ValueError, match="total_norm"):
            per_b200.clip_grads_with_norm_(p, 2.0, bad)


def test_layouts():
    dense = normal(40, 30).t()                                  # transposed: dense, any order
    channels = normal(4, 6, 5, 5).to(memory_format=torch.channels_last)
    grads = [dense, channels, normal(3, 4, 5), torch.tensor(2.0, device="cuda")]
    check_norm(per_b200.grad_norm(grads), grads)
    check_clip(grads, 0.5)
    with pytest.raises(ValueError, match="gaps"):
        per_b200.grad_norm([normal(10, 10)[:, :5]])
    with pytest.raises(ValueError, match="gaps"):
        per_b200.grad_norm([normal(1).expand(10)])
    assert float(per_b200.grad_norm(torch.tensor([3.0, 4.0], device="cuda"))) == 5.0


def test_shared_memory_is_refused():
    flat = normal(100)
    p = params([flat[:60]])[0]
    for grads in ([p, p], params([flat[:60], flat[59:]]), params([flat[50:], flat[:51]])):
        old = flat.clone()
        with pytest.raises(ValueError, match="share memory"):
            per_b200.clip_grad_norm_(grads, 1e-3)
        with pytest.raises(ValueError, match="share memory"):
            per_b200.clip_grads_with_norm_(grads, 1e-3, torch.tensor(1.0, device="cuda"))
        assert torch.equal(flat, old)
    check_clip([flat[50:], flat[:50]], 0.5)  # side by side, in another order
    twice = [flat, flat]                     # reading alone may
    check_norm(per_b200.grad_norm(twice), twice)


def test_bad_gradients():
    with pytest.raises(TypeError):
        per_b200.grad_norm([normal(4).double()])
    with pytest.raises(TypeError):
        per_b200.grad_norm([torch.ones(4, device="cuda", dtype=torch.int32)])
    with pytest.raises(TypeError):
        per_b200.grad_norm([torch.eye(4, device="cuda").to_sparse()])
    with pytest.raises(RuntimeError, match="CUDA"):
        per_b200.grad_norm([normal(4), torch.ones(4)])


def test_beyond_32_bits():
    n = (1 << 32) + 12345
    big = torch.full((n,), 0.5, device="cuda", dtype=BF16)
    big[-1] = 3.0
    p = params([big[1:]])
    got = float(per_b200.clip_grad_norm_(p, 1.0))
    want = math.sqrt(0.25 * (n - 2) + 9.0)
    # a thread adds squares of 1/4, exactly while its sum is below 2^22; the threads' sums are
    # joined in float64, so only the root and its rounding are left
    assert abs(got - want) <= 4 * ref.U32 * want
    k = torch.tensor(0.5 / (want + 1e-6))
    assert abs(float(big[n // 2]) - float(k)) <= 0.01 * float(k)
    assert float(big[0]) == 0.5
    assert abs(float(big[-1]) / 3.0 - float(k) / 0.5) <= 0.01 * float(k) / 0.5
    assert float(big[1:].min()) > 0


def test_same_bits_every_time():
    grads, flat = bucket([3_000_000, 17, 99_999], F32)
    want = per_b200.grad_norm(grads)
    for _ in range(10):
        assert torch.equal(per_b200.grad_norm(grads), want)


def test_the_step_sees_the_change():
    """In-place scaling is visible to autograd's check for changed tensors."""
    g = normal(10)
    p = params([g])
    v = g._version
    per_b200.clip_grad_norm_(p, 1e-3)
    assert p[0].grad._version > v


def test_streams_and_captured_graphs():
    made = []
    for seed in (1, 2):
        grads, flat = bucket([200_000, 7, 3000], F32, seed=seed)
        start = flat.clone()
        p = params(grads)
        per_b200.clip_grad_norm_(p, 1.0)
        eager = flat.clone()
        flat.copy_(start)
        want = per_b200.grad_norm(grads)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norm = per_b200.clip_grad_norm_(p, 1.0)
        made.append((g, flat, start, eager, norm, want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for _, flat, start, _, _, _ in made:
            flat.copy_(start)
        for (g, *_), s in zip(made, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, flat, _, eager, norm, want in made:
            assert torch.equal(flat, eager) and torch.equal(norm, want)
    # eager calls on two streams at once
    for _, flat, start, _, _, _ in made:
        flat.copy_(start)
    torch.cuda.synchronize()
    got = []
    for (_, flat, *_), s in zip(made, streams):
        with torch.cuda.stream(s):
            torch.cuda._sleep(100_000)
            got.append(per_b200.grad_norm([flat]))
    torch.cuda.synchronize()
    for n, (_, flat, *_rest) in zip(got, made):
        check_norm(n, [flat])
