"""The learner's operators next to the replay buffer, as a training step calls them: layer norm (forward, and
forward with its gradients) and the global gradient norm (alone, and with clipping).

`run` computes them in their plain form, or, with `own` set, through the public calls of per_b200.
"""

import os
import sys

import torch

own = False

EPS = 1e-5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


_library = None


def library():
    """per_b200 of this repository (the folder triton-per_b200 holds the package)."""
    global _library
    if _library is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-per_b200"))
        import per_b200

        _library = per_b200
    return _library


# ------------------------------------------------------------------- cases
def norm_case(op, rows, dim, dtype="float32", params="float32", affine="both", stride=0, offset=0):
    """Layer norm of `rows` rows of `dim` values; stride > 0: the rows are columns offset..offset+dim of
    packed rows of `stride` values, as the field views of a sampled batch are."""
    return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "params": params, "affine": affine,
            "stride": stride, "offset": offset}


def grad_case(op, copies, inputs, width, depth, outputs, dtype="float32", norms=False):
    """The gradients of `copies` networks of `depth` hidden layers of `width`, each layer a matrix and a bias,
    with `norms` also the two float32 vectors of a layer norm behind every hidden layer."""
    return {"op": op, "copies": copies, "inputs": inputs, "width": width, "depth": depth, "outputs": outputs,
            "dtype": dtype, "norms": norms}


def listed():
    return [
        # the actor choosing the action for one observation: one row, latency alone
        {"name": "forward 1x256", **norm_case("forward", 1, 256)},
        # next_obs of a sampled batch of 65,536 packed 74-value rows, normalised where it lies: rows that start
        # on any 4-byte boundary
        {"name": "forward views 65536x32", **norm_case("forward", 65536, 32, stride=74, offset=41)},
        # evaluation over wide 16-bit rows: memory bound
        {"name": "forward bf16 65536x4096", **norm_case("forward", 65536, 4096, "bfloat16")},
        # a hidden layer of a critic at the replay benchmark's batch: one training step, latency again
        {"name": "train 256x256", **norm_case("train", 256, 256)},
        # the same layer at the largest batch of the sampling sweep
        {"name": "train 65536x256", **norm_case("train", 65536, 256)},
        # odd sizes, rows that start on 2-byte boundaries
        {"name": "train fp16 8191x1001", **norm_case("train", 8191, 1001, "float16")},
        # few long rows: the row itself has to be spread
        {"name": "train 48x20000", **norm_case("train", 48, 20000)},
        # a wide network trained in bfloat16, its parameters too: memory bound
        {"name": "train bf16 16384x8192", **norm_case("train", 16384, 8192, "bfloat16", "bfloat16")},
        # the synthetic learner's two critics at its own sizes: a few small tensors, latency alone
        {"name": "clip 2 critics", **grad_case("clip", 2, 40, 256, 2, 1)},
        # ten critics of a high update-to-data learner, with layer norms: 100 tensors
        {"name": "clip 10 critics", **grad_case("clip", 10, 40, 512, 2, 1, norms=True)},
        # a wide bfloat16 network with float32 layer norms, its gradients far beyond the L2 cache
        {"name": "clip bf16 8192 wide", **grad_case("clip", 1, 4096, 8192, 8, 1000, "bfloat16", True)},
        # the norm alone, logged every step
        {"name": "norm 2048 wide", **grad_case("norm", 1, 500, 2048, 10, 17)},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(["forward", "train", "train", "clip", "clip", "norm"])
    dtype = rng.choice(list(DTYPES))
    if op in ("forward", "train"):
        dim = spread(8, 30000)
        rows = spread(1, min(300000, 80_000_000 // dim))
        params = rng.choice(["float32", dtype])
        affine = rng.choice(["both", "both", "weight", "none"])
        packed = op == "forward" and rng.random() < 0.4
        stride = dim + rng.randrange(1, 200) if packed else 0
        offset = rng.randrange(stride - dim + 1) if packed else 0
        return norm_case(op, rows, dim, dtype, params, affine, stride, offset)
    width = spread(16, 6000)
    depth = rng.randrange(1, 9)
    inputs, outputs = spread(1, 4000), spread(1, 1000)
    copies = min(spread(1, 30), max(1, 200_000_000 // (width * (width * (depth - 1) + inputs + outputs))))
    return grad_case(op, copies, inputs, width, depth, outputs, dtype, rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def shapes(case):
    """(shape, is a layer norm's) of every gradient of the case, in the order of a network's parameters."""
    got = []
    for _ in range(case["copies"]):
        last = case["inputs"]
        for _ in range(case["depth"]):
            got += [((case["width"], last), False), ((case["width"],), False)]
            got += [((case["width"],), True)] * (2 if case["norms"] else 0)
            last = case["width"]
        got += [((case["outputs"], last), False), ((case["outputs"],), False)]
    return got


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] in ("forward", "train"):
        rows, dim = case["rows"], case["dim"]
        dtype, params = DTYPES[case["dtype"]], DTYPES[case["params"]]
        width = case["stride"] or dim
        # what a linear layer gives: each row with a mean and a spread of its own
        x = (normal(rows, width) * (0.5 + normal(rows, 1).abs()) + normal(rows, 1)).to(dtype)
        if case["stride"]:
            x = x[:, case["offset"]:case["offset"] + dim]
        state = {"op": case["op"], "x": x, "dim": dim, "w": None, "b": None}
        if case["affine"] != "none":
            state["w"] = (1 + 0.2 * normal(dim)).to(params)
        if case["affine"] == "both":
            state["b"] = (0.2 * normal(dim)).to(params)
        if case["op"] == "train":
            state["dy"] = normal(rows, dim).to(dtype)
            state["leaves"] = [state[k].requires_grad_() for k in ("x", "w", "b") if state[k] is not None]
        return state

    # the gradients lie one behind the other in a flat buffer for each type, as the buckets of data-parallel
    # training keep them: a tensor starts wherever the one before it ended
    kinds = [(torch.float32 if is_norm else DTYPES[case["dtype"]], shape) for shape, is_norm in shapes(case)]
    sizes = [(t, int(torch.Size(s).numel())) for t, s in kinds]
    flats = {}
    for t in dict.fromkeys(t for t, _ in kinds):
        flats[t] = torch.empty(sum(n for k, n in sizes if k is t), dtype=t, device="cuda")
    total = sum(n for _, n in sizes)
    at, params = dict.fromkeys(flats, 0), []
    for i, ((t, shape), (_, n)) in enumerate(zip(kinds, sizes)):
        grad = flats[t][at[t]:at[t] + n]
        at[t] += n
        # the gradients' scale differs from layer to layer; their norm is some 10, the threshold 1
        torch.randn(n, generator=g, device="cuda", out=grad) if t is torch.float32 else grad.copy_(normal(n))
        grad.mul_(10 / total ** 0.5 * 2.0 ** (i % 5 - 2))
        p = torch.nn.Parameter(torch.empty(shape, dtype=t, device="cuda"))
        p.grad = grad.view(shape)
        params.append(p)
    return {"op": case["op"], "flats": list(flats.values()), "params": params,
            "grads": [p.grad for p in params], "max_norm": 1.0}


# --------------------------------------------------------------------- run
def run(state):
    if state["op"] == "forward":
        if own:
            with torch.no_grad():
                return library().layer_norm(state["x"], (state["dim"],), state["w"], state["b"], EPS)
        with torch.no_grad():
            return plain_forward(state)[0].to(state["x"].dtype)
    if state["op"] == "train":
        if own:
            y = library().layer_norm(state["x"], (state["dim"],), state["w"], state["b"], EPS)
            return [y, *torch.autograd.grad(y, state["leaves"], state["dy"])]
        with torch.no_grad():
            return plain_train(state)
    if state["op"] == "norm":
        if own:
            return library().grad_norm(state["grads"])
        return plain_norm(state["flats"])
    # a threshold that falls a little with every step: each pass clips, as it would a new step's gradients,
    # though the ones in the buffers are those that the last pass has clipped
    max_norm = state["max_norm"]
    state["max_norm"] = max_norm * (1 - 2.0 ** -16)
    if own:
        norm = library().clip_grad_norm_(state["params"], max_norm)
    else:
        norm = plain_clip(state["flats"], max_norm)
    return [norm, *state["flats"]]


def plain_forward(state):
    x = state["x"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = (centred.square().mean(1, keepdim=True) + EPS).rsqrt()
    normed = centred * rstd
    y = normed
    if state["w"] is not None:
        y = y * state["w"].float()
    if state["b"] is not None:
        y = y + state["b"].float()
    return y, normed, rstd


def plain_train(state):
    y, normed, rstd = plain_forward(state)
    dy = state["dy"].float()
    d = dy if state["w"] is None else dy * state["w"].float()
    dx = rstd * (d - d.mean(1, keepdim=True) - normed * (d * normed).mean(1, keepdim=True))
    out = [y.to(state["x"].dtype), dx.to(state["x"].dtype)]
    if state["w"] is not None:
        out.append((dy * normed).sum(0).to(state["w"].dtype))
    if state["b"] is not None:
        out.append(dy.sum(0).to(state["b"].dtype))
    return out


def plain_norm(flats):
    return torch.stack([f.float().square().sum() for f in flats]).sum().sqrt()


def plain_clip(flats, max_norm):
    norm = plain_norm(flats)
    scale = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    [f.copy_(f.float() * scale) for f in flats]
    return norm


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] in ("forward", "train"):
        rows, dim = case["rows"], case["dim"]
        values = rows * dim * DTYPES[case["dtype"]].itemsize
        vectors = dim * DTYPES[case["params"]].itemsize * {"both": 2, "weight": 1, "none": 0}[case["affine"]]
        if case["op"] == "forward":  # x read, y written; sums, squares, and the scaled and shifted result
            return {"bytes": 2 * values + vectors, "flops": 7 * rows * dim}
        # x and dy read, y and dx written, the vectors read and their gradients written
        return {"bytes": 4 * values + 2 * vectors, "flops": 20 * rows * dim}
    count = size = 0
    for shape, is_norm in shapes(case):
        n = int(torch.Size(shape).numel())
        count += n
        size += n * (4 if is_norm else DTYPES[case["dtype"]].itemsize)
    if case["op"] == "norm":
        return {"bytes": size + 4, "flops": 2 * count}
    return {"bytes": 2 * size + 4, "flops": 3 * count}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("forward", "train"):
            x = state["x"].double()
            n = case["dim"]
            var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
            std = torch.sqrt(var + EPS)
            x = (x - mean).div_(std)
            y = x * state["w"].double() if state["w"] is not None else x.clone()
            if state["b"] is not None:
                y += state["b"].double()
            if case["op"] == "forward":
                return y
            dy = state["dy"].double()
            dw = torch.einsum("rc,rc->c", dy, x) if state["w"] is not None else None
            db = torch.einsum("rc->c", dy) if state["b"] is not None else None
            if state["w"] is not None:
                dy = dy * state["w"].double()
            # the projection of the upstream gradient off the directions 1 and x that the norm removes
            along = torch.einsum("rc,rc->r", dy, x).unsqueeze(1) / n
            dx = (dy - dy.sum(1, keepdim=True) / n - along * x) / std
            return [v for v in (y, dx, dw, db) if v is not None]
        grads = [g.double() for g in state["grads"]]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g) for g in grads]))
        if case["op"] == "norm":
            return norm
        scale = min(1.0, state["max_norm"] / (float(norm) + 1e-6))
        return [norm, *[f.double() * scale for f in state["flats"]]]
