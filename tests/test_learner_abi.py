"""The learner's C entry points and Python functions refuse bad calls before
anything reaches a GPU (CPU only)."""

import ctypes
import math
import os
import subprocess
import tempfile

import pytest
import torch

import per_b200
from per_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
L = _lib.lib
OK, INVALID, NULL, EMPTY, LARGE, MISALIGNED = 0, 1, 2, 3, 4, 5
P = 1 << 20  # stands for a device address: never read here


def norm(rows=4, dim=8, dtype=0, param_dtype=0, eps=1e-5):
    return _lib.Norm(rows, dim, dtype, param_dtype, eps)


C_PROBE = r"""
#include <stddef.h>
#include <stdio.h>
#include "per_b200.h"
#define F(T, m) printf(#T "." #m " %zu\n", offsetof(T, m))
int main(void) {
  printf("per_norm_t %zu\nper_tensor_t %zu\n", sizeof(per_norm_t), sizeof(per_tensor_t));
  F(per_norm_t, dim); F(per_norm_t, dtype); F(per_norm_t, param_dtype); F(per_norm_t, eps);
  F(per_tensor_t, count); F(per_tensor_t, dtype);
  return 0;
}
"""


def test_structs_match_the_header():
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        open(src, "w").write(C_PROBE)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        lines = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n")
    py = {"per_norm_t": _lib.Norm, "per_tensor_t": _lib.Tensor}
    for k, v in (l.rsplit(" ", 1) for l in lines if l):
        if "." in k:
            t, m = k.split(".")
            assert getattr(py[t], m).offset == int(v), k
        else:
            assert ctypes.sizeof(py[k]) == int(v), k


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), INVALID), (dict(dim=0), INVALID), (dict(dtype=3), INVALID),
    (dict(dtype=-1), INVALID), (dict(dtype=0, param_dtype=1), INVALID),
    (dict(dtype=1, param_dtype=2), INVALID), (dict(dim=1 << 31), LARGE),
    (dict(rows=(1 << 40) + 1), LARGE), (dict(eps=-1e-5), INVALID), (dict(eps=math.nan), INVALID),
])
def test_layer_norm_refuses_bad_descriptors(kw, code):
    d = norm(**kw)
    assert L.per_layer_norm(ctypes.byref(d), P, 8, None, None, 2 * P, 8, None, None) == code


def test_layer_norm_refuses_bad_pointers_and_strides():
    d = norm()
    f = lambda *a: L.per_layer_norm(ctypes.byref(d), *a, None)  # noqa: E731
    assert L.per_layer_norm(None, P, 8, None, None, 2 * P, 8, None, None) == NULL
    assert f(None, 8, None, None, 2 * P, 8, None) == NULL
    assert f(P, 8, None, None, None, 8, None) == NULL
    assert f(P, 7, None, None, 2 * P, 8, None) == INVALID    # rows would overlap
    assert f(P, 8, None, None, 2 * P, 7, None) == INVALID
    assert f(P + 2, 8, None, None, 2 * P, 8, None) == MISALIGNED
    assert f(P, 8, None, 3 * P + 1, 2 * P, 8, None) == MISALIGNED
    assert f(P, 8, None, None, 2 * P, 8, 3 * P + 8) == MISALIGNED
    assert f(P, 8, None, None, P, 8, None) == INVALID        # in place
    assert f(P, 8, None, None, P + 3 * 32, 8, None) == INVALID
    assert f(P, 16, None, None, P + 28, 16, None) == INVALID  # columns 7..15 over 0..8
    assert f(P, 16, None, None, P - 28, 16, None) == INVALID
    empty = norm(rows=0)
    assert L.per_layer_norm(ctypes.byref(empty), None, 8, None, None, None, 8, None, None) == OK


def test_layer_norm_backward_refuses_bad_calls():
    d = norm()
    need = L.per_layer_norm_backward_workspace(ctypes.byref(d))
    assert need >= 0
    big = max(need, 1 << 20)

    def f(dy=P, ds=8, x=2 * P, xs=8, w=None, stats=3 * P, dx=5 * P, dxs=8, dw=6 * P,
          db=7 * P, ws=8 * P, nbytes=big, desc=d):
        return L.per_layer_norm_backward(ctypes.byref(desc), dy, ds, x, xs, w, stats, dx, dxs,
                                         dw, db, ws, nbytes, None)

    assert f(dx=None, dw=None, db=None) == OK  # nothing wanted
    for name in ("dy", "x", "stats"):
        assert f(**{name: None}) == NULL, name
    if need:
        assert f(ws=None) == NULL
        assert f(nbytes=need - 1) == INVALID
    assert f(ds=7) == INVALID
    assert f(ds=-8) == INVALID
    assert f(xs=7) == INVALID
    assert f(xs=0) == INVALID
    assert f(dxs=7) == INVALID
    assert f(dx=P) == INVALID      # over dy
    assert f(dx=2 * P) == INVALID  # over x
    assert f(ws=8 * P + 4) == MISALIGNED
    assert f(dw=6 * P + 2) == MISALIGNED
    assert f(stats=3 * P + 8) == MISALIGNED
    assert f(desc=norm(dtype=5)) == INVALID
    assert L.per_layer_norm_backward_workspace(ctypes.byref(norm(dim=0))) == -1
    assert L.per_layer_norm_backward_workspace(None) == -1


def tensors(*entries):
    return (_lib.Tensor * len(entries))(*[_lib.Tensor(*e, 0) for e in entries])


def test_gradient_norm_refuses_bad_calls():
    need = L.per_grad_norm_workspace(1)
    assert need > 0 and L.per_grad_norm_workspace(-1) == -1
    good = tensors((P, 10, 0))

    def f(t=good, n=1, kind=2, out=2 * P, ws=3 * P, nbytes=need):
        return L.per_grad_norm(t, n, kind, out, ws, nbytes, None)

    assert f(n=-1) == INVALID
    assert f(t=None) == NULL
    assert f(n=(1 << 24) + 1) == LARGE
    assert f(kind=0) == INVALID
    assert f(kind=4) == INVALID
    assert f(out=None) == NULL
    assert f(ws=None) == NULL
    assert f(ws=3 * P + 8) == MISALIGNED
    assert f(out=2 * P + 2) == MISALIGNED
    assert f(nbytes=need - 1) == INVALID
    assert f(t=tensors((None, 10, 0))) == NULL
    assert f(t=tensors((P, -1, 0))) == INVALID
    assert f(t=tensors((P, 10, 7))) == INVALID
    assert f(t=tensors((P + 2, 10, 0))) == MISALIGNED
    assert f(t=tensors((P, (1 << 44) + 1, 0))) == LARGE
    for max_norm in (-1.0, math.nan):
        assert L.per_clip_grad_norm(good, 1, 2, max_norm, 2 * P, 3 * P, need, None) == INVALID
        assert L.per_scale_grads(good, 1, max_norm, 2 * P, None) == INVALID
    assert L.per_scale_grads(good, 1, 1.0, None, None) == NULL
    assert L.per_scale_grads(None, 1, 1.0, 2 * P, None) == NULL


def test_no_cpu_fallback():
    x = torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        per_b200.layer_norm(x, (8,))
    with pytest.raises(RuntimeError, match="CUDA"):
        per_b200.LayerNorm(8)(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        per_b200.grad_norm([x])
    p = torch.nn.Parameter(x.clone())
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="CUDA"):
        per_b200.clip_grad_norm_([p], 1.0)
    assert torch.equal(p.grad, torch.ones_like(p))


def test_clipping_refuses_bad_arguments_and_passes_empty_lists():
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            per_b200.clip_grad_norm_([], bad)
    for bad in (0, 3, -math.inf, math.nan, "fro"):
        with pytest.raises(ValueError, match="norm_type"):
            per_b200.clip_grad_norm_([], 1.0, norm_type=bad)
    assert float(per_b200.clip_grad_norm_([], 1.0)) == 0.0
    assert float(per_b200.grad_norm([])) == 0.0
    without = torch.nn.Parameter(torch.ones(3))  # no gradient: skipped, as torch does
    assert float(per_b200.clip_grad_norm_(iter([without]), 1.0)) == 0.0
    assert float(per_b200.clip_grad_norm_(without, 1.0, error_if_nonfinite=True)) == 0.0


def test_module_has_the_parameters_of_torch():
    for kw in ({}, {"bias": False}, {"elementwise_affine": False}, {"eps": 1e-3}):
        ours, theirs = per_b200.LayerNorm((3, 5), **kw), torch.nn.LayerNorm((3, 5), **kw)
        assert {k: tuple(v.shape) for k, v in ours.state_dict().items()} == \
            {k: tuple(v.shape) for k, v in theirs.state_dict().items()}
        ours.load_state_dict(theirs.state_dict())
        assert ours.eps == theirs.eps and ours.normalized_shape == theirs.normalized_shape
        assert repr(ours) == repr(theirs)
    assert per_b200.LayerNorm(7, dtype=torch.bfloat16).weight.dtype == torch.bfloat16
