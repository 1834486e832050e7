"""Operators of the learner that trains on sampled batches, on sm_100a kernels.

Between `sample` and `update_priorities` a learner with a high update-to-data
ratio runs layer norms in its critics and clips its gradients by their global
norm. These are drop-ins for torch.nn.functional.layer_norm, torch.nn.LayerNorm
and torch.nn.utils.clip_grad_norm_ / get_total_norm / clip_grads_with_norm_ on
CUDA tensors of float32, bfloat16 or float16. Every call enqueues its work on
the current stream of the tensors' device, synchronises nothing (except
error_if_nonfinite=True) and can be captured into a CUDA graph. Tensors made on
another stream are the caller's to order, as for torch's own operators
(wait_stream, record_stream). As with the buffers there is no CPU path.

The calls are no torch operators, so nothing that records or transforms
operators sees them: torch.jit.trace, ONNX export, make_fx, torch.export, fake
tensors, vmap and the torch.func transforms are refused, and torch.compile
breaks its graph at each call (fullgraph=True raises).
"""

from __future__ import annotations

import math
import numbers

import torch

from . import _lib  # noqa: F401  (the library the binding calls)

try:
    from . import _per_torch
except ImportError:
    _per_torch = None


def _binding():
    if _per_torch is None:
        raise RuntimeError("per_b200: the torch binding (_per_torch) is missing; build it with "
                           "`python per_b200/build.py`. There is no fallback.")
    return _per_torch


# ------------------------------------------------------------- layer norm
def layer_norm(input: torch.Tensor, normalized_shape, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the trailing dimensions `normalized_shape`, as
    torch.nn.functional.layer_norm; differentiable once, in reverse mode.

    The result has the input's type and is contiguous; weight and bias are
    float32 or of the input's type (under autocast the types stay as they
    are). The rows may be strided, for instance the field views that a
    buffer's sample() returns, at any alignment: they are read where they
    lie. Inputs whose trailing dimensions are not contiguous are copied first.

    In a captured training step, drop the outputs of eager steps made on the
    default stream (`del loss`) before the capture; a leaf that is still part
    of one is refused."""
    if isinstance(normalized_shape, numbers.Integral):
        normalized_shape = (normalized_shape,)
    return _binding().layer_norm(input, normalized_shape, weight, bias, eps)


class LayerNorm(torch.nn.Module):
    """torch.nn.LayerNorm (same arguments, parameters and state_dict) on
    layer_norm()."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, device=None, dtype=None):
        super().__init__()
        if isinstance(normalized_shape, numbers.Integral):
            normalized_shape = (normalized_shape,)
        self.normalized_shape = tuple(normalized_shape)
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        shape = self.normalized_shape
        if elementwise_affine:
            self.weight = torch.nn.Parameter(torch.empty(shape, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        if elementwise_affine and bias:
            self.bias = torch.nn.Parameter(torch.empty(shape, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        if self.weight is not None:
            torch.nn.init.ones_(self.weight)
        if self.bias is not None:
            torch.nn.init.zeros_(self.bias)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return (f"{self.normalized_shape}, eps={self.eps}, "
                f"elementwise_affine={self.elementwise_affine}")


# ----------------------------------------------------------- gradient norm
_KINDS = {1.0: 1, 2.0: 2, math.inf: 3}  # norm_type -> PER_NORM_*


def _kind(norm_type) -> int:
    kind = _KINDS.get(norm_type)
    if kind is None:
        try:
            kind = _KINDS[float(norm_type)]
        except (KeyError, ValueError, TypeError):
            raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type!r}") from None
    return kind


def _max_norm(max_norm) -> float:
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm if type(max_norm) is float else float(max_norm)


def _listed(tensors) -> list:
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    return tensors if type(tensors) is list else list(tensors)


def grad_norm(tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all values of `tensors` (a tensor or an iterable of them,
    of mixed types, on one device, each dense in its memory) as one vector: a
    float32 scalar on their device, not differentiable. norm_type is 1, 2 or
    inf."""
    kind = _kind(norm_type)
    norm = _binding().grad_norm(_listed(tensors), False, kind)
    return torch.tensor(0.0) if norm is None else norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """Scale the gradients of `parameters` in place so that their global norm
    is at most max_norm; returns the norm before that (float32 scalar on their
    device), as torch.nn.utils.clip_grad_norm_.

    Every value is multiplied by min(1, max_norm / (norm + 1e-6)) in float32
    and rounded once; where that factor is 1 nothing is written. Parameters
    without a gradient are skipped. A norm of NaN makes every gradient NaN, an
    infinite one makes the finite values 0; error_if_nonfinite=True raises
    instead, before anything is changed (it waits for the GPU). Gradients have
    to be dense and must not share memory: a parameter listed twice is
    refused. foreach is accepted for compatibility; there is one path."""
    kind, max_norm = _kind(norm_type), _max_norm(max_norm)
    parameters = _listed(parameters)
    if error_if_nonfinite:
        norm = _binding().grad_norm(parameters, True, kind)
        if norm is not None:
            if not math.isfinite(norm.item()):
                raise RuntimeError(f"the norm of order {norm_type} of the gradients is not finite, "
                                   "so they cannot be clipped (error_if_nonfinite=False clips anyway)")
            _per_torch.clip_grads_with_norm(parameters, max_norm, norm)
    else:
        norm = _binding().clip_grad_norm(parameters, kind, max_norm)
    return torch.tensor(0.0) if norm is None else norm


def clip_grads_with_norm_(parameters, max_norm: float, total_norm: torch.Tensor,
                          foreach: bool | None = None) -> None:
    """clip_grad_norm_() with a norm that is known already, for instance joined
    over the ranks of a sharded job: `total_norm` is one float32 value on the
    gradients' device."""
    _binding().clip_grads_with_norm(_listed(parameters), _max_norm(max_norm), total_norm)
