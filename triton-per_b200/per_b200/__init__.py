"""per_b200 - a B200-native prioritized experience replay engine.

Drop-in for triton-per's `PERBuffer` (triton backend): PyTorch host code over
hand-written sm_100a CUDA kernels behind a C ABI (include/per_b200.h). The
learner's layer norm and gradient clipping (per_b200.learner) run on kernels
of the same library.
"""

from .buffer import BLOCK_P, PERBuffer, SampleOut
from .learner import LayerNorm, clip_grad_norm_, clip_grads_with_norm_, grad_norm, layer_norm

__all__ = ["BLOCK_P", "PERBuffer", "SampleOut", "LayerNorm", "clip_grad_norm_",
           "clip_grads_with_norm_", "grad_norm", "layer_norm"]
