"""Softmax cross entropy of the vocabulary projection, with its gradient, without keeping the scores.

The language-model wrapper of the reference projects its last hidden states onto the vocabulary
(grm/utils/train.py:223) and hands the ``[tokens, vocabulary]`` scores to the cross entropy.  Here
projection and loss are one operator: the scores exist tile by tile on the tensor cores, forward and (a second
time) backward.  The kernels are ``grmx_linear_xent_fwd`` / ``grmx_linear_xent_bwd`` of the C ABI.
CUDA tensors only.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import cuda_ops

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def linear_cross_entropy(hidden: Tensor, weight: Tensor, targets: Tensor, bias: Optional[Tensor] = None, *,
                         ignore_index: int = -100, reduction: str = "mean") -> Tensor:
    """``cross_entropy(hidden @ weight.T + bias, targets)``, for ``hidden [..., D]`` and ``targets [...]``.

    Scores, their exponentials and all sums are float32, and so is the loss.  With bfloat16 inputs the gradient of the
    scores is rounded to bfloat16 before it is multiplied by ``weight`` and ``hidden`` and added up for ``bias``, and with
    "none" so are the hidden states times their token's upstream gradient, for the gradient of ``weight``.

    ``hidden`` and ``weight [V, D]`` share one type, bfloat16 or float32; ``bias [V]`` has that type or is
    float32; gradients come in the types of what they belong to.  ``reduction`` is "none" (``[...]``), "sum" or
    "mean" (over the tokens that count; NaN if none does).  Tokens with ``target == ignore_index`` have loss 0 and
    a zero gradient.  Any other target outside the vocabulary is ignored too and reported by
    ``cuda_ops.check_device_errors``.  A word whose bias is ``-inf`` is masked: it has probability 0,
    and a token without any other word a loss of NaN.  A bias of the type's lowest value is a finite one.
    What the hidden states of ignored tokens hold, NaN included, reaches neither loss nor gradients.
    Differentiable once, in reverse mode; inputs with a forward-mode tangent are refused.
    """
    cuda_ops._require_extension("linear_cross_entropy")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if hidden.device.type != "cuda":
        raise RuntimeError(f"linear_cross_entropy: tensors must be on a CUDA device, got {hidden.device}; this engine has no "
                           "CPU path.")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden [..., D] and weight [V, D] do not fit: {tuple(hidden.shape)}, {tuple(weight.shape)}")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets must have the shape {tuple(hidden.shape[:-1])}, got {tuple(targets.shape)}")
    loss = cuda_ops._Extension.module.linear_cross_entropy(hidden, weight, targets, bias, int(ignore_index), _REDUCTIONS[reduction])
    if cuda_ops._checking_each_call() and not torch.cuda.is_current_stream_capturing():
        cuda_ops.check_device_errors()
    return loss
