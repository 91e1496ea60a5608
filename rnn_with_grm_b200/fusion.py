"""The mixing rule after a block and its LayerNorm as one operator, with gradients.

``RetrievedStateFusion`` of the reference adds, or gates, the retrieved contribution onto the online state and
normalises (grm/core/aggregator.py:116-145); the stack does the same between its layers
(grm/core/multilayer_grm.py:93,96).  ``torch.ops.grmx.add_layer_norm`` and ``retrieve_fuse`` are the inference forms of
the plain residual rule; this is the operator to train with: residual rule with an optional scale per feature, or
gate rule, forward and backward in one pass over the rows each (``grmx_fuse_norm_fwd`` / ``grmx_fuse_norm_bwd`` of
the C ABI).  CUDA tensors only.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import cuda_ops


def fuse_layer_norm(online: Tensor, update: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, *,
                    gate: Optional[Tensor] = None, scale: Optional[Tensor] = None, eps: float = 1e-5,
                    return_sum: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """``LayerNorm(s) * weight + bias`` over the last dimension, of ``s = online + scale * update``, or with ``gate``
    (the logits) of ``s = sigmoid(gate) * online + (1 - sigmoid(gate)) * scale * update``.

    Rows ``[..., H]`` (``online``, ``update``, ``gate``) share shape and type, bfloat16 or float32, with ``H <= 8192``;
    the vectors ``[H]`` (``scale``, ``weight``, ``bias``, all optional) share a type, that of the rows or float32.
    Arithmetic is float32, results have the type of the rows, gradients that of what they belong to.  With
    ``return_sum`` the result is ``(out, s)``: what the next block adds to, where the norm stands before it.
    Differentiable once, in reverse mode; inputs with a forward-mode tangent are refused.
    """
    cuda_ops._require_extension("fuse_layer_norm")
    if online.device.type != "cuda":
        raise RuntimeError(f"fuse_layer_norm: tensors must be on a CUDA device, got {online.device}; this engine has no CPU path.")
    out = cuda_ops._Extension.module.fuse_layer_norm(online, update, weight, bias, gate, scale, float(eps), bool(return_sum))
    if cuda_ops._checking_each_call() and not torch.cuda.is_current_stream_capturing():
        cuda_ops.check_device_errors()
    return (out[0], out[1]) if return_sum else out[0]
