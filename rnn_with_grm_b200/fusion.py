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
from torch.autograd.function import once_differentiable

from . import cuda_ops


class FuseLayerNormFn(torch.autograd.Function):
    """``(online, update, gate?, scale?, weight?, bias?) -> (out, sum)``; ``sum`` is empty unless asked for."""

    @staticmethod
    def forward(ctx, online: Tensor, update: Tensor, gate: Optional[Tensor], scale: Optional[Tensor],
                weight: Optional[Tensor], bias: Optional[Tensor], eps: float, want_sum: bool):
        out, total, row_stats = torch.ops.grmx.fuse_norm_fwd(online, update, gate, scale, weight, bias, eps, want_sum, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(online, update, gate, scale, weight, bias, row_stats)
        ctx.want_sum = want_sum
        if not want_sum:
            ctx.mark_non_differentiable(total)
        return out, total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out: Optional[Tensor], grad_sum: Optional[Tensor]):
        grad_sum = grad_sum if ctx.want_sum else None
        if grad_out is None and grad_sum is None:
            return (None,) * 8
        online, update, gate, scale, weight, bias, row_stats = ctx.saved_tensors
        want = list(ctx.needs_input_grad[:6])
        # without gate and scale both row tensors have the same gradient: one is written
        shared = gate is None and scale is None and want[0] and want[1]
        asked = want if not shared else [True, False, *want[2:]]
        grads = torch.ops.grmx.fuse_norm_bwd(grad_out, grad_sum, online, update, gate, scale, weight, bias, row_stats, asked)
        grads = [grad if wanted else None for grad, wanted in zip(grads, asked)]
        if shared:
            grads[1] = grads[0]
        return (*grads, None, None)


def fuse_layer_norm(online: Tensor, update: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, *,
                    gate: Optional[Tensor] = None, scale: Optional[Tensor] = None, eps: float = 1e-5,
                    return_sum: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """``LayerNorm(s) * weight + bias`` over the last dimension, of ``s = online + scale * update``, or with ``gate``
    (the logits) of ``s = sigmoid(gate) * online + (1 - sigmoid(gate)) * scale * update``.

    Rows ``[..., H]`` (``online``, ``update``, ``gate``) share shape and type, bfloat16 or float32, with ``H <= 8192``;
    the vectors ``[H]`` (``scale``, ``weight``, ``bias``, all optional) share a type, that of the rows or float32.
    Arithmetic is float32, results have the type of the rows, gradients that of what they belong to.  With
    ``return_sum`` the result is ``(out, s)``: what the next block adds to, where the norm stands before it.
    """
    cuda_ops._require_extension("fuse_layer_norm")
    if online.device.type != "cuda":
        raise RuntimeError(f"fuse_layer_norm: tensors must be on a CUDA device, got {online.device}; this engine has no CPU path.")
    leaves = (online, update, gate, scale, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in leaves):
        out, total = FuseLayerNormFn.apply(online, update, gate, scale, weight, bias, float(eps), bool(return_sum))
    else:
        out, total, _ = torch.ops.grmx.fuse_norm_fwd(online, update, gate, scale, weight, bias, float(eps), bool(return_sum), False)
    if cuda_ops._checking_each_call() and not torch.cuda.is_current_stream_capturing():
        cuda_ops.check_device_errors()
    return (out, total) if return_sum else out
