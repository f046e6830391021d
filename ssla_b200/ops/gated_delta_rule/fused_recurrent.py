"""Token-by-token gated delta rule for serving: one or a few tokens of every sequence.

Same arguments and results as ``chunk_gated_delta_rule``; carry ``final_state`` into the next call
as ``initial_state``.  The forward is ``ssla_recurrent_gated_delta_rule_fwd`` (the state stays in
registers over a sequence's tokens and crosses HBM once each way); gradients are those of the same
function and come from the chunked kernels, which work on chunks of 64 tokens however few a sequence
has: the backward's buffers hold three padded states (K to 64 or 128, V to a multiple of 64, fp32),
one [K, K] map and a 64 x 64 tile per sequence and value head.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from ... import _lib
from ..utils.guard import refuse_tangents
from .chunk import chunk_bwd, chunk_fwd, needs_grad, norm_inputs, tensor_args

_NAME = "fused_recurrent_gated_delta_rule"


def recurrent_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state):
    dev = q.device
    o = torch.empty_like(v)
    ht = None
    if output_final_state:
        ht = torch.empty_like(h0) if h0 is not None else torch.empty(
            (len(cu) - 1, v.shape[1], q.shape[2], v.shape[2]), device=dev, dtype=torch.float32)
    with _lib.on_device(dev):
        rc = _lib.load().ssla_recurrent_gated_delta_rule_fwd(
            *tensor_args(q, k, v, g, beta, cu, scale), _lib.ptr(h0), o.data_ptr(), _lib.ptr(ht), _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, _NAME)
    return o, ht


class FusedRecurrentGatedDeltaRuleFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, cu_seqlens, scale, initial_state, output_final_state):
        q, k, v, g, beta, cu, h0 = norm_inputs(q, k, v, g, beta, cu_seqlens, initial_state, _NAME)
        o, ht = recurrent_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state)
        ctx.save_for_backward(q, k, v, g, beta, cu, h0)
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        return o, ht

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dht):
        if do is None and dht is None:
            return (None,) * 9
        q, k, v, g, beta, cu, h0 = ctx.saved_tensors
        has_h0, has_ht = h0 is not None, dht is not None  # the states' accuracy goes by both
        states = chunk_fwd(q, k, v, g, beta, cu, ctx.scale, h0, has_ht, output=False)[2]
        dq, dk, dv, dg, dbeta, dh0 = chunk_bwd(q, k, v, g, beta, cu, ctx.scale, has_h0, has_ht, states, do, dht,
                                               ctx.needs_input_grad[7])
        return dq, dk, dv, dg, dbeta, None, None, dh0, None


@torch.compiler.disable
def fused_recurrent_gated_delta_rule(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    beta: torch.Tensor,
    cu_seqlens: torch.LongTensor,
    scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    r"""Recurrent gated delta rule; arguments and returns as ``chunk_gated_delta_rule``.  A gradient of
    many short sequences takes many times the memory of the call itself (see above)."""
    refuse_tangents(_NAME, q, k, v, g, beta, initial_state)
    if needs_grad(q, k, v, g, beta, initial_state):
        return FusedRecurrentGatedDeltaRuleFunction.apply(q, k, v, g, beta, cu_seqlens, scale, initial_state,
                                                          output_final_state)
    q, k, v, g, beta, cu, h0 = norm_inputs(q, k, v, g, beta, cu_seqlens, initial_state, _NAME)
    return recurrent_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state)
