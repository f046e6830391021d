"""Chunked gated delta rule over packed variable-length sequences.

Next to ``chunk_gla`` (whose layout, argument order and conventions it keeps) for states that are
corrected instead of only added to: before a token writes its value, what the state already
returns for its key is subtracted.  Per value head, with state S [K, V]::

    S <- exp(g_t) S;   u_t = beta_t (v_t - S^T k_t);   S <- S + k_t u_t^T;   o_t = scale S^T q_t

fp32 tokens are computed at fp32 accuracy.  16-bit tokens: products of 16-bit operands, which only the
outputs' own rounding shows; final states and initial states' gradients are fp32-accurate, fp32 ``dg`` and
``dbeta`` are off by about 1e-5.  Per 64 tokens (or shorter sequence) and value head a call holds two K x V
matrices and a K x K one, padded to K = 64 or 128 and V a multiple of 64, in fp32; training keeps one of each
for the backward.

``beta k^T k`` should stay below 2 (keys of unit length, beta in [0, 1] or [0, 2)): beyond that the
recurrence itself grows without bound.  The kernels are ``ssla_chunk_gated_delta_rule_fwd`` /
``_bwd`` of the C ABI; the project ssla follows has no delta rule.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from ... import _lib
from ..utils.guard import prepare_cu_seqlens, refuse_tangents


def _refuse(q, k, v, g, beta, initial_state, cu, what):
    """The exception for arguments that do not belong together; None where they do."""
    if q.dim() != 3 or k.shape != q.shape or v.dim() != 3 or v.shape[0] != q.shape[0]:
        return ValueError(
            f"{what} expects q, k [T, H, K] and v [T, HV, V]; got q {tuple(q.shape)}, k {tuple(k.shape)}, "
            f"v {tuple(v.shape)}"
        )
    T, H, K = q.shape
    _, HV, V = v.shape
    if H == 0 or HV == 0 or HV % H:
        return ValueError(f"{what}: the {HV} value heads must be a positive multiple of the {H} key heads")
    if g.shape != (T, HV) or beta.shape != (T, HV):
        return ValueError(f"{what} expects g, beta [T, HV] = [{T}, {HV}]; got {tuple(g.shape)}, {tuple(beta.shape)}")
    if not (1 <= K <= 128 and 1 <= V <= 256):
        return ValueError(f"{what}: K={K}, V={V} not supported (1 <= K <= 128, 1 <= V <= 256)")
    for x in (q, k, v, g, beta, initial_state):
        if x is not None and not x.is_cuda:
            return RuntimeError(f"{what}: tensors must be on a CUDA device (no CPU path)")
    if q.dtype not in _lib._DT:
        return TypeError(f"unsupported dtype {q.dtype}; expected float32, bfloat16 or float16")
    for x in (k, v, g, beta, initial_state):
        if x is not None and x.device != q.device:
            return RuntimeError(f"{what}: all tensors must be on one device, got {q.device} and {x.device}")
    if initial_state is not None and cu is not None:
        N = cu.numel() - 1
        if initial_state.dim() == 0 or initial_state.shape[0] != N:
            return ValueError(
                f"The number of initial states is expected to be equal to the number of input sequences, "
                f"i.e., {N} rather than {initial_state.shape[0] if initial_state.dim() else 0}."
            )
        if initial_state.shape != (N, HV, K, V):
            return ValueError(f"{what}: initial_state must be [N, HV, K, V] = {(N, HV, K, V)}; got "
                              f"{tuple(initial_state.shape)}")
    return None


def norm_inputs(q, k, v, g, beta, cu_seqlens, initial_state, what):
    """Checked, contiguous inputs of one dtype (q's) on q's device; gates in their own dtype.  A
    decoding step is bound by this code, so the usual case passes one chain of comparisons."""
    dev, dt, code, cu = q.device, q.dtype, _lib._DT, cu_seqlens
    qs, vs = q.shape, v.shape
    fits = (
        len(qs) == 3 and len(vs) == 3 and k.shape == qs and vs[0] == qs[0] and 0 < qs[2] <= 128 and 0 < vs[2] <= 256
        and qs[1] > 0 and vs[1] > 0 and vs[1] % qs[1] == 0 and g.shape == vs[:2] and beta.shape == vs[:2]
        and q.is_cuda and k.device == dev and v.device == dev and g.device == dev and beta.device == dev and dt in code
    )
    if not fits:
        raise _refuse(q, k, v, g, beta, initial_state, None, what)
    if cu is None or cu.dim() != 1 or cu.device != dev or cu.dtype != torch.int64 or not cu.is_contiguous() or not len(cu):
        cu = prepare_cu_seqlens(cu_seqlens, dev)
    if initial_state is not None:
        if initial_state.device != dev or initial_state.shape != (len(cu) - 1, vs[1], qs[2], vs[2]):
            raise _refuse(q, k, v, g, beta, initial_state, cu, what)
        initial_state = initial_state.float().contiguous()
    if k.dtype != dt:
        k = k.to(dt)
    if v.dtype != dt:
        v = v.to(dt)
    if g.dtype not in code:
        g = g.float()
    if beta.dtype not in code:
        beta = beta.float()
    return q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous(), beta.contiguous(), cu, initial_state


def tensor_args(q, k, v, g, beta, cu, scale):
    """The arguments that every entry point of the family starts with."""
    code = _lib._DT
    T, H, K = q.shape
    _, HV, V = v.shape
    scale = K ** -0.5 if scale is None else float(scale)
    return (q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), code[q.dtype], code[g.dtype],
            code[beta.dtype], cu.data_ptr(), cu.shape[0] - 1, T, H, HV, K, V, scale)


def chunk_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state, output=True):
    """(o, final state or None, states): ``states`` is what the backward needs of the chunks; without
    ``output`` o is None and not computed."""
    T, H, K = q.shape
    HV, V = v.shape[1:]
    N = cu.numel() - 1
    L = _lib.load()
    dev = q.device
    o = torch.empty_like(v) if output else None
    ht = torch.empty((N, HV, K, V), device=dev, dtype=torch.float32) if output_final_state else None
    nb = L.ssla_gated_delta_rule_states_bytes(_lib.dtype_code(q), N, T, H, HV, K, V, h0 is not None,
                                              output_final_state)
    states = torch.empty(nb, device=dev, dtype=torch.uint8)
    wb = L.ssla_gated_delta_rule_workspace_bytes(N, T, H, HV, K, V, 0)
    ws = torch.empty(wb, device=dev, dtype=torch.uint8)
    with _lib.on_device(dev):
        _lib.check(
            L.ssla_chunk_gated_delta_rule_fwd(
                *tensor_args(q, k, v, g, beta, cu, scale), _lib.ptr(h0), _lib.ptr(o), _lib.ptr(ht),
                states.data_ptr(), nb, ws.data_ptr(), wb, _lib.raw_stream(q.device),
            ),
            "chunk_gated_delta_rule forward",
        )
    return o, ht, states


def chunk_bwd(q, k, v, g, beta, cu, scale, has_h0, has_ht, states, do, dht, want_dh0=True):
    """Gradients from ``states`` of a forward with (``has_h0``) and into (``has_ht``) a state; ``do``,
    ``dht``: None where nothing used that result."""
    T, H, K = q.shape
    HV, V = v.shape[1:]
    N = cu.numel() - 1
    L = _lib.load()
    dev = q.device
    do = do.to(q.dtype).contiguous() if do is not None else torch.zeros_like(v)
    dht = dht.float().contiguous() if dht is not None else None
    dq, dk, dv, dg, dbeta = (torch.empty_like(x) for x in (q, k, v, g, beta))
    dh0 = torch.empty((N, HV, K, V), device=dev, dtype=torch.float32) if has_h0 and want_dh0 else None
    wb = L.ssla_gated_delta_rule_workspace_bytes(N, T, H, HV, K, V, 1)
    ws = torch.empty(wb, device=dev, dtype=torch.uint8)
    with _lib.on_device(dev):
        _lib.check(
            L.ssla_chunk_gated_delta_rule_bwd(
                *tensor_args(q, k, v, g, beta, cu, scale), has_h0, has_ht, states.data_ptr(), states.numel(), do.data_ptr(),
                _lib.ptr(dht), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(),
                _lib.ptr(dh0), ws.data_ptr(), wb, _lib.raw_stream(q.device),
            ),
            "chunk_gated_delta_rule backward",
        )
    return dq, dk, dv, dg, dbeta, dh0


class ChunkGatedDeltaRuleFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, cu_seqlens, scale, initial_state, output_final_state):
        q, k, v, g, beta, cu, h0 = norm_inputs(q, k, v, g, beta, cu_seqlens, initial_state, "chunk_gated_delta_rule")
        o, ht, states = chunk_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state)
        ctx.save_for_backward(q, k, v, g, beta, cu, states)
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        ctx.has_h0, ctx.has_ht = h0 is not None, bool(output_final_state)
        return o, ht

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dht):
        if do is None and dht is None:
            return (None,) * 9
        q, k, v, g, beta, cu, states = ctx.saved_tensors
        dq, dk, dv, dg, dbeta, dh0 = chunk_bwd(q, k, v, g, beta, cu, ctx.scale, ctx.has_h0, ctx.has_ht, states, do, dht,
                                               ctx.needs_input_grad[7])
        return dq, dk, dv, dg, dbeta, None, None, dh0, None


def needs_grad(q, k, v, g, beta, initial_state) -> bool:
    return torch.is_grad_enabled() and (
        q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or beta.requires_grad
        or (initial_state is not None and initial_state.requires_grad)
    )


@torch.compiler.disable
def chunk_gated_delta_rule(
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
    r"""Chunked gated delta rule.

    Args:
        q, k: ``[T, H, K]`` (K <= 128); v: ``[T, HV, V]`` (V <= 256), HV a multiple of H: every key
            head serves ``HV / H`` consecutive value heads.
        g: log forget gates ``[T, HV]`` (g <= 0; ``-inf`` empties the state before the token).
        beta: writing strengths ``[T, HV]``.
        cu_seqlens: cumulative sequence lengths ``[N+1]``; tokens outside every sequence get zero
            outputs and zero gradients, whatever they hold.  Inside a sequence a NaN or infinity also
            reaches earlier tokens of its chunk of 64 (not with ``fused_recurrent_gated_delta_rule``).
        scale: read-out scale, default ``K ** -0.5``.
        initial_state: ``[N, HV, K, V]`` or None.
        output_final_state: also return the final state ``[N, HV, K, V]`` (fp32).
    Returns:
        ``(o [T, HV, V], final_state or None)``.
    """
    refuse_tangents("chunk_gated_delta_rule", q, k, v, g, beta, initial_state)
    if needs_grad(q, k, v, g, beta, initial_state):
        return ChunkGatedDeltaRuleFunction.apply(q, k, v, g, beta, cu_seqlens, scale, initial_state,
                                                 output_final_state)
    q, k, v, g, beta, cu, h0 = norm_inputs(q, k, v, g, beta, cu_seqlens, initial_state, "chunk_gated_delta_rule")
    return chunk_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state)[:2]
