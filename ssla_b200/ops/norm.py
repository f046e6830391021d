"""Group norm with an activation over channels-last token features (inference and training).

``z = weight * (x - mean) / sqrt(var + eps) + bias``, ``y = act(z)``, with biased variance.  Without
``cu_seqlens`` every token's groups are normalised for themselves (with a head a group: the norm over each
head's values behind a linear-attention mixer; the activation is of the normalised values, a separate gate
is the caller's product); with it the statistics of a group run over all tokens of a
packed sequence (group norm of a sample's event features).  Kernels: ``ssla_group_norm_act_fwd`` /
``_bwd``.  The reference closes its layers with ``nn.LayerNorm`` (layers/mos_attention.py:144); it
has no group norm.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .utils.guard import prepare_cu_seqlens, refuse_tangents

_ACT = {None: 0, "none": 0, "silu": 1, "relu": 2}
MAX_TOKEN_GROUP = 1024  # channels of a group that is normalised per token


def _param(p, C, x, name):
    if p is None:
        return None
    if p.shape != (C,):
        raise ValueError(f"group_norm_act: {name} must be [{C}], got {tuple(p.shape)}")
    if p.device != x.device:
        raise RuntimeError(f"group_norm_act: {name} is on {p.device}, x on {x.device}")
    return p.float().contiguous()


def _inputs(x, num_groups, weight, bias, cu_seqlens, activation):
    if x.dim() < 2:
        raise ValueError(f"group_norm_act expects x [T, ...channels], got {tuple(x.shape)}")
    T, C = x.shape[0], math.prod(x.shape[1:])
    if C < 1 or num_groups < 1 or C % num_groups:
        raise ValueError(f"group_norm_act: {C} channels cannot be split into {num_groups} groups")
    if activation not in _ACT:
        raise ValueError(f"group_norm_act: activation must be one of None, 'silu', 'relu'; got {activation!r}")
    if cu_seqlens is None and C // num_groups > MAX_TOKEN_GROUP:
        raise ValueError(f"group_norm_act: per token, a group has at most {MAX_TOKEN_GROUP} channels")
    _lib.require_cuda(x, weight, bias, what="group_norm_act")
    _lib.dtype_code(x)
    w, b = _param(weight, C, x, "weight"), _param(bias, C, x, "bias")
    cu = prepare_cu_seqlens(cu_seqlens, x.device) if cu_seqlens is not None else None
    return x.contiguous(), w, b, cu, T, C


def _fwd(x, w, b, cu, T, C, G, eps, act):
    L = _lib.load()
    N = cu.numel() - 1 if cu is not None else 0
    y = torch.empty_like(x)
    saved = ws = None
    sb = nb = 0
    if cu is not None:
        sb = L.ssla_group_norm_act_saved_bytes(T, C, G, N)
        saved = torch.empty(sb, device=x.device, dtype=torch.uint8)
        nb = L.ssla_group_norm_act_workspace_bytes(T, C, G, 1, N, 0)
        ws = torch.empty(nb, device=x.device, dtype=torch.uint8)
    with _lib.on_device(x.device):
        _lib.check(
            L.ssla_group_norm_act_fwd(
                x.data_ptr(), _lib.dtype_code(x), T, C, G, _lib.ptr(w), _lib.ptr(b), float(eps), act, _lib.ptr(cu), N,
                y.data_ptr(), _lib.ptr(saved), sb, _lib.ptr(ws), nb, _lib.raw_stream(x.device),
            ),
            "group_norm_act forward",
        )
    return y, saved


class GroupNormActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, cu_seqlens, eps, activation):
        x, w, b, cu, T, C = _inputs(x, num_groups, weight, bias, cu_seqlens, activation)
        y, saved = _fwd(x, w, b, cu, T, C, num_groups, eps, _ACT[activation])
        ctx.save_for_backward(x, w, b, cu, saved)
        ctx.args = (num_groups, eps, _ACT[activation], T, C)
        ctx.dtypes = [p.dtype if p is not None else None for p in (weight, bias)]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, b, cu, saved = ctx.saved_tensors
        G, eps, act, T, C = ctx.args
        L = _lib.load()
        N = cu.numel() - 1 if cu is not None else 0
        dy = dy.to(x.dtype).contiguous()
        dx = torch.empty_like(x)
        dw, db = torch.empty((2, C), device=x.device, dtype=torch.float32)
        nb = L.ssla_group_norm_act_workspace_bytes(T, C, G, int(cu is not None), N, 1)
        ws = torch.empty(nb, device=x.device, dtype=torch.uint8)
        with _lib.on_device(x.device):
            _lib.check(
                L.ssla_group_norm_act_bwd(
                    x.data_ptr(), dy.data_ptr(), _lib.dtype_code(x), T, C, G, _lib.ptr(w), _lib.ptr(b), float(eps),
                    act, _lib.ptr(cu), N, _lib.ptr(saved), saved.numel() if saved is not None else 0, dx.data_ptr(),
                    dw.data_ptr(), db.data_ptr(), ws.data_ptr(), nb, _lib.raw_stream(x.device),
                ),
                "group_norm_act backward",
            )
        wd, bd = ctx.dtypes
        return (dx, None, dw.to(wd) if wd is not None else None, db.to(bd) if bd is not None else None, None, None,
                None)


@torch.compiler.disable
def group_norm_act(
    x: torch.Tensor,
    num_groups: int,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
    activation: Optional[str] = "silu",
) -> torch.Tensor:
    r"""Group norm over channels-last features with the activation in the same pass.

    Args:
        x: ``[T, C]`` or ``[T, H, V]`` (C = H * V channels per token); float32, bfloat16 or float16.
        num_groups: groups of consecutive channels; C must divide evenly.  Per token a group has at
            most 1024 channels.
        weight, bias: ``[C]`` scale and shift, or None.
        cu_seqlens: None (statistics per token) or cumulative sequence lengths ``[N+1]``
            (statistics per sequence); tokens outside every sequence get zeros.
        activation: ``"silu"``, ``"relu"`` or None.
    Returns:
        y in x's shape and dtype (statistics in fp32 or more, one rounding at the end).
    """
    refuse_tangents("group_norm_act", x, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return GroupNormActFunction.apply(x, num_groups, weight, bias, cu_seqlens, eps, activation)
    x, w, b, cu, T, C = _inputs(x, num_groups, weight, bias, cu_seqlens, activation)
    return _fwd(x, w, b, cu, T, C, num_groups, eps, _ACT[activation])[0]
