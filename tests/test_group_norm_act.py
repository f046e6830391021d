"""Group norm with an activation against float64.

Tolerances (RMS relative, ``conftest.assert_close``): statistics are fp32 or better and every
element sees a handful of fp32 operations, so fp32 results stay within a few 2^-24 of the value
before the activation: 2e-6 (dw, db: sums of T such products: likewise, joined in 64 bits).  16-bit
results are rounded once, by at most 2^-8 (bf16) or 2^-11 (fp16) of the value."""
import pytest
import torch

from conftest import assert_close

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(x, groups, w, b, cu, act, dy, eps=1e-5):
    T, C = x.shape
    x, w, b = (None if t is None else t.double().requires_grad_() for t in (x, w, b))
    parts = [x[a:c] for a, c in zip(cu[:-1], cu[1:])] if cu is not None else [x]
    ys = []
    for p in parts:
        p = p.reshape(p.shape[0], groups, C // groups)
        dims = (0, 2) if cu is not None else (2,)
        if p.numel():
            p = (p - p.mean(dims, keepdim=True)) / torch.sqrt(p.var(dims, unbiased=False, keepdim=True) + eps)
        ys.append(p.reshape(-1, C))
    z = torch.cat(ys)
    if cu is not None and cu[-1] < T:
        z = torch.cat([z, z.new_zeros(T - cu[-1], C)])
    z = (z * w if w is not None else z) + (b if b is not None else 0.0)
    y = z * torch.sigmoid(z) if act == "silu" else torch.relu(z) if act == "relu" else z
    if cu is not None and cu[-1] < T:
        y = torch.cat([y[: cu[-1]], y.new_zeros(T - cu[-1], C)])
    ins = [t for t in (x, w, b) if t is not None]
    return y.detach(), torch.autograd.grad((y * dy.double()).sum(), ins)


# T, C, groups, cu (None: per token)
SHAPES = [
    (37, 64, 4, None),
    (5, 33, 1, None),
    (300, 1024, 1, None),
    (64, 24, 8, None),
    (1, 8, 2, None),
    (200, 96, 8, [0, 3, 3, 50, 200]),
    (999, 12, 3, [0, 1, 2, 600, 990]),
    (70, 66, 2, [0, 70]),
    (20, 4096, 2, [0, 11, 20]),
    (40, 5000, 1, [0, 40]),
    (513, 320, 5, [0, 0, 512, 513]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act,params", [("silu", True), ("relu", True), (None, False)])
@pytest.mark.parametrize("T,C,groups,cu", SHAPES)
def test_forward_backward(dtype, act, params, T, C, groups, cu):
    from ssla_b200.ops.norm import group_norm_act

    gen = torch.Generator().manual_seed(T + C)
    x = (torch.randn(T, C, generator=gen) * 2 + torch.randn(C, generator=gen)).to(dtype)
    dy = torch.randn(T, C, generator=gen).to(dtype)
    w = 1 + 0.3 * torch.randn(C, generator=gen) if params else None
    b = 0.3 * torch.randn(C, generator=gen) if params else None
    y_r, g_r = reference(x, groups, w, b, cu, act, dy)
    ins = [t.cuda().requires_grad_() for t in (x, w, b) if t is not None]
    y = group_norm_act(ins[0], groups, *(ins[1:] if params else (None, None)),
                       cu_seqlens=torch.tensor(cu).cuda() if cu is not None else None, activation=act)
    assert y.dtype == dtype
    assert_close(y, y_r, TOL[dtype], "y")
    grads = torch.autograd.grad(y, ins, dy.cuda())
    for name, a, r in zip(("dx", "dw", "db"), grads, g_r):
        assert_close(a, r, TOL[a.dtype], name)
