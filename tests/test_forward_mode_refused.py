"""Operators without a forward-mode derivative refuse inputs that carry a tangent: a result without
one would read as a derivative of zero."""
import pytest
import torch
from torch.autograd import forward_ad

OPS = ("chunk", "recurrent", "norm", "norm packed")


def call(op, device="cpu"):
    """(function of a list of tensors, those tensors)."""
    from ssla_b200.ops.gated_delta_rule import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule
    from ssla_b200.ops.norm import group_norm_act

    cu = torch.tensor([0, 5], device=device)
    if op.startswith("norm"):
        packed = cu if op == "norm packed" else None
        x = [torch.randn(5, 8, device=device), torch.randn(8, device=device), torch.randn(8, device=device)]
        return lambda x, w, b: group_norm_act(x, 2, w, b, cu_seqlens=packed), x
    f = chunk_gated_delta_rule if op == "chunk" else fused_recurrent_gated_delta_rule
    x = [torch.randn(*s, device=device) for s in ((5, 1, 8), (5, 1, 8), (5, 2, 8), (5, 2), (5, 2), (1, 2, 8, 8))]
    return lambda q, k, v, g, b, h: f(q, k, v, g, b, cu, initial_state=h)[0], x


@pytest.mark.parametrize("op", OPS)
def test_a_tangent_is_refused(op):
    f, x = call(op)
    for i in range(len(x)):
        for grad in (False, True):
            with forward_ad.dual_level():
                y = [t.clone().requires_grad_(grad) for t in x]
                y[i] = forward_ad.make_dual(y[i], torch.ones_like(y[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*y)


@pytest.mark.parametrize("op", OPS)
def test_a_level_without_tangents_changes_nothing(op):
    f, x = call(op)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="CUDA"):  # the next check
        f(*x)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_on_the_gpu(op):
    f, x = call(op, "cuda")
    want = f(*x)
    with forward_ad.dual_level():
        assert torch.equal(f(*x), want)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(forward_ad.make_dual(x[0], torch.ones_like(x[0])), *x[1:])
