"""Gated delta rule (chunked, recurrent) against the float64 token recurrence of
``oracle.delta_rule``.

Tolerances (RMS relative, ``conftest.assert_close``; single elements within 5x of the largest
magnitude).  fp32 and the fp32 states of every type: products of split TF32 operands are off by
about 2^-21 and fp32 sums of up to 128 terms by a few 2^-24, over a dozen chained products well
below 1e-5.  16-bit outputs are rounded once (half a step: bf16 2^-8, fp16 2^-11); the products
behind a bf16 output round their operands to TF32 (2^-11 each, about ten in a row), together below
one bf16 step's half, and behind an fp16 output they are split: 2^-8 and 2^-10 are above both."""
import pytest
import torch
import torch.nn.functional as F

from conftest import assert_close
from oracle.delta_rule import gated_delta_rule_ref

TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
NAMES = ("dq", "dk", "dv", "dg", "dbeta", "dh0")


def make(T, H, HV, K, V, cu, dtype, seed=0, h0=True, rate=0.3, gdtype=None):
    gen = torch.Generator().manual_seed(seed)
    q = F.normalize(F.silu(torch.randn(T, H, K, generator=gen)), dim=-1)
    k = F.normalize(F.silu(torch.randn(T, H, K, generator=gen)), dim=-1)
    v = torch.randn(T, HV, V, generator=gen)
    g = -rate * F.softplus(torch.randn(T, HV, generator=gen))
    beta = torch.sigmoid(torch.randn(T, HV, generator=gen))
    N = len(cu) - 1
    hz = torch.randn(N, HV, K, V, generator=gen) * 0.3 if h0 else None
    do = torch.randn(T, HV, V, generator=gen).to(dtype)
    dht = torch.randn(N, HV, K, V, generator=gen) * 0.3
    q, k, v = (x.to(dtype) for x in (q, k, v))
    g, beta = (x.to(gdtype or dtype) for x in (g, beta))
    return (q, k, v, g, beta), hz, do, dht, torch.tensor(cu)


def reference(x, h0, do, dht, cu, scale=None):
    leaves = [y.double().requires_grad_() for y in x]
    h = h0.double().requires_grad_() if h0 is not None else None
    o, ht = gated_delta_rule_ref(*leaves, cu, scale, h)
    ins = leaves + ([h] if h is not None else [])
    loss = (o * do.double()).sum() + (ht * dht.double()).sum()
    grads = torch.autograd.grad(loss, ins, allow_unused=True)
    return o.detach(), ht.detach(), [torch.zeros_like(i) if y is None else y for i, y in zip(ins, grads)]


def on_gpu(fn, x, h0, do, dht, cu, scale=None):
    leaves = [y.cuda().requires_grad_() for y in x]
    h = h0.cuda().requires_grad_() if h0 is not None else None
    o, ht = fn(*leaves, cu.cuda(), scale=scale, initial_state=h, output_final_state=True)
    ins = leaves + ([h] if h is not None else [])
    grads = torch.autograd.grad([o, ht], ins, [do.cuda(), dht.cuda()])
    return o.detach(), ht.detach(), list(grads)


def operators():
    from ssla_b200.ops.gated_delta_rule import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule

    return {"chunk": chunk_gated_delta_rule, "recurrent": fused_recurrent_gated_delta_rule}


# T, H, HV, K, V, cu: empty and one-token sequences, chunk borders, odd heads, shared key heads
SHAPES = [
    (150, 2, 2, 64, 64, [0, 70, 150]),
    (200, 1, 2, 32, 48, [0, 0, 1, 65, 129, 129, 200]),
    (130, 2, 4, 128, 128, [0, 64, 128, 130]),
    (70, 1, 3, 17, 5, [0, 3, 70]),
    (67, 3, 3, 128, 200, [0, 67]),
    (193, 1, 1, 72, 40, [0, 193]),
    (1, 1, 1, 1, 1, [0, 1]),
    (64, 1, 1, 100, 256, [0, 64]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("T,H,HV,K,V,cu", SHAPES)
def test_forward(op, dtype, T, H, HV, K, V, cu):
    for h0 in (False, True):
        x, h, _, _, cu_t = make(T, H, HV, K, V, cu, dtype, seed=T + K, h0=h0)
        o_r, ht_r = gated_delta_rule_ref(*x, cu_t, None, h)
        o, ht = operators()[op](*[y.cuda() for y in x], cu_t.cuda(), initial_state=h.cuda() if h0 else None,
                                output_final_state=True)
        assert o.dtype == dtype and ht.dtype == torch.float32
        assert_close(o, o_r, TOL[dtype], "o")
        assert_close(ht, ht_r, TOL[torch.float32], "ht")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("T,H,HV,K,V,cu", SHAPES)
def test_backward(dtype, T, H, HV, K, V, cu):
    for h0 in (False, True):
        args = make(T, H, HV, K, V, cu, dtype, seed=T + V, h0=h0)
        o_r, ht_r, g_r = reference(*args)
        o, ht, g = on_gpu(operators()["chunk"], *args)
        assert_close(o, o_r, TOL[dtype], "o")
        for name, a, b in zip(NAMES, g, g_r):
            assert a.dtype == (torch.float32 if name == "dh0" else dtype)
            if not b.any():
                # one token without a state: dg = q.dq - k.dk, two equal products; what is left is
                # the rounding of their 2 K fp32 additions, at most 2 K 2^-24 sum |q dq| each
                bound = 4 * K * 2.0 ** -24 * float((args[0][0].double().repeat_interleave(HV // H, 1) * g_r[0]).abs().sum())
                assert float(a.abs().max()) <= bound, name
                continue
            assert_close(a, b, TOL[a.dtype], name)
