"""Gradients of the gates where a head forgets fast: dg of a token that keeps exp(-20) of the state is
that small itself, and nothing larger may leave its rounding there.

Tolerances (RMS relative, ``conftest.assert_close``), per head, so that no weak gate hides a strong one.
Every pair of tokens (row r, column c < r) adds its own term x to dg of the tokens c < t <= r, formed as
a sum over rows minus one over columns, so that the pairs behind t cancel: with one gate for all tokens
they are as large as the pairs that stay, at most 64 of them by one rounding each, 64 x 2 x 2^-24 = 8e-6 if
all went one way.  fp32 tokens: the suite's 1e-5.  16-bit tokens with fp32 gates: the products behind dg
hold 16 bits (ten in a row, 2^-17 each), and without any state the start states 11 (2^-12): 2^-10 is above
their sum."""
import pytest
import torch

from conftest import assert_close
from oracle.delta_rule import gated_delta_rule_ref
from test_gated_delta_rule import make, operators, reference

TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -10, torch.float16: 2.0 ** -10}


def dg_of(f, x, h0, do, dht, cu, state):
    leaves = [y.cuda().requires_grad_() for y in x]
    o, ht = f(*leaves, cu.cuda(), initial_state=h0.cuda() if state else None, output_final_state=state)
    outs, seeds = ([o, ht], [do.cuda(), dht.cuda()]) if state else ([o], [do.cuda()])
    return torch.autograd.grad(outs, leaves[3], seeds)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("gate", [-1.0, -5.0, -10.0, -20.0])
@pytest.mark.parametrize("T,H,HV,K,V,cu", [(150, 1, 2, 64, 64, [0, 64, 150]), (130, 1, 1, 128, 96, [0, 1, 130])])
def test_one_gate_for_all_tokens(T, H, HV, K, V, cu, gate, dtype, state):
    x, h0, do, dht, cu_t = make(T, H, HV, K, V, cu, dtype, seed=T + K, h0=state, gdtype=torch.float32)
    x = (*x[:3], torch.full_like(x[3], gate), x[4])
    want = reference(x, h0, do, dht if state else torch.zeros_like(dht), cu_t)[2][3]
    got = dg_of(operators()["chunk"], x, h0, do, dht, cu_t, state)
    for h in range(HV):
        assert_close(got[:, h], want[:, h], TOL[dtype], f"dg of head {h}")


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_heads_that_forget_at_unlike_rates(op, dtype):
    rates = torch.tensor([0.02, 1.0, 4.0, 8.0, 12.0, 18.0])
    x, h0, do, dht, cu = make(200, 3, 6, 32, 48, [0, 30, 200], dtype, seed=7, gdtype=torch.float32)
    # between 0.9 and 1.1 of the head's rate: the pairs of a head stay within exp(3.6) of each other
    u = 0.9 + 0.2 * torch.rand(200, 6, generator=torch.Generator().manual_seed(1))
    x = (*x[:3], -rates * u, x[4])
    want = reference(x, h0, do, dht, cu)[2][3]
    got = dg_of(operators()[op], x, h0, do, dht, cu, True)
    for h in range(6):
        # gates that differ by exp(3.6) let terms 37 times a token's own cancel: the norm over the head is
        # that of its largest terms, so the bar of one gate holds
        assert_close(got[:, h], want[:, h], TOL[dtype], f"dg of head {h}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_one_token_sequences_without_a_state(dtype):
    """Nothing was there to forget: dg is 0, whatever q, k and do are."""
    x, _, do, _, cu = make(40, 2, 2, 64, 64, list(range(41)), dtype, seed=2, h0=False, gdtype=torch.float32)
    got = dg_of(operators()["chunk"], x, None, do, None, cu, False)
    assert not got.any()


def test_the_oracle_against_differences():
    """dg of the oracle at -20 by a central difference in 64 bits (exp(g) itself: relative step 1e-5)."""
    x, h0, do, dht, cu = make(5, 1, 1, 8, 8, [0, 5], torch.float32, seed=3)
    x = (*x[:3], torch.full_like(x[3], -20.0), x[4])
    want = reference(x, h0, do, dht, cu)[2][3]

    def loss(e, t):
        g = x[3].double().clone()
        g[t] += e
        o, ht = gated_delta_rule_ref(*x[:3], g, x[4], cu, None, h0)
        return (o * do.double()).sum() + (ht * dht.double()).sum()

    size = float((loss(0.0, 0)).abs())
    for t in range(5):
        diff = float(loss(1e-3, t) - loss(-1e-3, t)) / 2e-3
        # third derivative as large as the first: 1e-6 / 6 of it; 2^-53 of the loss over the step
        assert abs(diff - float(want[t])) < 1e-6 * abs(float(want[t])) + 40 * 2.0 ** -53 * (size + 10) / 2e-3
