"""Value columns of unlike size.  Column c of v, o and the states has nothing to do with the others, so
each is compared for itself: a column 1e-12 times its neighbour keeps its own accuracy, forward and
reverse, and how many columns a block of the state's chain takes changes nothing.

Tolerances: those of ``test_gated_delta_rule``, per column.  The chain brings every column's largest entry
of 16 rows near 2^14 before it is split into fp16 planes, so two planes are off by at most 2^-38 of it."""
import pytest
import torch

from conftest import assert_close
from oracle.delta_rule import gated_delta_rule_ref
from test_gated_delta_rule import NAMES, TOL, make, on_gpu, operators, reference

# N HV: 4 (8 columns a block), 80 (16 columns), 160 (32 columns)
HEADS = [2, 40, 80]


def unlike_columns(V, shift):
    """1, 1e-4, 1e-8, 1e-12 in turn within every 8 columns."""
    return 10.0 ** -(4.0 * ((torch.arange(V) + shift) % 4))


def inputs(HV, K, dtype, seed, state=True):
    x, h0, do, dht, cu = make(200, HV, HV, K, 64, [0, 130, 200], dtype, seed=seed, h0=state)
    c, d = unlike_columns(64, 0), unlike_columns(64, 1)
    x = (x[0], x[1], (x[2].float() * c).to(dtype), x[3], x[4])
    return x, h0 * c if state else None, (do.float() * d).to(dtype), dht * d, cu


def columns(a, b, tol, name):
    for c in range(a.shape[-1]):
        assert_close(a[..., c], b[..., c], tol, f"{name} column {c}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("HV", HEADS)
def test_columns_keep_their_own_accuracy(HV, K, dtype):
    args = inputs(HV, K, dtype, seed=HV + K)
    o_r, ht_r, g_r = reference(*args)
    o, ht, g = on_gpu(operators()["chunk"], *args)
    columns(o, o_r, TOL[dtype], "o")
    columns(ht, ht_r, TOL[torch.float32], "ht")
    g, g_r = dict(zip(NAMES, g)), dict(zip(NAMES, g_r))
    columns(g["dv"], g_r["dv"], TOL[dtype], "dv")
    columns(g["dh0"], g_r["dh0"], TOL[torch.float32], "dh0")


@pytest.mark.gpu
@pytest.mark.parametrize("HV", HEADS)
def test_columns_without_any_state(HV):
    """bf16 without states: the chain's operands have 11 bits, of every column."""
    x, _, do, _, cu = inputs(HV, 64, torch.bfloat16, seed=HV, state=False)
    o_r = gated_delta_rule_ref(*x, cu)[0]
    leaves = [y.cuda().requires_grad_() for y in x]
    o, _ = operators()["chunk"](*leaves, cu.cuda())
    columns(o, o_r, TOL[torch.bfloat16], "o")
    zero = torch.zeros(2, HV, 64, 64)
    dv_r = reference(x, None, do, zero, cu)[2][2]
    columns(torch.autograd.grad(o, leaves[2], do.cuda())[0], dv_r, TOL[torch.bfloat16], "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_the_same_bits_next_to_any_number_of_heads(dtype):
    """One head alone, and the same head 80 and 160 times in one call."""
    f = operators()["chunk"]
    x, h0, do, dht, cu = make(200, 1, 1, 64, 64, [0, 200], dtype, seed=5)
    c, d = unlike_columns(64, 0), unlike_columns(64, 1)
    x, h0, do, dht = (x[0], x[1], (x[2].float() * c).to(dtype), x[3], x[4]), h0 * c, (do.float() * d).to(dtype), dht * d
    o, ht, g = on_gpu(f, x, h0, do, dht, cu)
    for n in (80, 160):
        many = [y.repeat_interleave(n, 1) for y in (*x, h0, do, dht)]
        o_n, ht_n, g_n = on_gpu(f, many[:5], many[5], many[6], many[7], cu)
        for name, a, b in zip(("o", "ht", *NAMES), (o_n, ht_n, *g_n), (o, ht, *g)):
            assert torch.equal(a, b.repeat_interleave(n, 1)), (name, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_no_decay_over_many_chunks(dtype):
    """g = 0, 60 chunks, writing strengths up to 1.8: what the state's products lose does not add up, for
    every write erases along its key what was there."""
    x, h0, do, dht, cu = make(3800, 1, 1, 64, 32, [0, 3800], dtype, seed=9, h0=False)
    q, k, v, g, beta = x
    x = (q, k, v, torch.zeros_like(g), (1.8 * beta.float()).to(dtype))
    o_r, ht_r = gated_delta_rule_ref(*x, cu)
    f = operators()["chunk"]
    args = [y.cuda() for y in x]
    o, ht = f(*args, cu.cuda(), output_final_state=True)
    assert_close(o, o_r, TOL[dtype], "o")
    assert_close(ht, ht_r, TOL[torch.float32], "ht")
    o, _ = f(*args, cu.cuda())
    assert_close(o, o_r, TOL[dtype], "o without states")


@pytest.mark.gpu
@pytest.mark.parametrize("HV", HEADS)
@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e20, 1e30])
def test_states_far_from_one(HV, size):
    """The chain's scales follow the state over the exponents of fp32."""
    x, h0, do, dht, cu = make(200, HV, HV, 64, 64, [0, 130, 200], torch.float32, seed=HV)
    x, h0 = (x[0], x[1], x[2] * size, x[3], x[4]), h0 * size
    o_r, ht_r = gated_delta_rule_ref(*x, cu, None, h0)
    o, ht = operators()["chunk"](*[y.cuda() for y in x], cu.cuda(), initial_state=h0.cuda(), output_final_state=True)
    # at 1e-30 the low parts of split operands (2^-22 of them) are still normal numbers
    for name, a, b in (("o", o, o_r), ("ht", ht, ht_r)):
        assert_close(a.double() / size, b / size, TOL[torch.float32], name)
    do, dht = do * size, dht * size
    leaves = [y.cuda().requires_grad_() for y in (*x[:2], x[2] / size, *x[3:])]
    o, ht = operators()["chunk"](*leaves, cu.cuda(), output_final_state=True)
    dv = torch.autograd.grad([o, ht], leaves[2], [do.cuda(), dht.cuda()])[0]
    one = reference((*x[:2], x[2] / size, *x[3:]), None, do / size, dht / size, cu)[2][2]
    assert_close(dv.double() / size, one, TOL[torch.float32], "dv")
