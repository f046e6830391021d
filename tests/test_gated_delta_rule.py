"""Gated delta rule (chunked, recurrent) against the float64 token recurrence of
``oracle.delta_rule``.

Tolerances (RMS relative, ``conftest.assert_close``; single elements within 5x of the largest
magnitude).  fp32 and the fp32 states of every type: products of split TF32 operands are off by
about 2^-21 and fp32 sums of up to 128 terms by a few 2^-24, over a dozen chained products well
below 1e-5.  16-bit outputs are rounded once (half a step: bf16 2^-8, fp16 2^-11); the products
behind them take operands of two bf16 planes (2^-17 each, about ten in a row), and behind bf16 outputs
of calls without any state the chunks' start states have 11 bits (2^-12 once per chunk, decaying with
the state): together below half a bf16 step, and below half an fp16 step, so 2^-8 and 2^-10 are above both."""
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


# Enough states for chains of 16 and of 32 columns; with and without states that go in and out.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("T,H,HV,K,cu", [
    (80, 20, 40, 40, [0, 70, 80]),
    (80, 40, 40, 128, [0, 70, 80]),
    (90, 60, 60, 40, [0, 66, 70, 90]),
    (90, 30, 60, 128, [0, 66, 70, 90]),
    (200, 2, 2, 64, [0, 200]),
    (200, 1, 2, 128, [0, 150, 200]),
])
def test_many_states_and_none(T, H, HV, K, cu, state, dtype):
    f = operators()["chunk"]
    x, h0, do, dht, cu_t = make(T, H, HV, K, 64, cu, dtype, seed=T + K, h0=state)
    if state:
        o, ht, g = on_gpu(f, x, h0, do, dht, cu_t)
    else:
        dht = torch.zeros_like(dht)
        leaves = [y.cuda().requires_grad_() for y in x]
        o, ht = f(*leaves, cu_t.cuda())
        assert ht is None
        g = torch.autograd.grad(o, leaves, do.cuda())
    o_r, ht_r, g_r = reference(x, h0, do, dht, cu_t)
    assert_close(o, o_r, TOL[dtype], "o")
    if state:
        assert_close(ht, ht_r, TOL[torch.float32], "ht")
    for name, a, b in zip(NAMES, g, g_r):
        assert_close(a, b, TOL[a.dtype], name)


# ------------------------------------------------------------------ refusals (no GPU)
def inputs(T=8, H=1, HV=2, K=4, V=4, N=1, **change):
    x = {"q": torch.zeros(T, H, K), "k": torch.zeros(T, H, K), "v": torch.zeros(T, HV, V), "g": torch.zeros(T, HV),
         "beta": torch.zeros(T, HV), "cu_seqlens": torch.tensor([0] + [T] * N)}
    x.update(change)
    return x


@pytest.mark.parametrize("op", ["recurrent", "chunk"])
@pytest.mark.parametrize("change,message", [
    ({"k": torch.zeros(8, 1, 5)}, "expects q, k"),
    ({"q": torch.zeros(8, 4)}, "expects q, k"),
    ({"v": torch.zeros(7, 2, 4)}, "expects q, k"),
    ({"v": torch.zeros(8, 2, 257)}, "not supported"),
    ({"q": torch.zeros(8, 1, 129), "k": torch.zeros(8, 1, 129)}, "not supported"),
    ({"q": torch.zeros(8, 1, 0), "k": torch.zeros(8, 1, 0)}, "not supported"),
    ({"q": torch.zeros(())}, "expects q, k"),
    ({"g": torch.zeros(8, 1)}, "expects g, beta"),
    ({"beta": torch.zeros(8, 2, 1)}, "expects g, beta"),
    ({"q": torch.zeros(8, 3, 4), "k": torch.zeros(8, 3, 4)}, "multiple of the 3 key heads"),
    ({"v": torch.zeros(8, 0, 4), "g": torch.zeros(8, 0), "beta": torch.zeros(8, 0)}, "positive multiple"),
])
def test_refused_shapes(op, change, message):
    with pytest.raises(ValueError, match=message):
        operators()[op](**inputs(**change))


@pytest.mark.parametrize("op", ["recurrent", "chunk"])
def test_refused_devices(op):
    with pytest.raises(RuntimeError, match="CUDA"):
        operators()[op](**inputs())


def test_entry_points_report_errors():
    from ssla_b200 import _lib

    L = _lib.load()

    def call(name, dtype=0, N=1, T=8, H=1, HV=1, K=4, V=4, tail=()):
        rc = getattr(L, name)(None, None, None, None, None, dtype, 0, 0, None, N, T, H, HV, K, V, 1.0, *tail)
        return rc, L.ssla_last_error()

    fwd = (None, None, None, None, 0, None, 0, None)
    bwd = (0, 0, None, 0, None, None, None, None, None, None, None, None, None, 0, None)
    rec = (None, None, None, None)
    for name, tail in (("ssla_chunk_gated_delta_rule_fwd", fwd), ("ssla_chunk_gated_delta_rule_bwd", bwd),
                       ("ssla_recurrent_gated_delta_rule_fwd", rec)):
        for change, message in (({"dtype": 9}, b"dtype"), ({"K": 129}, b"not supported"), ({"V": 0}, b"not supported"),
                                ({"H": 2, "HV": 3}, b"value heads"), ({"T": -1}, b"negative"), ({}, b"null"),
                                ({"N": 1 << 30, "HV": 64, "H": 64}, b"too many")):
            rc, said = call(name, tail=tail, **change)
            assert rc == -1 and message in said, (name, change, rc, said)
        assert call(name, H=0, HV=0, tail=tail)[0] == 0  # nothing to do
    # buffers that are too small (any address: sizes are checked first)
    one = torch.zeros(64, dtype=torch.uint8).data_ptr()
    rc = L.ssla_chunk_gated_delta_rule_fwd(one, one, one, one, one, 0, 0, 0, one, 1, 8, 1, 1, 4, 4, 1.0, None, one, None,
                                           one, 64, one, 64, None)
    assert rc == -3 and b"needed" in L.ssla_last_error()
    assert L.ssla_gated_delta_rule_states_bytes(0, 1, 8, 1, 1, 0, 4, 0, 0) == 0
    assert (L.ssla_gated_delta_rule_states_bytes(1, 2, 500, 1, 1, 64, 64, 1, 0)
            > L.ssla_gated_delta_rule_states_bytes(1, 2, 500, 1, 1, 64, 64, 0, 0) > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
def test_refused_on_gpu(op):
    f = operators()[op]

    def cuda(**change):
        return {n: x.cuda() for n, x in inputs(**change).items()}

    with pytest.raises(ValueError, match="number of initial states"):
        f(**cuda(), initial_state=torch.zeros(2, 2, 4, 4).cuda())
    with pytest.raises(ValueError, match="initial_state must be"):
        f(**cuda(), initial_state=torch.zeros(1, 2, 4, 5).cuda())
    with pytest.raises(ValueError, match="1-D"):
        f(**cuda(cu_seqlens=torch.zeros(2, 2, dtype=torch.int64)))
    with pytest.raises(TypeError, match="dtype"):
        f(**{n: x.double() if n in "qkv" else x for n, x in cuda().items()})
    with pytest.raises(RuntimeError, match="CUDA"):
        f(**dict(cuda(), beta=torch.zeros(8, 2)))
    with pytest.raises(RuntimeError, match="CUDA"):
        f(**cuda(), initial_state=torch.zeros(1, 2, 4, 4))


# ------------------------------------------------------------------ where it can go wrong
@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rows_of_no_sequence(op, dtype):
    """Padding before the first and behind the last sequence: NaN there reaches nothing, outputs and
    gradients of it are 0."""
    T, cu = 150, [5, 75, 75, 130]
    x, h0, do, dht, cu_t = make(T, 1, 2, 32, 40, cu, dtype, seed=3)
    inside = torch.zeros(T, dtype=torch.bool)
    inside[cu[0]:cu[-1]] = True
    ref = reference([torch.where(inside.reshape(-1, *[1] * (y.dim() - 1)), y, 0.0) for y in x], h0,
                    torch.where(inside[:, None, None], do, 0.0), dht, cu_t)
    dirty = [torch.where(inside.reshape(-1, *[1] * (y.dim() - 1)), y, float("nan")) for y in x]
    torch.empty(1 << 24, device="cuda").fill_(float("nan"))  # freed: what fresh outputs may hold
    o, ht, g = on_gpu(operators()[op], dirty, h0, do, dht, cu_t)
    assert_close(o, ref[0], TOL[dtype], "o")
    assert_close(ht, ref[1], TOL[torch.float32], "ht")
    assert not o[~inside.cuda()].any()
    for name, a, b in zip(NAMES, g, ref[2]):
        assert_close(a, b, TOL[a.dtype], name)
        if name != "dh0":
            assert not a[~inside.cuda()].any(), name


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
def test_no_sequences_and_no_tokens(op):
    f = operators()[op]
    x, h0, do, dht, _ = make(9, 1, 1, 8, 8, [0, 9], torch.float32)
    args = [y.cuda() for y in x]
    o, ht = f(*args, torch.tensor([4]).cuda(), output_final_state=True)
    assert o.shape == (9, 1, 8) and not o.any() and ht.shape == (0, 1, 8, 8)
    empty = [y[:0].requires_grad_() for y in args]
    h = h0.cuda().requires_grad_()
    o, ht = f(*empty, torch.tensor([0, 0]).cuda(), initial_state=h, output_final_state=True)
    assert o.shape == (0, 1, 8) and torch.equal(ht, h)
    assert torch.equal(torch.autograd.grad(ht, h, dht.cuda())[0], dht.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_strides_and_alignment(dtype):
    """Views with other strides and bases off a 16-byte boundary give what their copies give."""
    f = operators()["chunk"]
    x, h0, do, dht, cu = make(100, 2, 2, 64, 64, [0, 30, 100], dtype, seed=8)
    o_r, ht_r, g_r = on_gpu(f, x, h0, do, dht, cu)

    def moved(y, how):
        if how == "strided":
            return y.transpose(0, 1).contiguous().transpose(0, 1)
        z = torch.empty(y.numel() + 1, dtype=y.dtype, device=y.device)[1:].view(y.shape)
        return z.copy_(y)

    for how in ("strided", "shifted"):
        xs = [moved(y.cuda(), how).detach().requires_grad_() for y in x]
        h = moved(h0.cuda(), how).detach().requires_grad_()
        o, ht = f(*xs, cu.cuda(), initial_state=h, output_final_state=True)
        g = torch.autograd.grad([o, ht], xs + [h], [moved(do.cuda(), how), moved(dht.cuda(), how)])
        for a, b in zip([o, ht, *g], [o_r, ht_r, *g_r]):
            assert torch.equal(a, b), how
        r = operators()["recurrent"](*[y.detach() for y in xs], cu.cuda(), initial_state=h.detach())[0]
        assert torch.equal(r, operators()["recurrent"](*[y.cuda() for y in x], cu.cuda(), initial_state=h0.cuda())[0])


@pytest.mark.gpu
@pytest.mark.parametrize("H,off", [(1, 1), (2, 1), (2, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_results_off_a_vector_boundary(dtype, H, off, monkeypatch):
    """The C entry points write wherever the caller's results lie."""
    from ssla_b200.ops.gated_delta_rule import chunk

    x, h0, do, dht, cu = make(100, H, 2, 64, 64, [0, 30, 100], dtype, seed=9)
    want = on_gpu(operators()["chunk"], x, h0, do, dht, cu)

    def shifted(y):
        z = torch.empty(y.numel() + off, dtype=y.dtype, device=y.device)[off:].view(y.shape)
        assert z.data_ptr() % 16
        return z

    monkeypatch.setattr(chunk.torch, "empty_like", shifted)
    xs = [y.cuda() for y in x]
    scale = x[0].shape[-1] ** -0.5
    o, ht, states = chunk.chunk_fwd(*xs, cu.cuda(), scale, h0.cuda(), True)
    got = chunk.chunk_bwd(*xs, cu.cuda(), scale, True, True, states, do.cuda(), dht.cuda())
    for a, b in zip([o, ht, *got], [want[0], want[1], *want[2]]):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gates_that_empty_the_state(op, dtype):
    """g = -inf forgets everything before its token; very strong and very weak decays side by side."""
    x, h0, do, dht, cu = make(140, 1, 1, 32, 32, [0, 140], dtype, seed=5, rate=0.01)
    q, k, v, g, beta = x
    g = g.clone()
    g[[0, 17, 18, 64, 100]] = float("-inf")
    g[[40, 90]] = -80.0
    o_r, ht_r, g_r = reference((q, k, v, torch.where(g.isinf(), -1e4, g), beta), h0, do, dht, cu)
    o, ht, gr = on_gpu(operators()[op], (q, k, v, g, beta), h0, do, dht, cu)
    assert_close(o, o_r, TOL[dtype], "o")
    assert_close(ht, ht_r, TOL[torch.float32], "ht")
    for name, a, b in zip(NAMES, gr, g_r):
        if b.any():
            assert_close(a, b, TOL[a.dtype], name)
        else:  # dh0: the first gate empties the state
            assert not a.any(), name


@pytest.mark.gpu
@pytest.mark.parametrize("beta", [0.0, 1.0, 2.0])
def test_repeated_keys(beta):
    """One key over and over: the inverse of a chunk's triangular system is as far from the identity
    as unit keys allow (beta 1: every write replaces the last, beta 2: alternating signs)."""
    x, h0, do, dht, cu = make(130, 1, 1, 16, 24, [0, 130], torch.float32, seed=6, rate=1e-3)
    q, k, v, g, b = x
    k = k[:1].expand_as(k).contiguous()
    args = (q, k, v, g, torch.full_like(b, beta))
    o_r, ht_r, g_r = reference(args, h0, do, dht, cu)
    o, ht, gr = on_gpu(operators()["chunk"], args, h0, do, dht, cu)
    # T's entries and those of its powers stay within 2, but 64 of them add up with alternating signs
    # in every product: 64 x the bound of one
    assert_close(o, o_r, 64 * 2.0 ** -21, "o")
    assert_close(ht, ht_r, 64 * 2.0 ** -21, "ht")
    for name, a, r in zip(NAMES, gr, g_r):
        assert_close(a, r, 64 * 2.0 ** -21, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
def test_fp32_gates_and_scale(op, dtype):
    x, h0, do, dht, cu = make(99, 2, 4, 48, 64, [0, 33, 99], dtype, seed=11, gdtype=torch.float32)
    o_r, ht_r, g_r = reference(x, h0, do, dht, cu, scale=0.7)
    o, ht, g = on_gpu(operators()[op], x, h0, do, dht, cu, scale=0.7)
    assert_close(o, o_r, TOL[dtype], "o")
    assert_close(ht, ht_r, TOL[torch.float32], "ht")
    for name, a, b in zip(NAMES, g, g_r):
        # fp32 gradients of the gates still come from products of 16-bit planes
        assert_close(a, b, TOL[torch.float32] if name == "dh0" else TOL[dtype], name)


@pytest.mark.gpu
def test_wide_ranges_of_values():
    """Values of one column 1e6 times the others': the scaled planes of the state keep both (2^-28
    of the largest still has all its bits)."""
    x, h0, _, _, cu = make(200, 1, 1, 64, 64, [0, 200], torch.float32, seed=12)
    q, k, v, g, beta = x
    v = v * torch.where(torch.arange(64) % 8 == 3, 1e3, 1e-3)
    h0 = h0 * torch.where(torch.arange(64) % 8 == 3, 1e3, 1e-3)
    o_r, ht_r = gated_delta_rule_ref(q, k, v, g, beta, cu, None, h0)
    o, ht = operators()["chunk"](*[y.cuda() for y in (q, k, v, g, beta)], cu.cuda(), initial_state=h0.cuda(),
                                 output_final_state=True)
    for c in range(64):
        assert_close(o[..., c], o_r[..., c], TOL[torch.float32], f"o column {c}")
        assert_close(ht[..., c], ht_r[..., c], TOL[torch.float32], f"ht column {c}")
    # an infinity stays in its column
    v2 = v.clone()
    v2[70, 0, 5] = float("inf")
    o2, _ = operators()["chunk"](*[y.cuda() for y in (q, k, v2, g, beta)], cu.cuda(), initial_state=h0.cuda())
    rest = [c for c in range(64) if c != 5]
    assert torch.equal(o2[..., rest], o[..., rest]) and not o2[71:, 0, 5].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gradient_against_differences(dtype):
    """<gradient, direction> against a central difference of the forward in float64 (the oracle's, on
    which the forward is tested): eps = 1e-4 leaves eps^2 of the third derivative and 1e-16 / eps."""
    x, h0, do, dht, cu = make(75, 1, 2, 16, 16, [0, 20, 75], dtype, seed=13)
    _, _, g = on_gpu(operators()["chunk"], x, h0, do, dht, cu)
    gen = torch.Generator().manual_seed(1)
    d = [torch.randn(y.shape, generator=gen, dtype=torch.float64) for y in (*x, h0)]

    def loss(e):
        y = [a.double() + e * b for a, b in zip((*x, h0), d)]
        o, ht = gated_delta_rule_ref(*y[:5], cu, None, y[5])
        return float((o * do.double()).sum() + (ht * dht.double()).sum())

    diff = (loss(1e-4) - loss(-1e-4)) / 2e-4
    ours = sum(float((a.double().cpu() * b).sum()) for a, b in zip(g, d))
    # errors of the elements are independent: they add up like the norms
    size = sum(float((a.double().cpu() * b).square().sum()) for a, b in zip(g, d)) ** 0.5
    assert abs(ours - diff) < 4 * TOL[dtype] * size + 1e-6 * abs(diff)


@pytest.mark.gpu
def test_same_bits_every_time_and_on_another_stream():
    f = operators()["chunk"]
    args = make(300, 2, 4, 64, 64, [0, 100, 300], torch.bfloat16, seed=14)
    o, ht, g = on_gpu(f, *args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o2, ht2, g2 = on_gpu(f, *args)
    s.synchronize()
    for a, b in zip([o, ht, *g], [o2, ht2, *g2]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls that overlap share nothing: states and workspaces belong to the call."""
    f = operators()["chunk"]
    sets = [make(2000, 2, 2, 64, 64, [0, 900, 2000], torch.bfloat16, seed=s) for s in (15, 16)]
    gpu = [([y.cuda() for y in x], h.cuda(), cu.cuda()) for x, h, _, _, cu in sets]
    want = [f(*x, cu, initial_state=h, output_final_state=True) for x, h, cu in gpu]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i, (x, h, cu) in enumerate(gpu):
            with torch.cuda.stream(streams[i]):
                got[i].append(f(*x, cu, initial_state=h, output_final_state=True))
    torch.cuda.synchronize()
    for w, rs in zip(want, got):
        for r in rs:
            assert torch.equal(r[0], w[0]) and torch.equal(r[1], w[1])


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
def test_captured_and_replayed(op):
    """A captured call reads its inputs at replay, sequence lengths included."""
    f = operators()[op]
    x, h0, _, _, cu = make(128, 1, 2, 64, 64, [0, 60, 128], torch.bfloat16, seed=17)
    static = [y.cuda() for y in x]
    h, cu_g = h0.cuda(), cu.cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f(*static, cu_g, initial_state=h, output_final_state=True)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, ht = f(*static, cu_g, initial_state=h, output_final_state=True)
    x2, h2, _, _, cu2 = make(128, 1, 2, 64, 64, [0, 100, 128], torch.bfloat16, seed=18)
    for a, b in zip(static + [h, cu_g], (*x2, h2, cu2)):
        a.copy_(b)
    graph.replay()
    want = f(*static, cu_g, initial_state=h, output_final_state=True)
    assert torch.equal(o, want[0]) and torch.equal(ht, want[1])


@pytest.mark.gpu
def test_training_step_captured():
    """Forward and backward in one graph, leaves of their own; an eager step of other leaves first."""
    f = operators()["chunk"]
    x, h0, do, dht, cu = make(200, 1, 2, 64, 64, [0, 60, 200], torch.bfloat16, seed=19)
    want = on_gpu(f, x, h0, do, dht, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaves = [y.cuda().requires_grad_() for y in (*x, h0)]
        cu_g, do_g, dht_g = cu.cuda(), do.cuda(), dht.cuda()

        def step():
            o, ht = f(*leaves[:5], cu_g, initial_state=leaves[5], output_final_state=True)
            return [o, ht, *torch.autograd.grad([o, ht], leaves, [do_g, dht_g])]

        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = [y.detach() for y in step()]
    for y in out:
        y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, [want[0], want[1], *want[2]]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_prompt_then_tokens_then_norm():
    """Prefill in chunks, then token by token, then the heads' norm: as one pass over everything."""
    from ssla_b200.ops.gated_delta_rule import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule
    from ssla_b200.ops.norm import group_norm_act

    N, L, steps, H, HV, K, V = 3, 90, 5, 2, 4, 64, 64
    x, h0, _, _, _ = make(N * (L + steps), H, HV, K, V, [0, N * (L + steps)], torch.bfloat16, seed=20)
    h0 = torch.randn(N, HV, K, V, generator=torch.Generator().manual_seed(2)) * 0.3
    w = 1 + 0.1 * torch.randn(HV * V, generator=torch.Generator().manual_seed(3))
    whole = torch.arange(N + 1) * (L + steps)
    o_r, ht_r = gated_delta_rule_ref(*x, whole, None, h0)
    parts = [y.reshape(N, L + steps, *y.shape[1:]) for y in x]
    pre = [p[:, :L].reshape(N * L, *p.shape[2:]).cuda() for p in parts]
    o, state = chunk_gated_delta_rule(*pre, (torch.arange(N + 1) * L).cuda(), initial_state=h0.cuda(),
                                      output_final_state=True)
    rows = [o.reshape(N, L, HV, V)]
    one = torch.arange(N + 1).cuda()
    for t in range(L, L + steps):
        o, state = fused_recurrent_gated_delta_rule(*[p[:, t].contiguous().cuda() for p in parts], one,
                                                    initial_state=state, output_final_state=True)
        rows.append(o[:, None])
    o = torch.cat(rows, 1).reshape(-1, HV, V)
    assert_close(o, o_r, TOL[torch.bfloat16], "o")
    assert_close(state, ht_r, TOL[torch.float32], "state")
    y = group_norm_act(o, HV, w.cuda())
    assert y.shape == o.shape
    z = o.double().cpu()
    z = (z - z.mean(-1, keepdim=True)) / torch.sqrt(z.var(-1, unbiased=False, keepdim=True) + 1e-5)
    z = z.reshape(-1, HV * V) * w.double()
    assert_close(y.reshape(-1, HV * V), z * torch.sigmoid(z), TOL[torch.bfloat16], "norm")


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """States of more than 2^31 elements (131080 x 128 x 128); the last sequences against the oracle."""
    N, K = 131080, 128
    x, _, _, _, _ = make(4, 1, 1, K, K, [0, 4], torch.bfloat16, seed=21)
    big = [torch.zeros(N, *y.shape[1:], dtype=y.dtype, device="cuda") for y in x]
    for b, y in zip(big, x):
        b[-4:] = y.cuda()
    h0 = torch.zeros(N, 1, K, K, device="cuda")
    h0[-4:] = torch.randn(4, 1, K, K, generator=torch.Generator().manual_seed(4)).cuda() * 0.3
    o, ht = operators()["recurrent"](*big, torch.arange(N + 1).cuda(), initial_state=h0, output_final_state=True)
    o_r, ht_r = gated_delta_rule_ref(*x, torch.arange(5), None, h0[-4:].cpu())
    assert_close(o[-4:], o_r, TOL[torch.bfloat16], "o")
    assert_close(ht[-4:], ht_r, TOL[torch.float32], "ht")
