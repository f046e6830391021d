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


# ------------------------------------------------------------------ refusals (no GPU)
@pytest.mark.parametrize("args,kw,message", [
    ((torch.zeros(4), 1), {}, "expects x"),
    ((torch.zeros(4, 6), 4), {}, "cannot be split"),
    ((torch.zeros(4, 0), 1), {}, "cannot be split"),
    ((torch.zeros(4, 6), 0), {}, "cannot be split"),
    ((torch.zeros(4, 6), 2), {"activation": "gelu"}, "activation"),
    ((torch.zeros(4, 1025), 1), {}, "at most 1024"),
])
def test_refused(args, kw, message):
    from ssla_b200.ops.norm import group_norm_act

    with pytest.raises(ValueError, match=message):
        group_norm_act(*args, **kw)


def test_refused_device():
    from ssla_b200.ops.norm import group_norm_act

    with pytest.raises(RuntimeError, match="CUDA"):
        group_norm_act(torch.zeros(4, 6), 2)


def test_entry_points_report_errors():
    from ssla_b200 import _lib

    L = _lib.load()
    one = torch.zeros(64, dtype=torch.uint8).data_ptr()
    for args, message in (((None, 9, 4, 8, 2), b"dtype"), ((None, 0, 4, 9, 2), b"groups"), ((None, 0, -1, 8, 2), b"groups"),
                          ((None, 0, 4, 2048, 1), b"at most"), ((None, 0, 4, 8, 2), b"null")):
        rc = L.ssla_group_norm_act_fwd(*args, None, None, 1e-5, 1, None, 0, None, None, 0, None, 0, None)
        assert rc == -1 and message in L.ssla_last_error(), args
    rc = L.ssla_group_norm_act_fwd(one, 0, 4, 8, 2, None, None, 1e-5, 7, None, 0, one, None, 0, None, 0, None)
    assert rc == -1 and b"activation" in L.ssla_last_error()
    rc = L.ssla_group_norm_act_fwd(one, 0, 4, 8, 2, None, None, 1e-5, 1, one, 1, one, one, 64, one, 16, None)
    assert rc == -3 and b"needed" in L.ssla_last_error()
    rc = L.ssla_group_norm_act_bwd(one, one, 0, 4, 8, 2, None, None, 1e-5, 1, None, 0, None, 0, one, one, one, None, 0, None)
    assert rc == -3
    rc = L.ssla_group_norm_act_bwd(one, one, 0, 4, 8, 2, None, None, 1e-5, 1, None, 0, None, 0, one, None, one, one, 64, None)
    assert rc == -1


@pytest.mark.gpu
def test_refused_on_gpu():
    from ssla_b200.ops.norm import group_norm_act

    x = torch.zeros(4, 6).cuda()
    with pytest.raises(ValueError, match="weight"):
        group_norm_act(x, 2, torch.zeros(5).cuda())
    with pytest.raises(RuntimeError, match="CUDA"):
        group_norm_act(x, 2, torch.zeros(6))
    with pytest.raises(TypeError, match="dtype"):
        group_norm_act(x.double(), 2)
    with pytest.raises(ValueError, match="1-D"):
        group_norm_act(x, 2, cu_seqlens=torch.zeros(2, 2, dtype=torch.int64).cuda())


# ------------------------------------------------------------------ where it can go wrong
@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_mean_far_from_zero(packed):
    """Mean 1000 times the deviation: fp32 inputs hold the deviation to 2^-24 x 1000, and no more is
    lost."""
    from ssla_b200.ops.norm import group_norm_act

    gen = torch.Generator().manual_seed(1)
    x = (torch.randn(500, 48, generator=gen) + 1000.0).float()
    cu = [0, 123, 500] if packed else None
    dy = torch.randn(500, 48, generator=gen)
    y_r, (dx_r,) = reference(x, 4, None, None, cu, "silu", dy)
    xg = x.cuda().requires_grad_()
    y = group_norm_act(xg, 4, cu_seqlens=torch.tensor(cu).cuda() if cu else None)
    (dx,) = torch.autograd.grad(y, xg, dy.cuda())
    assert_close(y, y_r, 2.0 ** -24 * 1000, "y")
    assert_close(dx, dx_r, 2.0 ** -24 * 1000, "dx")


@pytest.mark.gpu
def test_shapes_layouts_and_parameter_types():
    from ssla_b200.ops.norm import group_norm_act

    gen = torch.Generator().manual_seed(2)
    x = torch.randn(6, 4, 32, generator=gen).bfloat16()
    w, b = (torch.randn(128, generator=gen).bfloat16().cuda().requires_grad_() for _ in range(2))
    y_r, g_r = reference(x.reshape(6, 128), 4, w.detach().cpu(), b.detach().cpu(), None, "silu", torch.ones(6, 128))
    y = group_norm_act(x.cuda(), 4, w, b)
    assert y.shape == x.shape and y.dtype == torch.bfloat16
    assert_close(y.reshape(6, 128), y_r, TOL[torch.bfloat16], "y")
    dw, db = torch.autograd.grad(y.sum(), (w, b))
    assert dw.dtype == torch.bfloat16
    assert_close(dw, g_r[1], 2.0 ** -8, "dw")
    assert_close(db, g_r[2], 2.0 ** -8, "db")
    t = x.cuda().transpose(0, 1).contiguous().transpose(0, 1)  # other strides
    assert torch.equal(group_norm_act(t, 4, w, b), y)
    shifted = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)
    assert_close(group_norm_act(shifted, 4, w, b).reshape(6, 128), y_r, TOL[torch.bfloat16], "off a boundary")
    for cu in (None, torch.tensor([0, 0]).cuda(), torch.tensor([0]).cuda()):
        e = torch.zeros(0, 128, device="cuda", requires_grad=True)
        y0 = group_norm_act(e, 4, w, cu_seqlens=cu)
        assert y0.shape == (0, 128)
        assert not torch.autograd.grad(y0.sum(), w)[0].any()


@pytest.mark.gpu
def test_rows_of_no_sequence_and_nan():
    """Rows outside every sequence: NaN there reaches nothing, results 0.  A NaN inside spoils its own
    sequence and group only."""
    from ssla_b200.ops.norm import group_norm_act

    gen = torch.Generator().manual_seed(3)
    x, dy = torch.randn(60, 16, generator=gen), torch.randn(60, 16, generator=gen)
    y_r, (dx_r, dw_r) = reference(x[10:50], 2, torch.ones(16), None, [0, 15, 40], "silu", dy[10:50])
    x[:10], x[50:] = float("nan"), float("nan")
    xg, w = x.cuda().requires_grad_(), torch.ones(16, device="cuda", requires_grad=True)
    cu = torch.tensor([10, 25, 50]).cuda()
    y = group_norm_act(xg, 2, w, cu_seqlens=cu)
    dx, dw = torch.autograd.grad(y, (xg, w), dy.cuda())
    assert_close(y[10:50], y_r, TOL[torch.float32], "y")
    assert_close(dx[10:50], dx_r, TOL[torch.float32], "dx")
    assert_close(dw, dw_r, TOL[torch.float32], "dw")
    for t in (y, dx):
        assert not t[:10].any() and not t[50:].any()
    none = group_norm_act(xg.detach(), 2, cu_seqlens=torch.tensor([7]).cuda())
    assert not none.any()
    x[20, 3] = float("nan")
    y2 = group_norm_act(x.cuda(), 2, cu_seqlens=cu)
    assert y2[10:25, :8].isnan().all() and torch.equal(y2[10:25, 8:], y.detach()[10:25, 8:])
    assert torch.equal(y2[25:50], y.detach()[25:50])


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_captured_streams_and_repeats(packed):
    from ssla_b200.ops.norm import group_norm_act

    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(5000, 96, generator=gen, device="cuda").requires_grad_()
    w = torch.randn(96, generator=gen, device="cuda").requires_grad_()
    dy = torch.randn(5000, 96, generator=gen, device="cuda")
    cu = torch.tensor([0, 1000, 1001, 5000]).cuda() if packed else None

    def step():
        y = group_norm_act(x, 8, w, cu_seqlens=cu)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy)]

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    with torch.no_grad():
        x.mul_(-2.0)
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_more_than_32_bits_of_elements():
    from ssla_b200.ops.norm import group_norm_act

    T, C = (1 << 20) + 3, 2048
    x = torch.zeros(T, C, dtype=torch.bfloat16, device="cuda")
    x[-5:] = torch.randn(5, C, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    y_r = reference(x[-5:].cpu(), 16, None, None, None, "silu", torch.zeros(5, C))[0]
    assert_close(group_norm_act(x, 16)[-5:], y_r, TOL[torch.bfloat16], "per token")
    y_r = reference(x[-5:].cpu(), 16, None, None, [0, 5], "silu", torch.zeros(5, C))[0]
    y = group_norm_act(x, 16, cu_seqlens=torch.tensor([0, T - 5, T]).cuda())
    assert_close(y[-5:], y_r, TOL[torch.bfloat16], "packed")
