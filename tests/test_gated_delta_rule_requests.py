"""The backward computes what is asked for: no gradient of a final state that nothing used, no state
gradient where the initial state needs none, and the token-by-token operator's recomputation leaves out
the outputs."""
import pytest
import torch

from conftest import assert_close
from test_gated_delta_rule import NAMES, TOL, make, operators, reference

NAME = {"chunk": "ssla_b200.ops.gated_delta_rule.chunk", "recurrent": "ssla_b200.ops.gated_delta_rule.fused_recurrent"}


def spy(monkeypatch, op):
    """Records (dht, dh0) of every backward of ``op``."""
    import importlib

    m, seen = importlib.import_module(NAME[op]), []
    plain = m.chunk_bwd

    def recorded(*args, **kw):
        out = plain(*args, **kw)
        seen.append((args[11], out[5]))
        return out

    monkeypatch.setattr(m, "chunk_bwd", recorded)
    return seen


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_unused_states_are_left_out(op, dtype, monkeypatch):
    seen = spy(monkeypatch, op)
    x, h0, do, dht, cu = make(90, 1, 2, 32, 32, [0, 20, 90], dtype, seed=1)
    want = reference(x, h0, do, torch.zeros_like(dht), cu)[2]
    leaves = [y.cuda().requires_grad_() for y in x]
    o, ht = operators()[op](*leaves, cu.cuda(), initial_state=h0.cuda(), output_final_state=True)
    got = torch.autograd.grad(o, leaves, do.cuda())
    for name, a, b in zip(NAMES, got, want):
        assert_close(a, b, TOL[a.dtype], name)
    assert seen == [(None, None)]


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
@pytest.mark.parametrize("h0", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_only_the_final_state_is_used(op, h0, dtype):
    x, h, do, dht, cu = make(90, 1, 2, 32, 32, [0, 20, 90], dtype, seed=2, h0=h0)
    want = reference(x, h, torch.zeros_like(do), dht, cu)[2]
    leaves = [y.cuda().requires_grad_() for y in (*x, *([h] if h0 else []))]
    o, ht = operators()[op](*leaves[:5], cu.cuda(), initial_state=leaves[5] if h0 else None, output_final_state=True)
    got = torch.autograd.grad(ht, leaves, dht.cuda(), allow_unused=True)
    for name, a, b in zip(NAMES, got, want):
        if b.any():
            assert_close(a, b, TOL[a.dtype], name)
        else:  # dq
            assert a is None or not a.any(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("state", [False, True])
def test_recurrent_gradients_are_the_chunked_ones(dtype, state):
    """Same function, same kernels, same accuracy of the states: same bits."""
    x, h0, do, dht, cu = make(300, 2, 4, 64, 64, [0, 100, 300], dtype, seed=3, h0=state, gdtype=torch.float32)
    got = {}
    for op, f in operators().items():
        leaves = [y.cuda().requires_grad_() for y in (*x, *([h0] if state else []))]
        o, ht = f(*leaves[:5], cu.cuda(), initial_state=leaves[5] if state else None, output_final_state=True)
        got[op] = torch.autograd.grad([o, ht], leaves, [do.cuda(), dht.cuda()])
    for name, a, b in zip(NAMES, got["recurrent"], got["chunk"]):
        assert torch.equal(a, b), name


@pytest.mark.gpu
def test_states_alone():
    """The forward's C entry without an output buffer leaves the same states and final state."""
    from ssla_b200.ops.gated_delta_rule import chunk

    for dtype in (torch.float32, torch.bfloat16):
        x, h0, _, _, cu = make(200, 1, 2, 64, 64, [0, 64, 200], dtype, seed=4)
        args = [y.cuda() for y in x]
        _, ht, states = chunk.chunk_fwd(*args, cu.cuda(), 0.125, h0.cuda(), True)
        o, ht2, states2 = chunk.chunk_fwd(*args, cu.cuda(), 0.125, h0.cuda(), True, output=False)
        assert o is None and torch.equal(ht, ht2)
        assert states.numel() == states2.numel()
        # through the backward: the buffer holds unused padding
        do, dht = torch.ones_like(args[2]), torch.ones_like(ht)
        a, b = (chunk.chunk_bwd(*args, cu.cuda(), 0.125, True, True, s, do, dht) for s in (states, states2))
        for name, y, z in zip(NAMES, a, b):
            assert torch.equal(y, z), name


@pytest.mark.gpu
def test_memory_of_a_recurrent_gradient():
    """The recomputation of many one-token sequences holds the states and one workspace, no outputs."""
    from ssla_b200 import _lib

    N, HV, K = 4000, 2, 64
    x, h0, do, dht, cu = make(N, HV, HV, K, K, list(range(N + 1)), torch.float32, seed=5)
    leaves = [y.cuda().requires_grad_() for y in x]
    h, cu, do, dht = h0.cuda(), cu.cuda(), do.cuda(), dht.cuda()
    o, ht = operators()["recurrent"](*leaves, cu, initial_state=h, output_final_state=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    torch.autograd.grad([o, ht], leaves, [do, dht])
    L = _lib.load()
    states = L.ssla_gated_delta_rule_states_bytes(0, N, N, HV, HV, K, K, 1, 1)
    work = L.ssla_gated_delta_rule_workspace_bytes(N, N, HV, HV, K, K, 1)
    # five gradients, the recomputed final state (freed before the backward) and the allocator's rounding
    grads = 3 * leaves[2].numel() * 4 + 2 * leaves[3].numel() * 4
    most = states + work + grads + (16 << 20)
    assert torch.cuda.max_memory_allocated() - start <= most


def step_of(f, x, h0, seeds, cu, use):
    """A training step on leaves of its own: (leaves, function that runs it)."""
    leaves = [y.cuda().requires_grad_() for y in (*x, *([h0] if h0 is not None else []))]
    seeds, cu = [y.cuda() for y in seeds], cu.cuda()

    def step():
        out = f(*leaves[:5], cu, initial_state=leaves[5] if h0 is not None else None, output_final_state=True)
        outs = [y for y, u in zip(out, use) if u]
        return [y.detach() for y in out] + list(torch.autograd.grad(outs, leaves, [s for s, u in zip(seeds, use) if u],
                                                                    allow_unused=True))

    return leaves, step


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
@pytest.mark.parametrize("use", [(True, False), (False, True), (True, True)], ids=str)
def test_captured_steps_replayed_at_once(op, use):
    """Two captured steps, replayed on two streams at the same time with new inputs: as eager steps."""
    sets = [make(500, 1, 2, 64, 64, [0, 200, 500], torch.bfloat16, seed=s, h0=h0) for s, h0 in ((6, True), (7, False))]
    graphs, outs, steps, streams = [], [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, (x, h0, do, dht, cu) in zip(streams, sets):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            leaves, step = step_of(operators()[op], x, h0, (do, dht), cu, use)
            step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step())
        graphs.append(g)
        steps.append(step)
        with torch.no_grad():
            leaves[2].mul_(-0.5)  # the graph reads its inputs at replay
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, step in zip(outs, steps):
        for a, b in zip(out, step()):
            assert a is None and b is None or torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["recurrent", "chunk"])
def test_one_graph_backward_twice(op):
    x, h0, do, dht, cu = make(150, 2, 4, 48, 40, [0, 64, 150], torch.bfloat16, seed=8)
    leaves = [y.cuda().requires_grad_() for y in (*x, h0)]
    o, ht = operators()[op](*leaves[:5], cu.cuda(), initial_state=leaves[5], output_final_state=True)
    first = torch.autograd.grad([o, ht], leaves, [do.cuda(), dht.cuda()], retain_graph=True)
    alone = torch.autograd.grad(o, leaves, do.cuda(), retain_graph=True)
    again = torch.autograd.grad([o, ht], leaves, [do.cuda(), dht.cuda()])
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    want = reference(x, h0, do, torch.zeros_like(dht), cu)[2]
    for name, a, b in zip(NAMES, alone, want):
        assert_close(a, b, TOL[a.dtype], name)
