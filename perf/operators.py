"""The gated delta rule (chunked and recurrent) and the group norm with an activation that closes
such a token mixer: cases, inputs, plain forms and 64-bit values for timing and checking the
kernels of ``ssla_b200.ops.gated_delta_rule`` and ``ssla_b200.ops.norm``.

Packed layout throughout: tokens ``[T, H, D]`` of ``N`` sequences with ``cu_seqlens [N + 1]``.

* recurrent:  S = exp(g) S;  u = beta (v - S^T k);  S = S + k u^T;  o = scale S^T q
* chunk:      the same function over long sequences, forward (prefill) or forward and backward
* norm:       y = act(w (x - mean) / sqrt(var + eps) + b), statistics over a sequence's tokens and
              a group's channels (or over a group's channels of one token)
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ELEM = {"float32": 4, "bfloat16": 2, "float16": 2}
CHUNK = 64


# ------------------------------------------------------------------------------------ cases
def _delta(name, op, n, t, h, hv, k, v, dtype, ragged=False, h0=True, grad=False):
    c = {"op": op, "n": n, "t": t, "h": h, "hv": hv, "k": k, "v": v, "dtype": dtype, "ragged": ragged, "h0": h0,
         "grad": grad}
    return dict(c, name=name) if name else c


def _norm(name, n, t, c, groups, dtype, act, packed, grad):
    d = {"op": "norm", "n": n, "t": t, "c": c, "groups": groups, "dtype": dtype, "act": act, "packed": packed,
         "grad": grad}
    return dict(d, name=name) if name else d


def listed():
    return [
        # one token of four streams: a single user's decoding step, latency alone
        _delta("decode_4_streams", "recurrent", 4, 4, 4, 4, 64, 64, "bfloat16"),
        # a served batch: one token of 256 requests, key heads shared by two value heads
        _delta("decode_256_requests", "recurrent", 256, 256, 16, 32, 128, 128, "bfloat16"),
        # event streams, one fp32 token each, the streaming benchmark's sizes
        _delta("decode_65536_streams", "recurrent", 65536, 65536, 4, 4, 32, 32, "float32"),
        # a few tokens a request (drafted tokens to verify, short prompts), odd sizes
        _delta("short_ragged", "recurrent", 48, 203, 6, 6, 72, 40, "float16", ragged=True),
        # small fp32 prefill with states in and out
        _delta("prefill_small_fp32", "chunk", 3, 331, 4, 4, 64, 64, "float32", ragged=True),
        # one long prompt: few sequences and heads, the time axis is all there is to share out
        _delta("prefill_long", "chunk", 1, 32768, 4, 8, 128, 128, "bfloat16", h0=False),
        # training step at the chunked benchmark's sizes
        _delta("train_8x2048", "chunk", 8, 16384, 4, 4, 64, 64, "bfloat16", h0=False, grad=True),
        # training step over documents of unlike lengths, shared key heads, large heads
        _delta("train_ragged_128", "chunk", 7, 8191, 8, 16, 128, 128, "bfloat16", ragged=True, h0=False, grad=True),
        # fp32 training with odd head sizes and states that carry gradients
        _delta("train_odd_fp32", "chunk", 5, 2500, 3, 3, 48, 80, "float32", ragged=True, grad=True),
        # the heads' norm after the mixer, 16384 tokens of 32 heads, training
        _norm("head_norm_train", 1, 16384, 4096, 32, "bfloat16", "silu", False, True),
        # per-sample group norm of event features, training: the pixel events of a batch of 64
        _norm("sample_norm_train", 64, 333917, 96, 8, "float32", "silu", True, True),
        # the heads' norm of one decoded batch
        _norm("head_norm_decode", 1, 256, 2048, 16, "bfloat16", "silu", False, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    kind = rng.choice(["decode", "short", "prefill", "train", "train", "norm", "norm"])
    if kind == "norm":
        cg = rng.choice([4, 8, 12, 24, 33, 64, 96, 128, 192, 256])
        groups = rng.choice([1, 2, 3, 4, 8, 16, 32])
        c = cg * groups
        packed = rng.random() < 0.5
        t = _log(rng, 16, max(32, min(330000, 30000000 // c)))
        n = min(t, _log(rng, 1, 96)) if packed else 1
        return _norm(None, n, t, c, groups, dtype, rng.choice(["silu", "silu", "relu", "none"]), packed,
                     rng.random() < 0.6)
    k = rng.choice([16, 24, 32, 48, 64, 64, 72, 96, 128, 128])
    v = rng.choice([k, k, 32, 40, 64, 80, 128, 192])
    h = rng.choice([1, 2, 3, 4, 6, 8, 16])
    hv = h * rng.choice([1, 1, 2, 3])
    if kind in ("decode", "short"):
        n = max(1, min(_log(rng, 1, 20000), int(2.5e8 / (hv * k * v))))
        t = n if kind == "decode" else n * rng.choice([2, 3, 5, 8]) + rng.randrange(3)
        return _delta(None, "recurrent", n, t, h, hv, k, v, dtype, ragged=kind == "short")
    grad = kind == "train"
    most = int((1.3e8 if grad else 2.5e8) / (hv * (64 * (k + v) + 3 * k * v) / 64))
    t = max(1, min(_log(rng, 60, 30000), most))
    n = min(t, _log(rng, 1, 12))
    h0 = rng.random() < 0.5 and (not grad or dtype == "float32")
    return _delta(None, "chunk", n, t, h, hv, k, v, dtype, ragged=rng.random() < 0.7, h0=h0, grad=grad)


def _lengths(case):
    """Lengths of the packed sequences, a function of the case alone; ragged ones differ up to
    about a factor of three and may be empty where there are more sequences than tokens."""
    n, t = case["n"], case["t"]
    if not case.get("ragged", case["op"] == "norm"):
        return [t // n + (1 if i < t % n else 0) for i in range(n)]
    w = [1.0 + 2.0 * ((i * 0.6180339887 + 0.31) % 1.0) for i in range(n)]
    ends, acc = [], 0.0
    for x in w:
        acc += x
        ends.append(int(round(acc / sum(w) * t)))
    return [b - a for a, b in zip([0] + ends[:-1], ends)]


# ------------------------------------------------------------------------------------ inputs
def _unit(x):
    x = x * torch.sigmoid(x)
    return x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    dt = DTYPES[case["dtype"]]
    lens = _lengths(case)
    cu = torch.tensor([0] + lens).cumsum(0).cuda()
    t = case["t"]
    if case["op"] == "norm":
        c = case["c"]
        x = (rnd(t, c) * 1.5 + 0.5 * rnd(c)).to(dt)
        s = {"case": case, "x": x, "cu": cu if case["packed"] else None, "w": 1.0 + 0.2 * rnd(c), "b": 0.2 * rnd(c)}
        if case["grad"]:
            s["dy"] = rnd(t, c).to(dt)
            for n in ("x", "w", "b"):
                s[n].requires_grad_()
        return s
    h, hv, k, v, n = case["h"], case["hv"], case["k"], case["v"], case["n"]
    s = {"case": case, "cu": cu, "longest": max(lens)}
    s["q"] = _unit(rnd(t, h, k)).to(dt)
    s["k"] = _unit(rnd(t, h, k)).to(dt)  # SiLU and unit length: keys with a common direction
    s["v"] = rnd(t, hv, v).to(dt)
    rate = torch.exp(torch.linspace(-4.0, 0.5, hv, device="cuda"))  # heads forget at unlike rates
    s["g"] = (-rate * torch.log1p(torch.exp(rnd(t, hv)))).to(dt)
    s["beta"] = torch.sigmoid(rnd(t, hv)).to(dt)
    s["h0"] = 0.3 * rnd(n, hv, k, v) if case["h0"] else None
    if case["grad"]:
        s["do"] = rnd(t, hv, v).to(dt)
        s["dht"] = 0.3 * rnd(n, hv, k, v) if case["h0"] else None
        for name in ("q", "k", "v", "g", "beta", "h0"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------ plain forms
def _rows(cu, longest):
    """Padded view of packed sequences: token index [N, longest], whether it is one, and each
    token's place in the flattened padded view."""
    at = cu[:-1, None] + torch.arange(longest, device=cu.device)
    real = at < cu[1:, None]
    return at, real


def _places(cu, t, longest):
    i = torch.arange(t, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    return seq * longest + i - cu[seq]


def _plain_recurrent(q, k, v, g, beta, cu, longest, h0):
    (t, h, kd), (hv, vd) = q.shape, v.shape[1:]
    n, r, out = cu.numel() - 1, hv // h, v.dtype
    s = h0.float() if h0 is not None else torch.zeros(n, hv, kd, vd, device=q.device)
    q, k, v, g, beta = (x.float() for x in (q, k, v, g, beta))
    q, k = (x.repeat_interleave(r, 1) for x in (q * kd ** -0.5, k))
    at, real = _rows(cu, longest)
    at = at.clamp(max=t - 1)
    os = []
    for i in range(longest):
        a, m = at[:, i], real[:, i, None, None]
        ki = torch.where(m, k[a], 0.0)[..., None]
        s = s * torch.exp(torch.where(m[..., 0], g[a], 0.0))[..., None, None]
        u = beta[a][..., None] * (v[a] - (s * ki).sum(-2))
        s = s + ki * u[..., None, :]
        os.append((s * q[a][..., None]).sum(-2))
    o = torch.stack(os, 1).reshape(n * longest, hv, vd)[_places(cu, t, longest)]
    return o.to(out), s


def _unit_lower_inverse(a):
    """(I + a)^-1 for strictly lower a [..., 64, 64]: inverses of diagonal blocks, twice as large
    at every step."""
    size, b = a.shape[-1], 1
    inv = torch.eye(size, device=a.device, dtype=a.dtype).expand_as(a)
    while b < size:
        i = torch.arange(size, device=a.device) // b
        low = (i[:, None] // 2 == i[None, :] // 2) & (i[:, None] > i[None, :])
        inv = inv - inv @ torch.where(low, a, 0.0) @ inv
        b *= 2
    return inv


def _plain_chunk(q, k, v, g, beta, cu, longest, h0):
    (t, h, kd), (hv, vd) = q.shape, v.shape[1:]
    n, r, out = cu.numel() - 1, hv // h, v.dtype
    nc = max(1, -(-longest // CHUNK))
    at, real = _rows(cu, nc * CHUNK)
    at = at.clamp(max=t - 1)

    def cut(x, heads):  # [T, heads, ...] -> [N, heads, chunks, 64, ...], zeros behind the end
        x = torch.where(real.reshape(n, -1, *[1] * (x.dim() - 1)), x.float()[at], 0.0)
        return x.reshape(n, nc, CHUNK, heads, *x.shape[3:]).movedim(3, 1)

    q, k = (cut(x, h).repeat_interleave(r, 1) for x in (q, k))
    v, beta = cut(v, hv), cut(beta, hv)[..., None]
    gc = cut(g, hv).double().cumsum(-1)
    tri = torch.ones(CHUNK, CHUNK, device=q.device, dtype=torch.bool).tril()
    fade = torch.exp(torch.where(tri, gc[..., :, None] - gc[..., None, :], -math.inf)).float()
    start, left = torch.exp(gc).float()[..., None], torch.exp(gc[..., -1:] - gc).float()[..., None]
    whole = torch.exp(gc[..., -1]).float()[..., None, None]
    inv = _unit_lower_inverse(torch.where(tri.tril(-1), beta * fade * (k @ k.mT), 0.0))
    w, u0 = inv @ (beta * start * k), inv @ (beta * v)
    kl = (left * k).mT
    s = h0.float() if h0 is not None else torch.zeros(n, hv, kd, vd, device=q.device)
    ss = []
    for c in range(nc):  # the state goes from chunk to chunk
        ss.append(s)
        s = whole[:, :, c] * s + kl[:, :, c] @ (u0[:, :, c] - w[:, :, c] @ s)
    ss = torch.stack(ss, 2)
    o = kd ** -0.5 * ((start * q) @ ss + (fade * (q @ k.mT)) @ (u0 - w @ ss))
    o = o.movedim(1, 3).reshape(n * nc * CHUNK, hv, vd)[_places(cu, t, nc * CHUNK)]
    return o.to(out), s


def _plain_norm(x, groups, w, b, cu, act):
    t, c = x.shape
    xf = x.float().reshape(t, groups, c // groups)
    if cu is None:
        mean = xf.mean(-1, keepdim=True)
        var = (xf - mean).square().mean(-1, keepdim=True)
    else:
        seq = torch.searchsorted(cu[1:].contiguous(), torch.arange(t, device=x.device), right=True)
        count = ((cu[1:] - cu[:-1]) * (c // groups)).clamp(min=1)[:, None]

        def over_sequences(a):  # sums over a group's channels and a sequence's tokens, in 64 bits
            s = torch.nn.functional.pad(a.double().sum(-1).t().contiguous().cumsum(1), (1, 0)).t()
            return ((s[cu[1:]] - s[cu[:-1]]) / count)[seq][..., None]

        mean = over_sequences(xf).float()
        var = over_sequences((xf - mean).square()).float()
    y = ((xf - mean) / (var + 1e-5).sqrt()).reshape(t, c) * w + b
    y = y * torch.sigmoid(y) if act == "silu" else torch.where(y > 0, y, 0.0) if act == "relu" else y
    return y.to(x.dtype)


# ------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if c["op"] == "norm":
        act = None if c["act"] == "none" else c["act"]
        if own:
            from ssla_b200.ops.norm import group_norm_act

            y = group_norm_act(s["x"], c["groups"], s["w"], s["b"], cu_seqlens=s["cu"], activation=act)
        else:
            y = _plain_norm(s["x"], c["groups"], s["w"], s["b"], s["cu"], act)
        if not c["grad"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    a = [s[x] for x in ("q", "k", "v", "g", "beta")]
    if own:
        from ssla_b200.ops import gated_delta_rule as d

        f = d.fused_recurrent_gated_delta_rule if c["op"] == "recurrent" else d.chunk_gated_delta_rule
        o, ht = f(*a, s["cu"], initial_state=s["h0"], output_final_state=not c["grad"] or c["h0"])
    else:
        f = _plain_recurrent if c["op"] == "recurrent" else _plain_chunk
        o, ht = f(*a, s["cu"], s["longest"], s["h0"])
    if not c["grad"]:
        return {"o": o, "ht": ht}
    names = [x for x in ("q", "k", "v", "g", "beta", "h0") if s[x] is not None]
    outs, seeds = ([o, ht], [s["do"], s["dht"]]) if c["h0"] else ([o], [s["do"]])
    grads = torch.autograd.grad(outs, [s[x] for x in names], seeds)
    return dict({"d" + x: y for x, y in zip(names, grads)}, o=o.detach(), **({"ht": ht.detach()} if c["h0"] else {}))


def work(case):
    e, t, n = ELEM[case["dtype"]], case["t"], case["n"]
    if case["op"] == "norm":
        # forward x in, y out; backward dy in too and dx out (x read once for both)
        c = case["c"]
        return {"bytes": (4 if case["grad"] else 2) * t * c * e + 8 * c * (2 if case["grad"] else 1),
                "flops": (30 if case["grad"] else 12) * t * c}
    h, hv, k, v = case["h"], case["hv"], case["k"], case["v"]
    tokens = e * t * (2 * h * k + 2 * hv * v + 2 * hv)  # q, k, v, o, g, beta
    state = 4 * n * hv * k * v
    b = tokens + state * (0 if case["grad"] and not case["h0"] else 1 + bool(case["h0"]))
    f = 6 * t * hv * k * v  # S^T k, the update and S^T q of every token
    if case["grad"]:
        b += e * t * (2 * h * k + 2 * hv * v + 2 * hv) + (2 * state if case["h0"] else 0)  # do in, gradients out
        f += 14 * t * hv * k * v  # the recurrence again, its adjoint and the products of the gradients
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------ 64 bits
def _steps64(q, k, v, g, beta, s):
    """The recurrence itself over [N, L, heads, ...] tokens in 64 bits."""
    os = []
    for i in range(q.shape[1]):
        s = torch.exp(g[:, i])[..., None, None] * s
        u = beta[:, i, :, None] * (v[:, i] - torch.einsum("nhkv,nhk->nhv", s, k[:, i]))
        s = s + torch.einsum("nhk,nhv->nhkv", k[:, i], u)
        os.append(torch.einsum("nhkv,nhk->nhv", s, q[:, i]))
    return torch.stack(os, 1), s


def _exact_delta(case, seed):
    s = prepare(case, seed)
    lens, longest = _lengths(case), s["longest"]
    n, hv, kd, vd, r = case["n"], case["hv"], case["k"], case["v"], case["hv"] // case["h"]
    if longest * (3 if case["grad"] else 1) > 60000:
        return None

    def padded(x):
        p = torch.zeros(n, longest, *x.shape[1:], dtype=torch.float64, device="cuda")
        at = 0
        for i, m in enumerate(lens):
            p[i, :m] = x.detach()[at:at + m]
            at += m
        return p

    def packed(p):
        return torch.cat([p[i, :m] for i, m in enumerate(lens)])

    x = [padded(s[y]) for y in ("q", "k", "v", "g", "beta")]
    x[0] = x[0].repeat_interleave(r, 2) / math.sqrt(kd)
    x[1] = x[1].repeat_interleave(r, 2)
    h0 = s["h0"].detach().double() if case["h0"] else torch.zeros(n, hv, kd, vd, dtype=torch.float64, device="cuda")
    starts, os, st = [], [], h0
    with torch.no_grad():
        for a in range(0, longest, 64):
            starts.append(st)
            o, st = _steps64(*[y[:, a:a + 64] for y in x], st)
            os.append(o)
    got = {"o": packed(torch.cat(os, 1))}
    if not case["grad"]:
        return dict(got, ht=st)
    if case["h0"]:
        got["ht"] = st
    do = padded(s["do"])
    ds = s["dht"].double() if case["h0"] else torch.zeros_like(h0)
    grads = [torch.zeros_like(y) for y in x]
    for j in reversed(range(len(starts))):  # 64 tokens at a time, their states made again
        a = 64 * j
        part = [y[:, a:a + 64].clone().requires_grad_() for y in x] + [starts[j].clone().requires_grad_()]
        o, end = _steps64(*part)
        *d, ds = torch.autograd.grad([o, end], part, [do[:, a:a + 64], ds])
        for y, z in zip(grads, d):
            y[:, a:a + 64] = z
    grads[0] = grads[0].unflatten(2, (-1, r)).sum(3) / math.sqrt(kd)
    grads[1] = grads[1].unflatten(2, (-1, r)).sum(3)
    got.update({"d" + y: packed(z) for y, z in zip(("q", "k", "v", "g", "beta"), grads)})
    return dict(got, dh0=ds) if case["h0"] else got


def _exact_norm(case, seed):
    s = prepare(case, seed)
    t, c, groups, act = case["t"], case["c"], case["groups"], case["act"]
    x, w, b = (s[n].detach().double() for n in ("x", "w", "b"))
    lens = _lengths(case) if case["packed"] else None
    shape = (t, groups, c // groups)
    x = x.reshape(shape)

    def mean(a):  # over each sequence's tokens and the group's channels
        if lens is None:
            return a.mean(2, keepdim=True).expand(shape)
        return torch.cat([p.mean((0, 2), keepdim=True).expand(p.shape) for p in a.split(lens)])

    m = mean(x)
    rstd = (mean((x - m) ** 2) + 1e-5) ** -0.5
    xh = (x - m) * rstd
    z = xh.reshape(t, c) * w + b
    sg = 1 / (1 + torch.exp(-z))
    got = {"y": z * sg if act == "silu" else z.clamp(min=0) if act == "relu" else z}
    if case["grad"]:
        dz = s["dy"].double()
        dz = dz * (sg + z * sg * (1 - sg)) if act == "silu" else dz * (z > 0) if act == "relu" else dz
        e = (dz * w).reshape(shape)
        got["dx"] = (rstd * (e - mean(e) - xh * mean(e * xh))).reshape(t, c)
        got["dw"], got["db"] = (dz * xh.reshape(t, c)).sum(0), dz.sum(0)
    return got


def exact(case, seed):
    return _exact_norm(case, seed) if case["op"] == "norm" else _exact_delta(case, seed)
