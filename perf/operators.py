"""Cases and plain forms of the training operators: the selective scan with its gradients, the causal conv1d
with its gradients from an 8-bit checkpoint of its input, that checkpoint itself, and the preference loss with
its gradient.

``run`` makes one pass: with ``own`` the calls of ``mamba_metal_b200.training``, without it the same operators
in elementary float32 torch operations, rounded once at the end. ``exact`` gives the same outputs from the
operators' definitions in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32  # values of one row that share a scale in an 8-bit checkpoint
IGNORE = -100


def listed():
    return [
        # A short answer of one user on the 130m shape (1536 channels): launch latency decides.
        dict(name="scan_short", op="scan", dtype="bf16", batch=1, dim=1536, dstate=16, length=48, layout="channel_first",
             z=True, D=True, bias=True, softplus=True, state=True),
        # The 5,601-token prompt of the 130m configuration in float32: one odd-length row, little parallelism
        # over channels, so the work has to be split over time.
        dict(name="scan_prompt", op="scan", dtype="f32", batch=1, dim=1536, dstate=16, length=5601,
             layout="channels_last", z=True, D=True, bias=True, softplus=True, state=False),
        # The scan benchmark's own shape as a training batch.
        dict(name="scan_batch", op="scan", dtype="f16", batch=8, dim=1536, dstate=16, length=4096,
             layout="channel_first", z=True, D=True, bias=False, softplus=True, state=False),
        # Long documents at the 2.8b shape's 5120 channels, with the state handed on.
        dict(name="scan_long", op="scan", dtype="bf16", batch=1, dim=5120, dstate=16, length=16384,
             layout="channel_first", z=True, D=True, bias=True, softplus=True, state=True),
        # The conv of a short answer: latency, a length that is not a multiple of anything.
        dict(name="conv_short", op="conv", dtype="bf16", batch=1, dim=1536, length=33, layout="channel_first", silu=True,
             bias=True),
        # The conv benchmark's own shape as a training batch.
        dict(name="conv_batch", op="conv", dtype="f16", batch=8, dim=1536, length=4096, layout="channel_first", silu=True,
             bias=True),
        # Odd prompts at the 2.8b shape, whose rows the block lays out (tokens, channels).
        dict(name="conv_odd", op="conv", dtype="bf16", batch=4, dim=5120, length=5601, layout="channels_last", silu=True,
             bias=True),
        # A checkpoint of few, short, ragged rows.
        dict(name="checkpoint_short", op="checkpoint", dtype="f32", rows=1536, cols=33),
        # The in_proj output of 16 x 2048 tokens at the 2.8b shape, held until the backward pass.
        dict(name="checkpoint_layer", op="checkpoint", dtype="bf16", rows=10240, cols=32768),
        # One pair of two-token answers: latency over few long rows.
        dict(name="preference_short", op="preference", dtype="bf16", pairs=1, length=2, vocab=50280, prompt=0.0,
             beta=0.1, smoothing=0.0),
        # Ragged float32 logits whose rows begin at odd addresses, with label smoothing.
        dict(name="preference_odd", op="preference", dtype="f32", pairs=2, length=777, vocab=50277, prompt=0.4,
             beta=0.2, smoothing=0.1),
        # A training batch of eight pairs of 1024 tokens, about half of them prompt.
        dict(name="preference_batch", op="preference", dtype="bf16", pairs=8, length=1024, vocab=50280, prompt=0.5,
             beta=0.1, smoothing=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "conv", "checkpoint", "preference"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    layout = rng.choice(["channel_first", "channels_last"])
    flag = lambda: rng.random() < 0.7
    if op == "scan":
        most = 5120 * 16384 * 16
        dstate = rng.choice([16, 16, 16, 8, 24, 64])
        batch, dim = rng.randint(1, 8), _log_int(rng, 8, 5120)
        length = _log_int(rng, 1, max(1, min(16384, most // (batch * dim * dstate))))
        return dict(op=op, dtype=dtype, batch=batch, dim=dim, dstate=dstate, length=length, layout=layout, z=flag(),
                    D=flag(), bias=flag(), softplus=True, state=flag())
    if op == "conv":
        most = 4 * 5120 * 5601
        batch, dim = rng.randint(1, 8), _log_int(rng, 8, 5120)
        length = _log_int(rng, 1, max(1, min(16384, most // (batch * dim))))
        return dict(op=op, dtype=dtype, batch=batch, dim=dim, length=length, layout=layout, silu=flag(), bias=flag())
    if op == "checkpoint":
        rows = _log_int(rng, 1, 10240)
        return dict(op=op, dtype=dtype, rows=rows, cols=_log_int(rng, 1, 32768))
    pairs = rng.randint(1, 8)
    vocab = rng.choice([50280, 50277, _log_int(rng, 300, 50280)])
    length = _log_int(rng, 1, max(1, 8 * 1024 // (pairs * (2 if dtype == "f32" else 1))))
    return dict(op=op, dtype=dtype, pairs=pairs, length=length, vocab=vocab, prompt=rng.choice([0.0, 0.3, 0.6]),
                beta=rng.choice([0.05, 0.1, 0.5]), smoothing=rng.choice([0.0, 0.1]))


# ---- inputs ------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _activation(case, g, scale=1.0):
    """(batch, dim, length) normal values in the case's type and layout."""
    b, d, n, dt = case["batch"], case["dim"], case["length"], DTYPES[case["dtype"]]
    if case["layout"] == "channels_last":
        return (_randn(g, b, n, d) * scale).to(dt).transpose(1, 2)
    return (_randn(g, b, d, n) * scale).to(dt)


def _prompt_lengths(case):
    """Prompt tokens of every row, spread evenly up to twice the case's mean share."""
    rows = 2 * case["pairs"]
    return [min(case["length"], int(case["length"] * case["prompt"] * (2 * r + 1) / rows)) for r in range(rows)]


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "scan":
        b, d, n, length = case["batch"], case["dim"], case["dstate"], case["length"]
        st["u"], st["delta"], st["dy"] = _activation(case, g), _activation(case, g, 0.5), _activation(case, g)
        st["z"] = _activation(case, g) if case["z"] else None
        # A after some training: the S4D-real start -(n + 1), moved by a tenth of its logarithm
        st["A"] = -torch.exp(torch.log(torch.arange(1, n + 1, device=DEV, dtype=torch.float32)) + 0.1 * _randn(g, d, n))
        st["B"], st["C"] = _randn(g, b, n, length).to(dt), _randn(g, b, n, length).to(dt)
        st["D"] = 1 + 0.1 * _randn(g, d) if case["D"] else None
        if case["bias"]:  # softplus(bias) log-uniform over 1e-3 .. 1e-1, the model's own start
            step = torch.exp(torch.rand(d, generator=g, device=DEV) * math.log(100.0) + math.log(1e-3))
            st["bias"] = step + torch.log(-torch.expm1(-step))
        else:
            st["bias"] = None
        st["dstate"] = _randn(g, b, d, n) if case["state"] else None
        leaves = ("u", "delta", "A", "B", "C", "D", "z", "bias")
    elif case["op"] == "conv":
        d = case["dim"]
        st["x"], st["dout"] = _activation(case, g), _activation(case, g)
        st["weight"] = torch.rand(d, 1, 4, generator=g, device=DEV) - 0.5
        st["bias"] = 0.2 * torch.rand(d, generator=g, device=DEV) - 0.1 if case["bias"] else None
        leaves = ("x", "weight", "bias")
    elif case["op"] == "checkpoint":
        # rows of different sizes, as channels have
        size = torch.exp(_randn(g, case["rows"], 1))
        st["x"] = (_randn(g, case["rows"], case["cols"]) * size).to(dt)
        leaves = ()
    else:
        rows, length, vocab = 2 * case["pairs"], case["length"], case["vocab"]
        st["logits"] = torch.empty(rows, length, vocab, device=DEV, dtype=dt)
        for r in range(rows):
            st["logits"][r] = 2 * _randn(g, length, vocab)
        st["labels"] = torch.randint(0, vocab, (rows, length), generator=g, device=DEV)
        for r, p in enumerate(_prompt_lengths(case)):
            st["labels"][r, :p] = IGNORE
        # the reference model's sums: near what these logits give
        answers = (st["labels"] != IGNORE).sum(1)
        st["ref"] = -answers * (math.log(vocab) + 2.0) + 2 * _randn(g, rows)
        leaves = ("logits",)
    if own:
        for k in leaves:
            if st[k] is not None:
                st[k].requires_grad_(True)
    return st


# ---- the framework's calls -----------------------------------------------------------------------------


def _run_own(st):
    from mamba_metal_b200 import training

    case = st["case"]
    if case["op"] == "scan":
        names = [k for k in ("u", "delta", "A", "B", "C", "D", "z", "bias") if st[k] is not None]
        y, state = training.selective_scan(st["u"], st["delta"], st["A"], st["B"], st["C"], D=st["D"], z=st["z"],
                                           delta_bias=st["bias"], delta_softplus=case["softplus"], return_state=True)
        outs, seeds = ([y, state], [st["dy"], st["dstate"]]) if case["state"] else ([y], [st["dy"]])
        grads = torch.autograd.grad(outs, [st[k] for k in names], seeds)
        return {"y": y, "state": state, **{"d" + k: v for k, v in zip(names, grads)}}
    if case["op"] == "conv":
        names = [k for k in ("x", "weight", "bias") if st[k] is not None]
        out = training.causal_conv1d(st["x"], st["weight"], st["bias"], silu=case["silu"], checkpoint8=True)
        grads = torch.autograd.grad(out, [st[k] for k in names], st["dout"])
        return {"out": out, **{"d" + k: v for k, v in zip(names, grads)}}
    if case["op"] == "checkpoint":
        c = training.checkpoint8(st["x"])
        return {"values": c.restore(), "exponents": c.exponents}
    loss, chosen, rejected = training.preference_loss(st["logits"], st["labels"], st["ref"], beta=case["beta"],
                                                      label_smoothing=case["smoothing"])
    (dlogits,) = torch.autograd.grad(loss, st["logits"])
    return {"loss": loss, "chosen": chosen, "rejected": rejected, "dlogits": dlogits}


# ---- the plain forms -------------------------------------------------------------------------------------


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _linear_recurrence(a, b, reverse=False):
    """v_t = a_t v_{t-1} + b_t from zero over (steps, chunks, ...) with time = chunk * steps + step; backwards in
    time with ``reverse``. Within the chunks step by step, then from chunk to chunk. Writes over ``b``."""
    steps, chunks = a.shape[:2]
    order = list(range(steps))[::-1] if reverse else list(range(steps))
    decay = a.clone()  # product of a from the chunk's first step up to this one
    for before, now in zip(order, order[1:]):
        b[now] += a[now] * b[before]
        decay[now] *= decay[before]
    carry = torch.zeros_like(b[0, 0])
    for c in range(chunks - 1, -1, -1) if reverse else range(chunks):
        b[:, c] += decay[:, c] * carry
        carry = b[order[-1], c]
    return b


def _plain_scan(st):
    case = st["case"]
    b, d, n, length = case["batch"], case["dim"], case["dstate"], case["length"]
    steps = math.isqrt(length - 1) + 1
    chunks = -(-length // steps)

    def lay(t):  # (batch, channels, length) -> float32 (steps, chunks, batch, channels), zeros after the end
        p = torch.zeros(chunks * steps, b, t.shape[1], device=DEV, dtype=torch.float32)
        p[:length] = t.float().permute(2, 0, 1)
        return p.view(chunks, steps, b, -1).transpose(0, 1).contiguous()

    def back(t):  # and back to (batch, channels, length)
        return t.transpose(0, 1).reshape(chunks * steps, b, -1)[:length].permute(1, 2, 0)

    u, dy, A, Bm, Cm = lay(st["u"]), lay(st["dy"]), st["A"].float(), lay(st["B"]), lay(st["C"])
    raw = lay(st["delta"])
    if st["bias"] is not None:
        raw = raw + st["bias"].float()
    dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(torch.clamp(raw, max=20.0)))) if case["softplus"] else raw
    inside = torch.zeros(chunks * steps, device=DEV)
    inside[:length] = 1
    dt = dt * inside.view(chunks, steps).t()[:, :, None, None]  # nothing moves after the end
    a = torch.exp(dt[..., None] * A)
    h = _linear_recurrence(a, (dt * u)[..., None] * Bm[..., None, :])
    out = (h * Cm[..., None, :]).sum(-1)
    if st["D"] is not None:
        out = out + st["D"].float() * u
    state = h[-1, -1].clone()
    if st["z"] is not None:
        z = lay(st["z"])
        s = _sigmoid(z)
        y, dz, dyg = out * (z * s), dy * out * s * (1 + z * (1 - s)), dy * (z * s)
    else:
        y, dz, dyg = out, None, dy
    dC = (h * dyg[..., None]).sum(-2)
    later = torch.empty_like(a)  # the decay of the step that follows each one
    later[:-1] = a[1:]
    later[-1, :-1] = a[0, 1:]
    later[-1, -1] = 0
    seed = Cm[..., None, :] * dyg[..., None]
    if st["dstate"] is not None:
        seed[-1, -1] += st["dstate"]
    g = _linear_recurrence(later, seed, reverse=True)
    del later, seed
    dB = (g * (dt * u)[..., None]).sum(-2)
    gB = (g * Bm[..., None, :]).sum(-1)
    moved = (h - (dt * u)[..., None] * Bm[..., None, :]) * g  # a_t h_{t-1} g_t
    dA = (moved * dt[..., None]).sum((0, 1, 2))
    ddelta = u * gB + (moved * A).sum(-1)
    if case["softplus"]:
        ddelta = torch.where(raw > 20, ddelta, ddelta * _sigmoid(raw))
    ddelta = ddelta * inside.view(chunks, steps).t()[:, :, None, None]
    du = dt * gB
    if st["D"] is not None:
        du = du + st["D"].float() * dyg
    dt_ = DTYPES[case["dtype"]]
    r = {"y": back(y).to(dt_), "state": state, "du": back(du).to(dt_), "ddelta": back(ddelta).to(dt_), "dA": dA,
         "dB": back(dB).to(dt_), "dC": back(dC).to(dt_)}
    if st["D"] is not None:
        r["dD"] = (dyg * u).sum((0, 1, 2))
    if st["z"] is not None:
        r["dz"] = back(dz).to(dt_)
    if st["bias"] is not None:
        r["dbias"] = ddelta.sum((0, 1, 2))
    return r


def _plain_checkpoint(x):
    """(values as float32, stored exponents): blocks of BLOCK values of the last axis share the smallest power of
    two of which 127 reach their largest magnitude; values are whole multiples of it, ties to even."""
    cols = x.shape[-1]
    blocks = -(-cols // BLOCK)
    p = torch.zeros(*x.shape[:-1], blocks * BLOCK, device=x.device, dtype=torch.float32)
    p[..., :cols] = x.float()
    p = p.view(*x.shape[:-1], blocks, BLOCK)
    top = p.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e with m in [1/2, 1)
    e = torch.where(m <= 127 / 128, e - 7, e - 6)
    e = torch.where(top > 0, e, -126).clamp(min=-126)
    unit = lambda k: ((k + 127) << 23).to(torch.int32).view(torch.float32)  # 2^k, exactly
    values = torch.round(p * unit(-e)) * unit(e)
    return values.view(*x.shape[:-1], -1)[..., :cols], (e[..., 0] + 127).to(torch.uint8)


def _plain_conv(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    length = case["length"]
    w = st["weight"].float().view(-1, 4, 1)

    def before(x):
        v = torch.zeros_like(x) + (0 if st["bias"] is None else st["bias"].float()[:, None])
        for k in range(4):
            lag = 3 - k
            if lag < length:
                v[..., lag:] += w[:, k] * x[..., :length - lag]
        return v

    pre = before(st["x"].float())
    out = pre * _sigmoid(pre) if case["silu"] else pre
    x = _plain_checkpoint(st["x"])[0]  # the backward pass has the checkpoint
    pre = before(x)
    dpre = st["dout"].float()
    if case["silu"]:
        s = _sigmoid(pre)
        dpre = dpre * s * (1 + pre * (1 - s))
    dx, dw = torch.zeros_like(x), torch.zeros(case["dim"], 1, 4, device=DEV)
    for k in range(4):
        lag = 3 - k
        if lag < length:
            dx[..., :length - lag] += w[:, k] * dpre[..., lag:]
            dw[:, 0, k] = (dpre[..., lag:] * x[..., :length - lag]).sum((0, 2))
    r = {"out": out.to(dt), "dx": dx.to(dt), "dweight": dw}
    if st["bias"] is not None:
        r["dbias"] = dpre.sum((0, 2))
    return r


def _plain_preference(st):
    case, pairs = st["case"], st["case"]["pairs"]
    beta, eps = case["beta"], case["smoothing"]
    labels = st["labels"]
    answer = labels != IGNORE
    at = torch.where(answer, labels, 0)[..., None]
    x = st["logits"].float()
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    logp = (x.gather(-1, at) - torch.log(total))[..., 0]
    gain = torch.where(answer, logp, 0).sum(1) - st["ref"]
    chosen, rejected = beta * gain[:pairs], beta * gain[pairs:]
    m = chosen - rejected
    softplus = lambda v: torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))
    loss = ((1 - eps) * softplus(-m) + eps * softplus(m)).mean()
    dm = (eps * _sigmoid(m) - (1 - eps) * _sigmoid(-m)) * (beta / pairs)
    row = torch.where(answer, torch.cat([dm, -dm])[:, None], 0)[..., None]
    e *= -row / total
    e.scatter_add_(-1, at, row)
    return {"loss": loss, "chosen": chosen, "rejected": rejected, "dlogits": e.to(DTYPES[case["dtype"]])}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "scan":
        return _plain_scan(state)
    if op == "conv":
        return _plain_conv(state)
    if op == "checkpoint":
        values, exponents = _plain_checkpoint(state["x"])
        return {"values": values.to(DTYPES[state["case"]["dtype"]]), "exponents": exponents}
    return _plain_preference(state)


# ---- what a pass cannot do without --------------------------------------------------------------------


def work(case):
    s = SIZE[case["dtype"]]
    if case["op"] == "scan":
        b, d, n, length = case["batch"], case["dim"], case["dstate"], case["length"]
        el, bc = b * d * length, b * n * length
        # read u, delta, dy (z), B, C; write y, du, ddelta (dz), dB, dC; A and dA, states
        nbytes = s * (el * (8 if case["z"] else 6) + 4 * bc) + 4 * d * n * 2 + 4 * b * d * n * (2 if case["state"] else 1)
        # each state and step: decay 2, input 1, h 2, y 2; gradient's recurrence 3, dC 2, dB 2, g B 2, a h g 2,
        # dA 2, ddelta 2; and about 30 for each element outside the states
        return {"bytes": nbytes, "flops": el * (22 * n + 30)}
    if case["op"] == "conv":
        el = case["batch"] * case["dim"] * case["length"]
        # read x and dout, write out and dx; the checkpoint (8 bits and a scale in 32) written and read
        return {"bytes": el * (4 * s + 2 * (1 + 1 / BLOCK)), "flops": el * 50}
    if case["op"] == "checkpoint":
        el = case["rows"] * case["cols"]
        return {"bytes": el * (2 * s + 2 * (1 + 1 / BLOCK)), "flops": el * 6}
    tokens = sum(case["length"] - p for p in _prompt_lengths(case))
    every = 2 * case["pairs"] * case["length"]
    # read the answers' logits once, write the gradient of all
    return {"bytes": s * case["vocab"] * (tokens + every) + 8 * every, "flops": 8 * tokens * case["vocab"]}


# ---- 64 bits ---------------------------------------------------------------------------------------------


def _exact_scan(st):
    case = st["case"]
    b, d, n, length = case["batch"], case["dim"], case["dstate"], case["length"]
    f = lambda k: None if st[k] is None else st[k].detach().double()
    u, raw, dy, z, A, Bm, Cm, D = (f(k) for k in ("u", "delta", "dy", "z", "A", "B", "C", "D"))
    if st["bias"] is not None:
        raw = raw + f("bias")[:, None]
    dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(torch.clamp(raw, max=20.0)))) if case["softplus"] else raw
    gate = z * torch.sigmoid(z) if z is not None else torch.ones_like(u)
    time_major = lambda t: t.permute(2, 0, 1).contiguous()
    uT, dtT, BT, CT, eT = (time_major(t) for t in (u, dt, Bm, Cm, dy * gate))
    hs = torch.empty(length, b, d, n, device=DEV, dtype=torch.float64)
    out = torch.empty(length, b, d, device=DEV, dtype=torch.float64)
    h = torch.zeros(b, d, n, device=DEV, dtype=torch.float64)
    for t in range(length):
        h = torch.exp(dtT[t, :, :, None] * A) * h + (dtT[t] * uT[t])[:, :, None] * BT[t, :, None, :]
        hs[t] = h
        out[t] = torch.matmul(h, CT[t, :, :, None])[..., 0]
    du, ddt = torch.empty_like(uT), torch.empty_like(uT)
    dB, dC = torch.empty_like(BT), torch.empty_like(CT)
    dA = torch.zeros(d, n, device=DEV, dtype=torch.float64)
    g = f("dstate") if st["dstate"] is not None else torch.zeros_like(h)  # what later steps want of h_t
    for t in range(length - 1, -1, -1):
        g = g + eT[t, :, :, None] * CT[t, :, None, :]
        dC[t] = torch.matmul(eT[t][:, None, :], hs[t])[:, 0]
        dB[t] = torch.matmul((dtT[t] * uT[t])[:, None, :], g)[:, 0]
        gB = torch.matmul(g, BT[t, :, :, None])[..., 0]
        g = g * torch.exp(dtT[t, :, :, None] * A)
        du[t], ddt[t] = dtT[t] * gB, uT[t] * gB
        if t:
            w = g * hs[t - 1]
            ddt[t] += (w * A).sum(-1)
            dA += (w * dtT[t][:, :, None]).sum(0)
    channel = lambda t: t.permute(1, 2, 0)
    out, du, ddt, dB, dC = (channel(t) for t in (out, du, ddt, dB, dC))
    if D is not None:
        out, du = out + D[:, None] * u, du + D[:, None] * dy * gate
    if case["softplus"]:
        ddt = torch.where(raw > 20, ddt, ddt * torch.sigmoid(raw))
    r = {"y": out * gate, "state": h, "du": du, "ddelta": ddt, "dA": dA, "dB": dB, "dC": dC}
    if D is not None:
        r["dD"] = (dy * gate * u).sum((0, 2))
    if z is not None:
        s = torch.sigmoid(z)
        r["dz"] = dy * out * (s + z * s * (1 - s))
    if st["bias"] is not None:
        r["dbias"] = ddt.sum((0, 2))
    return r


def _exact_checkpoint(x):
    x = x.detach().double()
    pad = -x.shape[-1] % BLOCK
    p = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, BLOCK))
    top = p.abs().amax(-1)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 127)).to(torch.int64)
    unit = lambda k: ((k + 1023) << 52).view(torch.float64)  # 2^k by its bits: a power that is off moves ties
    e = torch.where(127 * unit(e - 1) >= top, e - 1, e)  # where the logarithm's rounding went one too far
    e = torch.where(127 * unit(e) < top, e + 1, e)
    e = torch.where(top > 0, e, -126).clamp(min=-126)
    values = (torch.round(p / unit(e)[..., None]) * unit(e)[..., None]).flatten(-2)
    return values[..., :x.shape[-1]], (e + 127).to(torch.uint8)


def _exact_conv(st):
    case, length = st["case"], st["case"]["length"]
    w = st["weight"].detach().double()[:, 0]

    def taps(x):  # (batch, dim, length, 4): what each tap sees
        return torch.nn.functional.pad(x, (3, 0)).unfold(-1, length, 1).transpose(-1, -2)

    def before(x):
        v = sum(taps(x)[..., k] * w[:, k, None] for k in range(4))
        return v if st["bias"] is None else v + st["bias"].detach().double()[:, None]

    pre = before(st["x"].detach().double())
    out = pre * torch.sigmoid(pre) if case["silu"] else pre
    x = _exact_checkpoint(st["x"])[0]
    pre, dpre = before(x), st["dout"].double()
    if case["silu"]:
        s = torch.sigmoid(pre)
        dpre = dpre * (s + pre * s * (1 - s))
    ahead = torch.nn.functional.pad(dpre, (0, 3))
    dx = sum(ahead[..., 3 - k:3 - k + length] * w[:, k, None] for k in range(4))
    dw = torch.stack([(taps(x)[..., k] * dpre).sum((0, 2)) for k in range(4)], -1)[:, None]
    r = {"out": out, "dx": dx, "dweight": dw}
    if st["bias"] is not None:
        r["dbias"] = dpre.sum((0, 2))
    return r


def _exact_preference(st):
    case, pairs = st["case"], st["case"]["pairs"]
    beta, eps, labels = case["beta"], case["smoothing"], st["labels"]
    rows, length = labels.shape
    gain = torch.zeros(rows, device=DEV, dtype=torch.float64)
    lse = torch.empty(rows, length, device=DEV, dtype=torch.float64)
    for r in range(rows):
        x = st["logits"][r].detach().double()
        lse[r] = torch.logsumexp(x, -1)
        keep = (labels[r] != IGNORE).nonzero()[:, 0]
        gain[r] = (x[keep, labels[r, keep]] - lse[r, keep]).sum() - st["ref"][r].double()
    chosen, rejected = beta * gain[:pairs], beta * gain[pairs:]
    m = chosen - rejected
    loss = -((1 - eps) * torch.nn.functional.logsigmoid(m) + eps * torch.nn.functional.logsigmoid(-m)).mean()
    dm = (eps * torch.sigmoid(m) - (1 - eps) * torch.sigmoid(-m)) * beta / pairs
    dlogits = torch.zeros(rows, length, case["vocab"], device=DEV, dtype=torch.float64)
    for r in range(rows):
        c = dm[r] if r < pairs else -dm[r - pairs]
        keep = (labels[r] != IGNORE).nonzero()[:, 0]
        dlogits[r, keep] = -c * torch.exp(st["logits"][r, keep].detach().double() - lse[r, keep, None])
        dlogits[r, keep, labels[r, keep]] += c
    return {"loss": loss, "chosen": chosen, "rejected": rejected, "dlogits": dlogits}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "scan":
        return _exact_scan(st)
    if case["op"] == "conv":
        return _exact_conv(st)
    if case["op"] == "checkpoint":
        values, exponents = _exact_checkpoint(st["x"])
        return {"values": values, "exponents": exponents}
    return _exact_preference(st)
