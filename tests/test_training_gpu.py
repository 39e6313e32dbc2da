"""Training operators (GPU): gradients of the selective scan and the causal conv1d, 8-bit checkpoints, preference
loss, against plain float64 restatements differentiated by torch, and against differences.

Tolerances are those of tests/helpers.py: one relative factor per element type, above the rounding of the result
to that type (2^-12 for float16, 2^-9 for bfloat16) and above float32 arithmetic over the lengths tested
(a few hundred rounding errors of 2^-24), with the same factor of the reference's RMS as the floor."""

import math

import numpy as np
import pytest
import torch

from mamba_metal_b200 import causal_conv1d, selective_scan, training
from tests.helpers import RTOL, assert_close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LAYOUTS = ["channel_first", "channels_last", "strided"]


def name(dt):
    return str(dt).split(".")[-1]


def randn(g, *shape):
    return torch.randn(shape, generator=g, dtype=torch.float64)


def put(t, dtype, layout="channel_first"):
    """A float64 CPU tensor (b, d, n) on the GPU in ``dtype`` and ``layout``, and its rounded float64 values."""
    x = t.to(dtype).to(DEV)
    if layout == "channels_last":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "strided":  # every other step of every other channel of a larger buffer
        big = torch.full((t.shape[0], 2 * t.shape[1] + 1, 2 * t.shape[2] + 3), float("nan"), dtype=dtype, device=DEV)
        big[:, 1::2, 1:-2:2] = x
        x = big[:, 1::2, 1:-2:2]
    return x, x.double().cpu()


def scan_ref(u, delta, A, B, C, D, z, bias, softplus):
    """The definition, step by step; whatever dtype it is given."""
    raw = delta if bias is None else delta + bias[:, None]
    dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20)))) if softplus else raw
    h = torch.zeros(u.shape[0], u.shape[1], A.shape[1], dtype=u.dtype)
    ys = []
    for t in range(u.shape[2]):
        h = torch.exp(dt[:, :, t, None] * A) * h + (dt * u)[:, :, t, None] * B[:, None, :, t]
        ys.append((h * C[:, None, :, t]).sum(-1))
    y = torch.stack(ys, -1)
    if D is not None:
        y = y + D[:, None] * u
    if z is not None:
        y = y * z * torch.sigmoid(z)
    return y, h


def scan_inputs(shape, dtype, layout, opts, seed=0):
    b, d, n, length = shape
    g = torch.Generator().manual_seed(seed)
    out = {}
    for k in ("u", "delta", "z"):
        out[k] = put(randn(g, b, d, length) * (0.5 if k == "delta" else 1), dtype, layout)
    for k in ("B", "C"):
        out[k] = put(randn(g, b, n, length), dtype, layout)
    f32 = lambda t: put(t, torch.float32)
    out["A"] = f32(-torch.exp(torch.log(torch.arange(1, n + 1, dtype=torch.float64)) + 0.1 * randn(g, d, n)))
    out["D"], out["bias"] = f32(1 + 0.1 * randn(g, d)), f32(randn(g, d) - 2)
    if "delta" not in opts and "softplus" not in opts:  # steps as they are: positive
        out["delta"] = put(randn(g, b, d, length).abs() * 0.3, dtype, layout)
    for k in ("D", "z", "bias"):
        if k not in opts:
            out[k] = (None, None)
    dy, dstate = put(randn(g, b, d, length), dtype), f32(randn(g, b, d, n))
    return {k: v[0] for k, v in out.items()}, {k: v[1] for k, v in out.items()}, dy, dstate


NAMES = ("u", "delta", "A", "B", "C", "D", "z", "bias")


def run_scan(gpu, dy, dstate, opts):
    leaves = {k: gpu[k].detach().requires_grad_(True) for k in NAMES if gpu[k] is not None}
    y, state = training.selective_scan(leaves["u"], leaves["delta"], leaves["A"], leaves["B"], leaves["C"],
                                       D=leaves.get("D"), z=leaves.get("z"), delta_bias=leaves.get("bias"),
                                       delta_softplus="softplus" in opts, return_state=True)
    outs, seeds = ([y, state], [dy, dstate]) if "state" in opts else ([y], [dy])
    return y, state, dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), seeds)))


def check_scan(shape, dtype, layout, opts, seed=0):
    gpu, cpu, dy, dstate = scan_inputs(shape, dtype, layout, opts, seed)
    y, state, grads = run_scan(gpu, dy[0], dstate[0], opts)
    leaves = {k: cpu[k].requires_grad_(True) for k in NAMES if cpu[k] is not None}
    yr, hr = scan_ref(*(leaves.get(k) for k in NAMES), "softplus" in opts)
    loss = (yr * dy[1]).sum() + ((hr * dstate[1]).sum() if "state" in opts else 0)
    ref = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
    what = f"{shape} {name(dtype)} {layout} {sorted(opts)}"
    assert_close(y, yr.detach(), RTOL[name(dtype)], f"y {what}")
    assert_close(state, hr.detach(), RTOL["float32"], f"state {what}")
    for k, g in grads.items():
        assert g.dtype == gpu[k].dtype and g.shape == gpu[k].shape
        assert_close(g, ref[k], RTOL[name(g.dtype)], f"d{k} {what}")


ALL = frozenset(("D", "z", "bias", "softplus", "state"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (2, 5, 3, 2), (1, 64, 16, 64), (2, 17, 16, 65), (1, 70, 8, 200),
                                   (2, 33, 24, 130), (1, 20, 64, 193), (1, 136, 16, 1000)])
def test_scan_gradient(shape, layout, dtype):
    check_scan(shape, dtype, layout, ALL)


@pytest.mark.parametrize("opts", [(), ("z",), ("D",), ("softplus",), ("softplus", "bias"), ("state",),
                                  ("D", "z", "softplus"), ("bias", "softplus", "state")])
@pytest.mark.parametrize("shape", [(2, 19, 16, 50), (1, 19, 20, 150)])
def test_scan_gradient_options(shape, opts):
    check_scan(shape, torch.float32, "channel_first", frozenset(opts), seed=3)


def test_scan_gradient_many_tiles():
    """Sizes at which a block works off several tiles of channels and the groups end inside one."""
    check_scan((8, 1000, 4, 330), torch.float32, "channel_first", ALL, seed=5)


# (batch, channels, states, steps) at which the cut walks join long chunks of two or four chunks, the last one ragged, and a
# block of the gradient works off several tiles, copied ahead where rows lie on 16 bytes. test_training_cpu.py holds
# them to that.
LARGE = [(4, 2000, 2, 936), (4, 2000, 16, 456), (4, 2000, 20, 936), (8, 1536, 16, 1192), (4, 2001, 3, 937), (8, 1021, 5, 1001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["channel_first", "channels_last"])
@pytest.mark.parametrize("shape", LARGE)
def test_scan_gradient_large(shape, layout, dtype):
    """Sizes that training runs at, against the float64 definition on the GPU."""
    gpu, cpu, dy, dstate = scan_inputs(shape, dtype, layout, ALL, seed=17)
    y, state, grads = run_scan(gpu, dy[0], dstate[0], ALL)
    with torch.device(DEV):
        leaves = {k: cpu[k].to(DEV).requires_grad_(True) for k in NAMES}
        yr, hr = scan_ref(*(leaves[k] for k in NAMES), True)
        ref = torch.autograd.grad((yr * dy[1].to(DEV)).sum() + (hr * dstate[1].to(DEV)).sum(), list(leaves.values()))
    assert_close(y, yr, RTOL[name(dtype)], "y")
    assert_close(state, hr, RTOL["float32"], "state")
    for k, r in zip(leaves, ref):
        assert_close(grads[k], r, RTOL[name(grads[k].dtype)], f"d{k}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shape", [(2, 9, 16, 256), (2, 9, 16, 257), (1, 33, 7, 255), (1, 8191, 2, 263), (1, 8197, 9, 259)])
def test_scan_gradient_where_the_walks_change(shape, layout, dtype):
    """Lengths and channel counts around those from which whole sequences are walked, cut into long chunks or not."""
    check_scan(shape, dtype, layout, ALL, seed=11)


@pytest.mark.parametrize("shape", [(1, 40, 16, 100), (1, 40, 16, 300), (1, 8200, 6, 290)])
def test_scan_states_alone(shape):
    """The states are the same whether or not the outputs are asked for."""
    gpu, _, _, _ = scan_inputs(shape, torch.float16, "channel_first", ALL, 13)
    u, delta, A, B, C, D, z, bias = (gpu[k] for k in NAMES)
    call = lambda outputs: training.selective_scan_states(u, delta, A, B, C, D=D, z=z, delta_bias=bias, delta_softplus=True,
                                                          outputs=outputs)
    y, state, states = call(True)
    none, nothing, alone = call(False)
    assert none is None and nothing is None and torch.equal(states, alone)


def test_scan_gradient_softplus_cutoff():
    """Steps on both sides of the cutoff at 20, and steps whose decay leaves nothing of the state."""
    shape, opts = (1, 6, 4, 70), frozenset(("softplus",))
    gpu, cpu, dy, dstate = scan_inputs(shape, torch.float32, "channel_first", opts)
    raw = torch.linspace(-40, 60, 6 * 70, dtype=torch.float64).reshape(1, 6, 70)[:, :, torch.randperm(70)]
    gpu["delta"], cpu["delta"] = put(raw, torch.float32)
    _, _, grads = run_scan(gpu, dy[0], dstate[0], opts)
    leaves = {k: cpu[k].requires_grad_(True) for k in ("u", "delta", "A", "B", "C")}
    y, _ = scan_ref(*(leaves.get(k) for k in NAMES), True)
    ref = dict(zip(leaves, torch.autograd.grad((y * dy[1]).sum(), list(leaves.values()))))
    for k in leaves:
        assert_close(grads[k], ref[k], RTOL["float32"], f"d{k}")


def test_scan_gradient_against_differences():
    """Central differences of the float64 definition along one direction, with all inputs moving: the quotient is off
    by about 1e-8 (step 1e-4 squared), the float32 gradient by RTOL of its terms."""
    opts = ALL
    gpu, cpu, dy, dstate = scan_inputs((2, 9, 5, 77), torch.float32, "channel_first", opts, seed=7)
    _, _, grads = run_scan(gpu, dy[0], dstate[0], opts)
    g = torch.Generator().manual_seed(1)
    way = {k: randn(g, *cpu[k].shape) * cpu[k].abs().mean() for k in NAMES}

    def value(step):
        y, h = scan_ref(*(cpu[k] + step * way[k] for k in NAMES), True)
        return float((y * dy[1]).sum() + (h * dstate[1]).sum())

    quotient = (value(1e-4) - value(-1e-4)) / 2e-4
    terms = {k: grads[k].double().cpu() * way[k] for k in NAMES}
    got = sum(float(t.sum()) for t in terms.values())
    scale = math.sqrt(sum(float((t ** 2).sum()) for t in terms.values()))
    assert abs(got - quotient) < RTOL["float32"] * max(scale, abs(quotient))


def test_scan_values_are_the_inference_scans():
    gpu, _, _, _ = scan_inputs((2, 40, 16, 300), torch.bfloat16, "channel_first", ALL)
    y = training.selective_scan(gpu["u"], gpu["delta"], gpu["A"], gpu["B"], gpu["C"], D=gpu["D"], z=gpu["z"],
                                delta_softplus=True)
    ref = selective_scan(gpu["u"], gpu["delta"], gpu["A"], gpu["B"], gpu["C"], D=gpu["D"], z=gpu["z"], delta_softplus=True)
    assert_close(y, ref.float(), RTOL["bfloat16"], "y")
    assert not ref.requires_grad


def test_scan_mixed_types_broadcast_and_absent_gradients():
    gpu, cpu, dy, _ = scan_inputs((2, 12, 4, 90), torch.float32, "channel_first", frozenset(("softplus",)))
    u = gpu["u"][:1].bfloat16().expand(2, -1, -1).detach().requires_grad_(True)  # one row for both
    y = training.selective_scan(u, gpu["delta"], gpu["A"], gpu["B"], gpu["C"], delta_softplus=True)
    assert y.dtype == torch.bfloat16
    y.sum().backward()  # a gradient of stride 0
    ur = u.detach().double().cpu().requires_grad_(True)
    yr, _ = scan_ref(ur, cpu["delta"], cpu["A"], cpu["B"], cpu["C"], None, None, None, True)
    yr.sum().backward()
    assert_close(u.grad, ur.grad, RTOL["bfloat16"], "du")
    # only the state is used
    leaf = gpu["u"].detach().requires_grad_(True)
    _, state = training.selective_scan(leaf, gpu["delta"], gpu["A"], gpu["B"], gpu["C"], delta_softplus=True,
                                       return_state=True)
    state.sum().backward()
    ur = cpu["u"].detach().requires_grad_(True)
    scan_ref(ur, cpu["delta"], cpu["A"], cpu["B"], cpu["C"], None, None, None, True)[1].sum().backward()
    assert_close(leaf.grad, ur.grad, RTOL["float32"], "du from the state")


def test_scan_gradient_repeats_and_other_streams():
    gpu, _, dy, dstate = scan_inputs((2, 100, 16, 700), torch.float16, "channels_last", ALL)
    first = run_scan(gpu, dy[0], dstate[0], ALL)[2]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run_scan(gpu, dy[0], dstate[0], ALL)[2]
    torch.cuda.current_stream().wait_stream(side)
    for k in first:
        assert torch.equal(first[k], second[k]), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first", [0, 1, 2, 3, 5, 7])
def test_rows_at_any_alignment(first, dtype):
    """Views whose rows begin at every place inside an aligned word, with the neighbours of the views left alone."""
    b, d, n = 2, 5, 301
    g = torch.Generator().manual_seed(first)
    big = randn(g, b, d, n + 16).to(dtype).to(DEV)
    x = big[..., first:first + n]
    c = training.checkpoint8(x)
    values, exponents = checkpoint_ref(x.double().cpu())
    assert np.array_equal(c.exponents.cpu().numpy(), exponents)
    out = torch.full((b, d, n + 16), 7.0, dtype=dtype, device=DEV)
    view = out[..., first:first + n]
    a = training._checkpoint_args(view, c.codes, c.exponents)
    training._run("mm_checkpoint8_unpack", view.device, a)
    assert np.array_equal(view.double().cpu().numpy(), values)
    assert (out[..., :first] == 7).all() and (out[..., first + n:] == 7).all()
    w = torch.randn(d, 4, device=DEV)
    whole = x.contiguous()
    y, held = training.conv1d_checkpoint8(x, w, None)
    z, same = training.conv1d_checkpoint8(whole, w, None)
    assert torch.equal(y, z) and torch.equal(held.codes, same.codes)
    for p, q in zip(training.causal_conv1d_backward(x, x, w, None), training.causal_conv1d_backward(whole, whole, w, None)):
        assert torch.equal(p, q)
    A = -torch.rand(d, 4, device=DEV)
    B = torch.randn(b, 4, n, device=DEV, dtype=dtype)
    left = training.selective_scan_backward(x, x, x, A, B, B, z=x, delta_softplus=True)
    right = training.selective_scan_backward(whole, whole, whole, A, B, B, z=whole, delta_softplus=True)
    for k in ("u", "delta", "A", "B", "C", "z"):
        assert torch.equal(left[k], right[k]), k


def test_empty_sequences():
    u = torch.empty(2, 3, 0, device=DEV, requires_grad=True)
    A = torch.full((3, 4), -1.0, device=DEV, requires_grad=True)
    B = torch.empty(2, 4, 0, device=DEV)
    y, state = training.selective_scan(u, u, A, B, B, return_state=True)
    assert y.shape == u.shape and not state.any()
    (y.sum() + state.sum()).backward()
    assert not A.grad.any()
    w = torch.ones(3, 4, device=DEV, requires_grad=True)
    for held in (False, True):
        w.grad = None
        training.causal_conv1d(u, w, checkpoint8=held).sum().backward()
        assert not w.grad.any()
    assert training.checkpoint8(torch.empty(3, 0, device=DEV)).restore().shape == (3, 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,length", [(4, 40), (24, 33), (16, 1)])
def test_no_channels(n, length, dtype, monkeypatch):
    """Gradients of B and C are sums over no channels: zeros, whatever their memory held."""
    empty = torch.empty
    monkeypatch.setattr(training.torch, "empty", lambda *a, **k: empty(*a, **k).fill_(7))
    u, A = empty(2, 0, length, device=DEV, dtype=dtype), empty(0, n, device=DEV)
    B = torch.ones(2, n, length, device=DEV, dtype=dtype)
    for z in (None, u):
        g = training.selective_scan_backward(u, u, u, A, B, B, z=z, delta_softplus=True)
        assert g["B"].shape == g["C"].shape == B.shape and not g["B"].any() and not g["C"].any()
        assert g["u"].shape == u.shape and g["A"].shape == A.shape
    y, state = training.selective_scan(u, u, A, B, B, return_state=True)
    assert y.shape == u.shape and state.shape == (2, 0, n)


# ---- checkpoints -------------------------------------------------------------------------------------------


def checkpoint_ref(x):
    """(values, exponent bytes) of float64 ``x`` (..., n), by the definition."""
    x = np.asarray(x, dtype=np.float64)
    n = x.shape[-1]
    blocks = -(-n // 32)
    p = np.zeros(x.shape[:-1] + (blocks * 32,))
    p[..., :n] = x
    p = p.reshape(x.shape[:-1] + (blocks, 32))
    top = np.abs(p).max(-1)
    e = np.full(top.shape, -126)
    while True:
        low = 127 * np.ldexp(1.0, e) < top
        if not low.any():
            break
        e[low] += 1
    v = np.ldexp(np.rint(np.ldexp(p, -e[..., None])), e[..., None])
    return v.reshape(x.shape[:-1] + (-1,))[..., :n], e + 127


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 31), (1, 5, 32), (2, 7, 33), (1, 40, 256), (3, 6, 1000), (2, 3, 2309),
                                   (1, 9, 1025)])
def test_checkpoint(shape, layout, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x, ref = put(randn(g, *shape) * torch.exp(3 * randn(g, shape[0], shape[1], 1)), dtype, layout)
    c = training.checkpoint8(x)
    values, exponents = checkpoint_ref(ref)
    assert np.array_equal(c.exponents.cpu().numpy(), exponents)
    assert np.array_equal(c.restore().double().cpu().numpy(), values)
    assert np.array_equal(c.restore(torch.float32).double().cpu().numpy(), values)
    assert c.restore().dtype == dtype and c.shape == x.shape and c.nbytes < 1.1 * x.numel() + 32 * x.shape[0] * x.shape[1]
    step = np.repeat(np.ldexp(1.0, exponents - 127), 32, -1)[..., :shape[2]]
    assert (np.abs(values - ref.numpy()) <= step / 2).all()


@pytest.mark.parametrize("shape", [(70,), (3, 70), (2, 2, 3, 70)])
def test_checkpoint_axes(shape):
    x = torch.randn(shape, device=DEV)
    c = training.checkpoint8(x)
    assert c.codes.shape == x.shape and c.exponents.shape == (*shape[:-1], 3)
    assert np.array_equal(c.restore().double().cpu().numpy(), checkpoint_ref(x.cpu())[0])


def test_checkpoint_extremes():
    tiny, big = 2.0 ** -149, float(torch.finfo(torch.float32).max)
    rows = [0.0, tiny, 2.0 ** -120, 1.0, 126.5, 127.0, 127.5, 254.0, 255.0, big / 2, big]
    x = torch.zeros(len(rows), 64)
    for i, v in enumerate(rows):
        x[i, :32] = v * torch.linspace(-1, 1, 32)
        x[i, 40] = v
    c = training.checkpoint8(x.to(DEV))
    values, exponents = checkpoint_ref(x)
    assert np.array_equal(c.exponents.cpu().numpy(), exponents)
    got = c.restore().double().cpu().numpy()
    assert np.array_equal(got, np.clip(values, -big, big))
    half = torch.full((1, 32), 65504.0, device=DEV, dtype=torch.float16)
    assert torch.equal(training.checkpoint8(half).restore(), half)
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = torch.ones(2, 70)
        x[0, 33] = bad
        c = training.checkpoint8(x.to(DEV))
        assert c.exponents.tolist() == [[121, 255, 121], [121, 121, 121]]
        got = c.restore().cpu()
        assert got[0, 32:64].isnan().all() and torch.equal(got[0, :32], x[0, :32]) and torch.equal(got[1], x[1])


def test_checkpoint_error_bound():
    """Less than 1/127 of a block's largest magnitude, and more than 1/128 where that lies just above 127 steps: its step is
    twice the one before."""
    g = torch.Generator().manual_seed(9)
    top = torch.cat([torch.full((40,), 127 * (1 + 2.0 ** -12)), torch.rand(400, generator=g) + 1, torch.full((40,), 1.99)])
    x = (2 * torch.rand(480, 32, generator=g) - 1) * top[:, None]
    x[:, 0] = top
    x[:40, 1], x[440:, 1] = 0.99999, 0.0156  # just under half a step
    off = (training.checkpoint8(x.to(DEV)).restore().cpu().double() - x.double()).abs().amax(1) / top.double()
    assert (off < 1 / 127).all() and (off[:40] > 1 / 128).all() and (off[440:] > 1 / 128).all()


@pytest.mark.parametrize("packed", DTYPES)
def test_checkpoint_restored_in_other_types(packed):
    """Exact in float32 and bfloat16, rounded to float16, in all of the packed type's range."""
    g = torch.Generator().manual_seed(10)
    top = torch.ldexp(torch.ones(250), torch.arange(-126, 124)) if packed != torch.float16 else torch.ldexp(torch.ones(40), torch.arange(-24, 16))
    x = ((2 * torch.rand(len(top), 32, generator=g) - 1) * top[:, None]).to(packed)
    c = training.checkpoint8(x.to(DEV))
    values = checkpoint_ref(x.double())[0]
    for dtype in (torch.float32, torch.bfloat16):
        assert np.array_equal(c.restore(dtype).double().cpu().numpy(), values)
    half = torch.as_tensor(values).clamp(-65504, 65504).half()
    assert torch.equal(c.restore(torch.float16).cpu(), half)


# ---- conv --------------------------------------------------------------------------------------------------


def conv_ref(x, w, bias, silu):
    pre = torch.nn.functional.conv1d(x, w[:, None, :], bias, padding=3, groups=x.shape[1])[..., :x.shape[2]]
    return pre * torch.sigmoid(pre) if silu else pre


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 2), (1, 5, 4), (2, 8, 33), (1, 66, 256), (2, 7, 259), (1, 24, 1032),
                                   (2, 3, 2309), (1, 9, 1025), (1, 300, 70)])
def test_conv_gradient(shape, layout, dtype, held):
    b, d, n = shape
    silu, with_bias = n != 4, d != 3
    g = torch.Generator().manual_seed(n)
    x, xr = put(randn(g, *shape), dtype, layout)
    dout, dr = put(randn(g, *shape), dtype)
    w = (torch.rand(d, 4, generator=g, dtype=torch.float64) - 0.5).float()
    bias = (0.2 * randn(g, d)).float() if with_bias else None
    leaves = [x.detach().requires_grad_(True), w[:, None].to(DEV).requires_grad_(True)]
    leaves += [bias.to(DEV).requires_grad_(True)] if with_bias else []
    out = training.causal_conv1d(*leaves, silu=silu, checkpoint8=held)
    grads = torch.autograd.grad(out, leaves, dout)
    ref = [w.double().requires_grad_(True)] + ([bias.double().requires_grad_(True)] if with_bias else [])
    outr = conv_ref(xr, ref[0], ref[1] if with_bias else None, silu)
    assert_close(out, outr.detach(), RTOL[name(dtype)], "out")
    at = torch.as_tensor(checkpoint_ref(xr)[0]) if held else xr
    at.requires_grad_(True)
    want = torch.autograd.grad((conv_ref(at, ref[0], ref[1] if with_bias else None, silu) * dr).sum(), [at, *ref])
    assert grads[0].dtype == dtype and grads[1].shape == (d, 1, 4)
    assert_close(grads[0], want[0], RTOL[name(dtype)], "dx")
    for k, (a, r) in enumerate(zip(grads[1:], want[1:])):
        assert_close(a.reshape(r.shape), r, RTOL["float32"], ("dweight", "dbias")[k])


def test_conv_values_and_checkpoint_are_the_separate_operators():
    x = torch.randn(2, 24, 133, device=DEV, dtype=torch.bfloat16)
    w, b = torch.randn(24, 4, device=DEV), torch.randn(24, device=DEV)
    out, c = training.conv1d_checkpoint8(x, w, b)
    assert torch.equal(out, causal_conv1d(x, w, b))
    p = training.checkpoint8(x)
    assert torch.equal(c.codes, p.codes) and torch.equal(c.exponents, p.exponents)
    dout = torch.randn_like(x)
    once, again = (training.causal_conv1d_backward(dout, c, w, b) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(once, again))


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("first", [1, 2, 3])
def test_conv_weights_in_a_flat_buffer(first, layout, held):
    """Weights that begin at any float of a buffer give the bits of weights of their own."""
    g = torch.Generator().manual_seed(first)
    d = 24
    x, dout = put(randn(g, 2, d, 140), torch.bfloat16, layout)[0], put(randn(g, 2, d, 140), torch.bfloat16)[0]
    flat, b = randn(g, 4 * d + 8).float().to(DEV), randn(g, d).float().to(DEV)
    view = flat[first:first + 4 * d].view(d, 1, 4)
    assert view.data_ptr() % 16
    got = []
    for w in (view, view.clone()):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        out = training.causal_conv1d(*leaves, checkpoint8=held)
        got.append([out, *torch.autograd.grad(out, leaves, dout)])
    for p, q in zip(*got):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shape", [(1, 8, 70), (2, 9, 700), (1, 130, 333)])
def test_conv_gradient_at_the_largest_values(shape, layout, dtype):
    """Where a code stands for more than the type's largest value, the gradient is taken at that value, as restored: the
    bits are those of the gradient at the restored tensor."""
    b, d, n = shape
    g = torch.Generator().manual_seed(d)
    x = randn(g, *shape)
    x[:, ::3, ::37] = float(torch.finfo(dtype).max)
    x[:, 1::3, 30::41] = -float(torch.finfo(dtype).max)
    x, dout = put(x, dtype, layout)[0], put(0.01 * randn(g, *shape), dtype)[0]
    c = training.checkpoint8(x)
    at = c.restore()
    assert at.isfinite().all() and at.abs().max() == torch.finfo(dtype).max
    w, bias = (0.2 * randn(g, d, 4)).clamp(-0.2, 0.2).float().to(DEV), randn(g, d).float().to(DEV)
    for silu in (True, False):
        for p, q in zip(training.causal_conv1d_backward(dout, c, w, bias, silu=silu),
                        training.causal_conv1d_backward(dout, at, w, bias, silu=silu)):
            assert p.isfinite().all() and torch.equal(p, q)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("length", [5, 70, 257, 1003])
def test_conv_weights_that_the_last_steps_do_not_reach(length, layout, bad):
    """Without SiLU the first tap's gradient is a sum over values that end three steps before the last: what is no number
    among those three does not enter it, nor dx."""
    g = torch.Generator().manual_seed(length)
    x, dout = put(randn(g, 2, 9, length), torch.float16, layout)[0], put(randn(g, 2, 9, length), torch.float16)[0]
    w = randn(g, 9, 4).float().to(DEV)
    x[..., -3:] = 0
    dx, dw, db = training.causal_conv1d_backward(dout, x, w, None, silu=False)
    x[..., -3:] = bad
    dx2, dw2, db2 = training.causal_conv1d_backward(dout, x, w, None, silu=False)
    assert torch.equal(dx, dx2) and torch.equal(dw[:, 0], dw2[:, 0]) and torch.equal(db, db2)
    assert not dw2[:, 1:].isfinite().any()


def test_conv_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    x, w, b, dout = randn(g, 2, 5, 70), randn(g, 5, 4) / 2, randn(g, 5), randn(g, 2, 5, 70)
    leaves = [t.float().to(DEV).requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(training.causal_conv1d(*leaves), leaves, dout.float().to(DEV))
    way = [randn(g, *t.shape) for t in (x, w, b)]
    value = lambda s: float((conv_ref(*(t + s * v for t, v in zip((x, w, b), way)), True) * dout).sum())
    quotient = (value(1e-4) - value(-1e-4)) / 2e-4
    terms = [a.double().cpu() * v for a, v in zip(grads, way)]
    scale = math.sqrt(sum(float((t ** 2).sum()) for t in terms))
    assert abs(sum(float(t.sum()) for t in terms) - quotient) < RTOL["float32"] * max(scale, abs(quotient))


# ---- preference loss ---------------------------------------------------------------------------------------


def preference_ref(logits, labels, ref, beta, eps, ignore=-100):
    keep = labels != ignore
    logp = torch.log_softmax(logits, -1).gather(-1, torch.where(keep, labels, 0)[..., None])[..., 0]
    gain = beta * (torch.where(keep, logp, 0.0).sum(1) - ref)
    n = logits.shape[0] // 2
    m = gain[:n] - gain[n:]
    ls = torch.nn.functional.logsigmoid
    return (-(1 - eps) * ls(m) - eps * ls(-m)).mean(), gain[:n], gain[n:]


def check_preference(logits, labels, ref, beta=0.3, eps=0.0, scale=None):
    x = logits.detach().requires_grad_(True)
    loss, chosen, rejected = training.preference_loss(x, labels, ref, beta=beta, label_smoothing=eps)
    assert not chosen.requires_grad and loss.dtype == torch.float32
    (dx,) = torch.autograd.grad(loss, x, scale)
    xr = logits.double().cpu().requires_grad_(True)
    lr, cr, rr = preference_ref(xr, labels.cpu(), ref.double().cpu(), beta, eps)
    (dr,) = torch.autograd.grad(lr, xr, None if scale is None else scale.double().cpu())
    for got, want, what in ((loss, lr, "loss"), (chosen, cr, "chosen"), (rejected, rr, "rejected")):
        assert_close(got, want.detach(), RTOL["float32"], what)
    assert dx.dtype == logits.dtype
    assert_close(dx, dr, RTOL[name(logits.dtype)], "dlogits")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs,length,vocab", [(1, 1, 1), (1, 1, 7), (2, 3, 64), (3, 5, 1001), (1, 2, 50277), (4, 90, 513)])
def test_preference(pairs, length, vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    logits = (2 * randn(g, 2 * pairs, length, vocab)).to(dtype).to(DEV)
    labels = torch.randint(0, vocab, (2 * pairs, length), generator=g)
    labels[torch.rand(labels.shape, generator=g) < 0.3] = -100
    labels[0] = -100  # an answer without tokens
    ref = -length * (math.log(vocab) + 1) + randn(g, 2 * pairs).float()
    check_preference(logits, labels.to(DEV), ref.to(DEV), eps=0.1 if pairs > 1 else 0.0,
                     scale=torch.tensor(1.7, device=DEV) if vocab == 64 else None)


def test_preference_all_tokens_ignored_and_no_tokens():
    logits = torch.randn(4, 6, 50, device=DEV, requires_grad=True)
    labels = torch.full((4, 6), -100, device=DEV)
    loss, chosen, rejected = training.preference_loss(logits, labels, torch.zeros(4, device=DEV))
    assert abs(loss.item() - math.log(2)) < 1e-6 and not chosen.any() and not rejected.any()
    loss.backward()
    assert not logits.grad.any()
    none = torch.empty(4, 0, 50, device=DEV, requires_grad=True)
    loss, _, _ = training.preference_loss(none, labels[:, :0], torch.zeros(4, device=DEV))
    loss.backward()
    assert abs(loss.item() - math.log(2)) < 1e-6 and none.grad.shape == (4, 0, 50)


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min])
def test_preference_masked_vocabulary(low):
    """Entries struck out with -inf or the type's lowest value; a token whose entries are all the lowest value; NaN in
    ignored tokens."""
    g = torch.Generator().manual_seed(4)
    logits = randn(g, 2, 4, 300).float()
    logits[:, :, 100:200] = low
    if math.isfinite(low):
        logits[0, 1] = low
    labels = torch.randint(0, 100, (2, 4), generator=g)
    labels[1, 3] = -100
    logits[1, 3] = float("nan")
    x = logits.to(DEV).requires_grad_(True)
    loss, _, _ = training.preference_loss(x, labels.to(DEV), torch.zeros(2, device=DEV))
    (dx,) = torch.autograd.grad(loss, x)
    clean = logits.double()
    clean[1, 3] = 0
    clean.requires_grad_(True)
    lr, _, _ = preference_ref(clean, labels, torch.zeros(2, dtype=torch.float64), 0.1, 0.0)
    (dr,) = torch.autograd.grad(lr, clean)
    assert_close(loss, lr.detach(), RTOL["float32"], "loss")
    assert_close(dx, dr, RTOL["float32"], "dlogits")


def test_preference_strides_and_labels_outside():
    g = torch.Generator().manual_seed(6)
    wide = randn(g, 4, 9, 203).to(torch.bfloat16).to(DEV)
    labels = torch.randint(0, 200, (4, 8), generator=g).to(DEV)
    ref = torch.full((4,), -40.0, device=DEV)
    check_preference(wide[:, :-1, 1:202], labels, ref)        # the usual shift; rows begin anywhere
    check_preference(wide.transpose(0, 1)[:8].transpose(0, 1)[..., :200], labels, ref)
    check_preference(wide[:, 1:, ::2][..., :100].expand(4, 8, 100), labels % 100, ref)
    for bad in (-1, 200, 1 << 40):
        wrong = labels.clone()
        wrong[1, 2] = bad
        loss, chosen, rejected = training.preference_loss(wide[:, :-1, :200], wrong, ref)
        assert loss.isnan() and chosen[1].isnan() and not chosen[0].isnan() and not rejected.isnan().any()


def test_preference_gradient_against_differences():
    g = torch.Generator().manual_seed(8)
    x, labels, ref = randn(g, 4, 5, 40), torch.randint(0, 40, (4, 5), generator=g), randn(g, 4) - 18
    way = randn(g, 4, 5, 40)
    leaf = x.float().to(DEV).requires_grad_(True)
    loss, _, _ = training.preference_loss(leaf, labels.to(DEV), ref.float().to(DEV), beta=0.5, label_smoothing=0.2)
    loss.backward()
    value = lambda s: float(preference_ref(x + s * way, labels, ref, 0.5, 0.2)[0])
    quotient = (value(1e-4) - value(-1e-4)) / 2e-4
    terms = leaf.grad.double().cpu() * way
    assert abs(float(terms.sum()) - quotient) < RTOL["float32"] * max(float(terms.norm()), abs(quotient))
