"""Training pass of the block and the model (GPU): against a float64 restatement differentiated by torch, and the example
that runs all training operators together."""

import importlib.util
from pathlib import Path

import pytest
import torch

from mamba_metal_b200 import MambaBlock, MambaConfig, MambaModel, init_weights_, training
from tests.helpers import RTOL, assert_close, assert_close_lowp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def block_ref(p, x, R, N):
    """MambaBlock in the parameters' dtype, step by step."""
    E = p["D"].shape[0]
    xz = x @ p["in_proj.weight"].T
    xin, z = xz[..., :E].transpose(1, 2), xz[..., E:].transpose(1, 2)
    pre = torch.nn.functional.conv1d(xin, p["conv1d.weight"], p["conv1d.bias"], padding=3, groups=E)[..., :x.shape[1]]
    xc = pre * torch.sigmoid(pre)
    dbl = xc.transpose(1, 2) @ p["x_proj.weight"].T
    dt = torch.nn.functional.softplus(dbl[..., :R] @ p["dt_proj.weight"].T + p["dt_proj.bias"])
    B, C, A = dbl[..., R:R + N], dbl[..., R + N:], -torch.exp(p["A_log"])
    h = torch.zeros(x.shape[0], E, N, dtype=x.dtype)
    ys = []
    for t in range(x.shape[1]):
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * xc[:, :, t])[..., None] * B[:, t, None]
        ys.append((h * C[:, t, None]).sum(-1))
    y = (torch.stack(ys, -1) + p["D"][:, None] * xc) * z * torch.sigmoid(z)
    return y.transpose(1, 2) @ p["out_proj.weight"].T


def make_block(dtype, d_model=40, seed=0):
    cfg = MambaConfig(d_model=d_model, n_layer=1, vocab_size=8)
    model = init_weights_(MambaModel(cfg, dtype=dtype, device=DEV), seed=seed)
    return model.layers[0].mixer


@pytest.mark.parametrize("length", [1, 33, 64, 150])
@pytest.mark.parametrize("held", [False, True])
def test_block_gradient_float32(length, held):
    """Without checkpoints the float32 tolerance holds. With them the gradients are those of slightly other
    activations: each is off by at most half a step, so by 1.4% of a block's values in the RMS (a step of 1/127 to
    1/64 of the largest, values of a third of it), and gradients by that much in L2 or less."""
    block = make_block(torch.float32)
    g = torch.Generator().manual_seed(length)
    x, dy = torch.randn(2, length, 40, generator=g), torch.randn(2, length, 40, generator=g)
    leaf = x.to(DEV).requires_grad_(True)
    out = block.forward_train(leaf, checkpoint8=held)
    names = [n for n, _ in block.named_parameters()]
    grads = torch.autograd.grad(out, [leaf, *block.parameters()], dy.to(DEV))
    ref = {n: p.detach().double().cpu().requires_grad_(True) for n, p in block.named_parameters()}
    xr = x.double().requires_grad_(True)
    outr = block_ref(ref, xr, block.dt_rank, block.d_state)
    want = torch.autograd.grad(outr, [xr, *ref.values()], dy.double())
    assert_close(out, outr.detach(), RTOL["float32"], "out")
    for n, a, r in zip(["x", *names], grads, want):
        assert a.shape == r.shape and a.dtype == torch.float32
        if held:
            assert_close_lowp(a, r, f"d{n}", rel_l2=2.8e-2)
        else:
            assert_close(a, r, RTOL["float32"], f"d{n}")


def test_block_values_are_the_inference_blocks():
    for dtype, length in ((torch.float32, 80), (torch.bfloat16, 77)):
        block = make_block(dtype)
        x = torch.randn(2, length, 40, device=DEV).to(dtype)
        with torch.no_grad():
            ref = block(x)
        a, b = block.forward_train(x, checkpoint8=True), block.forward_train(x, checkpoint8=False)
        assert a.dtype == dtype and a.shape == ref.shape
        assert_close_lowp(a, ref.float(), "8 bits", rel_l2=RTOL[str(dtype).split(".")[-1]])
        assert torch.equal(a, b)


@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length", [33, 64])
def test_block_under_autocast(length, low):
    """float32 parameters, activations of the autocast type; the backward pass called outside. Gradients from 8-bit
    activations against those without: 2.8e-2 as above, and the type's own factor for what is computed again in it."""
    block = make_block(torch.float32)
    g = torch.Generator().manual_seed(length)
    x, dy = torch.randn(2, length, 40, generator=g).to(DEV), torch.randn(2, length, 40, generator=g).to(DEV)
    outs, grads = [], []
    for held in (True, False):
        leaf = x.detach().requires_grad_(True)
        with torch.autocast("cuda", dtype=low):
            outs.append(block.forward_train(leaf, checkpoint8=held))
        grads.append(torch.autograd.grad(outs[-1], [leaf, *block.parameters()], dy.to(outs[-1].dtype)))
    assert outs[0].dtype == low and torch.equal(*outs)
    for n, a, r in zip(["x", *(n for n, _ in block.named_parameters())], *grads):
        assert a.dtype == torch.float32 and a.shape == r.shape
        assert_close_lowp(a, r, f"d{n}", rel_l2=2.8e-2 + RTOL[str(low).split(".")[-1]])


def test_model_trains_under_autocast():
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=50)
    model = init_weights_(MambaModel(cfg, dtype=torch.float32, device=DEV), seed=1)
    ids = torch.randint(0, 50, (2, 40), device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = model.forward_train(ids, checkpoint8=True).float().square().mean()
    loss.backward()
    for n, p in model.named_parameters():
        assert p.grad is not None and p.grad.dtype == p.dtype and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, n


def test_exact_activations_are_the_default():
    """A lossy form is asked for: by default the gradients are those of the activations as they are."""
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=50)
    model = init_weights_(MambaModel(cfg, dtype=torch.float32, device=DEV), seed=2)
    ids = torch.randint(0, 50, (2, 40), device=DEV)
    x = torch.randn(2, 40, 64, device=DEV)
    grads = []
    for asked in ({}, {"checkpoint8": False}):
        loss = model.forward_train(ids, **asked).square().mean() + model.layers[0].mixer.forward_train(x, **asked).square().mean()
        grads.append(torch.autograd.grad(loss, list(model.parameters())))
    # the embeddings' gradient is torch's own, whose order of additions is free
    for (n, _), a, b in zip(model.named_parameters(), *grads):
        assert n.startswith("embeddings") or torch.equal(a, b), n


def test_rms_norm_gradient():
    g = torch.Generator().manual_seed(3)
    x, w, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 5, 96), (96,), (3, 5, 96)))
    leaf, wl = x.float().to(DEV).requires_grad_(True), w.float().to(DEV).requires_grad_(True)
    y = training.rms_norm(leaf, wl, 1e-5, torch.float32)
    grads = torch.autograd.grad(y, (leaf, wl), dy.float().to(DEV))
    x.requires_grad_(True), w.requires_grad_(True)
    ref = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w
    want = torch.autograd.grad(ref, (x, w), dy)
    assert_close(y, ref.detach(), RTOL["float32"], "y")
    for a, r in zip(grads, want):
        assert_close(a, r, RTOL["float32"], "gradient")


def test_model_gradient_reaches_every_parameter():
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=50)
    model = init_weights_(MambaModel(cfg, dtype=torch.bfloat16, device=DEV), seed=1)
    ids = torch.randint(0, 50, (2, 40), device=DEV)
    logits = model.forward_train(ids)
    with torch.no_grad():
        assert_close_lowp(logits, model(ids).float(), "logits", rel_l2=2e-2)
    logits.float().square().mean().backward()
    for n, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, n


def test_checkpoints_hold_less():
    """What a block of 8 bits keeps between the passes against the same block without."""
    block = make_block(torch.bfloat16, d_model=256)
    x = torch.randn(4, 512, 256, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    kept = {}
    for held in (True, False):
        block.forward_train(x, checkpoint8=held).sum().backward()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = block.forward_train(x, checkpoint8=held)
        kept[held] = torch.cuda.memory_allocated() - before - out.numel() * 2
        out.sum().backward()
        del out
    tokens, E, D = 4 * 512, 512, 256
    assert kept[True] < tokens * (1.1 * (3 * E + D) + 2.1 * (16 + 32)) + (1 << 20)
    assert kept[False] > 3 * kept[True]


def test_tensor_parallel_block_is_refused():
    block = make_block(torch.float32)
    block.tp_reduce = lambda *a: None
    with pytest.raises(ValueError, match="tensor-parallel"):
        block.forward_train(torch.zeros(1, 8, 40, device=DEV))


@pytest.mark.parametrize("held", [True, False])
def test_example(held):
    spec = importlib.util.spec_from_file_location(
        "preference_step", Path(__file__).resolve().parents[1] / "examples" / "preference_step.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(steps=12, checkpoint8=held)
    assert abs(losses[0] - 0.6931) < 1e-3  # the reference is the model itself
    assert min(losses[-3:]) < 0.9 * losses[0]
