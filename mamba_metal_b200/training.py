"""Differentiable counterparts of the package's operators, and what a training step needs beside them: 8-bit
activation checkpoints and the preference loss. No counterpart in the reference, which has no backward pass.

``selective_scan`` and ``causal_conv1d`` take the arguments of the functions of the same name in the package and
compute the same values; gradients flow to every floating-point input that asks for them. They are functions of
their own so that the package's inference functions keep returning tensors without a graph. Everything runs in
libmamba_b200.so on the current stream of the tensors' device; there is no CPU path. The backward passes can
be differentiated once, and equal calls give equal bits.
"""

from __future__ import annotations

import ctypes
import struct
from array import array
from dataclasses import dataclass
from functools import lru_cache

import torch
import torch.nn.functional as F
from torch.amp import custom_bwd, custom_fwd
from torch.autograd.function import once_differentiable

from mamba_metal_b200 import _lib, ops
from mamba_metal_b200.selective_scan import MAX_DSTATE, _scan_dtype

CHECKPOINT8_BLOCK = 32  # values of a row that share an exponent (MM_CHECKPOINT8_BLOCK)


# ---- calls -------------------------------------------------------------------------------------------------
# A short call is bound by its host side, so arguments go into their struct in one piece (all fields are 8 bytes wide,
# in the order of include/mamba_b200.h), and device and stream are looked up without the context managers' cost.

_ZERO3 = (0, 0, 0)


def _p(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _s3(t: torch.Tensor | None):
    return _ZERO3 if t is None else t.stride()


def _bits(x: float) -> int:
    return struct.unpack("q", struct.pack("d", x))[0]


def _args(cls, *values):
    return cls.from_buffer(array("q", values))


def _size(name: str, args) -> int:
    n = ctypes.c_size_t(0)
    _lib.check(getattr(_lib.lib(), name)(ctypes.byref(args), ctypes.byref(n)), name)
    return n.value


def _run(name: str, dev: torch.device, args, *rest) -> None:
    fn, index = getattr(_lib.lib(), name), dev.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(ctypes.byref(args), *rest, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(ctypes.byref(args), *rest, stream)
    _lib.check(rc, name)


def _run_with_workspace(name: str, nbytes: int, dev: torch.device, args, *before) -> None:
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _run(name, dev, args, *before, _p(ws), nbytes)


def _by_channel(t: torch.Tensor) -> bool:
    """Whether a (..., channels, time) view is laid out with the channels contiguous."""
    return t.shape[-2] > 1 and t.shape[-1] > 1 and t.stride(-2) == 1 and t.stride(-1) != 1


def _empty(shape, dtype, device, by_channel: bool) -> torch.Tensor:
    b, d, n = shape
    if by_channel:
        return torch.empty((b, n, d), dtype=dtype, device=device).transpose(1, 2)
    return torch.empty((b, d, n), dtype=dtype, device=device)


def _laid_out(t: torch.Tensor, by_channel: bool) -> torch.Tensor:
    """``t`` (batch, channels, time) with the wanted axis contiguous; a gradient can arrive in any layout (of a sum,
    for instance, with stride 0)."""
    if by_channel:
        return t if t.stride(1) == 1 else t.transpose(1, 2).contiguous().transpose(1, 2)
    return t if t.stride(2) == 1 else t.contiguous()


def _cast(t: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor | None:
    return t if t is None or t.dtype == dtype else t.detach().to(dtype)


def _f32(t: torch.Tensor | None) -> torch.Tensor | None:
    t = _cast(t, torch.float32)
    return t if t is None or t.is_contiguous() else t.detach().contiguous()


def _like(grad: torch.Tensor | None, t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else _cast(grad if grad.shape == t.shape else grad.view(t.shape), t.dtype)


# ---- 8-bit activation checkpoints --------------------------------------------------------------------------


def _three(t: torch.Tensor):
    """(sizes, strides) of ``t``, up to three axes, as (batch, rows, length)."""
    size, stride = t.shape, t.stride()
    return ((1,) * (3 - len(size)) + tuple(size), (0,) * (3 - len(size)) + stride)


def _checkpoint_args(x, codes, exponents):
    size, stride = _three(x)
    return _args(_lib.MMCheckpoint8Args, _p(x), _p(codes), _p(exponents), _lib.DTYPE_CODE[x.dtype], *size, *stride,
                 *_three(codes)[1], *_three(exponents)[1])


def _checkpoint_buffers(shape, device, by_channel: bool):
    """Codes and exponents for a tensor of up to three axes, laid out like it. Rows of codes of eight values or more start
    on multiples of eight bytes, so that they can be written and read in vectors whatever the length; shorter rows have
    no vectors. So codes and exponents never take up more than 16 bits a value."""
    n = shape[-1]
    blocks = -(-n // CHECKPOINT8_BLOCK)
    if by_channel:
        lead, d = tuple(shape[:-2]), shape[-2]
        return (torch.empty((*lead, n, d), dtype=torch.int8, device=device).transpose(-1, -2),
                torch.empty((*lead, blocks, d), dtype=torch.uint8, device=device).transpose(-1, -2))
    pitch, strides = n if n < 8 else (n + 7) // 8 * 8, [1]
    for size in reversed(shape[1:]):
        strides.insert(0, strides[0] * (pitch if len(strides) == 1 else size))
    return (torch.empty_strided(shape, strides, dtype=torch.int8, device=device),
            torch.empty((*shape[:-1], blocks), dtype=torch.uint8, device=device))


@dataclass(frozen=True)
class Checkpoint8:
    """A tensor held in 8 bits: ``codes`` (int8, the tensor's shape) and ``exponents`` (uint8, one per 32 values of the
    last axis). A value stands for ``code * 2 ** (exponent - 127)``; exponent 255 marks a block that held an infinity
    or a NaN, and stands for NaN. ``dtype`` is the type of the tensor that was packed."""

    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype

    def __post_init__(self):
        # the kernels go by the codes' shape alone: fewer exponents than that asks for would be read past their end
        shape = self.codes.shape
        assert len(shape) >= 1 and self.exponents.shape == (*shape[:-1], -(-shape[-1] // CHECKPOINT8_BLOCK)), \
            "exponents are one for every 32 codes of the last axis"
        assert self.codes.dtype == torch.int8 and self.exponents.dtype == torch.uint8

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def nbytes(self) -> int:
        """Bytes that codes and exponents take up, with what lies between their rows."""
        return _span(self.codes) + _span(self.exponents)

    def restore(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values, in ``dtype`` (default: the packed tensor's), laid out like the packed tensor. Exact in the packed
        tensor's type, in float32 and in bfloat16; in float16 rounded where its small values are too far apart. Past the
        type's largest finite value that one is returned instead."""
        dtype = dtype or self.dtype
        if dtype not in _lib.DTYPE_CODE:
            raise TypeError(f"unsupported dtype {dtype}")
        codes, exponents = _up_to_three(self.codes), _up_to_three(self.exponents)
        dev = _lib.require_cuda(codes, exponents)
        if codes.dim() > 1 and _by_channel(codes):
            out = torch.empty((*codes.shape[:-2], codes.shape[-1], codes.shape[-2]), dtype=dtype, device=dev).transpose(-1, -2)
        else:
            out = torch.empty(codes.shape, dtype=dtype, device=dev)
        _run("mm_checkpoint8_unpack", dev, _checkpoint_args(out, codes, exponents))
        return out if self.codes.dim() <= 3 else out.view(self.shape)


def _span(t: torch.Tensor) -> int:
    """Elements from the first to the last of ``t`` in memory."""
    return 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0


def _made(codes: torch.Tensor, exponents: torch.Tensor, dtype: torch.dtype) -> Checkpoint8:
    """A Checkpoint8 of parts that this module made for each other; they are not checked again, which would take a short
    call 2 us."""
    c = object.__new__(Checkpoint8)
    c.__dict__.update(codes=codes, exponents=exponents, dtype=dtype)
    return c


def _up_to_three(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() <= 3 else t.flatten(0, -3)


def checkpoint8(x: torch.Tensor) -> Checkpoint8:
    """Packs ``x`` (float32, float16 or bfloat16, one axis or more) into 8 bits a value: blocks of 32 values of the last
    axis share the smallest power of two of which 127 reach their largest magnitude, and every value becomes a whole
    multiple of it, ties to even. No value moves by more than half that power of two: by less than 1/127 of the block's
    largest magnitude, where that is at least 127 * 2 ** -126 (the power of two is never less than 2 ** -126)."""
    assert x.dim() >= 1, "a checkpoint holds a tensor of one axis or more"
    if x.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {x.dtype}")
    dev = _lib.require_cuda(x)
    rows = _up_to_three(x)
    codes, exponents = _checkpoint_buffers(rows.shape, dev, rows.dim() > 1 and _by_channel(rows))
    _run("mm_checkpoint8_pack", dev, _checkpoint_args(rows, codes, exponents))
    if x.dim() > 3:
        codes, exponents = codes.unflatten(0, x.shape[:-2]), exponents.unflatten(0, x.shape[:-2])
    return _made(codes, exponents, x.dtype)


# ---- causal conv1d -----------------------------------------------------------------------------------------


def conv1d_checkpoint8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, *, silu: bool = True):
    """``causal_conv1d`` and ``checkpoint8`` of its input in one pass over ``x`` (batch, dim, seqlen). Returns
    (out, checkpoint); no graph."""
    dim = x.shape[1]
    assert x.dim() == 3 and weight.numel() == dim * ops.D_CONV and weight.shape[0] == dim, "only d_conv == 4 is implemented"
    assert bias is None or tuple(bias.shape) == (dim,)
    if x.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {x.dtype}")
    dev = _lib.require_cuda(x, weight, bias)
    w, b = _f32(weight), _f32(bias)
    by_channel = _by_channel(x)
    out = _empty(x.shape, x.dtype, dev, by_channel)
    codes, exponents = _checkpoint_buffers(x.shape, dev, by_channel)
    a = _args(_lib.MMConvCheckpointArgs, _p(x), _p(w), _p(b), _p(out), _p(codes), _p(exponents), _lib.DTYPE_CODE[x.dtype],
              *x.shape, ops.D_CONV, *x.stride(), *out.stride(), *codes.stride(), *exponents.stride(), bool(silu))
    _run("mm_causal_conv1d_fwd_checkpoint8", dev, a)
    return out, _made(codes, exponents, x.dtype)


def causal_conv1d_backward(dout: torch.Tensor, x: torch.Tensor | Checkpoint8, weight: torch.Tensor,
                           bias: torch.Tensor | None, *, silu: bool = True):
    """Gradient of ``causal_conv1d`` at ``x``, or at the values that a checkpoint of it stands for: (dx of dout's
    dtype, dweight (dim, 4) float32, dbias (dim,) float32)."""
    held = isinstance(x, Checkpoint8)
    src = x.codes if held else x
    batch, dim, seqlen = src.shape
    assert dout.shape == src.shape and dout.dtype == x.dtype
    assert weight.numel() == dim * ops.D_CONV and (bias is None or tuple(bias.shape) == (dim,))
    if dout.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {dout.dtype}")
    dev = _lib.require_cuda(dout, src, x.exponents if held else None, weight, bias)
    w, b = _f32(weight), _f32(bias)
    by_channel = _by_channel(src)
    dout = _laid_out(dout, by_channel)
    dx = _empty(src.shape, dout.dtype, dev, by_channel)
    dw = torch.empty((dim, ops.D_CONV), dtype=torch.float32, device=dev)
    db = torch.empty((dim,), dtype=torch.float32, device=dev)
    a = _args(_lib.MMConvBwdArgs, 0 if held else _p(src), _p(src) if held else 0, _p(x.exponents) if held else 0, _p(w), _p(b),
              _p(dout), _p(dx), _p(dw), _p(db), _lib.DTYPE_CODE[dout.dtype], batch, dim, seqlen, ops.D_CONV,
              *(_ZERO3 if held else src.stride()), *(src.stride() if held else _ZERO3),
              *(x.exponents.stride() if held else _ZERO3), *dout.stride(), *dx.stride(), bool(silu))
    _run_with_workspace("mm_causal_conv1d_bwd", _size("mm_causal_conv1d_bwd_workspace_size", a), dev, a)
    return dx, dw, db


class _CausalConv1d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, held):
        ctx.silu, ctx.held = silu, held
        if held:
            out, c = conv1d_checkpoint8(x, weight, bias, silu=silu)
            ctx.save_for_backward(c.codes, c.exponents, weight, bias)
        else:
            out = _empty(x.shape, x.dtype, x.device, _by_channel(x))
            ops.causal_conv1d(x, weight, bias, silu=silu, out=out)
            ctx.save_for_backward(x, None, weight, bias)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        src, exponents, weight, bias = ctx.saved_tensors
        if ctx.held:
            src = _made(src, exponents, dout.dtype)
        dx, dw, db = causal_conv1d_backward(dout, src, weight, bias, silu=ctx.silu)
        return dx, _like(dw, weight), _like(db, bias), None, None


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, silu: bool = True,
                  checkpoint8: bool = False) -> torch.Tensor:
    """Differentiable ``mamba_metal_b200.causal_conv1d``: x (batch, dim, seqlen), weight (dim, 1, 4) or (dim, 4), bias
    (dim,) or None. The output and dx are laid out like ``x``. With ``checkpoint8`` the backward pass is given
    ``x`` in 8 bits (made in the forward pass, see :func:`checkpoint8`) in place of ``x`` itself: the output is
    the same, the gradients are those at the values that the checkpoint stands for."""
    _lib.require_cuda(x, weight, bias)
    assert x.dim() == 3 and weight.shape[0] == x.shape[1] and weight.numel() == x.shape[1] * ops.D_CONV, \
        "only d_conv == 4 is implemented"
    assert bias is None or tuple(bias.shape) == (x.shape[1],)
    return _CausalConv1d.apply(x, weight, bias, bool(silu), bool(checkpoint8))


# ---- selective scan ----------------------------------------------------------------------------------------


def selective_scan_backward(dy: torch.Tensor, u, delta, A, B, C, *, D=None, z=None, delta_bias=None,
                            delta_softplus: bool = False, dstate: torch.Tensor | None = None,
                            states: torch.Tensor | None = None) -> dict:
    """Gradient of ``selective_scan`` for given dy (batch, dim, seqlen) and, optionally, dstate (batch, dim, dstate) of
    the last state. All activations share one dtype; A, D and delta_bias are float32. ``states`` is what
    ``selective_scan_states`` returned for the same inputs; without it they are computed again. Returns a dict of
    "u", "delta", "B", "C", "z" (that dtype; "z" None without z) and "A", "D", "delta_bias" (float32; None where
    not given)."""
    dev = _lib.require_cuda(dy, u, delta, A, B, C, D, z, delta_bias, dstate, states)
    batch, dim, seqlen = u.shape
    n = A.shape[1]
    assert dy.shape == u.shape == delta.shape and tuple(B.shape) == (batch, n, seqlen) == tuple(C.shape)
    assert (z is None or z.shape == u.shape) and tuple(A.shape) == (dim, n) and n <= MAX_DSTATE
    for t in (delta, B, C, z, dy):
        assert t is None or t.dtype == u.dtype
    for t, shape in ((D, (dim,)), (delta_bias, (dim,)), (dstate, (batch, dim, n))):
        assert t is None or (t.dtype == torch.float32 and tuple(t.shape) == shape and t.is_contiguous())
    assert A.dtype == torch.float32
    if u.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {u.dtype}")
    if states is None:
        states = selective_scan_states(u, delta, A, B, C, D=D, z=z, delta_bias=delta_bias, delta_softplus=delta_softplus,
                                       outputs=False)[2]
    assert states.dtype == torch.float32 and states.is_contiguous()
    by_channel = _by_channel(u)
    dy = _laid_out(dy, by_channel)
    act = lambda: _empty(u.shape, u.dtype, dev, by_channel)
    f32 = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dev)
    g = {"u": act(), "delta": act(), "z": None if z is None else act(), "A": f32(dim, n),
         "B": _empty(B.shape, u.dtype, dev, _by_channel(B)), "C": _empty(C.shape, u.dtype, dev, _by_channel(C)),
         "D": None if D is None else f32(dim), "delta_bias": None if delta_bias is None else f32(dim)}
    f = _scan_args(u, delta, A, B, C, D, z, delta_bias, delta_softplus)
    a = _args(_lib.MMScanBwdArgs, *f, _p(states), _p(dy), _p(dstate), *(_p(g[k]) for k in ("u", "delta", "A", "B", "C", "D", "z")),
              _p(g["delta_bias"]), *dy.stride(), *g["u"].stride(), *g["delta"].stride(), *_s3(g["z"]), *g["B"].stride(),
              *g["C"].stride())
    states_bytes, _, nbytes = _scan_sizes(_lib.DTYPE_CODE[u.dtype], batch, dim, n, seqlen)
    assert states.numel() * 4 == states_bytes, "states of another call"
    _run_with_workspace("mm_selective_scan_bwd", nbytes, dev, a)
    return g


def selective_scan_states(u, delta, A, B, C, *, D=None, z=None, delta_bias=None, delta_softplus: bool = False,
                          outputs: bool = True):
    """The training forward pass: (y, last state, states), without a graph. All activations share one dtype; A, D and
    delta_bias are float32. ``states`` (a flat float32 tensor: h before every 32nd step) is what
    ``selective_scan_backward`` starts from. With ``outputs=False`` only states is computed, y and the last state
    are None."""
    dev = _lib.require_cuda(u, delta, A, B, C, D, z, delta_bias)
    batch, dim, seqlen = u.shape
    n = A.shape[1]
    assert delta.shape == u.shape and tuple(B.shape) == (batch, n, seqlen) == tuple(C.shape)
    assert (z is None or z.shape == u.shape) and tuple(A.shape) == (dim, n) and n <= MAX_DSTATE
    for t in (delta, B, C, z):
        assert t is None or t.dtype == u.dtype
    for t in (D, delta_bias):
        assert t is None or (t.dtype == torch.float32 and tuple(t.shape) == (dim,) and t.is_contiguous())
    assert A.dtype == torch.float32
    if u.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {u.dtype}")
    return _scan_forward(u, delta, A, B, C, D, z, delta_bias, delta_softplus, outputs)


def _scan_forward(u, delta, A, B, C, D, z, delta_bias, delta_softplus, outputs=True):
    dev = u.device
    y = _empty(u.shape, u.dtype, dev, _by_channel(u)) if outputs else None
    state = torch.empty((u.shape[0], u.shape[1], A.shape[1]), dtype=torch.float32, device=dev) if outputs else None
    a = _args(_lib.MMScanArgs, *_scan_args(u, delta, A, B, C, D, z, delta_bias, delta_softplus, y, state))
    states_bytes, nbytes, _ = _scan_sizes(_lib.DTYPE_CODE[u.dtype], u.shape[0], u.shape[1], A.shape[1], u.shape[2])
    states = torch.empty(states_bytes // 4, dtype=torch.float32, device=dev)
    _run_with_workspace("mm_selective_scan_train_fwd", nbytes, dev, a, states.data_ptr())
    return y, state, states


def _scan_args(u, delta, A, B, C, D, z, delta_bias, softplus, y=None, state=None):
    """The fields of MMScanArgs, in order."""
    return (_p(u), _p(delta), _p(A), _p(B), _p(C), _p(D), _p(z), _p(y), _p(state), _lib.DTYPE_CODE[u.dtype], u.shape[0],
            u.shape[1], A.shape[1], u.shape[2], *u.stride(), *delta.stride(), *_s3(z), *_s3(y), *B.stride(), *C.stride(),
            *A.stride(), bool(softplus), 0, 0, _p(delta_bias))


@lru_cache(maxsize=256)
def _scan_sizes(dtype: int, batch: int, dim: int, dstate: int, seqlen: int):
    """Bytes of the states and of the forward and the backward pass's workspaces, which follow from the sizes alone."""
    f = _lib.MMScanArgs(dtype=dtype, batch=batch, dim=dim, dstate=dstate, seqlen=seqlen)
    return (_size("mm_selective_scan_states_size", f), _size("mm_selective_scan_train_workspace_size", f),
            _size("mm_selective_scan_bwd_workspace_size", _lib.MMScanBwdArgs(fwd=f)))


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, softplus):
        ctx.set_materialize_grads(False)
        dtype = _scan_dtype(u, delta, B, C, z)
        uc, dc, Bc, Cc, zc = (_cast(t, dtype) for t in (u, delta, B, C, z))
        Af, Df, bf = _cast(A, torch.float32), _f32(D), _f32(delta_bias)
        y, state, states = _scan_forward(uc, dc, Af, Bc, Cc, Df, zc, bf, softplus)
        ctx.softplus = softplus
        ctx.dtypes = tuple(None if t is None else t.dtype for t in (u, delta, A, B, C, D, z, delta_bias))
        ctx.save_for_backward(uc, dc, Af, Bc, Cc, Df, zc, bf, states)
        return _cast(y, u.dtype), state

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate):
        u, delta, A, B, C, D, z, bias, states = ctx.saved_tensors
        if dy is None and dstate is None:
            return (None,) * 9
        dy = torch.zeros_like(u) if dy is None else _cast(dy, u.dtype)
        g = selective_scan_backward(dy, u, delta, A, B, C, D=D, z=z, delta_bias=bias, delta_softplus=ctx.softplus,
                                    dstate=_f32(dstate), states=states)
        names = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")
        return (*(None if t is None else _cast(g[k], t) for k, t in zip(names, ctx.dtypes)), None)


def selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   D: torch.Tensor | None = None, z: torch.Tensor | None = None,
                   delta_bias: torch.Tensor | None = None, delta_softplus: bool = False, return_state: bool = False):
    """Differentiable ``mamba_metal_b200.selective_scan``: shapes, dtypes and results as there, and ``delta_bias``
    (dim,), added to delta before softplus. The last state is differentiable too. y and the gradients of u, delta
    and z are laid out like u. Kept for the backward pass: the inputs and the state before every 32nd step."""
    batch, dim, seqlen = u.shape
    _, dstate = A.shape
    assert delta.shape == u.shape
    assert tuple(B.shape) == (batch, dstate, seqlen) == tuple(C.shape)
    assert A.shape[0] == dim and dstate <= MAX_DSTATE
    assert z is None or z.shape == u.shape
    assert D is None or tuple(D.shape) == (dim,)
    assert delta_bias is None or tuple(delta_bias.shape) == (dim,)
    _lib.require_cuda(u, delta, A, B, C, D, z, delta_bias)
    y, state = _SelectiveScan.apply(u, delta, A, B, C, D, z, delta_bias, bool(delta_softplus))
    return (y, state) if return_state else y


# ---- preference loss ---------------------------------------------------------------------------------------


@lru_cache(maxsize=256)
def _preference_bytes(dtype: int, pairs: int, length: int, vocab: int) -> int:
    return _size("mm_preference_loss_workspace_size",
                 _lib.MMPreferenceArgs(dtype=dtype, pairs=pairs, length=length, vocab=vocab, beta=1.0))


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ref, beta, smoothing, ignore_index):
        ctx.set_materialize_grads(False)
        rows, length, vocab = logits.shape
        dev, pairs = logits.device, rows // 2
        f32 = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dev)
        loss, chosen, rejected = f32(), f32(pairs), f32(pairs)
        stats = f32(rows * (2 * length + 1))  # and the answers' slopes behind them
        x = logits.detach()
        if vocab > 1 and x.stride(2) != 1:
            x = x.contiguous()
        values = (_lib.DTYPE_CODE[x.dtype], pairs, length, vocab, *x.stride()[:2])
        rest = (ignore_index, _bits(beta), _bits(smoothing))
        a = _args(_lib.MMPreferenceArgs, _p(x), _p(labels), _p(ref), _p(loss), _p(chosen), _p(rejected), _p(stats),
                  _p(stats) + 8 * rows * length, 0, 0, *values, 0, 0, *rest)
        _run_with_workspace("mm_preference_loss_fwd", _preference_bytes(*values[:4]), dev, a)
        ctx.args = values, rest
        ctx.save_for_backward(x, labels, stats)
        ctx.mark_non_differentiable(chosen, rejected)
        return loss, chosen, rejected

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        if grad_loss is None:
            return (None,) * 6
        x, labels, stats = ctx.saved_tensors
        grad = _f32(grad_loss)
        dlogits = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        values, rest = ctx.args
        a = _args(_lib.MMPreferenceArgs, _p(x), _p(labels), 0, 0, 0, 0, _p(stats), _p(stats) + 8 * labels.numel(), _p(grad),
                  _p(dlogits), *values, *dlogits.stride()[:2], *rest)
        _run("mm_preference_loss_bwd", x.device, a)
        return dlogits, None, None, None, None, None


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logps: torch.Tensor, *, beta: float = 0.1,
                    label_smoothing: float = 0.0, ignore_index: int = -100):
    """Preference loss over pairs of answers, from the policy's logits (2 * pairs, length, vocab): rows 0 .. pairs-1 are the
    chosen answers, the rest the rejected ones of the same pairs. ``labels`` (2 * pairs, length) int64 are the tokens
    that the logits are to predict (already shifted), ``ignore_index`` where a token is no part of the answer.
    ``ref_logps`` (2 * pairs,) are the answers' log-probabilities under the reference model.

    With r = beta * (logp - ref_logp) of an answer and m = r_chosen - r_rejected, the loss is the mean over the pairs of
    -(1 - label_smoothing) * log sigmoid(m) - label_smoothing * log sigmoid(-m). Returns (loss, chosen, rejected): a
    float32 scalar, differentiable in the logits, and the (pairs,) float32 values of r, which are not. The answers'
    log-probabilities are sums over tokens; of an answer without tokens it is 0. Logits of ignored tokens are not
    read. A label outside the vocabulary makes its answer's value, and the loss, NaN."""
    assert logits.dim() == 3 and logits.shape[0] >= 2 and logits.shape[0] % 2 == 0 and logits.shape[2] >= 1, \
        "logits are (2 * pairs, length, vocab)"
    assert labels.shape == logits.shape[:2] and tuple(ref_logps.shape) == (logits.shape[0],)
    assert labels.dtype == torch.int64 and ref_logps.is_floating_point()
    assert 0.0 <= label_smoothing <= 0.5 and beta > 0.0
    if logits.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {logits.dtype}")
    _lib.require_cuda(logits, labels, ref_logps)
    return _PreferenceLoss.apply(logits, labels.contiguous(), _f32(ref_logps), float(beta), float(label_smoothing),
                                 int(ignore_index))


# ---- a Mamba block ---------------------------------------------------------------------------------------------


def _proj(w: torch.Tensor, a: torch.Tensor) -> torch.Tensor:
    """w (out, c) applied to the channels of a (batch, c, time), in a's layout."""
    return F.linear(a.transpose(1, 2), w).transpose(1, 2) if _by_channel(a) else torch.matmul(w, a)


def _outer(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """sum over batch and time of a (batch, i, time) times b (batch, j, time): (i, j), one product over all tokens."""
    i, j = a.shape[1], b.shape[1]
    if _by_channel(a) and _by_channel(b):
        return a.transpose(1, 2).reshape(-1, i).t() @ b.transpose(1, 2).reshape(-1, j)
    return a.transpose(0, 1).reshape(i, -1) @ b.transpose(0, 1).reshape(j, -1).t()


class _Block(torch.autograd.Function):
    """MambaBlock.forward that keeps its activations (its input, the conv's, the gate, the scan's output) in 8 bits and
    computes the rest again in the backward pass, from the values they stand for. Under autocast the projections give
    activations of its type, and the backward pass runs under it as well."""

    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx, x, in_w, conv_w, conv_b, x_w, dt_w, dt_b, A_log, D, out_w, by_channel):
        E, R, N = conv_w.shape[0], dt_w.shape[1], A_log.shape[1]
        dtype = in_w.dtype
        xt = _cast(x, dtype).transpose(1, 2)
        xt = _laid_out(xt, by_channel)
        xz = _proj(in_w, xt)
        xc, cx = conv1d_checkpoint8(xz[:, :E], conv_w, conv_b)
        x_dbl = _proj(x_w, xc)
        dt = _proj(dt_w, x_dbl[:, :R])
        A, Df, bf = -torch.exp(A_log.float()), _f32(D), _f32(dt_b)
        y, _, _ = selective_scan_states(xc, dt, A, x_dbl[:, R:R + N], x_dbl[:, R + N:], D=Df, z=xz[:, E:], delta_bias=bf,
                                        delta_softplus=True)
        out = _proj(out_w, y).transpose(1, 2)
        held = [cx, checkpoint8(xt), checkpoint8(xz[:, E:]), checkpoint8(y)]
        ctx.x_dtype, ctx.dtypes = x.dtype, tuple(c.dtype for c in held)
        ctx.save_for_backward(x_dbl, in_w, conv_w, conv_b, x_w, dt_w, dt_b, A_log, D, out_w,
                              *(t for c in held for t in (c.codes, c.exponents)))
        return out

    @staticmethod
    @once_differentiable
    @custom_bwd(device_type="cuda")
    def backward(ctx, dout):
        x_dbl, in_w, conv_w, conv_b, x_w, dt_w, dt_b, A_log, D, out_w, *held = ctx.saved_tensors
        E, R, N = conv_w.shape[0], dt_w.shape[1], A_log.shape[1]
        cx, cxt, cz, cy = (_made(held[2 * i], held[2 * i + 1], t) for i, t in enumerate(ctx.dtypes))
        dtype = cx.dtype  # of the activations
        by_channel = _by_channel(cx.codes)
        xt, z, y = cxt.restore(), cz.restore(), cy.restore()
        xc = _empty(z.shape, dtype, z.device, by_channel)
        ops.causal_conv1d(cx.restore(), conv_w, conv_b, silu=True, out=xc)
        A, Df, bf = -torch.exp(A_log.float()), _f32(D), _f32(dt_b)
        dt = _proj(dt_w, x_dbl[:, :R])
        do = _laid_out(_cast(dout, dtype).transpose(1, 2), by_channel)
        d_out_w = _outer(do, y)
        g = selective_scan_backward(_proj(out_w.t(), do), xc, dt, A, x_dbl[:, R:R + N], x_dbl[:, R + N:], D=Df, z=z,
                                    delta_bias=bf, delta_softplus=True)
        d_dt_w = _outer(g["delta"], x_dbl[:, :R])
        d_dbl = _laid_out(torch.cat([_proj(dt_w.t(), g["delta"]), g["B"], g["C"]], 1), by_channel)
        d_x_w = _outer(d_dbl, xc)
        dx_in, dw, db = causal_conv1d_backward(g["u"] + _proj(x_w.t(), d_dbl), cx, conv_w, conv_b)
        dxz = _laid_out(torch.cat([dx_in, g["z"]], 1), by_channel)
        d_in_w = _outer(dxz, xt)
        dx = _proj(in_w.t(), dxz).transpose(1, 2)
        return (_cast(dx, ctx.x_dtype), _like(d_in_w, in_w), _like(dw, conv_w), _like(db, conv_b), _like(d_x_w, x_w),
                _like(d_dt_w, dt_w), _like(g["delta_bias"], dt_b), _cast(g["A"] * A, A_log.dtype), _like(g["D"], D),
                _like(d_out_w, out_w), None)


def mamba_block(block, x: torch.Tensor, checkpoint8: bool = False) -> torch.Tensor:
    """Differentiable ``MambaBlock`` forward: x (batch, length, d_model) to the same, with gradients for x and all of the
    block's parameters (``MambaBlock.forward_train`` calls it). Autograd holds the activations that the backward pass
    needs, and every intermediate, as they are. With ``checkpoint8`` its input, the conv's input, the gate and the
    scan's output are held in 8 bits instead (1.03 bytes an element, a little more for rows of few steps, and
    never more than two), and the rest is computed again; the output is the same, the gradients are those at the
    values that the 8 bits stand for."""
    if block.tp_reduce is not None:
        raise ValueError("tensor-parallel blocks have no training pass")
    _lib.require_cuda(x, block.in_proj.weight)
    E, R, N = block.d_inner, block.dt_rank, block.d_state
    # as in the inference pass: rows along time where they are 16-byte aligned, else along channels
    by_channel = (x.shape[1] * block.in_proj.weight.dtype.itemsize) % 16 != 0 and x.shape[1] > 1
    if checkpoint8:
        return _Block.apply(x, block.in_proj.weight, block.conv1d.weight, block.conv1d.bias, block.x_proj.weight,
                            block.dt_proj.weight, block.dt_proj.bias, block.A_log, block.D, block.out_proj.weight, by_channel)
    xz = _proj(block.in_proj.weight, _laid_out(x.to(block.in_proj.weight.dtype).transpose(1, 2), by_channel))
    xc = causal_conv1d(xz[:, :E], block.conv1d.weight, block.conv1d.bias)
    x_dbl = _proj(block.x_proj.weight, xc)
    y = selective_scan(xc, _proj(block.dt_proj.weight, x_dbl[:, :R]), -torch.exp(block.A_log.float()), x_dbl[:, R:R + N],
                       x_dbl[:, R + N:], D=block.D, z=xz[:, E:], delta_bias=block.dt_proj.bias, delta_softplus=True)
    return _proj(block.out_proj.weight, y).transpose(1, 2)


class _RMSNorm(torch.autograd.Function):
    """The package's RMSNorm over the last axis of a float32 tensor, result in ``dtype``; the gradient in float32."""

    @staticmethod
    def forward(ctx, x, weight, eps, dtype):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return ops.add_rmsnorm(x.contiguous(), None, weight, eps, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight = ctx.saved_tensors
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + ctx.eps)
        unit, g = x * r, g.float()
        dw = (g * unit).flatten(0, -2).sum(0)
        g = g * weight
        return r * (g - unit * (g * unit).mean(-1, keepdim=True)), dw, None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, dtype: torch.dtype) -> torch.Tensor:
    """Differentiable RMSNorm of a float32 ``x`` over its last axis, in ``dtype``. ``x`` is kept for the backward pass, which
    is torch operations over float32 (bf16 8x2048x768 337 us, forward and backward)."""
    assert x.dtype == torch.float32 and weight.dtype == torch.float32 and tuple(weight.shape) == tuple(x.shape[-1:])
    _lib.require_cuda(x, weight)
    return _RMSNorm.apply(x, weight, eps, dtype)
