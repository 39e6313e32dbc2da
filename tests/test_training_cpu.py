"""Training operators: refusals and host-side plans that need no GPU."""

import ctypes

import pytest
import torch

from mamba_metal_b200 import _lib, training
from tests.test_training_gpu import LARGE


def size_of(fn, a):
    n = ctypes.c_size_t(0)
    return fn(ctypes.byref(a), ctypes.byref(n)), n.value


def test_struct_layouts_are_padding_free():
    scan = 9 + 5 + 6 * 3 + 2 + 3 + 1
    for s, n in ((_lib.MMCheckpoint8Args, 3 + 4 + 9), (_lib.MMConvCheckpointArgs, 6 + 5 + 12 + 1),
                 (_lib.MMConvBwdArgs, 9 + 5 + 15 + 1), (_lib.MMPreferenceArgs, 10 + 4 + 4 + 1 + 2),
                 (_lib.MMScanBwdArgs, scan + 11 + 18)):
        assert ctypes.sizeof(s) == 8 * n, s.__name__


def test_cpu_tensors_are_refused():
    u, A, B = torch.zeros(1, 2, 8), torch.zeros(2, 4), torch.zeros(1, 4, 8)
    for call in (lambda: training.selective_scan(u, u, A, B, B), lambda: training.causal_conv1d(u, torch.zeros(2, 4)),
                 lambda: training.selective_scan_backward(u, u, u, A, B, B),
                 lambda: training.causal_conv1d_backward(u, u, torch.zeros(2, 4), None),
                 lambda: training.checkpoint8(u), lambda: training.conv1d_checkpoint8(u, torch.zeros(2, 4), None),
                 lambda: training.Checkpoint8(u.to(torch.int8), torch.zeros(1, 2, 1, dtype=torch.uint8), u.dtype).restore(),
                 lambda: training.preference_loss(torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_shapes_and_types_are_checked():
    u, A, B = torch.zeros(1, 2, 8), torch.zeros(2, 4), torch.zeros(1, 4, 8)
    bad = [lambda: training.selective_scan(u, u[..., 1:], A, B, B), lambda: training.selective_scan(u, u, A, B, B[..., 1:]),
           lambda: training.selective_scan(u, u, torch.zeros(3, 4), B, B),
           lambda: training.selective_scan(u, u, torch.zeros(2, 65), torch.zeros(1, 65, 8), torch.zeros(1, 65, 8)),
           lambda: training.selective_scan(u, u, A, B, B, D=torch.zeros(3)),
           lambda: training.selective_scan(u, u, A, B, B, z=u[:, :1]),
           lambda: training.selective_scan(u, u, A, B, B, delta_bias=torch.zeros(1)),
           lambda: training.conv1d_checkpoint8(u, torch.zeros(2, 3), None),
           lambda: training.conv1d_checkpoint8(u, torch.zeros(2, 4), torch.zeros(3)),
           lambda: training.causal_conv1d_backward(u[..., 1:], u, torch.zeros(2, 4), None),
           lambda: training.checkpoint8(torch.zeros(()))]
    labels = torch.zeros(2, 3, dtype=torch.int64)
    bad += [lambda: training.preference_loss(torch.zeros(3, 3, 5), labels, torch.zeros(3)),
            lambda: training.preference_loss(torch.zeros(2, 3, 5), labels[:, :2], torch.zeros(2)),
            lambda: training.preference_loss(torch.zeros(2, 3, 5), labels.int(), torch.zeros(2)),
            lambda: training.preference_loss(torch.zeros(2, 3, 5), labels, torch.zeros(1)),
            lambda: training.preference_loss(torch.zeros(2, 3, 5), labels, torch.zeros(2), beta=0.0),
            lambda: training.preference_loss(torch.zeros(2, 3, 5), labels, torch.zeros(2), label_smoothing=0.6)]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: training.checkpoint8(u.double()), lambda: training.checkpoint8(u.long()),
                 lambda: training.conv1d_checkpoint8(u.double(), torch.zeros(2, 4), None),
                 lambda: training.preference_loss(torch.zeros(2, 3, 5, dtype=torch.float64), labels, torch.zeros(2))):
        with pytest.raises(TypeError):
            call()


def test_checkpoint_parts_that_do_not_belong_together_are_refused():
    """The kernels find a value's exponent by the codes' shape, so any other shape or type would be read past its end."""
    codes, exponents = torch.zeros(2, 3, 70, dtype=torch.int8), torch.zeros(2, 3, 3, dtype=torch.uint8)
    whole = training.Checkpoint8(codes, exponents, torch.float32)
    assert whole.shape == (2, 3, 70) and whole == training._made(codes, exponents, torch.float32)
    bad = [(codes, exponents[..., :2]), (codes, exponents[:1]), (codes, exponents[:, :2]), (codes, exponents[0]),
           (codes[..., :64], exponents), (codes[..., :0], exponents), (codes.short(), exponents), (codes, exponents.short()),
           (codes.view(torch.uint8), exponents), (codes[0, 0, 0], exponents[0, 0, 0])]
    for c, e in bad:
        with pytest.raises(AssertionError):
            training.Checkpoint8(c, e, torch.float32)


@pytest.mark.parametrize("by_channel", [False, True])
def test_checkpoints_of_short_rows(by_channel):
    """At no length do codes and exponents take up more than 16 bits a value, and ``nbytes`` says what they take up, but for
    the padding after the last row."""
    for n in [*range(1, 80), 255, 257, 5601]:
        codes, exponents = training._checkpoint_buffers((2, 96, n), "cpu", by_channel)
        c = training.Checkpoint8(codes, exponents, torch.bfloat16)
        held = codes.untyped_storage().nbytes() + exponents.untyped_storage().nbytes()
        assert held <= 2 * 2 * 96 * n
        assert held - 8 < c.nbytes <= held
        assert by_channel or n < 8 or all(s % 8 == 0 for s in codes.stride()[:2])
    codes, exponents = training._checkpoint_buffers((3, 0), "cpu", False)
    assert training.Checkpoint8(codes, exponents, torch.float32).nbytes == 0


def test_everything_that_a_kernel_reads_is_asked_for_its_device(monkeypatch):
    """Exponents and states too: a pointer of another GPU would be read by this one's kernel."""
    class Stop(Exception):
        pass

    def stop(*tensors):
        asked.extend(id(t) for t in tensors)
        raise Stop

    monkeypatch.setattr(_lib, "require_cuda", stop)
    u, A, B = torch.zeros(1, 2, 40), torch.zeros(2, 4), torch.zeros(1, 4, 40)
    states, w = torch.zeros(16), torch.zeros(2, 4)
    c = training.Checkpoint8(torch.zeros(1, 2, 40, dtype=torch.int8), torch.zeros(1, 2, 2, dtype=torch.uint8), u.dtype)
    for call, read in ((lambda: training.selective_scan_backward(u, u, u, A, B, B, states=states), (u, A, B, states)),
                       (lambda: training.causal_conv1d_backward(u, c, w, None), (u, c.codes, c.exponents, w)),
                       (c.restore, (c.codes, c.exponents))):
        asked = []
        with pytest.raises(Stop):
            call()
        assert all(id(t) in asked for t in read)


def test_c_entries_refuse():
    lib = _lib.lib()
    c = _lib.MMCheckpoint8Args()
    c.dtype, c.batch, c.dim, c.length = 5, 1, 1, 1
    assert lib.mm_checkpoint8_pack(ctypes.byref(c), None) == -3
    c.dtype, c.length = 1, -1
    assert lib.mm_checkpoint8_unpack(ctypes.byref(c), None) == -2
    c.length = 1
    assert lib.mm_checkpoint8_pack(ctypes.byref(c), None) == -1
    assert lib.mm_checkpoint8_pack(None, None) == -1
    v = _lib.MMConvBwdArgs()
    v.dtype, v.batch, v.dim, v.seqlen, v.width = 1, 1, 8, 16, 3
    assert size_of(lib.mm_causal_conv1d_bwd_workspace_size, v)[0] == -2
    v.width = 4
    assert lib.mm_causal_conv1d_bwd(ctypes.byref(v), None, 0, None) == -1
    f = _lib.MMConvCheckpointArgs()
    f.dtype, f.batch, f.dim, f.seqlen, f.width = 1, 1, 8, 16, 4
    assert lib.mm_causal_conv1d_fwd_checkpoint8(ctypes.byref(f), None) == -1
    p = _lib.MMPreferenceArgs()
    p.dtype, p.pairs, p.length, p.vocab = 2, 0, 3, 5
    assert size_of(lib.mm_preference_loss_workspace_size, p)[0] == -2
    p.pairs = 1
    assert lib.mm_preference_loss_fwd(ctypes.byref(p), None, 0, None) == -1
    assert lib.mm_preference_loss_bwd(ctypes.byref(p), None) == -1
    s = _lib.MMScanBwdArgs()
    s.fwd.dtype, s.fwd.batch, s.fwd.dim, s.fwd.dstate, s.fwd.seqlen = 1, 1, 8, 65, 16
    assert size_of(lib.mm_selective_scan_bwd_workspace_size, s)[0] == -2
    s.fwd.dstate, s.fwd.dtype = 16, 7
    assert size_of(lib.mm_selective_scan_bwd_workspace_size, s)[0] == -3
    s.fwd.dtype = 2
    assert lib.mm_selective_scan_bwd(ctypes.byref(s), None, 0, None) == -1
    rc, one = size_of(lib.mm_selective_scan_bwd_workspace_size, s)
    s.fwd.seqlen = 65
    assert rc == 0 and size_of(lib.mm_selective_scan_bwd_workspace_size, s)[1] > one > 0


def test_scan_gradient_of_no_channels_asks_for_what_it_clears():
    """dB and dC have a size of their own; with no channels they are zeros that the call has to write."""
    s = _lib.MMScanBwdArgs()
    s.fwd.dtype, s.fwd.batch, s.fwd.dim, s.fwd.dstate, s.fwd.seqlen = 1, 2, 0, 4, 40
    lib = _lib.lib()
    assert lib.mm_selective_scan_bwd(ctypes.byref(s), None, 0, None) == -1
    s.fwd.seqlen = 0
    assert lib.mm_selective_scan_bwd(ctypes.byref(s), None, 0, None) == 0


def scan_plan(dtype, batch, dim, n, length):
    """How the scan's training pass cuts a call: (chunks of a long chunk, long chunks, whether the forward pass walks whole
    sequences, tiles that a block of the gradient works off, blocks beside each other over the channels)."""
    chunks = -(-length // 32)
    if n <= 16 and length <= 256:
        per_long = chunks
    else:
        per_long = 4
        while chunks > 2 and per_long > 1 and batch * -(-dim // 32) * -(-chunks // per_long) < 12 * 148:
            per_long //= 2
    whole = n <= 16 and (length <= 256 or batch * dim >= 8192)
    every = dim * batch * chunks
    width = 16 if (dtype == torch.float32 and n <= 16) or every < 3 * 148 * 32 else 32
    tiles = 1 if n > 16 else min(max(every // (4 * 3 * 148) // width, 1), 512 // width)
    return per_long, -(-chunks // per_long), whole, tiles, -(-dim // (width * tiles))


def scan_sizes(dtype, batch, dim, n, length):
    """The workspaces' sizes that follow from the plan."""
    _, longs, whole, _, groups = scan_plan(dtype, batch, dim, n, length)
    room = lambda *floats: sum(-(-4 * f // 256) * 256 for f in floats)
    chunks, np4, passes = -(-length // 32), -(-n // 4) * 4, -(-n // 16)
    rows, lrows = batch * chunks * dim, batch * longs * dim
    cut = lrows if longs > 1 and not whole else 0
    bc = batch * chunks * groups * passes * 16 * 32
    many = chunks > 1
    return room(cut * np4, cut), 256 + room(many * rows * np4, many * rows, many * lrows * np4, many * lrows, bc, bc, rows * np4,
                                            rows, rows)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_plans(dtype):
    """The plan restated above is the library's (whose workspaces follow from it), and the gradient tests reach all of its
    kinds: long chunks of two and of four chunks, the last of them ragged, with both forward passes; several tiles a block."""
    sizes = [(1, 1536, 16, 48), (1, 1536, 16, 5601), (8, 1536, 16, 4096), (1, 5120, 16, 16384), (2, 100, 40, 700)] + LARGE
    for s in sizes:
        a = _lib.MMScanBwdArgs()
        f = a.fwd
        f.dtype, (f.batch, f.dim, f.dstate, f.seqlen) = _lib.DTYPE_CODE[dtype], s
        rc, forward = size_of(_lib.lib().mm_selective_scan_train_workspace_size, f)
        assert rc == 0 and size_of(_lib.lib().mm_selective_scan_bwd_workspace_size, a)[0] == 0
        assert (forward, size_of(_lib.lib().mm_selective_scan_bwd_workspace_size, a)[1]) == scan_sizes(dtype, *s), s
    plans = [(s, *scan_plan(dtype, *s)) for s in LARGE]
    ragged = [(per, longs, whole, tiles) for (_, _, _, length), per, longs, whole, tiles, _ in plans
              if longs > 2 and length % 32 and -(-length // 32) % per]
    assert {(4, False), (2, False), (4, True)} <= {(per, whole) for per, _, whole, _ in ragged}
    assert any(n > 16 and per == 4 for (_, _, n, _), per, *_ in plans)
    in_words = [(s, tiles) for s, *_, tiles, groups in plans if s[1] % 8 == 0 and s[3] % 8 == 0 and groups > 1]
    assert max(tiles for _, tiles in in_words) >= 4 and any(s[1] % 8 and tiles > 1 for s, *_, tiles, _ in plans)
