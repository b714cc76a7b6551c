"""Refusals of the training entry points through the C ABI, and their workspace queries, on CPU:
every call fails its checks, or asks for a size, before a device is touched."""
import ctypes

import pytest
import torch

from hp_rms_norm_b200 import capi
import hp_rms_norm_b200 as hp

P = 1 << 20  # an address nothing reads: 256-byte aligned, far from the others
A = [P + (k << 28) for k in range(8)]
BF16, FP16 = capi.DTYPE_BF16, capi.DTYPE_FP16


def status(entry, *args, workspace=0, size=0, flags=capi.LAUNCH_DEFAULT):
    n = ctypes.c_int64(size)
    return getattr(capi.load(), entry)(*args, workspace, ctypes.byref(n), None, flags)


def gated(out=A[0], gate_up=0, x=A[2], w=A[3], rows=4, hidden=64, d=32, os=32, gs=64, xs=64, ws=64,
          act=capi.ACT_SILU, dtype=BF16):
    return ["hprn_gated_linear", out, gate_up, x, w, rows, hidden, d, os, gs, xs, ws, act, dtype]


def gated_backward(gx=A[0], gw=A[1], dout=A[2], gate_up=A[3], x=A[4], w=A[5], rows=4, hidden=64, d=32,
                   gxs=64, gws=64, ds=32, gs=64, xs=64, ws=64, act=capi.ACT_SILU, dtype=BF16):
    return ["hprn_gated_linear_backward", gx, gw, dout, gate_up, x, w, rows, hidden, d, gxs, gws, ds, gs,
            xs, ws, act, dtype]


def loss(loss=A[0], lse=A[1], x=A[2], w=A[3], t=A[4], ignore=-100, rows=4, hidden=64, vocab=100, xs=64,
         ws=64, dtype=BF16):
    return ["hprn_linear_cross_entropy", loss, lse, x, w, t, ignore, rows, hidden, vocab, xs, ws, dtype]


def loss_backward(gx=A[0], gw=A[1], c=A[2], x=A[3], w=A[4], t=A[5], lse=A[6], ignore=-100, rows=4,
                  hidden=64, vocab=100, gxs=64, gws=64, xs=64, ws=64, dtype=BF16):
    return ["hprn_linear_cross_entropy_backward", gx, gw, c, x, w, t, lse, ignore, rows, hidden, vocab,
            gxs, gws, xs, ws, dtype]


def norm(gx=A[0], gw=A[1], dout=A[2], x=A[3], w=A[4], extra=0, rows=4, hidden=64, gxs=64, ds=64, xs=64,
         es=64, eps=1e-6, dtype=BF16):
    return ["hprn_rms_norm_backward", gx, gw, dout, x, w, extra, rows, hidden, gxs, ds, xs, es, eps, dtype]


CALLS = [gated, gated_backward, loss, loss_backward, norm]


@pytest.mark.parametrize("call", CALLS)
def test_dtype_sizes_flags(call):
    assert status(*call(dtype=7)) == capi.ERR_UNSUPPORTED_DTYPE
    assert status(*call(dtype=capi.DTYPE_FP32)) == capi.ERR_UNSUPPORTED_DTYPE
    for bad in (dict(rows=-1), dict(hidden=-1), dict(rows=1 << 40), dict(hidden=1 << 40)):
        assert status(*call(**bad)) == capi.ERR_INVALID_ARGUMENT
    assert status(*call(), flags=64) == capi.ERR_INVALID_ARGUMENT
    c = call()
    assert getattr(capi.load(), c[0])(*c[1:], None, None, None, 0) == capi.ERR_INVALID_ARGUMENT
    assert b"workspace_bytes" in capi.load().hprn_last_error()


@pytest.mark.parametrize("bad", [
    gated(out=0), gated(x=0), gated(w=0), gated(out=A[0] + 1), gated(gate_up=A[1] + 2), gated(xs=63),
    gated(ws=63), gated(os=31), gated(gate_up=A[1], gs=63), gated(act=9), gated(out=A[2]), gated(gate_up=A[3]),
    gated_backward(gx=0), gated_backward(gw=0), gated_backward(dout=0), gated_backward(ds=31),
    gated_backward(gws=60), gated_backward(gx=A[4]), gated_backward(gw=A[0]), gated_backward(act=-1),
    gated_backward(gate_up=A[3] + 1),
    loss(loss=0), loss(lse=0), loss(x=0), loss(w=0), loss(t=0), loss(t=A[4] + 4), loss(ws=60), loss(lse=A[0]),
    loss(loss=A[4]), loss(loss=A[0] + 2),
    loss_backward(gx=0), loss_backward(gw=0), loss_backward(c=0), loss_backward(lse=0), loss_backward(t=0),
    loss_backward(gx=A[3]), loss_backward(gw=A[4]), loss_backward(gxs=10), loss_backward(c=A[2] + 2),
    norm(gx=0), norm(gw=0), norm(dout=0), norm(x=0), norm(w=0), norm(gx=A[2]), norm(gw=A[4]),
    norm(extra=A[5], es=8), norm(extra=A[0]), norm(x=A[3] + 1),
], ids=lambda c: f"{c[0][5:]}")
def test_bad_arguments(bad):
    assert status(*bad, workspace=A[7], size=1 << 40) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("call", CALLS)
def test_workspace(call):
    c = call()
    need = capi.workspace_bytes(*c)
    if need:
        assert status(*c) == capi.ERR_INVALID_ARGUMENT
        assert status(*c, workspace=A[7], size=need - 1) == capi.ERR_INVALID_ARGUMENT
        assert status(*c, workspace=A[7] + 8, size=need) == capi.ERR_INVALID_ARGUMENT
        assert b"workspace" in capi.load().hprn_last_error()


def test_workspace_grows_with_what_needs_copying():
    """Rows that start off 16-byte boundaries are copied: their bytes are asked for."""
    assert capi.workspace_bytes(*gated()) == 0
    copied = capi.workspace_bytes(*gated(w=A[3] + 2))
    assert copied >= 64 * 64 * 2
    assert capi.workspace_bytes(*gated(hidden=63, xs=63, ws=63)) >= (4 + 64) * 64 * 2


def test_vocabulary_pieces_bound_the_workspace():
    """The logits' gradients take at most 512 MiB, whatever the vocabulary; beside them lie the
    input's gradient in float32 and, where its sums are split, at most 16 shares of it."""
    big = capi.workspace_bytes(*loss_backward(rows=8192, vocab=1 << 20, hidden=64))
    assert big <= (512 << 20) + 17 * 8192 * 64 * 4 + 4096
    assert capi.workspace_bytes(*loss_backward(rows=8192, vocab=1 << 20, hidden=64)) >= 256 << 20


def test_gradient_lists():
    lib = capi.load()
    n = ctypes.c_int64(0)

    def run(*grads, count=None, norm=A[6]):
        table = (capi.Grad * max(1, len(grads)))(*grads)
        return lib.hprn_grad_norm(norm, table, len(grads) if count is None else count, A[7],
                                  ctypes.byref(ctypes.c_int64(1 << 20)), None, 0)

    def clip(*grads, norm=A[6], most=1.0):
        table = (capi.Grad * max(1, len(grads)))(*grads)
        return lib.hprn_grad_clip(table, len(grads), norm, most, None, 0)

    ok = dict(grad=A[0], out=A[1], rows=1, cols=10, row_stride=10, out_row_stride=10, dtype=2, out_dtype=0)
    g = lambda **k: capi.Grad(**{**ok, **k})
    assert run(count=-1) == capi.ERR_INVALID_ARGUMENT
    assert run(g(dtype=5)) == capi.ERR_UNSUPPORTED_DTYPE
    assert run(g(grad=0)) == capi.ERR_INVALID_ARGUMENT
    assert run(g(grad=A[0] + 2)) == capi.ERR_INVALID_ARGUMENT
    assert run(g(rows=2, row_stride=9)) == capi.ERR_INVALID_ARGUMENT
    assert run(g(rows=-1)) == capi.ERR_INVALID_ARGUMENT
    assert run(g(), norm=0) == capi.ERR_INVALID_ARGUMENT
    assert clip(g(out=0)) == capi.ERR_INVALID_ARGUMENT
    assert clip(g(out_dtype=9)) == capi.ERR_UNSUPPORTED_DTYPE
    assert clip(g(out=A[0] + 4)) == capi.ERR_INVALID_ARGUMENT
    assert clip(g(out=A[0])) == capi.ERR_INVALID_ARGUMENT        # in place needs one type
    assert clip(g(), most=-1.0) == capi.ERR_INVALID_ARGUMENT
    assert clip(g(), most=float("nan")) == capi.ERR_INVALID_ARGUMENT
    assert clip(g(), norm=0) == capi.ERR_INVALID_ARGUMENT
    assert n.value == 0


def test_norm_and_clip_in_one_call():
    lib = capi.load()
    ok = dict(grad=A[0], out=A[1], rows=1, cols=10, row_stride=10, out_row_stride=10, dtype=2, out_dtype=0)

    def both(norm=A[6], most=1.0, ws=A[7], given=1 << 20, flags=0, **k):
        n = ctypes.c_int64(given)
        size = None if given is None else ctypes.byref(n)
        return lib.hprn_clip_grad_norm(norm, (capi.Grad * 1)(capi.Grad(**{**ok, **k})), 1, most, ws, size, None, flags)

    for bad in (dict(norm=0), dict(norm=A[6] + 2), dict(most=-1.0), dict(most=float("nan")), dict(out=0),
                dict(out=A[0]), dict(out=A[1] + 1), dict(rows=2, out_row_stride=9), dict(ws=0), dict(given=0),
                dict(flags=64)):
        assert both(**bad) == capi.ERR_INVALID_ARGUMENT, bad
    assert both(out_dtype=9) == capi.ERR_UNSUPPORTED_DTYPE


def test_torch_operators_are_cuda_only_and_trace():
    names = ("gated_linear", "gated_linear_backward", "linear_cross_entropy",
             "linear_cross_entropy_backward", "rms_norm_backward", "grad_norm", "clip_grad_norm")
    for name in names:
        assert "(a!)" in str(getattr(torch.ops.hp_rms_norm, name).default._schema)
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        hp.gated_linear(x, w)
    with pytest.raises(NotImplementedError):
        hp.grad_norm([x])
    m = lambda t: t.to("meta")
    assert hp.gated_linear(m(x), m(w)).shape == (4, 3)
    t = torch.zeros(4, dtype=torch.int64, device="meta")
    assert hp.linear_cross_entropy(m(x), m(w), t)[0].shape == (4,)
    assert hp.rms_norm_backward(m(x), m(x), m(x[0]), 1e-6)[1].shape == (8,)


def test_stall_hook_refuses_long_waits():
    assert capi.load().hprn_test_stall_loads(1, 1_000_000_001) == capi.ERR_INVALID_ARGUMENT
    capi.test_stall_loads(False)
