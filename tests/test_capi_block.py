"""Refusals of the entry points around a block (gated norms, log probabilities, 8-bit integers)
through the C ABI, and their workspace queries, on CPU: every call fails its checks, or asks for a
size, before a device is touched."""
import ctypes

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import hp_rms_norm_b200 as hp
from hp_rms_norm_b200 import capi

P = 1 << 20  # an address nothing reads: 256-byte aligned, far from the others
A = [P + (k << 28) for k in range(14)]
BF16, FP16 = capi.DTYPE_BF16, capi.DTYPE_FP16


def with_size(entry, *args, workspace=0, size=0, flags=capi.LAUNCH_DEFAULT):
    n = ctypes.c_int64(size)
    return getattr(capi.load(), entry)(*args, workspace, ctypes.byref(n), None, flags)


def without(entry, *args, flags=capi.LAUNCH_DEFAULT):
    return getattr(capi.load(), entry)(*args, None, flags)


def norm(out=A[0], t=A[1], x=A[2], r=A[3], p=A[4], w=A[5], g=A[6], rows=8, hidden=64, per=8, width=64, os=64, ts=64, xs=64, rs=64,
         gs=64, scale=1.0, eps=1e-6, dtype=BF16):
    return without, ["hprn_gated_add_rms_norm", out, t, x, r, p, w, g, rows, hidden, per, width, os, ts, xs, rs, gs, scale, eps, dtype]


def norm_backward(dx=A[0], dr=A[1], dp=A[2], dw=A[3], dg=A[4], d=A[5], e=A[6], x=A[7], t=A[8], p=A[9], w=A[10], g=A[11], rows=8,
                  hidden=64, per=8, width=64, dxs=64, drs=64, dgs=64, ds=64, es=64, xs=64, ts=64, gs=64, scale=1.0, eps=1e-6, dtype=BF16):
    return with_size, ["hprn_gated_add_rms_norm_backward", dx, dr, dp, dw, dg, d, e, x, t, p, w, g, rows, hidden, per, width, dxs, drs,
                       dgs, ds, es, xs, ts, gs, scale, eps, dtype]


def probs(lp=A[0], h=A[1], lse=A[2], tv=A[3], ti=A[4], x=A[5], w=A[6], t=A[7], ignore=-100, temperature=1.0, top=2, rows=4, hidden=64,
          vocab=100, xs=64, ws=64, dtype=BF16):
    return with_size, ["hprn_linear_log_probs", lp, h, lse, tv, ti, x, w, t, ignore, temperature, top, rows, hidden, vocab, xs, ws, dtype]


def probs_backward(dx=A[0], dw=A[1], g=A[2], gh=A[3], x=A[4], w=A[5], t=A[6], lse=A[7], h=A[8], ignore=-100, temperature=1.0, rows=4,
                   hidden=64, vocab=100, dxs=64, dws=64, xs=64, ws=64, dtype=BF16):
    return with_size, ["hprn_linear_log_probs_backward", dx, dw, g, gh, x, w, t, lse, h, ignore, temperature, rows, hidden, vocab, dxs,
                       dws, xs, ws, dtype]


def quant(q=A[0], s=A[1], t=A[2], x=A[3], w=A[4], r=A[5], rows=4, hidden=64, qs=64, ts=64, xs=64, rs=64, eps=1e-6, dtype=BF16):
    return without, ["hprn_rms_norm_int8", q, s, t, x, w, r, rows, hidden, qs, ts, xs, rs, eps, dtype]


def product(out=A[0], x=A[1], xs=A[2], w=A[3], wsc=A[4], b=A[5], rows=64, hidden=64, channels=32, os=32, xl=64, wl=64, dtype=BF16):
    return with_size, ["hprn_linear_int8", out, x, xs, w, wsc, b, rows, hidden, channels, os, xl, wl, dtype]


CALLS = [norm, norm_backward, probs, probs_backward, quant, product]


def status(call, **keywords):
    how, args = call
    return how(*args, **keywords)


@pytest.mark.parametrize("call", CALLS)
def test_dtype_sizes_flags(call):
    assert status(call(dtype=7)) == capi.ERR_UNSUPPORTED_DTYPE
    assert status(call(dtype=capi.DTYPE_FP32)) == capi.ERR_UNSUPPORTED_DTYPE
    for bad in (dict(rows=-1), dict(hidden=-1), dict(rows=1 << 40), dict(hidden=1 << 40)):
        assert status(call(**bad)) == capi.ERR_INVALID_ARGUMENT
    assert status(call(), flags=64) == capi.ERR_INVALID_ARGUMENT
    how, args = call()
    if how is with_size:
        assert getattr(capi.load(), args[0])(*args[1:], None, None, None, 0) == capi.ERR_INVALID_ARGUMENT
        assert b"workspace_bytes" in capi.load().hprn_last_error()


@pytest.mark.parametrize("bad", [
    norm(out=0), norm(t=0), norm(x=0), norm(r=0), norm(w=0), norm(out=A[0] + 1), norm(g=A[6] + 1), norm(xs=63), norm(os=63), norm(ts=60),
    norm(per=3), norm(per=0), norm(width=32), norm(per=4, gs=63), norm(out=A[3]), norm(t=A[2]), norm(t=A[0]), norm(out=A[5]), norm(t=A[6]),
    norm(out=A[2] + 2), norm(t=A[3], ts=72), norm(out=A[2], os=80),
    norm_backward(dx=0), norm_backward(dr=0), norm_backward(dp=0), norm_backward(dw=0), norm_backward(dg=0), norm_backward(d=0),
    norm_backward(x=0), norm_backward(t=0), norm_backward(w=0), norm_backward(dx=A[0] + 1), norm_backward(dxs=63), norm_backward(es=63),
    norm_backward(per=4, dgs=63), norm_backward(per=5), norm_backward(width=2), norm_backward(dx=A[7]), norm_backward(dr=A[0]),
    norm_backward(dw=A[2]), norm_backward(dg=A[11]),
    probs(lp=0), probs(h=0), probs(lse=0), probs(x=0), probs(w=0), probs(t=0), probs(tv=0), probs(ti=0), probs(ti=A[4] + 4), probs(ws=60),
    probs(h=A[0]), probs(lp=A[7]), probs(top=-1), probs(top=65), probs(top=65, vocab=1000), probs(top=60, vocab=50), probs(temperature=0.0),
    probs(temperature=-1.0), probs(temperature=float("nan")), probs(temperature=float("inf")), probs(temperature=1e-40), probs(vocab=1 << 40),
    probs_backward(dx=0), probs_backward(dw=0), probs_backward(g=0), probs_backward(lse=0), probs_backward(h=0), probs_backward(gh=A[3] + 2),
    probs_backward(dws=60), probs_backward(dx=A[4]), probs_backward(dw=A[0]), probs_backward(temperature=0.0),
    quant(q=0), quant(s=0), quant(x=0), quant(r=0), quant(t=0), quant(s=A[1] + 2), quant(x=A[3] + 1), quant(qs=63), quant(ts=60), quant(q=A[3]),
    quant(s=A[0]), quant(t=A[3]), quant(t=A[5] + 2), quant(hidden=0),
    product(out=0), product(x=0), product(w=0), product(xs=0), product(wsc=0), product(out=A[0] + 1), product(xs=A[2] + 2), product(xl=63),
    product(os=31), product(out=A[1]), product(out=A[4]), product(hidden=131072, xl=131072, wl=131072), product(channels=-1),
], ids=lambda c: c[1][0])
def test_bad_arguments(bad):
    how, args = bad
    keywords = dict(workspace=A[13], size=1 << 30) if how is with_size else {}
    assert how(*args, **keywords) == capi.ERR_INVALID_ARGUMENT
    assert capi.load().hprn_last_error()


@pytest.mark.parametrize("call", [norm_backward, probs, probs_backward, product])
def test_workspace_queries(call):
    """A query asks for no tensor and launches nothing; one byte less than it says is refused."""
    _, args = call(hidden=65, **(dict(width=65) if call is norm_backward else {}))
    args = [65 if a == 64 and call is not product else a for a in args]
    if call is product:
        args = product(hidden=65, xl=65, wl=65)[1]
    need = ctypes.c_int64(-1)
    assert getattr(capi.load(), args[0])(*args[1:], None, ctypes.byref(need), None, capi.WORKSPACE_QUERY) == capi.OK
    assert need.value > 0
    assert with_size(*args, workspace=A[13], size=need.value - 1) == capi.ERR_INVALID_ARGUMENT
    assert b"workspace" in capi.load().hprn_last_error()
    assert with_size(*args, workspace=A[13] + 64, size=1 << 40) == capi.ERR_INVALID_ARGUMENT


def test_workspaces_stay_bounded():
    """A vocabulary's logits are held for a block of rows: 1 GiB and what a tile row needs beside it."""
    for rows, vocab in ((100, 131072), (8192, 131072), (1 << 20, 131072)):
        need = capi.workspace_bytes(*probs(rows=rows, vocab=vocab, hidden=64)[1])
        assert need <= (1 << 30) + (1 << 28)
    # One row a block of 256 where that is more.
    assert capi.workspace_bytes(*probs(rows=4096, vocab=1 << 22, hidden=64)[1]) <= 256 * (1 << 24) * 1.2


@pytest.mark.parametrize("hidden", [64, 512, 1001, 4096, 8192, 16384])
@pytest.mark.parametrize("rows,per", [(65536, 2), (65536, 3 * 2 ** 4), (5000, 2), (1 << 20, 4), (30, 15), (4096, 2048)])
def test_gates_that_rows_share_stay_bounded(rows, per, hidden):
    """The sums for a gate are one row of floats and one more for each run of rows that ends inside
    it, a run for each of at most 14 groups of 148 CTAs; or, of at most two gates a CTA, a row for each
    group.  With gates of two rows that is the size of the rows themselves."""
    per = per if rows % per == 0 else 2
    strides = {k: hidden for k in ("dxs", "drs", "dgs", "ds", "es", "xs", "ts", "gs")}
    need = capi.workspace_bytes(*norm_backward(rows=rows, hidden=hidden, per=per, width=hidden, **strides)[1])
    assert need <= 4 * -(-hidden // 8) * 8 * (rows // per + 148 * (3 * 14 + 1)) + 1024


def test_signatures():
    import inspect

    names = lambda f: list(inspect.signature(f).parameters)  # noqa: E731
    assert names(hp.gated_add_rms_norm) == ["input", "residual", "post_weight", "weight", "eps", "gate", "residual_scale", "out", "residual_out"]
    assert names(hp.linear_log_probs) == ["input", "weight", "target", "top", "temperature", "ignore_index"]
    assert names(hp.linear_int8) == ["input", "input_scale", "weight", "weight_scale", "bias", "dtype", "out"]
    assert names(hp.rms_norm_int8) == ["input", "weight", "eps", "residual", "residual_out"]


def test_shapes_without_a_device():
    """The shape-only kernels, as tracing runs them."""
    x, w = torch.empty(3, 5, 64, device="meta", dtype=torch.bfloat16), torch.empty(64, device="meta", dtype=torch.bfloat16)
    out = hp.gated_add_rms_norm(x, x.clone(), w, w, 1e-6, gate=w, residual_out=x.clone())
    assert out.shape == x.shape
    grads = hp.gated_add_rms_norm_backward(x, x, x, w, w, 1e-6, gate=x[:, :1, :1])
    assert [g.shape for g in grads] == [x.shape, x.shape, w.shape, w.shape, (3, 1, 1)]
    assert hp.gated_add_rms_norm_backward(x, x, x, None, w, 1e-6)[2::2] == (None, None)
    codes, scales = hp.rms_norm_int8(x, w, 1e-6)
    assert codes.dtype == torch.int8 and codes.shape == x.shape and scales.shape == (3, 5) and scales.dtype == torch.float32
    y = hp.linear_int8(codes, scales, torch.empty(7, 64, device="meta", dtype=torch.int8), torch.empty(7, device="meta"), dtype=torch.float16)
    assert y.shape == (3, 5, 7) and y.dtype == torch.float16
    v = torch.empty(100, 64, device="meta", dtype=torch.bfloat16)
    found = hp.linear_log_probs(x, v, torch.empty(3, 5, device="meta", dtype=torch.int64), top=4)
    assert found.top_indices.shape == (3, 5, 4) and found.top_indices.dtype == torch.int64 and found.entropy.shape == (3, 5)
    dx, dw = hp.linear_log_probs_backward(found.log_prob, x, v, torch.empty(3, 5, device="meta", dtype=torch.int64), found.lse)
    assert dx.shape == x.shape and dw.shape == v.shape


def test_outputs_are_tensors_of_their_own():
    """Gradients of what is absent too: the schema declares five outputs that alias nothing."""
    x, w = torch.empty(4, 64, device="meta", dtype=torch.bfloat16), torch.empty(64, device="meta", dtype=torch.bfloat16)
    for post, gate in ((None, None), (w, None), (None, w), (w, w)):
        grads = torch.ops.hp_rms_norm.gated_add_rms_norm_backward.default(x, None, x, x, post, w, gate, 1.0, 1e-6)
        assert len({id(g) for g in grads}) == 5
        assert [g.numel() for g in grads] == [256, 256, 0 if post is None else 64, 64, 0 if gate is None else 64]


def test_only_what_is_written_is_declared_written():
    """A traced graph orders and copies for the writes that the schemas declare."""
    class Written(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            called.append(func)
            given_by = dict(zip((a.name for a in func._schema.arguments), args)) | (kwargs or {})
            for declared in func._schema.arguments:
                given = given_by.get(declared.name)
                if declared.alias_info is not None and declared.alias_info.is_write and isinstance(given, torch.Tensor):
                    found.append(given)
            return func(*args, **(kwargs or {}))

    x, w = torch.empty(4, 64, device="meta", dtype=torch.bfloat16), torch.empty(64, device="meta", dtype=torch.bfloat16)
    r, out, total = x.clone(), x.clone(), x.clone()
    for call, want in ((lambda: hp.gated_add_rms_norm(x, r, w, w, 1e-6, out=out, residual_out=total), [out, total]),
                       (lambda: hp.gated_add_rms_norm(x, r, w, w, 1e-6, out=out), [out, r]),
                       (lambda: hp.gated_add_rms_norm(x, r, w, w, 1e-6, out=out, residual_out=r), [out, r]),
                       (lambda: hp.rms_norm_int8(x, w, 1e-6, residual=r, residual_out=total), [total]),
                       (lambda: hp.rms_norm_int8(x, w, 1e-6, residual=r), [r]),
                       (lambda: hp.rms_norm_int8(x, w, 1e-6, residual=r, residual_out=r), [r]),
                       (lambda: hp.rms_norm_int8(x, w, 1e-6), [])):
        found, called = [], []
        with Written():
            call()
        assert {id(t) for t in found} == {id(t) for t in want}


    # By position an operator's name means the form that it always meant.
    ops = torch.ops.hp_rms_norm
    for call, want in ((lambda: ops.gated_add_rms_norm(out, r, total, x, w, w, None, 1.0, 1e-6), ops.gated_add_rms_norm.default),
                       (lambda: ops.rms_norm_int8(x, w, r, total, 1e-6), ops.rms_norm_int8.default)):
        found, called = [], []
        with Written():
            call()
        assert called == [want]


def test_no_cpu_kernels():
    x, w = torch.zeros(4, 8).bfloat16(), torch.ones(8).bfloat16()
    for call in (lambda: hp.gated_add_rms_norm(x, x.clone(), w, w, 1e-6), lambda: hp.rms_norm_int8(x, w, 1e-6),
                 lambda: hp.linear_log_probs(x, x, torch.zeros(4, dtype=torch.int64))):
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()
