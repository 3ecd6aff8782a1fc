"""Argument checks of include/msplat_ops.h and the generator of the dropout
masks. No GPU: a refused call returns before it touches any."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import _ops_ref as R  # noqa: E402

ARG = 1
P = 1 << 20  # an address that is aligned and never read


def lib():
    from msplat import ops
    return ops._lib()


def refused(code, text):
    assert code == ARG
    assert text in lib().msplat_last_error().decode()


def forward(m=4, n=3, k=8, x=P, ldx=8, w=P, ldw=8, bias=None, act=0, res=None, ldr=0, z=None, ldz=0, y=P, ldy=3, dt=0,
            ydt=0):
    return lib().msplat_linear_forward(m, n, k, x, ldx, w, ldw, bias, act, res, ldr, z, ldz, y, ldy, dt, ydt, None)


@pytest.mark.parametrize("args,text", [
    (dict(m=-1), "m must be"), (dict(n=0), "n must be"), (dict(k=0), "k must be"), (dict(m=1 << 31), "m must be"),
    (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(dt=1), "dtype"), (dict(dt=4, ydt=5), "y_dtype"),
    (dict(x=None), "x is null"), (dict(w=None), "w is null"), (dict(y=None), "y is null"), (dict(ldx=7), "x: the row stride"),
    (dict(ldw=7), "w: the row stride"), (dict(ldy=2), "y: the row stride"), (dict(x=P + 2), "x is not aligned"),
    (dict(bias=P + 1), "bias is not aligned"), (dict(res=P, ldr=2), "residual: the row stride"),
    (dict(z=P, ldz=2), "preact: the row stride"), (dict(ldx=1 << 62), "too large")])
def test_linear_forward_refusals(args, text):
    refused(forward(**args), text)


def test_linear_forward_without_rows_needs_nothing():
    assert forward(m=0, x=None, w=None, y=None) == 0


def backward(m=4, n=3, k=8, x=P, ldx=8, w=P, ldw=8, z=P, ldz=3, act=2, dy=P, lddy=3, dx=P, lddx=8, dw=P, lddw=8, db=P,
             dt=0, ws=P, size=1 << 30):
    return lib().msplat_linear_backward(m, n, k, x, ldx, w, ldw, z, ldz, act, dy, lddy, dx, lddx, dw, lddw, db, dt, ws,
                                        size, None)


@pytest.mark.parametrize("args,text", [
    (dict(n=0), "n must be"), (dict(act=9), "activation"), (dict(dt=3), "dtype"), (dict(x=None), "x is null"),
    (dict(w=None), "w is null"), (dict(dy=None), "dy is null"), (dict(z=None), "preact is null"),
    (dict(lddx=7), "dx: the row stride"), (dict(lddw=7), "dw: the row stride"), (dict(db=P + 1), "dbias is not aligned"),
    (dict(ws=None), "workspace is null"), (dict(ws=P + 16), "workspace is not aligned"), (dict(size=16), "too small")])
def test_linear_backward_refusals(args, text):
    refused(backward(**args), text)


def test_dropout_refusals():
    def call(rows=4, cols=8, x=P, ldx=8, res=None, ldr=0, y=P, ldy=8, p=0.5, dev=None, dt=0):
        return lib().msplat_dropout(rows, cols, x, ldx, res, ldr, y, ldy, p, 1, 2, dev, dt, None)
    for args, text in ((dict(rows=-1), "rows must be"), (dict(cols=-1), "cols must be"), (dict(p=-0.1), "p must be"),
                       (dict(p=1.01), "p must be"), (dict(p=float("nan")), "p must be"), (dict(x=None), "x is null"),
                       (dict(y=None), "y is null"), (dict(ldx=7), "x: the row stride"), (dict(dt=2), "dtype"),
                       (dict(res=P, ldr=7), "residual: the row stride"), (dict(dev=P + 4), "offset_dev")):
        refused(call(**args), text)
    assert call(rows=0, x=None, y=None) == 0 and call(cols=0, x=None, y=None) == 0


def test_loss_refusals():
    def call(m=4, v=5, d=8, x=P, ldx=8, w=P, ldw=8, t=P, scale=1.0, weight=1.0, loss=P, row=P, dx=P, lddx=8, dw=P, lddw=8,
             dt=0, ws=P, size=1 << 30):
        return lib().msplat_loss_cross_entropy(m, v, d, x, ldx, w, ldw, t, scale, weight, loss, row, dx, lddx, dw, lddw, dt,
                                               ws, size, None)
    for args, text in ((dict(v=0), "v must be"), (dict(d=0), "d must be"), (dict(m=-1), "m must be"), (dict(dt=9), "dtype"),
                       (dict(x=None), "x is null"), (dict(w=None), "w is null"), (dict(t=None), "targets is null"),
                       (dict(t=P + 2), "targets is not aligned"), (dict(scale=float("inf")), "finite"),
                       (dict(weight=float("nan")), "finite"), (dict(lddx=7), "dx: the row stride"),
                       (dict(loss=P + 1), "loss is not aligned"), (dict(row=P + 2), "row_loss is not aligned"),
                       (dict(ws=None), "workspace is null"), (dict(ws=P + 128), "workspace is not aligned"),
                       (dict(size=1000), "too small")):
        refused(call(**args), text)


def test_workspaces_are_bounded():
    """Working memory does not grow with the logits: a million rows against 100,000 labels."""
    size = C.c_uint64()
    assert lib().msplat_loss_cross_entropy_workspace(1_000_000, 100_000, 64, 1, 5, C.byref(size)) == 0
    assert size.value < 2 << 30
    assert lib().msplat_loss_cross_entropy_workspace(1_000_000, 100_000, 64, 0, 5, C.byref(size)) == 0
    assert size.value < 256 << 20
    refused(lib().msplat_loss_cross_entropy_workspace(1, 1, 0, 1, 5, C.byref(size)), "d must be")
    refused(lib().msplat_linear_backward_workspace(1, 1, 1, 0, 0, None), "bytes is null")
    assert lib().msplat_linear_backward_workspace(0, 1, 1, 0, 0, C.byref(size)) == 0 and size.value == 0


def test_cpu_tensors_are_refused():
    from msplat import ops
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    for f in (lambda: ops.linear_forward(x, w), lambda: ops.linear_backward(x, w, torch.zeros(2, 3)),
              lambda: ops.dropout(x, 0.5, 1), lambda: ops.loss_cross_entropy(x, w, torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ops.MsplatError, match="CUDA tensors"):
            f()


def test_generator_known_answers():
    """Philox4x32-10 against the known answers published with it (Random123's kat_vectors)."""
    for ctr, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        got = R.philox4x32_10([np.array([c]) for c in ctr], key)
        assert tuple(int(g[0]) for g in got) == want
    d = R.draws(80_000, 3, 9)
    assert d.min() >= 0 and d.max() < 65536 and abs(d.mean() - 32767.5) < 5 * 65536 / (12 * 80_000) ** 0.5
    assert np.array_equal(R.draws(20, 3, 9, first=13), d[13:33])
