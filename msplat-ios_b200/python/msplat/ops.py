"""Operators for learned per-Gaussian attributes (include/msplat_ops.h).

Fully connected layers with their gradients, dropout, and a label loss with
its gradients, on torch CUDA tensors. Matrices are 2-D tensors whose columns
are contiguous (a slice of columns of a wider tensor will do), of one type per
call: float32, float16 or bfloat16. The calls run on `stream` (by default the
current stream of the tensors' device); results and workspaces come from
torch's allocator on that stream, so calls on several streams, and calls
captured into CUDA graphs, do not share any. A `stream` that is given has to wait
for whatever writes the call's inputs (Stream.wait_stream), and whoever reads the
results elsewhere for it; the inputs' memory is kept until it has used them, even
if they are freed. Gradients come from the calls for them, not from autograd: the
results of tensors that require one are not part of its graph. There is no CPU or
PyTorch fallback: a refused or failed call raises MsplatError.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._backend import MsplatError, load

__all__ = ["linear_forward", "linear_backward", "dropout", "loss_cross_entropy", "ACTIVATIONS", "status", "MsplatError"]

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
_DTYPES = {torch.float32: 0, torch.float16: 4, torch.bfloat16: 5}
_ERR_ARGUMENT = 1

_L = None


def _lib():
    global _L
    if _L is not None:
        return _L
    L = load()
    vp, f, i32, i64, u64, pu64 = C.c_void_p, C.c_float, C.c_int32, C.c_int64, C.c_uint64, C.POINTER(C.c_uint64)
    L.msplat_linear_forward.argtypes = [i64, i64, i64, vp, i64, vp, i64, vp, i32, vp, i64, vp, i64, vp, i64, i32, i32,
                                        vp]
    L.msplat_linear_backward_workspace.argtypes = [i64, i64, i64, i32, i32, pu64]
    L.msplat_linear_backward.argtypes = [i64, i64, i64, vp, i64, vp, i64, vp, i64, i32, vp, i64, vp, i64, vp, i64, vp,
                                         i32, vp, u64, vp]
    L.msplat_dropout.argtypes = [i64, i64, vp, i64, vp, i64, vp, i64, f, u64, u64, vp, i32, vp]
    L.msplat_loss_cross_entropy_workspace.argtypes = [i64, i64, i64, i32, i32, pu64]
    L.msplat_loss_cross_entropy.argtypes = [i64, i64, i64, vp, i64, vp, i64, vp, f, f, vp, vp, vp, i64, vp, i64, i32,
                                            vp, u64, vp]
    L.msplat_ops_status.argtypes = [vp]
    L.msplat_ops_rehearse_timeout.argtypes = [i32, vp]
    for name in ("msplat_linear_forward", "msplat_linear_backward_workspace", "msplat_linear_backward",
                 "msplat_dropout", "msplat_loss_cross_entropy_workspace", "msplat_loss_cross_entropy",
                 "msplat_ops_status", "msplat_ops_rehearse_timeout"):
        getattr(L, name).restype = C.c_int
    _L = L
    return L


def _check(code: int):
    if code:
        raise MsplatError(code, _L.msplat_last_error().decode())


def _refuse(msg: str):
    raise MsplatError(_ERR_ARGUMENT, msg)


def _matrix(t, name, device, dtype, rows=None, cols=None):
    """(address, row stride) of a matrix argument, or (None, 0) for None."""
    if t is None:
        return None, 0
    if t.dtype != dtype:
        _refuse(f"{name} must be {dtype}")
    if t.device != device:
        _refuse(f"{name} must be on {device}")
    shape = t.shape
    if len(shape) != 2 or (rows is not None and (shape[0] != rows or shape[1] != cols)):
        _refuse(f"{name} must have the shape ({rows}, {cols})" if rows is not None else f"{name} must be a matrix")
    s0, s1 = t.stride()
    if s1 != 1 and shape[1] > 1:
        _refuse(f"the columns of {name} must be contiguous")
    if s0 < shape[1]:
        if shape[0] > 1:
            _refuse(f"the rows of {name} overlap")
        s0 = shape[1]
    return t.data_ptr(), s0


def _vector(t, name, device, dtype, size):
    if t is None:
        return None
    if t.device != device or t.dtype != dtype or t.shape != (size,) or (size > 1 and t.stride(0) != 1):
        _refuse(f"{name} must be a contiguous {dtype} vector of {size} on {device}")
    return t.data_ptr()


def _dtype(x):
    code = _DTYPES.get(x.dtype) if isinstance(x, torch.Tensor) else None
    if code is None:
        _refuse("float32, float16 or bfloat16 tensors are needed")
    if not x.is_cuda:
        _refuse("CUDA tensors are needed")
    return code


def _rows(w, name):
    if not isinstance(w, torch.Tensor) or w.dim() != 2:
        _refuse(f"{name} must be a matrix")
    return w.shape[0]


def _act(name):
    code = ACTIVATIONS.get(name)
    return code if code is not None else _refuse(f"unknown activation {name!r}")


def _enter(device, stream):
    """Makes the call's device and stream current, where they are not, so that
    what is allocated belongs to the stream: the contexts to leave again."""
    if stream is None and device.index == _current_device():
        return ()
    entered = []
    if device.index != _current_device():
        entered.append(torch.cuda.device(device))
    if stream is not None:
        if stream.device != device:
            _refuse("the stream belongs to another device than the tensors")
        entered.append(torch.cuda.stream(stream))
    for c in entered:
        c.__enter__()
    return entered


def _leave(entered):
    for c in reversed(entered):
        c.__exit__(None, None, None)


def _used(stream, *tensors):
    """Keeps the memory of the caller's tensors, should they be freed, until the
    stream that was given has used them."""
    if stream is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _handle(device):
    """The address of the current stream."""
    return _raw_stream(device.index)


def _current_device():
    return torch.cuda.current_device()


def _raw_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


# the same without the objects around them, where torch has that
_current_device = getattr(torch._C, "_cuda_getDevice", _current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def _workspace(size_fn, device, *args):
    size = C.c_uint64()
    _check(size_fn(*args, C.byref(size)))
    # torch's blocks are 512-byte aligned
    return torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None, size.value


def linear_forward(x, w, bias=None, activation="none", residual=None, preact=None, out=None, out_dtype=None,
                   stream=None):
    """y = act(x @ w.T + bias) + residual for x [m, k] and w [n, k].

    activation: one of ACTIVATIONS. out_dtype: x's type (default) or float32,
    the type of residual, preact and the result. preact [m, n], when given,
    receives the activation's argument, which linear_backward needs (in x's type:
    with out_dtype float32 and 16-bit x, convert preact and dy for it). out [m,
    n], when given, receives the result (it may be residual itself)."""
    L = _lib()
    dt = _dtype(x)
    device, (m, k) = x.device, x.shape if x.dim() == 2 else _refuse("x must be a matrix")
    n = _rows(w, "w")
    if out_dtype is None:
        out_dtype = x.dtype if out is None else out.dtype
    if out_dtype != x.dtype and out_dtype != torch.float32:
        _refuse("out_dtype must be x's type or float32")
    px, ldx = _matrix(x, "x", device, x.dtype)
    pw, ldw = _matrix(w, "w", device, x.dtype, n, k)
    pb = _vector(bias, "bias", device, x.dtype, n)
    pr, ldr = _matrix(residual, "residual", device, out_dtype, m, n)
    pz, ldz = _matrix(preact, "preact", device, out_dtype, m, n)
    act = _act(activation)
    entered = _enter(device, stream)
    try:
        if out is None:
            out = x.new_empty((m, n)) if out_dtype == x.dtype else x.new_empty((m, n), dtype=out_dtype)
            py, ldy = out.data_ptr(), n
        else:
            py, ldy = _matrix(out, "out", device, out_dtype, m, n)
        _check(L.msplat_linear_forward(m, n, k, px, ldx, pw, ldw, pb, act, pr, ldr, pz, ldz, py, ldy, dt,
                                       _DTYPES[out_dtype], _handle(device)))
        _used(stream, x, w, bias, residual, preact, out)
    finally:
        _leave(entered)
    return out


def linear_backward(x, w, dy, preact=None, activation="none", need_dx=True, need_dw=True, need_dbias=True,
                    stream=None):
    """Gradients (dx [m, k], dw [n, k], dbias [n]) of linear_forward from dy
    [m, n] and, unless activation is "none", the preact of the forward. A
    gradient that is not needed is None; the residual's gradient is dy."""
    L = _lib()
    dt = _dtype(x)
    device, (m, k) = x.device, x.shape if x.dim() == 2 else _refuse("x must be a matrix")
    n = _rows(w, "w")
    px, ldx = _matrix(x, "x", device, x.dtype)
    pw, ldw = _matrix(w, "w", device, x.dtype, n, k)
    pdy, lddy = _matrix(dy, "dy", device, x.dtype, m, n)
    act = _act(activation)
    if act and preact is None:
        _refuse("preact is needed for this activation")
    pz, ldz = _matrix(preact, "preact", device, x.dtype, m, n) if act else (None, 0)
    entered = _enter(device, stream)
    try:
        new = lambda *shape: x.new_empty(shape)  # noqa: E731
        dx = new(m, k) if need_dx else None
        dw = new(n, k) if need_dw else None
        dbias = new(n) if need_dbias else None
        ws, size = _workspace(L.msplat_linear_backward_workspace, device, m, n, k, act, dt)
        _check(L.msplat_linear_backward(m, n, k, px, ldx, pw, ldw, pz, ldz, act, pdy, lddy,
                                        dx.data_ptr() if need_dx else None, k, dw.data_ptr() if need_dw else None, k,
                                        dbias.data_ptr() if need_dbias else None, dt,
                                        ws.data_ptr() if size else None, size, _handle(device)))
        _used(stream, x, w, dy, preact)
    finally:
        _leave(entered)
    return dx, dw, dbias


def dropout(x, p, seed, offset=0, residual=None, out=None, offset_dev=None, stream=None):
    """residual + x * keep / (1 - p). The mask is a function of (seed, offset
    + offset_dev, element) and never stored: the same call on the gradient
    (without residual) is the backward pass. seed and offset: integers in [0,
    2^64); offset_dev: an int64 CUDA tensor of one element, read when the
    kernel runs, so that each replay of a captured graph can have its own
    mask. out may be x or residual."""
    L = _lib()
    dt = _dtype(x)
    device, (m, n) = x.device, x.shape if x.dim() == 2 else _refuse("x must be a matrix")
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        _refuse("seed and offset must be in [0, 2^64)")
    px, ldx = _matrix(x, "x", device, x.dtype)
    pr, ldr = _matrix(residual, "residual", device, x.dtype, m, n)
    po = _vector(offset_dev, "offset_dev", device, torch.int64, 1)
    entered = _enter(device, stream)
    try:
        if out is None:
            out = x.new_empty((m, n))
            py, ldy = out.data_ptr(), n
        else:
            py, ldy = _matrix(out, "out", device, x.dtype, m, n)
        _check(L.msplat_dropout(m, n, px, ldx, pr, ldr, py, ldy, p, seed, offset, po, dt, _handle(device)))
        _used(stream, x, residual, out, offset_dev)
    finally:
        _leave(entered)
    return out


def loss_cross_entropy(x, w, targets, logit_scale=1.0, weight=1.0, grad=True, stream=None):
    """Softmax cross entropy of the rows of x [m, d] against the label
    embeddings w [v, d]: (loss, row_loss [m], dx, dw), with
    row_loss = logsumexp(l) - l[target] of l = logit_scale * x @ w.T and loss =
    weight * the mean over the labelled rows. targets: int32 [m]; a row whose
    target is outside [0, v) has no label and counts for nothing. dx and dw are
    the gradients of loss (None without grad). The logits are never kept."""
    L = _lib()
    dt = _dtype(x)
    device, (m, d) = x.device, x.shape if x.dim() == 2 else _refuse("x must be a matrix")
    v = _rows(w, "w")
    px, ldx = _matrix(x, "x", device, x.dtype)
    pw, ldw = _matrix(w, "w", device, x.dtype, v, d)
    pt = _vector(targets, "targets", device, torch.int32, m)
    entered = _enter(device, stream)
    try:
        loss = torch.empty((), dtype=torch.float32, device=device)
        row_loss = torch.empty(m, dtype=torch.float32, device=device)
        dx = torch.empty((m, d), dtype=x.dtype, device=device) if grad else None
        dw = torch.empty((v, d), dtype=x.dtype, device=device) if grad else None
        ws, size = _workspace(L.msplat_loss_cross_entropy_workspace, device, m, v, d, 1 if grad else 0, dt)
        _check(L.msplat_loss_cross_entropy(m, v, d, px, ldx, pw, ldw, pt, logit_scale, weight, loss.data_ptr(),
                                           row_loss.data_ptr(), dx.data_ptr() if grad else None, d,
                                           dw.data_ptr() if grad else None, d, dt, ws.data_ptr() if size else None,
                                           size, _handle(device)))
        _used(stream, x, w, targets)
    finally:
        _leave(entered)
    return loss, row_loss, dx, dw


def status(stream=None):
    """Waits for the stream and raises MsplatError when a kernel on any stream of
    its device gave up waiting since the last call for this stream (its waits are
    bounded)."""
    s = stream if stream is not None else torch.cuda.current_stream()
    L = _lib()
    with torch.cuda.device(s.device):
        _check(L.msplat_ops_status(s.cuda_stream))
