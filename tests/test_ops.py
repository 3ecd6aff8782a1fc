"""The operators of msplat.ops against their 64-bit forms (GPU)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import _ops_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = ("f32", "f16", "bf16")
ACTS = ("none", "relu", "gelu", "silu", "sigmoid")


def ops():
    from msplat import ops as o
    return o


def normal(seed, rows, cols, t, std=1.0, pad=0, lead=None):
    """[rows, cols] inside a matrix of cols + pad columns, starting at column lead."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    full = (torch.randn(rows, cols + pad, generator=g, device="cuda") * std).to(R.TYPES[t])
    lead = pad // 2 if lead is None else lead
    return full[:, lead:lead + cols]


def guarded(rows, cols, t, pad=3, behind=2):
    """An output view inside a buffer of a marker value, and a check that only the view was written."""
    full = torch.full((rows + behind, cols + 2 * pad), 77.0, dtype=t, device="cuda")
    view = full[:rows, pad:pad + cols]

    def untouched():
        rest = full.clone()
        rest[:rows, pad:pad + cols] = 77.0
        return bool((rest == 77.0).all())
    return view, untouched


# m, n, k: one of everything, below and above every tile, odd and round, long reductions
LAYERS = [(1, 1, 1), (1, 3, 5), (1, 512, 512), (2, 64, 32), (5, 7, 1000), (8, 130, 64), (9, 16, 16), (33, 65, 17),
          (64, 64, 64), (100, 3, 61), (128, 128, 64), (129, 257, 65), (200, 40, 72), (257, 96, 200), (1000, 256, 128),
          (300, 512, 320), (3, 1000, 1024), (1, 40, 4099), (20, 200, 2056), (5000, 24, 40)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", LAYERS)
def test_linear_forward(m, n, k, t):
    act = ACTS[(m + n + k) % 5]
    x, w = normal(1, m, k, t), normal(2, n, k, t, std=k ** -0.5)
    bias, res = normal(3, 1, n, t)[0], normal(4, m, n, t)
    z = torch.empty(m, n, dtype=R.TYPES[t], device="cuda")
    y = ops().linear_forward(x, w, bias, activation=act, residual=res, preact=z)
    want, bound, wz, bz = R.linear(x, w, bias, act, res, R.TYPES[t])
    R.check(y, want, bound, "y")
    R.check(z, wz, bz, "preact")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(act, t):
    m, n, k = 130, 70, 24
    x, w = normal(5, m, k, t, std=3.0), normal(6, n, k, t)
    y = ops().linear_forward(x, w, activation=act)
    want, bound, _, _ = R.linear(x, w, None, act, None, R.TYPES[t])
    R.check(y, want, bound, "y")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad,lead", [(8, 0), (8, 8), (5, 1), (1, 1), (40, 16)])
@pytest.mark.parametrize("m,n,k", [(1, 64, 40), (70, 33, 40), (300, 130, 136), (513, 3, 64)])
def test_linear_strides(m, n, k, pad, lead, t):
    """Columns of wider records at any alignment, an output inside a wider record, residual in place."""
    x, w = normal(7, m, k, t, pad=pad, lead=lead), normal(8, n, k, t, std=k ** -0.5, pad=pad, lead=lead)
    out, untouched = guarded(m, n, R.TYPES[t], pad=pad)
    res = normal(9, m, n, t)
    out.copy_(res)
    z, z_untouched = guarded(m, n, R.TYPES[t], pad=3)
    y = ops().linear_forward(x, w, activation="silu", residual=out, preact=z, out=out)
    want, bound, wz, bz = R.linear(x, w, None, "silu", res, R.TYPES[t])
    assert y is out
    R.check(y, want, bound, "y")
    R.check(z, wz, bz, "preact")
    assert untouched() and z_untouched()


@pytest.mark.parametrize("t", ("f16", "bf16"))
@pytest.mark.parametrize("m,n,k", [(1, 3, 64), (700, 3, 61), (300, 130, 512)])
def test_linear_f32_output(m, n, k, t):
    x, w, res = normal(10, m, k, t), normal(11, n, k, t, std=k ** -0.5), normal(12, m, n, "f32")
    y = ops().linear_forward(x, w, normal(13, 1, n, t)[0], activation="sigmoid", residual=res, out_dtype=torch.float32)
    want, bound, _, _ = R.linear(x, w, normal(13, 1, n, t)[0], "sigmoid", res, torch.float32)
    assert y.dtype == torch.float32
    R.check(y, want, bound, "y")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", LAYERS)
def test_linear_backward(m, n, k, t):
    act = ACTS[(m + n + k + 1) % 5]
    x, w = normal(14, m, k, t), normal(15, n, k, t, std=k ** -0.5)
    z, dy = normal(16, m, n, t), normal(17, m, n, t)
    dx, dw, db = ops().linear_backward(x, w, dy, preact=z, activation=act)
    for got, (want, bound), name in zip((dx, dw, db), R.linear_grads(x, w, dy, z, act, R.TYPES[t]), ("dx", "dw", "dbias")):
        assert got.dtype == R.TYPES[t]
        R.check(got, want, bound, name)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", (20_000, 100_003))
def test_linear_backward_many_rows(m, t):
    n, k = 64, 40
    x, w = normal(18, m, k, t), normal(19, n, k, t, std=k ** -0.5)
    z, dy = normal(20, m, n, t), normal(21, m, n, t)
    dx, dw, db = ops().linear_backward(x, w, dy, preact=z, activation="gelu")
    for got, (want, bound), name in zip((dx, dw, db), R.linear_grads(x, w, dy, z, "gelu", R.TYPES[t]),
                                        ("dx", "dw", "dbias")):
        R.check(got, want, bound, name)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("pad,lead", [(0, 0), (13, 10), (8, 8)])
def test_linear_backward_strides(pad, lead, act, t):
    """dy as columns 10 .. of a wider record, as the colour gradients are."""
    m, n, k = 333, 3, 20
    x, w = normal(22, m, k, t, pad=pad, lead=lead), normal(23, n, k, t, pad=pad, lead=lead)
    z, dy = normal(24, m, n, t, pad=pad, lead=lead), normal(25, m, n, t, pad=pad, lead=lead)
    dx, dw, db = ops().linear_backward(x, w, dy, preact=z, activation=act)
    for got, (want, bound), name in zip((dx, dw, db), R.linear_grads(x, w, dy, z, act, R.TYPES[t]), ("dx", "dw", "dbias")):
        R.check(got, want, bound, name)


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 0, 0)])
def test_linear_backward_parts(need):
    """Each gradient alone equals the one computed with the others, bit for bit."""
    x, w, z, dy = normal(26, 300, 48, "f32"), normal(27, 40, 48, "f32"), normal(28, 300, 40, "f32"), normal(29, 300, 40, "f32")
    full = ops().linear_backward(x, w, dy, preact=z, activation="gelu")
    part = ops().linear_backward(x, w, dy, preact=z, activation="gelu", need_dx=bool(need[0]), need_dw=bool(need[1]),
                                 need_dbias=bool(need[2]))
    for a, b, n in zip(full, part, need):
        assert (b is None) == (not n)
        assert b is None or torch.equal(a, b)


@pytest.mark.parametrize("act", ACTS)
def test_linear_gradients_against_differences(act):
    """dx, dw and dbias against central differences of the 32-bit forward, with weights w_ij of a scalar loss."""
    m, n, k, e = 12, 9, 7, 2.0 ** -7
    x, w, b = normal(30, m, k, "f32"), normal(31, n, k, "f32"), normal(32, 1, n, "f32")[0]
    dy = normal(33, m, n, "f32")
    z = torch.empty(m, n, device="cuda")
    ops().linear_forward(x, w, b, activation=act, preact=z)
    dx, dw, db = ops().linear_backward(x, w, dy, preact=z, activation=act)

    def value(x, w, b):
        return (ops().linear_forward(x, w, b, activation=act).double() * dy.double()).sum()
    for p, grad, pick in ((x, dx, 0), (w, dw, 1), (b, db, 2)):
        step = torch.randn_like(p) * e
        args = [x, w, b]
        args[pick] = p + step
        up = value(*args)
        args[pick] = p - step
        down = value(*args)
        want = float((grad.double() * step.double()).sum())
        # third derivatives are below 2 and |step| <= ~4 e: the difference is off by e^3-sized terms, relu by the
        # few arguments that change their sign within the step
        size = float((grad.double().abs() * step.double().abs()).sum()) + 1e-6
        assert abs(float(up - down) / 2 - want) <= (0.25 if act == "relu" else 0.02) * size


@pytest.mark.parametrize("t", TYPES)
def test_linear_no_rows(t):
    x, w = normal(34, 0, 8, t), normal(35, 5, 8, t)
    assert ops().linear_forward(x, w, activation="gelu").shape == (0, 5)
    dx, dw, db = ops().linear_backward(x, w, normal(36, 0, 5, t))
    assert dx.shape == (0, 8) and not dw.any() and not db.any() and dw.shape == (5, 8)


# ---- dropout ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 8), (5, 9), (1000, 33), (257, 64), (1, 100_001), (2049, 40)])
@pytest.mark.parametrize("p", (0.0, 0.1, 0.5, 1.0))
def test_dropout(rows, cols, p, t):
    x, res = normal(40, rows, cols, t), normal(41, rows, cols, t)
    seed, offset = 0xFEDCBA9876543210, (5 << 32) + 3
    for r in (None, res):
        y = ops().dropout(x, p, seed, offset, residual=r)
        want, bound = R.dropout(x, p, seed, offset, r, R.TYPES[t])
        R.check(y, want, bound, "y")
        # a dropped element adds exactly nothing
        keep = torch.from_numpy(R.draws(x.numel(), seed, offset) >= int(p * 65536 + 0.5)).reshape(x.shape).cuda()
        assert torch.equal(y[~keep], (torch.zeros_like(x) if r is None else r)[~keep])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad,lead", [(8, 0), (8, 8), (5, 1), (1, 1)])
@pytest.mark.parametrize("rows,cols", [(1, 40), (300, 40), (77, 13)])
def test_dropout_strides_and_in_place(rows, cols, pad, lead, t):
    x = normal(42, rows, cols, t, pad=pad, lead=lead)
    plain = ops().dropout(x.contiguous(), 0.3, 9, 1)
    out, untouched = guarded(rows, cols, R.TYPES[t], pad=pad)
    out.copy_(x)
    ops().dropout(out, 0.3, 9, 1, out=out)
    assert torch.equal(out, plain) and untouched()
    assert torch.equal(ops().dropout(x, 0.3, 9, 1), plain)
    res = normal(43, rows, cols, t)
    want = ops().dropout(x, 0.3, 9, 1, residual=res)
    ops().dropout(x, 0.3, 9, 1, residual=res, out=res)
    assert torch.equal(res, want)


@pytest.mark.parametrize("t", TYPES)
def test_dropout_masked_values(t):
    """Infinities and NaN in dropped places do not come through; kept ones do."""
    x = torch.full((64, 40), float("nan"), dtype=R.TYPES[t], device="cuda")
    x[::2] = float("inf")
    y = ops().dropout(x, 0.5, 3, 4)
    keep = torch.from_numpy(R.draws(x.numel(), 3, 4) >= 32768).reshape(x.shape).cuda()
    assert not y[~keep].any() and not bool(torch.isfinite(y[keep]).any())


def test_dropout_far_elements():
    """Blocks of elements past 2^32: their draws, read through a column of a tall matrix's last rows."""
    rows, cols = (1 << 29) + 5, 9  # 4.8e9 elements of 16 bits
    x = torch.ones(rows, cols, dtype=torch.float16, device="cuda")
    y = ops().dropout(x, 0.5, 11, 12, out=x)
    first = (rows - 4) * cols
    keep = torch.from_numpy(R.draws(4 * cols, 11, 12, first=first) >= 32768).reshape(4, cols).cuda()
    assert torch.equal(y[-4:] != 0, keep)


def test_dropout_offset_on_the_device():
    x = normal(44, 100, 33, "f32")
    dev = torch.tensor([1000], device="cuda")
    assert torch.equal(ops().dropout(x, 0.5, 1, 5, offset_dev=dev), ops().dropout(x, 0.5, 1, 1005))
    assert not torch.equal(ops().dropout(x, 0.5, 1, 5), ops().dropout(x, 0.5, 1, 1005))


# ---- label loss ------------------------------------------------------------------------------------------------------

# m, v, d
LOSSES = [(1, 1, 1), (1, 2, 3), (1, 1000, 64), (16, 5000, 256), (5, 7, 200), (64, 64, 32), (100, 101, 32), (129, 257, 65),
          (300, 33, 8), (257, 1030, 72), (1000, 10, 16), (70, 20_000, 40), (5000, 130, 24), (200, 300, 1000)]


def labels(seed, m, v, off=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, v, (m,), generator=g, device="cuda", dtype=torch.int32)
    drop = torch.rand(m, generator=g, device="cuda") < off
    return torch.where(drop, torch.tensor([-1, v, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device="cuda")[
        torch.arange(m, device="cuda") % 4], t)


def check_loss(x, w, t, scale, weight):
    loss, row, dx, dw = ops().loss_cross_entropy(x, w, t, logit_scale=scale, weight=weight)
    want = R.loss(x, w, t, scale, weight, x.dtype)
    for got, name in ((loss, "loss"), (row, "row_loss"), (dx, "dx"), (dw, "dw")):
        R.check(got, *want[name], name)
    only = ops().loss_cross_entropy(x, w, t, logit_scale=scale, weight=weight, grad=False)
    assert only[2] is None and only[3] is None
    assert torch.equal(only[0], loss) and torch.equal(only[1], row)
    return loss, row, dx, dw


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,v,d", LOSSES)
def test_loss(m, v, d, t):
    x, w = normal(50, m, d, t, std=2.0), normal(51, v, d, t, std=d ** -0.5)
    check_loss(x, w, labels(52, m, v), 1.0 if m % 2 else 3.0, 4096.0 if t == "f16" else 1.0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad,lead", [(8, 0), (8, 8), (5, 1)])
def test_loss_strides(pad, lead, t):
    x, w = normal(53, 150, 40, t, pad=pad, lead=lead), normal(54, 210, 40, t, pad=pad, lead=lead)
    check_loss(x, w, labels(55, 150, 210), 1.0, 1.0)


@pytest.mark.parametrize("t", TYPES)
def test_loss_without_labels(t):
    """No row has a label; rows without one may hold anything."""
    x, w = normal(56, 140, 32, t), normal(57, 60, 32, t)
    x[::3] = float("nan")
    x[1::3] = float("inf")
    for off in (1.0, 0.5):
        t_ = labels(58, 140, 60, off=off)
        if off < 1:
            known = (t_ >= 0) & (t_ < 60)
            x[known] = normal(59, 140, 32, t)[known]
        loss, row, dx, dw = check_loss(x, w, t_, 1.0, 2.0)
        if off == 1:
            assert float(loss) == 0 and not row.any() and not dx.any() and not dw.any()
    none = ops().loss_cross_entropy(x[:0], w, t_[:0])
    assert float(none[0]) == 0 and none[1].shape == (0,) and none[2].shape == (0, 32) and not none[3].any()


@pytest.mark.parametrize("t", TYPES)
def test_loss_extreme_logits(t):
    """Logits far below the largest, as a mask of the type's lowest value gives, and far above zero: no overflow and exact
    zeros. The rows' logits are large * (1, 0, -1, ...) with the label on the largest."""
    big = {"f32": 1e30, "bf16": 1e30, "f16": 6e4}[t]
    x = torch.zeros(40, 16, dtype=R.TYPES[t], device="cuda")
    x[:, 0] = big
    w = torch.zeros(50, 16, dtype=R.TYPES[t], device="cuda")
    w[3, 0], w[4:, 0] = 1, -1
    targets = torch.full((40,), 3, dtype=torch.int32, device="cuda")
    loss, row, dx, dw = ops().loss_cross_entropy(x, w, targets)
    assert float(loss) == 0 and not row.any() and not dx.any() and not dw.any()
    targets[:] = 0
    loss, row, dx, dw = ops().loss_cross_entropy(x, w, targets, weight=1.0)
    # log2(e), ln(2) and the two products with them are each off by 2^-24 at most
    assert torch.allclose(row, x[:, 0].float(), rtol=4 * 2.0 ** -24, atol=0) and bool(torch.isfinite(dx).all())
    assert torch.allclose(dx[:, 0].float(), torch.full((40,), 1 / 40, device="cuda"), rtol=2 * R.HALF_STEP[R.TYPES[t]] + 1e-6)


@pytest.mark.parametrize("t", TYPES)
def test_loss_pieces(t):
    """More logits than are handled at a time, on both ways of cutting them."""
    big = 4 if t == "f32" else 2
    for m, v, d in ((3000, (300 << 20) // (3000 * big), 16), ((300 << 20) // (1000 * big), 1000, 16)):
        x, w = normal(60, m, d, t), normal(61, v, d, t)
        check_loss(x, w, labels(62, m, v), 1.0, 1024.0 if t == "f16" else 1.0)
        torch.cuda.empty_cache()


def test_loss_gradients_against_differences():
    m, v, d, e = 20, 30, 12, 2.0 ** -6
    x, w, t = normal(63, m, d, "f32"), normal(64, v, d, "f32"), labels(65, m, v)
    _, _, dx, dw = ops().loss_cross_entropy(x, w, t, logit_scale=1.5, weight=10.0)
    for p, grad in ((x, dx), (w, dw)):
        step = torch.randn_like(p) * e
        f = lambda q: float(ops().loss_cross_entropy(*((q, w) if p is x else (x, q)), t, logit_scale=1.5, weight=10.0,  # noqa: E731
                                                     grad=False)[0])
        want = float((grad.double() * step.double()).sum())
        size = float((grad.double().abs() * step.double().abs()).sum())
        assert abs((f(p + step) - f(p - step)) / 2 - want) <= 0.02 * size


# ---- how the calls behave --------------------------------------------------------------------------------------------


def everything(t, seed, offset_dev=None, stream=None):
    """One call of each operator: inputs and a function that makes the calls."""
    x, w, b = normal(seed, 700, 96, t), normal(seed + 1, 200, 96, t, std=0.1), normal(seed + 2, 1, 200, t)[0]
    table, tg = normal(seed + 3, 900, 200, t, std=0.1), labels(seed + 4, 700, 900)

    def call():
        with torch.cuda.stream(stream):  # what a stream writes is allocated on it
            z = torch.empty(700, 200, dtype=x.dtype, device="cuda")
        y = ops().linear_forward(x, w, b, activation="gelu", preact=z, stream=stream)
        y = ops().dropout(y, 0.2, 7, 0, offset_dev=offset_dev, stream=stream)
        loss, row, dy, dt = ops().loss_cross_entropy(y, table, tg, weight=100.0, stream=stream)
        dh = ops().dropout(dy, 0.2, 7, 0, offset_dev=offset_dev, stream=stream)
        return (z, y, loss, row, dy, dt, *ops().linear_backward(x, w, dh, preact=z, activation="gelu", stream=stream))
    return x, call


@pytest.mark.parametrize("t", TYPES)
def test_same_bits_every_time_and_on_any_stream(t):
    _, call = everything(t, 70)
    first = call()
    side = torch.cuda.Stream()
    _, on_side = everything(t, 70, stream=side)
    torch.cuda.synchronize()
    runs = [call(), on_side(), call(), on_side()]  # two streams at once, each with its own workspaces
    torch.cuda.synchronize()
    for r in runs:
        for a, b in zip(first, r):
            assert torch.equal(a, b)


@pytest.mark.parametrize("t", TYPES)
def test_captured_and_replayed(t):
    """A captured run on new inputs, with another mask each time, equals an eager one; two graphs replayed on two streams
    do not disturb each other."""
    dev = torch.zeros(1, dtype=torch.int64, device="cuda")
    x, call = everything(t, 80, offset_dev=dev)
    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for k in range(2):
        x.copy_(normal(90 + k, 700, 96, t))
        dev.fill_(17 + k)
        want = call()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(want, out):
                assert torch.equal(a, b)
    del graphs


def test_refusals_on_the_device():
    o = ops()
    x, w = normal(1, 4, 8, "f32"), normal(2, 3, 8, "f32")
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [lambda: o.linear_forward(x, w.half()), lambda: o.linear_forward(x, w[:, :7]), lambda: o.linear_forward(x.t(), w),
           lambda: o.linear_forward(x, w, activation="tanh"), lambda: o.linear_forward(x, w, bias=w[0]),
           lambda: o.linear_forward(x, w.cpu()), lambda: o.linear_forward(x, w, out_dtype=torch.float16),
           lambda: o.linear_forward(x[:, :0], w[:, :0]), lambda: o.linear_forward(x.double(), w.double()),
           lambda: o.linear_forward(x, w, residual=x), lambda: o.linear_forward(x[0], w),
           lambda: o.linear_forward(x[:1].expand(4, 8), w),
           lambda: o.linear_backward(x, w, x[:, :3], activation="gelu"), lambda: o.linear_backward(x, w, x),
           lambda: o.dropout(x, 1.5, 0), lambda: o.dropout(x, float("nan"), 0), lambda: o.dropout(x, 0.5, -1),
           lambda: o.dropout(x, 0.5, 0, residual=w), lambda: o.dropout(x, 0.5, 0, offset_dev=t),
           lambda: o.loss_cross_entropy(x, w, t.long()), lambda: o.loss_cross_entropy(x, w, t[:3]),
           lambda: o.loss_cross_entropy(x, w[:0], t), lambda: o.loss_cross_entropy(x, w, t, weight=float("inf")),
           lambda: o.loss_cross_entropy(x, w, t, logit_scale=float("nan"))]
    for k, f in enumerate(bad):
        with pytest.raises(o.MsplatError):
            f()
            pytest.fail(f"call {k} was not refused")
    R.check(o.linear_forward(x, w), *R.linear(x, w, None, "none", None, torch.float32)[:2], "y after refusals")


# ---- few outputs, many rows ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(4096, 1, 1), (5000, 3, 61), (4100, 4, 64), (4099, 7, 33), (4097, 16, 200), (4096, 9, 1030),
                                   (4100, 3, 2600)])
@pytest.mark.parametrize("pad,lead", [(0, 0), (3, 1), (8, 8)])
def test_linear_few_outputs(m, n, k, pad, lead, t):
    act = ACTS[(m + n + k) % 5]
    x, w, b = normal(100, m, k, t, pad=pad, lead=lead), normal(101, n, k, t, std=k ** -0.5), normal(102, 1, n, t)[0]
    res = normal(103, m, n, t)
    z, z_untouched = guarded(m, n, R.TYPES[t])
    out, untouched = guarded(m, n, R.TYPES[t])
    ops().linear_forward(x, w, b, activation=act, residual=res, preact=z, out=out)
    want, bound, wz, bz = R.linear(x, w, b, act, res, R.TYPES[t])
    R.check(out, want, bound, "y")
    R.check(z, wz, bz, "preact")
    assert untouched() and z_untouched()


@pytest.mark.parametrize("t", TYPES)
def test_linear_neighbours_in_the_record(t):
    """What lies beside the columns of a wider record, NaN here, does not reach the result at any alignment."""
    for m, n in ((300, 40), (4200, 3)):
        for lead in range(0, 9):
            full = torch.full((m, 61 + 9), float("nan"), dtype=R.TYPES[t], device="cuda")
            x = full[:, lead:lead + 61]
            x.copy_(normal(104, m, 61, t))
            w = normal(105, n, 61, t, std=0.1)
            R.check(ops().linear_forward(x, w), *R.linear(x, w, None, "none", None, R.TYPES[t])[:2], f"lead {lead}")
            dx, dw, _ = ops().linear_backward(x, w, normal(106, m, n, t))
            R.check(dw, *R.linear_grads(x, w, normal(106, m, n, t), None, "none", R.TYPES[t])[1], f"dw, lead {lead}")


# ---- many rows against a small matrix ----------------------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,v,d", [(8192, 1, 1), (8193, 2, 7), (9000, 64, 32), (8320, 65, 33), (20_001, 101, 32),
                                   (8200, 128, 64), (150_000, 17, 48), (100_000, 40, 16)])
def test_loss_small_table(m, v, d, t):
    x, w = normal(110, m, d, t, std=2.0), normal(111, v, d, t, std=d ** -0.5)
    check_loss(x, w, labels(112, m, v), 1.5 if m % 2 else 1.0, 4096.0 if t == "f16" else 1.0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad,lead", [(8, 0), (8, 8), (5, 1)])
def test_loss_small_table_strides_and_masked_rows(pad, lead, t):
    m, v, d = 8300, 70, 40
    x, w = normal(113, m, d, t, pad=pad, lead=lead), normal(114, v, d, t, pad=pad, lead=lead)
    targets = labels(115, m, v, off=0.4)
    off = ~((targets >= 0) & (targets < v))
    x[off] = torch.where(torch.arange(d, device="cuda") % 2 == 0, float("nan"), float("inf")).to(x.dtype)
    check_loss(x, w, targets, 1.0, 100.0)
    loss, row, dx, dw = ops().loss_cross_entropy(x, w, torch.full_like(targets, -5))
    assert float(loss) == 0 and not row.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("t", TYPES)
def test_loss_small_table_extreme_logits(t):
    big = {"f32": 1e30, "bf16": 1e30, "f16": 6e4}[t]
    x = torch.zeros(8192, 16, dtype=R.TYPES[t], device="cuda")
    x[:, 0] = big
    for v in (50, 100):
        w = torch.zeros(v, 16, dtype=R.TYPES[t], device="cuda")
        w[v - 1, 0], w[:v - 2, 0] = 1, -1
        targets = torch.full((8192,), v - 1, dtype=torch.int32, device="cuda")
        loss, row, dx, dw = ops().loss_cross_entropy(x, w, targets)
        assert float(loss) == 0 and not row.any() and not dx.any() and not dw.any()
        targets[:] = v - 2
        loss, row, dx, dw = ops().loss_cross_entropy(x, w, targets, weight=64.0)
        assert torch.allclose(row, x[:, 0].float(), rtol=4 * 2.0 ** -24, atol=0) and bool(torch.isfinite(dx).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(8192, 1, 1), (8193, 3, 20), (9000, 64, 32), (8320, 65, 33), (20_001, 100, 64),
                                   (8200, 128, 64), (150_000, 16, 48), (77_777, 33, 7)])
@pytest.mark.parametrize("pad,lead", [(0, 0), (13, 10)])
def test_linear_backward_narrow(m, n, k, pad, lead, t):
    act = ACTS[(m + n + k) % 5]
    x, w = normal(116, m, k, t, pad=pad, lead=lead), normal(117, n, k, t, std=k ** -0.5)
    z, dy = normal(118, m, n, t), normal(119, m, n, t, pad=pad, lead=lead)
    full = ops().linear_backward(x, w, dy, preact=z, activation=act)
    for got, (want, bound), name in zip(full, R.linear_grads(x, w, dy, z, act, R.TYPES[t]), ("dx", "dw", "dbias")):
        R.check(got, want, bound, name)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        part = ops().linear_backward(x, w, dy, preact=z, activation=act, need_dx=need[0], need_dw=need[1], need_dbias=need[2])
        for a, b in zip(full, part):
            assert b is None or torch.equal(a, b)


# ---- the C entry points' own freedoms ------------------------------------------------------------------------------------


def workspace(size_fn, *args):
    import ctypes as C
    size = C.c_uint64()
    assert size_fn(*args, C.byref(size)) == 0
    return torch.empty(size.value + 1, dtype=torch.uint8, device="cuda"), size.value


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(300, 200, 96), (9000, 40, 24), (9000, 100, 50), (8192, 3, 32)])
def test_backward_c_entry(m, n, k, t):
    """Gradients into views of wider records; x null without dw, w null without dx; nothing beside the views is written."""
    L, code = ops()._lib(), {"f32": 0, "f16": 4, "bf16": 5}[t]
    x, w = normal(120, m, k, t), normal(121, n, k, t, std=k ** -0.5)
    z, dy = normal(122, m, n, t), normal(123, m, n, t)
    want = R.linear_grads(x, w, dy, z, "gelu", R.TYPES[t])
    ws, size = workspace(L.msplat_linear_backward_workspace, m, n, k, 2, code)
    stream = torch.cuda.current_stream().cuda_stream
    for pad in (3, 8):
        dx, dx_clean = guarded(m, k, R.TYPES[t], pad=pad)
        dw, dw_clean = guarded(n, k, R.TYPES[t], pad=pad)
        db = torch.empty(n, dtype=R.TYPES[t], device="cuda")
        for has_dx, has_dw in ((1, 1), (1, 0), (0, 1), (0, 0)):
            dx.zero_(), dw.zero_(), db.zero_()
            assert L.msplat_linear_backward(
                m, n, k, x.data_ptr() if has_dw else None, k, w.data_ptr() if has_dx else None, k, z.data_ptr(), n, 2,
                dy.data_ptr(), n, dx.data_ptr() if has_dx else None, dx.stride(0), dw.data_ptr() if has_dw else None,
                dw.stride(0), db.data_ptr(), code, ws.data_ptr(), size, stream) == 0, L.msplat_last_error()
            if has_dx:
                R.check(dx, *want[0], "dx")
            if has_dw:
                R.check(dw, *want[1], "dw")
            R.check(db, *want[2], "dbias")
            assert dx_clean() and dw_clean() and bool(dx.any()) == bool(has_dx) and bool(dw.any()) == bool(has_dw)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,v,d", [(300, 200, 96), (9000, 40, 24), (9000, 100, 50)])
def test_loss_c_entry(m, v, d, t):
    """Every output alone, in views of wider records, with a workspace for exactly what is asked."""
    L, code = ops()._lib(), {"f32": 0, "f16": 4, "bf16": 5}[t]
    x, w, targets = normal(124, m, d, t), normal(125, v, d, t, std=d ** -0.5), labels(126, m, v)
    want = R.loss(x, w, targets, 1.0, 50.0, R.TYPES[t])
    stream = torch.cuda.current_stream().cuda_stream
    for pad in (3, 8):
        for asked in ("loss", "row_loss", "dx", "dw"):
            ws, size = workspace(L.msplat_loss_cross_entropy_workspace, m, v, d, asked in ("dx", "dw"), code)
            out, clean = {"loss": (torch.empty((), device="cuda"), None), "row_loss": (torch.empty(m, device="cuda"), None),
                          "dx": guarded(m, d, R.TYPES[t], pad=pad), "dw": guarded(v, d, R.TYPES[t], pad=pad)}[asked]
            at = {name: out.data_ptr() if name == asked else None for name in ("loss", "row_loss", "dx", "dw")}
            assert L.msplat_loss_cross_entropy(m, v, d, x.data_ptr(), d, w.data_ptr(), d, targets.data_ptr(), 1.0, 50.0,
                                               at["loss"], at["row_loss"], at["dx"], d + 2 * pad, at["dw"], d + 2 * pad, code,
                                               ws.data_ptr(), size, stream) == 0, L.msplat_last_error()
            R.check(out, *want[asked], asked)
            assert clean is None or clean()


def test_status():
    x, w = normal(127, 300, 64, "bf16"), normal(128, 64, 64, "bf16")
    ops().linear_forward(x, w)
    ops().status()


def test_two_threads():
    """The same call from two host threads at once, each on its stream."""
    import threading
    x, w, targets = normal(129, 9000, 48, "f32"), normal(130, 90, 48, "f32"), labels(131, 9000, 90)
    want = ops().loss_cross_entropy(x, w, targets)
    torch.cuda.synchronize()
    got, fail = {}, []

    def work(k):
        try:
            s = torch.cuda.Stream()
            for _ in range(5):
                got[k] = ops().loss_cross_entropy(x, w, targets, stream=s)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            fail.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not fail
    for r in got.values():
        for a, b in zip(want, r):
            assert torch.equal(a, b)


@pytest.mark.parametrize("t,m,n,k", [("f16", 300_000_000, 3, 9), ("bf16", 36_000_000, 64, 64), ("f32", 36_000_000, 24, 61),
                                     ("f16", 36_000_000, 20, 61)])
def test_far_rows(t, m, n, k):
    """Matrices of more than 2^31 elements: the last rows of y, dx and row_loss, and a column of dw that only they reach."""
    x = torch.zeros(m, k, dtype=R.TYPES[t], device="cuda")
    last = normal(140, 500, k, t)
    x[-500:] = last
    w, b = normal(141, n, k, t, std=k ** -0.5), normal(142, 1, n, t)[0]
    y = ops().linear_forward(x, w, b, activation="relu")
    R.check(y[-500:], *R.linear(last, w, b, "relu", None, R.TYPES[t])[:2], "y")
    dy = torch.zeros(m, n, dtype=R.TYPES[t], device="cuda")
    dy[-500:] = normal(143, 500, n, t)
    dx, dw, db = ops().linear_backward(x, w, dy, preact=y, activation="relu")
    for got, (want, bound), name in zip((dx[-500:], dw, db), R.linear_grads(last, w, dy[-500:], y[-500:], "relu", R.TYPES[t]),
                                        ("dx", "dw", "dbias")):
        R.check(got, want, bound, name)
    del y, dx, dy
    targets = torch.full((m,), -1, dtype=torch.int32, device="cuda")
    targets[-500:] = labels(144, 500, n)
    _, row, dx, dw = ops().loss_cross_entropy(x, w, targets, weight=256.0)
    want = R.loss(last, w, targets[-500:], 1.0, 256.0, R.TYPES[t])
    R.check(row[-500:], *want["row_loss"], "row_loss")
    R.check(dx[-500:], *want["dx"], "dx")
    R.check(dw, *want["dw"], "dw")
    del x, dx, row, targets
    torch.cuda.empty_cache()
