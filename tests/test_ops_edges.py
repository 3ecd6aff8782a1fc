"""Edges of the operators of msplat.ops (GPU): places, values and streams at which one kernel's answer could differ from
another's, or from the formula's."""
import math

import pytest

torch = pytest.importorskip("torch")

import _ops_ref as R  # noqa: E402
from test_ops import TYPES, labels, normal, ops  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(4101, 3, 61), (4097, 8, 9)])
def test_few_outputs_at_every_alignment(m, n, k, t):
    """A row of few outputs adds its products in the order of the columns wherever it starts: the same bits at every
    alignment, with rows behind the last of a warp and pieces that hang over both ends of the matrix."""
    values, w = normal(200, m, k, t), normal(201, n, k, t, std=k ** -0.5)
    want = None
    for lead in range(16 // values.element_size()):
        x = torch.empty(m, k + 9, dtype=values.dtype, device="cuda")[:, lead:lead + k]
        x.copy_(values)
        y = ops().linear_forward(x, w)
        want = y if want is None else want
        assert torch.equal(y, want), lead
    R.check(want, *R.linear(values, w, None, "none", None, values.dtype)[:2], "y")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,v", [(700, 70), (8192, 40), (8192, 101), (9001, 101)])
@pytest.mark.parametrize("value", (float("-inf"), float("inf"), float("nan")))
def test_loss_rows_without_a_label_and_a_table_that_is_not_finite(m, v, value, t):
    """A label's embedding that is not finite makes 0 times it NaN: rows without a label, and those behind the last, still
    give nothing to dw, and without any label everything is 0."""
    d = 24
    x, w = normal(202, m, d, t), normal(203, v, d, t, std=d ** -0.5)
    x[:, 5] = x[:, 5].abs() + 0.5
    w[7, 5] = value
    targets = labels(204, m, v, off=0.4)
    targets[targets == 7] = 8
    loss, row, dx, dw = ops().loss_cross_entropy(x, w, torch.full_like(targets, -1))
    assert float(loss) == 0 and not row.any() and not dx.any() and not dw.any()
    known = (targets >= 0) & (targets < v)
    loss, row, dx, dw = ops().loss_cross_entropy(x, w, targets, weight=100.0)
    assert not row[~known].any() and not dx[~known].any()
    if value == float("-inf") and t != "f32":
        # that label's logit is -inf in every row (32-bit infinities are split: see below), its probability 0: the loss and
        # dw are those of a table without it, and its own row of dw is 0
        rest = torch.cat((w[:7], w[8:]))
        want = R.loss(x, rest, torch.where(targets > 7, targets - 1, targets).masked_fill(~known, -1), 1.0, 100.0, x.dtype)
        R.check(loss, *want["loss"], "loss")
        R.check(row, *want["row_loss"], "row_loss")
        R.check(torch.cat((dw[:7], dw[8:])), *want["dw"], "dw")
        assert not dw[7].any()


def check_wide(got, want, bound, name):
    """R.check where the formula's value fits 32 bits; the same infinity where it is beyond them, NaN where it is NaN."""
    top = torch.finfo(torch.float32).max
    nan, far = want.isnan(), want.abs() > top * 1.5
    assert torch.equal(got.isnan(), nan), f"{name}: NaN in other places"
    assert torch.equal(got[far], torch.where(want[far] > 0, float("inf"), float("-inf")).float()), f"{name}: infinities"
    rest = ~(nan | far)
    R.check(got[rest], want[rest], bound[rest], name)


@pytest.mark.parametrize("m,n,k", [(8, 40, 20), (9, 40, 20), (300, 130, 200), (5000, 3, 33), (20_000, 64, 32)])
def test_linear_infinities_and_largest_values(m, n, k):
    """32-bit infinities, NaN and the type's largest values in one factor or both: the formula's values from every kernel
    (infinities beside factors below 256). Every product has at most one term that is not ordinary."""
    big = torch.finfo(torch.float32).max
    x, w = normal(210, m, k, "f32"), normal(211, n, k, "f32")
    x[:, 3] = torch.tensor([float("inf"), float("-inf"), big, -big, float("nan"), 0.5, 0.0], device="cuda")[
        torch.arange(m, device="cuda") % 7]
    w[:, 3] = torch.tensor([1.0, -0.25, 0.0, 200.7, float("inf"), -3.3e-5, float("-inf")], device="cuda")[
        torch.arange(n, device="cuda") % 7]
    want = x.double() @ w.double().T
    # the products of the ordinary terms, and the one that is not, bound the rounding
    size = x[:, 3:4].double().abs() @ w[:, 3:4].double().abs().T
    rest = torch.cat((x[:, :3], x[:, 4:]), 1).double().abs() @ torch.cat((w[:, :3], w[:, 4:]), 1).double().abs().T
    off = R.SUM * (k + 8) * (size + rest)
    check_wide(ops().linear_forward(x, w), want, off + R.rounded(want.abs(), torch.float32), "y")


@pytest.mark.parametrize("m,n,k", [(300, 40, 24), (9000, 40, 24), (9000, 100, 50)])
def test_linear_gradients_of_infinities(m, n, k):
    """One infinite weight and one infinite feature: infinities of dz's signs in their columns of dx and dw, and nowhere
    else."""
    x, w, dy = normal(212, m, k, "f32"), normal(213, n, k, "f32"), normal(214, m, n, "f32")
    (dx0, bx), (dw0, bw), _ = R.linear_grads(x, w, dy, None, "none", torch.float32)
    x[m - 3, 1], w[n - 2, 4] = float("-inf"), float("inf")
    dx, dw, _ = ops().linear_backward(x, w, dy)
    dx0[:, 4], dw0[:, 1] = dy[:, n - 2] * float("inf"), dy[m - 3] * float("-inf")
    check_wide(dx, dx0, bx, "dx")
    check_wide(dw, dw0, bw, "dw")


@pytest.mark.parametrize("m,v", [(700, 70), (8192, 40), (9001, 101)])
@pytest.mark.parametrize("value", (float("-inf"), torch.finfo(torch.float32).min))
def test_loss_of_a_table_padded_with_the_lowest_value(m, v, value):
    """A label that an embedding of the lowest value takes out: its probability is 0, the rest is the table without it."""
    d = 24
    x, w = normal(215, m, d, "f32"), normal(216, v, d, "f32", std=d ** -0.5)
    x[:, 5] = x[:, 5].abs() + 0.5
    w[7, 5] = value
    targets = labels(217, m, v, off=0.3)
    targets[targets == 7] = 8
    known = (targets >= 0) & (targets < v)
    want = R.loss(x, torch.cat((w[:7], w[8:])), torch.where(targets > 7, targets - 1, targets).masked_fill(~known, -1), 1.0,
                  100.0, torch.float32)
    loss, row, dx, dw = ops().loss_cross_entropy(x, w, targets, weight=100.0)
    R.check(loss, *want["loss"], "loss")
    R.check(row, *want["row_loss"], "row_loss")
    R.check(torch.cat((dw[:7], dw[8:])), *want["dw"], "dw")
    assert not dw[7].any()
    if value != float("-inf"):  # 0 times -inf is NaN in the formula too
        R.check(dx, *want["dx"], "dx")


# ---- activations, relative to their own size --------------------------------------------------------------------------

# Steps of 2^-24 that the functions may be off by in 32 bits. gelu: the reciprocal and its argument (t: 2 steps, which
# change erfc(x) e^(x^2) by 1.13 / 0.4 times as much), ten coefficients' roundings (1 at each end), the density (its
# power 4, its exponent's two corrections 1) and two products: 14. sigmoid: the power 4, the exponent 1, sum, reciprocal 2,
# product: 10.
STEPS = 16 * 2.0 ** -24


def phi(z):
    """The Gaussian distribution function in 64 bits with all its bits in the negative tail (1 + erf cancels there)."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2))


def tail_values(t, low):
    return torch.cat((torch.linspace(low, 0, 3001), torch.linspace(0, -low, 1001), torch.tensor([-1e-3, 1e-3, 0.0]))).to(
        R.TYPES[t])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", (1, 40, 5000))
@pytest.mark.parametrize("act,low", [("gelu", -12.5), ("silu", -80.0), ("sigmoid", -80.0)])
def test_activations_keep_their_small_values(act, low, rows, t):
    """act(z) for z passed through a layer of one input and weight 1: within half a step of the result's type and a few of
    32 bits of act(z), however small it is."""
    z = tail_values(t, low).cuda()
    for out_t in {R.TYPES[t], torch.float32}:
        if rows == 1:    # a row against many weights
            y = ops().linear_forward(torch.ones(1, 1, dtype=z.dtype, device="cuda"), z[:, None].contiguous(), activation=act,
                             out_dtype=out_t)[0]
            at = z
        elif rows == 40:
            at = z[:rows * 100].reshape(rows, 100)
            x = torch.zeros(rows, 100, dtype=z.dtype, device="cuda").copy_(at)
            y = ops().linear_forward(x, torch.eye(100, dtype=z.dtype, device="cuda"), activation=act, out_dtype=out_t)
        else:
            at = z.repeat(2)[:rows, None].contiguous()
            y = ops().linear_forward(at, torch.ones(1, 1, dtype=z.dtype, device="cuda"), activation=act, out_dtype=out_t)
        want = at.double() * phi(at.double()) if act == "gelu" else R.act(at.double(), act)
        off = (STEPS if out_t == torch.float32 else 2e-5) * want.abs() + 2.0 ** -126
        R.check(y, want, off + R.rounded(want.abs() + off, out_t), act)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", (40, 9000))
@pytest.mark.parametrize("act,low", [("gelu", -12.5), ("silu", -80.0), ("sigmoid", -80.0)])
def test_slopes_keep_their_small_values(act, low, m, t):
    """dy act'(z) through dx of a layer with the weights 1: relative to its own size, away from where it changes its sign."""
    n = 100
    z = tail_values(t, low).repeat(4)[:m * n] if m == 40 else tail_values(t, low).repeat(m * n // 4000)[:m * n]
    z = torch.cat((z, z.new_zeros(m * n - z.numel()))).reshape(m, n).cuda()
    eye = torch.eye(n, dtype=z.dtype, device="cuda") if m == 40 else torch.eye(64, dtype=z.dtype, device="cuda")
    z = z[:, :eye.shape[0]].contiguous()
    x, dy = torch.zeros_like(z), torch.ones_like(z)
    dx, _, _ = ops().linear_backward(x, eye, dy, preact=z, activation=act)
    want = R.slope(z.double(), act)
    if act == "sigmoid":  # q (1 - q), which cancels in the reference for large z
        q = torch.sigmoid(-z.double().abs())
        want = q * (1 - q)
    if act == "gelu":
        want = phi(z.double()) + z.double() * torch.exp(-z.double() ** 2 / 2) / math.sqrt(2 * math.pi)
    # gelu: Phi + z phi, silu: q + z q (1 - q): rounded from the sizes of both terms
    size = want.abs()
    if act == "gelu":
        size = phi(z.double()) + (z.double() * torch.exp(-z.double() ** 2 / 2) * 0.4).abs()
    if act == "silu":
        size = torch.sigmoid(z.double()) * (1 + (z.double() * torch.sigmoid(-z.double())).abs())
    off = (STEPS if t == "f32" else 2e-5) * size + 2.0 ** -126
    twice = off + 2 * R.rounded(want.abs() + off, R.TYPES[t])  # dz between the products, and dx
    R.check(dx, want, twice, act)


# ---- kernels that gave up waiting --------------------------------------------------------------------------------------


@pytest.mark.parametrize("kernels", (0, 1, 2))
def test_status_tells_every_stream_of_a_wait_that_ran_out(kernels):
    """A wait for a barrier at which nobody arrives gives up after a millisecond, whichever kernels' it is; each stream's
    next status raises, once, and another stream's call takes nothing away."""
    o = ops()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def raises(s):
        try:
            o.status(s)
            return False
        except o.MsplatError as e:
            assert "gave up" in str(e)
            return True
    for s in (*streams, None):
        raises(s)  # what earlier tests left
    assert not any(raises(s) for s in (*streams, None))
    assert o._lib().msplat_ops_rehearse_timeout(kernels, streams[0].cuda_stream) == 0
    assert raises(streams[0]) and raises(streams[1]) and raises(None)
    assert not any(raises(s) for s in (*streams, None))
    x, w = normal(220, 300, 64, "bf16"), normal(221, 64, 64, "bf16")
    R.check(o.linear_forward(x, w), *R.linear(x, w, None, "none", None, torch.bfloat16)[:2], "y")
    assert not raises(None)


# ---- inputs that are freed while another stream still reads them ----------------------------------------------------------


@pytest.mark.parametrize("op", ("linear_forward", "linear_backward", "dropout", "loss_cross_entropy"))
def test_inputs_freed_before_the_given_stream_has_read_them(op):
    """The caller's inputs are freed and their memory asked for again while the stream is still busy with something else."""
    o, m, n, k = ops(), 3001, 37, 41

    def inputs():
        x, w, y = normal(230, m, k, "f32").clone(), normal(231, n, k, "f32").clone(), normal(232, m, n, "f32").clone()
        return {"linear_forward": ((x, w), dict(bias=w[:, 0].contiguous(), residual=y, activation="gelu")),
                "linear_backward": ((x, w, y), dict(preact=y.clone(), activation="gelu")),
                "dropout": ((x, 0.3, 5), dict(residual=x.clone(), offset_dev=torch.tensor([7], device="cuda"))),
                "loss_cross_entropy": ((x, w, labels(233, m, n)), {})}[op]
    args, more = inputs()
    want = getattr(o, op)(*args, **more)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)  # some half a second
    got = getattr(o, op)(*args, **more, stream=side)
    held = [t for t in (*args, *more.values()) if isinstance(t, torch.Tensor)]
    sizes, at = [(t.shape, t.dtype) for t in held], {t.data_ptr() for t in held}
    del args, more, held
    again = [torch.empty(s, dtype=d, device="cuda") for s, d in sizes for _ in range(2)]
    # (a host that took longer than the stream may have the memory back)
    assert side.query() or not at & {t.data_ptr() for t in again}
    [t.fill_(-1) for t in again]
    torch.cuda.synchronize()
    want, got = ((v,) if isinstance(v, torch.Tensor) else v for v in (want, got))
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", (1, 40, 5000))
@pytest.mark.parametrize("act", ("relu", "gelu", "silu", "sigmoid"))
def test_activations_of_what_is_not_finite(act, m, t):
    """NaN stays NaN, at infinity the activations are their limits (silu at -inf may be NaN, as its formula is)."""
    values = torch.tensor([float("nan"), float("inf"), float("-inf"), 1.0, -100.0, 100.0], dtype=R.TYPES[t], device="cuda")
    one = torch.ones(1, 1, dtype=values.dtype, device="cuda")
    if m == 1:
        y = ops().linear_forward(one, values[:, None].contiguous(), activation=act)[0]
    else:  # a column of inputs, the same values again and again
        x = values.repeat(m // 6 + 1)[:m, None].contiguous()
        y = ops().linear_forward(x, one, activation=act)[:6, 0]
    y = y.double().tolist()
    assert math.isnan(y[0])
    assert y[1] == (1.0 if act == "sigmoid" else math.inf)
    assert y[2] == 0 or (act == "silu" and math.isnan(y[2]))
    assert abs(y[4]) <= 1e-40 and y[5] == (1.0 if act == "sigmoid" else 100.0) and y[3] > 0.7
    z = values.repeat(m)[:, None].contiguous()
    dx, _, _ = ops().linear_backward(torch.zeros_like(z), one, torch.ones_like(z), preact=z, activation=act)
    d = dx[:6, 0].double().tolist()
    assert math.isnan(d[0]) or act == "relu"
    assert d[5] == (0.0 if act == "sigmoid" else 1.0) or abs(d[5]) < 1e-40
    assert abs(d[4]) < 1e-40


@pytest.mark.parametrize("m,v,d", [(300, 300, 40), (20_000, 200, 24), (40, 3000, 100), (9000, 100, 32)])
@pytest.mark.parametrize("level", (1, 16, 64))
def test_loss_gradients_of_a_row_sum_to_nothing(m, v, d, level):
    """All embeddings have the same first column, so that logits of up to 4096 differ as those of the other columns do: softmax
    minus one-hot sums to 0, and so does the first column of dx. Its terms are off by the exponential's 2 steps of 2^-23 and
    their sum's few roundings; the product adds at most 188 times 16 of them, rounded towards zero (a step of a sum below 1,
    the rest small): 2^-17 of the column's 64 in all."""
    x, w = normal(240, m, d, "f32"), normal(241, v, d, "f32", std=d ** -0.5)
    x[:, 0], w[:, 0] = float(level), 64.0
    targets = labels(242, m, v, off=0.2)
    count = int(((targets >= 0) & (targets < v)).sum())
    _, _, dx, _ = ops().loss_cross_entropy(x, w, targets, weight=float(count))
    assert float(dx[:, 0].abs().max()) <= 64 * 2.0 ** -17
    assert float(dx.abs().max()) > 0.1
