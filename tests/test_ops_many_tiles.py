"""The operators of msplat.ops at sizes where every block takes many tiles (GPU): the rings of boxes and barriers go round
with a residual and a kept argument beside the result, and sums over many rows are held to what the kernels can do, not to
what a sum of so many products could at worst be."""
import math

import pytest

torch = pytest.importorskip("torch")

import _ops_ref as R  # noqa: E402
from test_ops import TYPES, guarded, labels, normal, ops  # noqa: E402, F401

pytestmark = pytest.mark.gpu

# rows, outputs, inputs: more than 148 tiles of 128 rows x 64, 128 and 256 columns, several columns of tiles, rows behind the
# last tile's, one to ten stages of the reduction
SHAPES = [(40_001, 48, 40), (30_000, 100, 72), (20_010, 300, 64), (33_000, 130, 200), (25_000, 64, 32), (20_000, 100, 600),
          (10_000, 520, 24), (60_000, 16, 130)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("residual,preact", [(1, 0), (0, 1), (1, 1)])
@pytest.mark.parametrize("pad", (8, 3))
def test_linear_forward_many_tiles(m, n, k, residual, preact, pad, t):
    """Outputs in wider records that TMA can (8) and cannot (3) address; the residual is the output's own memory."""
    x, w, bias = normal(300, m, k, t), normal(301, n, k, t, std=k ** -0.5), normal(302, 1, n, t)[0]
    out, untouched = guarded(m, n, R.TYPES[t], pad=pad)
    res = normal(303, m, n, t) if residual else None
    z, z_untouched = guarded(m, n, R.TYPES[t], pad=pad) if preact else (None, lambda: True)
    if residual:
        out.copy_(res)
    ops().linear_forward(x, w, bias, activation="silu", residual=out if residual else None, preact=z, out=out)
    want, bound, wz, bz = R.linear(x, w, bias, "silu", res, R.TYPES[t])
    R.check(out, want, bound, "y")
    if preact:
        R.check(z, wz, bz, "preact")
    assert untouched() and z_untouched()


@pytest.mark.parametrize("t", ("f16", "bf16"))
@pytest.mark.parametrize("m,n,k", [(40_001, 48, 40), (20_010, 300, 61), (30_000, 100, 72)])
def test_linear_forward_many_tiles_f32_output(m, n, k, t):
    x, w = normal(304, m, k, t), normal(305, n, k, t, std=k ** -0.5)
    res, z = normal(306, m, n, "f32"), torch.empty(m, n, device="cuda")
    y = ops().linear_forward(x, w, activation="gelu", residual=res, preact=z, out_dtype=torch.float32)
    want, bound, wz, bz = R.linear(x, w, None, "gelu", res, torch.float32)
    R.check(y, want, bound, "y")
    R.check(z, wz, bz, "preact")


def whole(seed, rows, cols, t, low=-3, high=4, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    full = torch.randint(low, high, (rows, cols + pad), generator=g, device="cuda").to(R.TYPES[t])
    return full[:, pad // 2:pad // 2 + cols]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(80_000, 64, 32), (150_000, 17, 33), (200_003, 100, 64), (160_000, 128, 20), (100_000, 3, 7),
                                   (40_000, 200, 136), (70_001, 40, 150)])
@pytest.mark.parametrize("pad", (0, 8, 5))
def test_linear_gradients_of_whole_numbers_are_exact(m, n, k, pad, t):
    """Products and sums of small whole numbers fit 24 bits: dx, dw and dbias are the exact ones, rounded once to the type;
    any row, tile or partial sum that is lost, doubled or late shows."""
    x, w, dy = whole(310, m, k, t, pad=pad), whole(311, n, k, t), whole(312, m, n, t, pad=pad)
    dx, dw, db = ops().linear_backward(x, w, dy)
    x, w, dy = x.double(), w.double(), dy.double()
    assert float((dy.abs().T @ x.abs()).max()) < 2 ** 24 and float(dy.abs().sum(0).max()) < 2 ** 24
    assert torch.equal(dx, (dy @ w).to(dx.dtype))
    assert torch.equal(dw, (dy.T @ x).to(dw.dtype))
    assert torch.equal(db, dy.sum(0).to(db.dtype))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,v,d", [(100_000, 64, 32), (200_003, 128, 24), (90_000, 32, 50), (30_000, 256, 40), (40_000, 64, 100)])
def test_loss_gradients_of_equal_logits(m, v, d, t):
    """A table of zeros makes every probability 1 / v, a power of 2, and dw a sum of whole numbers over v, scaled by powers
    of 2: off by the exponential's 2 steps for each 1 / v at most (not at all against a small table), and by the rounding
    to the type; dx is 0."""
    x, targets = whole(313, m, d, t), labels(314, m, v, off=0.3)
    known = (targets >= 0) & (targets < v)
    count = 1 << 16 if m >= 100_000 else 1 << 14
    more = torch.nonzero(known)[:, 0][count:]
    targets[more], known[more] = -7, False  # a power of 2 of labelled rows
    assert int(known.sum()) == count
    loss, row, dx, dw = ops().loss_cross_entropy(x, torch.zeros(v, d, dtype=x.dtype, device="cuda"), targets, weight=float(count))
    xd = torch.where(known[:, None], x.double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    hot = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_add_(0, targets[known].long(), xd[known])
    want = xd.sum(0) / v - hot
    # of each term: the exponential (2^-22) and log2(v) in its exponent (2^-24 of at most 8, 2^-21 of the power) where the
    # statistics come from a pass of their own, and the 16-bit types' rounding of the two values that g takes
    off = torch.zeros_like(want)
    if v > 128 or d > 64:
        off = off + xd.abs().sum(0) / v * (2.0 ** -22 + 2.0 ** -21)
    if t != "f32":  # 1 / v is exact; 1 / v - 1 is rounded for v above 256 (bf16) only
        assert v <= 256
    R.check(dw, want, off + R.rounded(want.abs() + off, dw.dtype), "dw")
    assert not dx.any()
    R.check(row, math.log(v) * known.double(), (2.0 ** -21 * math.log(v)) * known.double(), "row_loss")


def sums_bound(p2, m, size):
    """How far a sum of m products of random sign, p2 their sum of squares, may be: it is made in accumulators of at most
    1024 products, 16 at a time, each addition rounded towards zero (a step, 2^-23, of a running sum of at most five times
    its expected size), and the accumulators are added in 32 bits (half a step each of at most five times the size of the
    whole; size: the sum itself)."""
    run = 5 * p2.sqrt()
    return (m / 16) * 2.0 ** -23 * run * (1024 / m) ** 0.5 + (m / 512 + 300) * 2.0 ** -24 * run + 2.0 ** -22 * size.abs()


@pytest.mark.parametrize("m,n,k", [(9000, 33, 20), (80_000, 64, 32), (150_000, 16, 48), (200_003, 100, 64), (40_000, 200, 136)])
def test_linear_gradients_keep_32_bits(m, n, k):
    """dw and dbias of 32-bit normal values, to a bound that neither zeros, nor half of the rows, nor factors rounded to
    bf16 meet."""
    x, w, dy = normal(320, m, k, "f32"), normal(321, n, k, "f32"), normal(322, m, n, "f32")
    _, dw, db = ops().linear_backward(x, w, dy)
    xd, yd = x.double(), dy.double()
    want, p2 = yd.T @ xd, (yd ** 2).T @ (xd ** 2)
    bound = sums_bound(p2, m, want)
    R.check(dw, want, bound, "dw")
    R.check(db, yd.sum(0), sums_bound((yd ** 2).sum(0), m, yd.sum(0)), "dbias")
    for wrong in (torch.zeros_like(want), yd[:m // 2].T @ xd[:m // 2], dy.bfloat16().double().T @ x.bfloat16().double()):
        with pytest.raises(AssertionError):
            R.check(wrong, want, bound, "dw")


def positive(seed, rows, cols):
    return normal(seed, rows, cols, "f32").abs()


def one_sign_bound(k, want):
    """How far a sum of k positive 32-bit products may be: 512 of them are added 16 at a time in one accumulator, each
    addition rounded towards zero (32 steps of 2^-23); the five smaller products of a split factor's parts, 2^-7 of the whole
    together, 1536 at a time (480 steps of that); the accumulators in 32 bits, half a step each, and eight more."""
    return want * (32 * 2.0 ** -23 + 480 * 2.0 ** -23 * 2.0 ** -7 + (k / 512 + 8) * 2.0 ** -24)


@pytest.mark.parametrize("m,n,k", [(300, 200, 1536), (300, 200, 1537), (40, 9, 3100), (300, 200, 4096), (130, 70, 16_384),
                                   (20_000, 66, 1800), (5000, 500, 2100)])
@pytest.mark.parametrize("pad", (0, 3))
def test_linear_long_reductions_of_one_sign(m, n, k, pad):
    """32-bit sums of one sign, where truncating accumulators lose the same way at every step."""
    x, w = positive(330, m, k + pad)[:, pad:], positive(331, n, k + pad)[:, pad:]
    res, z = normal(332, m, n, "f32"), torch.empty(m, n, device="cuda")
    y = ops().linear_forward(x, w, residual=res, preact=z)
    want = x.double() @ w.double().T
    R.check(z, want, one_sign_bound(k, want), "preact")
    R.check(y, want + res.double(), one_sign_bound(k, want) + 2.0 ** -24 * (want + res.double()).abs(), "y")


def test_linear_gradients_long_reductions_of_one_sign():
    """dx over many outputs, and dw over rows in few pieces (a result of 32 MB leaves room for eight)."""
    m, n, k = 32_768, 2048, 4096
    x, dy, w = positive(333, m, k), positive(334, m, n), positive(335, n, k)
    dx, dw, _ = ops().linear_backward(x, w, dy)
    rows = torch.arange(0, m, 37, device="cuda")
    want = dy[rows].double() @ w.double()
    R.check(dx[rows], want, one_sign_bound(n, want), "dx")
    cols = torch.arange(0, n, 7, device="cuda")
    want = dy[:, cols].double().T @ x.double()
    R.check(dw[cols], want, one_sign_bound(m, want), "dw")


@pytest.mark.parametrize("m,v,d", [(300, 500, 1600), (20_000, 70, 2000), (40, 3000, 5000)])
def test_loss_of_long_rows(m, v, d):
    x, w = normal(336, m, d, "f32"), normal(337, v, d, "f32", std=d ** -0.5)
    targets = labels(338, m, v)
    got = ops().loss_cross_entropy(x, w, targets, weight=64.0)
    want = R.loss(x, w, targets, 1.0, 64.0, torch.float32)
    for a, name in zip(got, ("loss", "row_loss", "dx", "dw")):
        R.check(a, *want[name], name)


@pytest.mark.parametrize("t", ("f16", "bf16"))
def test_linear_gradients_of_a_million_rows_and_one_sign(t):
    """A 16-bit dw large enough for few pieces of its rows: half a step of the type, and what truncation takes from at most
    32768 products, 16 at a time (2048 steps of 2^-23)."""
    m, n, k = 1_000_000, 2048, 2048
    x, dy = (torch.empty(m, k, dtype=R.TYPES[t], device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(340)
    x.uniform_(0.25, 1.75, generator=g)
    dy.uniform_(0.25 / 2 ** 10, 1.75 / 2 ** 10, generator=g)  # sums of about 1000
    _, dw, _ = ops().linear_backward(x, torch.zeros(n, k, dtype=x.dtype, device="cuda"), dy, need_dx=False, need_dbias=False)
    some = torch.arange(0, n, 129, device="cuda")
    want = sum(a[:, some].double().T @ b.double() for a, b in zip(dy.split(125_000), x.split(125_000)))
    off = want * (2048 * 2.0 ** -23 + 64 * 2.0 ** -24)
    R.check(dw[some], want, off + R.rounded(want + off, dw.dtype), "dw")
    del x, dy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("t", ("f16", "bf16"))
@pytest.mark.parametrize("out", ("same", "f32"))
@pytest.mark.parametrize("m,n,k", [(130, 70, 4097), (300, 300, 20_000), (40, 130, 32_769), (200, 150, 40_000),
                                   (9, 20, 140_001), (20_000, 260, 5000)])
@pytest.mark.parametrize("pad", (0, 8, 3))
def test_linear_16_bit_long_reductions_of_one_sign(m, n, k, pad, out, t):
    """Half a step of the result's type, and what truncation takes from the products of one pass, 16 at a time: 4096 for 32-bit
    results (256 steps of 2^-23, and as many again, since f16 products are cut too), 32768 for 16-bit ones; passes in 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(350)
    x = torch.empty(m, k + pad, dtype=R.TYPES[t], device="cuda").uniform_(0.25, 1.75, generator=g)[:, pad:]
    w = (torch.empty(n, k + pad, device="cuda").uniform_(0.25, 1.75, generator=g) / k).to(R.TYPES[t])[:, pad:]
    out_t = torch.float32 if out == "f32" else R.TYPES[t]
    w = w * 64 if t == "f16" else w  # not below f16's normal numbers
    w = torch.nn.functional.pad(w, (pad, 0))[:, pad:]
    z = torch.empty(m, n, dtype=out_t, device="cuda")
    res = torch.full((m, n), -1.0, dtype=out_t, device="cuda")
    y = ops().linear_forward(x, w, residual=res, preact=z, out_dtype=out_t)
    want = torch.cat([a.double() @ w.double().T for a in x.split(2000)])
    length = 4096 if out == "f32" else 32_768
    off = want * (2 * length / 16 * 2.0 ** -23 + (k / length + 2) * 2.0 ** -24)
    R.check(z, want, off + R.rounded(want + off, out_t), "preact")
    off = off + 2.0 ** -24 * (want - 1).abs()
    R.check(y, want - 1, off + R.rounded((want - 1).abs() + off, out_t), "y")


@pytest.mark.parametrize("t", ("f16", "bf16"))
@pytest.mark.parametrize("m,v,d", [(300, 300, 4200), (100, 1000, 9000)])
@pytest.mark.parametrize("pad", (0, 3))
def test_loss_16_bit_of_long_rows(m, v, d, pad, t):
    x, w = normal(351, m, d, t, pad=pad, lead=pad), normal(352, v, d, t, std=d ** -0.5, pad=pad, lead=pad)
    targets = labels(353, m, v)
    got = ops().loss_cross_entropy(x, w, targets, weight=64.0)
    want = R.loss(x, w, targets, 1.0, 64.0, R.TYPES[t])
    for a, name in zip(got, ("loss", "row_loss", "dx", "dw")):
        R.check(a, *want[name], name)


@pytest.mark.parametrize("lead", (0, 1))
def test_linear_few_rows_of_many_inputs(lead):
    """Two rows of 64 million equal inputs: a lane adds at most 4096 products (half a step each) before that sum is added to
    the others."""
    k = 1 << 26
    x = torch.full((2, k + 4), 0.1, device="cuda")[:, lead:lead + k]
    w = torch.full((3, k + 4), 0.7, device="cuda")[:, lead:lead + k]
    y = ops().linear_forward(x, w)
    want = torch.full((2, 3), k, dtype=torch.float64, device="cuda") * float(x[0, 0]) * float(w[0, 0])
    R.check(y, want, want * (4096 + k / (512 * 32) + 8) * 2.0 ** -24, "y")
