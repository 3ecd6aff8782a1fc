"""Edges of the operators of msplat.ops (GPU): places, values and streams at which one kernel's answer could differ from
another's, or from the formula's."""
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
