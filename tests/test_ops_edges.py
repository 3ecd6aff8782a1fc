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
