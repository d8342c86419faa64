"""The softmax sums behind a selection's scores, over rows of the largest vocabulary and so many of
them that a warp adds up a whole row by itself."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

# What a score may be off by, all of it in units of 2^-24.  The sum: a term's exponential 4 (the
# special-function unit's 2^-22) and its argument 3 |x - max|, here at most 3 * 10; additions 8
# (pairs within a group, then compensated); the sum's step to the row's maximum 3.  log: an ulp of a
# value below 16, 16.  Then two additions below 16, half an ulp each, 16.  Joining two parts of a row 6
# (an exponential, a product, an addition): a row here has at most three parts, two joins, 12.  89
# units are 5.3e-6.
TOL = 6e-6
# Four rows by themselves are spread over the whole device: up to 16 parts one after the other in a
# lane, then five joins between lanes and one between warps, 132 units more.
TOL_SPREAD = 1.4e-5


def patterns(V, dtype):
    """Rows of many equal terms, and rows whose maximum rises from group to group."""
    one = torch.full((V,), -2.8)
    one[V // 3] = 0.0
    g = torch.Generator().manual_seed(V)
    ramp = torch.linspace(-1.0, 1.0, V)
    rising = torch.randn(V, generator=g).clamp(-5, 5).sort().values
    return torch.stack([one, torch.full((V,), 0.37), ramp, rising]).to(dtype)


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 524288), (torch.bfloat16, 300007), (torch.float32, 262144)])
def test_scores_of_long_rows(cuda_device, dtype, V):
    from dels_b200 import ops

    dev = cuda_device
    n = 7168
    rows = patterns(V, dtype)
    x = torch.empty(n, V, dtype=dtype, device=dev)
    for i in range(4):
        x[i::4] = rows[i].to(dev)
    out = ops.beam_select(x, torch.zeros(n, 1, device=dev), select=1)
    want = torch.log_softmax(rows.double(), 1).max(1)
    for i in range(4):
        got = out.scores[i::4, 0].double().cpu()
        assert (got - want.values[i]).abs().max() < TOL, (i, float((got - want.values[i]).abs().max()))
        # the first of the largest (a row's values repeat)
        first = int((rows[i] == rows[i].max()).nonzero()[0])
        assert (out.tokens[i::4] == first).all()
    # the same rows by themselves are summed in other shares
    few = ops.beam_select(x[:4], torch.zeros(4, 1, device=dev), select=1)
    assert (few.scores[:, 0].double().cpu() - want.values).abs().max() < TOL_SPREAD
