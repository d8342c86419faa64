"""Selections among thousands of equal logits and equal beams: the documented total order, pair by
pair, which scores alone do not show."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_beam import SCORE_TOL

pytestmark = pytest.mark.gpu


def check_order(out, x, cum):
    """No pair twice; every pair's score; a beam's tokens in its own order (larger x, then lower token)
    from the first on; and the list by score, then beam, then that order."""
    parents, tokens, scores = (t.cpu().numpy() for t in (out.parents, out.tokens, out.scores))
    x, cum = x.double().cpu(), cum.double().cpu().numpy()
    n_seq, beams = cum.shape
    logp = torch.log_softmax(x, 1)
    logp = torch.where(x == -math.inf, x, logp).numpy()
    x = x.numpy()
    for b in range(n_seq):
        pairs = list(zip(parents[b].tolist(), tokens[b].tolist()))
        assert len(set(pairs)) == len(pairs)
        rank = []
        for k in range(beams):
            mine = [t for p, t in pairs if p == k]
            order = np.lexsort((np.arange(x.shape[1]), -x[b * beams + k]))
            assert mine == order[: len(mine)].tolist(), (b, k)
        seen = dict.fromkeys(range(beams), 0)
        for j, (p, t) in enumerate(pairs):
            want = logp[b * beams + p, t] + cum[b, p]
            assert scores[b, j] == want or abs(scores[b, j] - want) < SCORE_TOL, (b, j)
            rank.append((-scores[b, j], p, seen[p]))
            seen[p] += 1
        assert rank == sorted(rank), b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("beams", [1, 2, 4])
@pytest.mark.parametrize("V", [600, 5003, 20000])
def test_order_among_equal_logits(cuda_device, dtype, beams, V):
    """Constant rows, two and three values, masks of the type's lowest value and of -inf, few values
    above them."""
    from dels_b200 import ops

    dev = cuda_device
    rng = np.random.default_rng(V + beams)
    x = torch.zeros(8, V)
    x[1, : V - 400] = -3.0
    x[2, ::2] = -1.0
    x[3] = torch.finfo(dtype).min
    x[4] = torch.from_numpy(np.sort(rng.integers(0, 3, V))).float()
    x[5] = -0.0
    x[6, : V - 300] = -math.inf
    x[7, 4:] = -math.inf
    for r in range(8):
        x[r, torch.from_numpy(rng.permutation(V)[: 3 * (r % 4)])] = 2.0 + r
    x = x.to(dtype)
    for cum in (torch.zeros(8 // beams, beams),
                torch.from_numpy(rng.standard_normal((8 // beams, beams)).astype(np.float32))):
        for select in (1, 16, 64):
            check_order(ops.beam_select(x.to(dev), cum.to(dev), select=select), x, cum)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,beams", [(1024, 4), (1003, 3), (20000, 8), (5003, 64)])
def test_equal_beams_share_the_lowest_tokens(cuda_device, dtype, V, beams):
    """Beams that are alike, with one value everywhere: all candidates of a sequence are equal, so the
    first beam's lowest tokens are the answer; with a few larger logits those come first, beam by beam."""
    from dels_b200 import ops

    dev = cuda_device
    n = 32
    scores = torch.full((5, beams), -2.0, device=dev)
    x = torch.full((5 * beams, V), 0.5, dtype=dtype, device=dev)
    out = ops.beam_select(x, scores, select=n)
    assert (out.parents == 0).all()
    assert torch.equal(out.tokens, torch.arange(n, device=dev).expand(5, n))
    assert (out.scores == out.scores[0, 0]).all()
    assert abs(float(out.scores[0, 0]) - (-2.0 - math.log(V))) < SCORE_TOL
    x[:, 7] = 3.0
    x[:, V - 1] = 3.0
    out = ops.beam_select(x, scores, select=n)
    top = min(n, 2 * beams)
    want_parents = torch.arange(beams, device=dev).repeat_interleave(2)[:top]
    want_tokens = torch.tensor([7, V - 1], device=dev).repeat(beams)[:top]
    for b in range(5):
        assert torch.equal(out.parents[b, :top].long(), want_parents)
        assert torch.equal(out.tokens[b, :top], want_tokens)
        if n > top:
            rest = torch.tensor([t for t in range(n) if t != 7], device=dev)[: n - top]
            assert (out.parents[b, top:] == 0).all()
            assert torch.equal(out.tokens[b, top:], rest)
