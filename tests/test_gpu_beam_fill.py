"""Selections of rows that allow fewer tokens than are selected, whose masked tokens fill the rest:
every sequence, every time."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_seq,beams,select,V", [(1500, 1, 16, 4096), (700, 3, 24, 1003), (600, 8, 64, 2500)])
def test_masked_tokens_fill_every_sequence(cuda_device, dtype, n_seq, beams, select, V):
    """One allowed token a beam: the allowed ones come first, by their beams' scores, then the lowest
    masked tokens of the first beam at -inf.  Many sequences, several times over."""
    from dels_b200 import ops

    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(n_seq + select)
    x = torch.full((n_seq * beams, V), -math.inf, dtype=dtype, device=dev)
    allowed = torch.randint(0, V, (n_seq * beams, 1), generator=g, device=dev)
    x.scatter_(1, allowed, 1.0)
    scores = torch.randperm(n_seq * beams, generator=g, device=dev).float().view(n_seq, beams) * -0.25
    # a single allowed token has probability one, so a beam's score stays what it was
    order = scores.argsort(1, descending=True)
    first = allowed.view(n_seq, beams)[:, :1]
    fill = torch.arange(select - beams, device=dev).expand(n_seq, -1)
    fill = fill + (fill >= first)
    tokens = torch.cat([allowed.view(n_seq, beams).gather(1, order), fill], 1)
    parents = torch.cat([order, torch.zeros_like(fill)], 1).int()
    want = torch.cat([scores.gather(1, order), torch.full_like(fill, -math.inf, dtype=torch.float32)], 1)
    for _ in range(20):
        out = ops.beam_select(x, scores, select=select)
        assert torch.equal(out.parents, parents)
        assert torch.equal(out.tokens, tokens)
        assert torch.equal(out.scores, want)
