"""The beam-drafting runner (kernel/dels_beam.py): its rollout step by step against the
selection's definition in float64, its greedy special case, and its own checks."""

from __future__ import annotations

import types

import numpy as np
import pytest
import torch
import torch.nn as nn

from test_gpu_beam import SCORE_TOL, reference_select

pytestmark = pytest.mark.gpu


def make_head(dev, V, E, G, r, seed):
    import dels as D

    target = types.SimpleNamespace(model=types.SimpleNamespace(embed_tokens=nn.Embedding(V, E)),
                                   lm_head=nn.Linear(G, V, bias=False))
    head = D.DeLSLocalHead(target_model=target, vocab_size=V, embed_dim=E, gru_hidden_dim=G, low_rank_dim=r,
                           lm_head_mode="low_rank", rank_activation="identity", dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(seed)
    with torch.no_grad():
        for p in head.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=dev) * 0.3)
    return head, g


def build(dev, V=1003, E=24, G=48, r=16, H=72, B=2, beams=4, steps=5, beta=0.2, seed=0):
    from kernel.dels_beam import DeLSBeamGraphRunner

    head, g = make_head(dev, V, E, G, r, seed)
    lm = torch.randn(V, H, generator=g, device=dev).bfloat16() * 0.3
    prior = torch.log_softmax(torch.randn(V, generator=g, device=dev), 0).bfloat16() if beta else None
    runner = DeLSBeamGraphRunner(local_head=head, batch_size=B, beams=beams, steps=steps, vocab_size=V,
                                 alpha_values=[0.5] * steps, beta_values=[beta] * steps, baseline_logits=prior,
                                 device=dev, target_lm_head_weight=lm)
    prefix = torch.randint(0, V, (B, 1), generator=g, device=dev)
    hidden = torch.randn(B, steps, H, generator=g, device=dev).bfloat16()
    return runner, prefix, hidden


@pytest.mark.parametrize("B,beams,steps,beta,V", [(1, 1, 3, 0.0, 1003), (2, 4, 5, 0.2, 1003), (3, 8, 4, 0.2, 2048),
                                                  (1, 16, 3, 0.0, 640)])
def test_rollout_follows_the_definition(cuda_device, B, beams, steps, beta, V):
    """Every step of a rollout done by hand: GRU, rank projection and local logits from the
    kernels the greedy runner uses, selection and reordering from numpy."""
    from dels_b200 import ops

    dev = cuda_device
    runner, prefix, hidden = build(dev, V=V, B=B, beams=beams, steps=steps, beta=beta, seed=B + beams)
    tokens, scores = runner(prefix, hidden)
    assert tokens.shape == (B, beams, steps) and scores.shape == (B, beams)
    # replayed with other inputs and back: nothing of a call is left behind
    runner(prefix.flip(0), hidden.flip(0) * 0.5)
    again = runner(prefix, hidden)
    assert torch.equal(tokens, again[0]) and torch.equal(scores, again[1])

    base = ops.linear_w8a8(hidden.view(B * steps, -1), runner._lm_q, runner._lm_scale).view(B, steps, V)
    rows = B * beams
    h = torch.empty(rows, runner.gru_hidden_dim, dtype=torch.bfloat16, device=dev)
    runner._gru(prefix.repeat_interleave(beams, 0)[:, 0], None, h)
    hist = np.zeros((rows, 0), np.int64)
    cum = np.zeros((B, 1), np.float32)
    prior = None if beta == 0 else runner._prior_f32.cpu().numpy()
    clear = True
    for t in range(steps):
        runner._rank(h, t)
        local = ops.linear_bf16(runner._s_scaled, runner.lm_head_weight).float().cpu().numpy()
        logits = local[::beams] if t == 0 else local
        parents, tok, sc, gaps = reference_select(logits, cum, beams, base[:, t].float().cpu().numpy(), prior, beta)
        clear &= bool((gaps > 4 * SCORE_TOL * (t + 1)).all())
        at = (parents + np.arange(B)[:, None] * beams).reshape(-1)
        hist = np.concatenate([hist[at], tok.reshape(-1, 1)], 1)
        cum = sc.astype(np.float32)
        moved = h[torch.from_numpy(at).to(dev)].contiguous()
        h = torch.empty_like(h)
        runner._gru(torch.from_numpy(tok.reshape(-1)).to(dev), moved, h)
    np.testing.assert_allclose(scores.cpu().numpy(), cum, rtol=2e-7, atol=SCORE_TOL * steps)
    assert clear  # (by the seeds: no two beams' scores meet)
    np.testing.assert_array_equal(tokens.cpu().numpy().reshape(rows, steps), hist)


def test_best_chain_of_wide_beams_is_no_worse_than_greedy(cuda_device):
    dev = cuda_device
    one, prefix, hidden = build(dev, B=3, beams=1, steps=4, seed=7)
    many, _, _ = build(dev, B=3, beams=12, steps=4, seed=7)
    greedy = one(prefix, hidden)[1][:, 0]
    tokens, scores = many(prefix, hidden)
    assert (scores[:, 0] >= greedy - SCORE_TOL * 4).all()
    assert (scores[:, 1:] <= scores[:, :-1]).all()
    for b in range(3):  # chains of a sequence differ
        assert len({tuple(x) for x in tokens[b].tolist()}) == 12


def test_runner_checks(cuda_device):
    dev = cuda_device
    for beams in (0, 65):
        with pytest.raises(ValueError, match="beams"):
            build(dev, beams=beams)
    from kernel.dels_beam import DeLSBeamGraphRunner

    head, _ = make_head(dev, 100, 8, 16, 8, 0)
    with pytest.raises(ValueError, match="does not match vocab_size"):
        DeLSBeamGraphRunner(local_head=head, batch_size=1, beams=2, steps=1, vocab_size=100, alpha_values=[1.0],
                            beta_values=[0.0], baseline_logits=None, device=dev,
                            target_lm_head_weight=torch.zeros(99, 16, device=dev))
