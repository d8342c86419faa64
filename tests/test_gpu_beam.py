"""Beam selection and state reordering on the B200 kernels against their definitions:
scores and order in float64 (numpy), moved states bit by bit."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = math.inf


def reference_select(logits, cum, n, base=None, prior=None, beta=0.0, finished=None, pad=0):
    """The best n candidates of every sequence.  x is formed in fp32, operation by operation,
    as the definition says; everything after it is float64."""
    n_seq, beams = cum.shape
    V = logits.shape[1]
    parents = np.zeros((n_seq, n), np.int32)
    tokens = np.zeros((n_seq, n), np.int64)
    scores = np.zeros((n_seq, n), np.float64)
    gaps = np.full((n_seq, n), INF)  # to the next candidate of another beam
    for b in range(n_seq):
        cand = []
        for k in range(beams):
            x = logits[b * beams + k].astype(np.float32)
            if base is not None:
                x = base[b].astype(np.float32) + x
            if prior is not None:
                x = x - np.float32(beta) * prior.astype(np.float32)
            if finished is not None and finished[b, k]:
                x = np.full(V, -INF, np.float32)
                x[pad] = 0.0
                p = np.where(x == 0, float(cum[b, k]), -INF)
            else:
                xd = x.astype(np.float64)
                top = xd.max()
                with np.errstate(invalid="ignore", divide="ignore"):
                    e = np.exp(xd - (top if np.isfinite(top) else 0.0))
                    p = np.where(xd == -INF, -INF, (xd - top) + (float(cum[b, k]) - np.log(e.sum())))
            best = np.lexsort((np.arange(V), -x.astype(np.float64)))[:n]
            cand += [(p[v], k, i, int(v)) for i, v in enumerate(best)]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        for j in range(n):
            scores[b, j], parents[b, j], _, tokens[b, j] = cand[j]
        for j in range(n):
            for other in (j - 1, j + 1):
                if 0 <= other < len(cand) and cand[other][1] != cand[j][1] and np.isfinite(cand[j][0]):
                    gaps[b, j] = min(gaps[b, j], abs(cand[other][0] - cand[j][0]))
    return parents, tokens, scores, gaps


# fp32 arithmetic of a score: sum_v exp has a relative error of at most a few 2^-23 (terms
# of 2 ulp, pairwise sums of at most 2^12 terms a lane), log, two additions and the final
# rounding each at most half an ulp of a magnitude below 64: under 64 * 2^-23 = 7.6e-6.
SCORE_TOL = 2e-5


def check_select(out, ref):
    parents, tokens, scores, gaps = ref
    got = out.scores.cpu().numpy().astype(np.float64)
    finite = np.isfinite(scores)
    np.testing.assert_array_equal(finite, np.isfinite(got))
    np.testing.assert_allclose(got[finite], scores[finite], rtol=2e-7, atol=SCORE_TOL)
    np.testing.assert_array_equal(got[~finite], scores[~finite])
    clear = gaps > 2 * SCORE_TOL  # the order within a beam is exact; across beams it goes by the score
    assert clear.mean() > 0.9
    np.testing.assert_array_equal(out.parents.cpu().numpy()[clear], parents[clear])
    np.testing.assert_array_equal(out.tokens.cpu().numpy()[clear], tokens[clear])


def to_dev(a, dev, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dev).to(dtype)


def make(seed, n_seq, beams, V, dtype, mix, dev, spread=3.0):
    rng = np.random.default_rng(seed)

    def typed(a):
        return torch.from_numpy(a.astype(np.float32)).to(dtype)

    logits = typed(rng.standard_normal((n_seq * beams, V)) * spread)
    base = typed(rng.standard_normal((n_seq, V)) * 3) if mix else None
    prior = typed(np.log((np.arange(1, V + 1) ** -1.1) / (np.arange(1, V + 1) ** -1.1).sum())).float() if mix else None
    cum = torch.from_numpy((rng.standard_normal((n_seq, beams)) * 1.5 - 6).astype(np.float32))
    return rng, logits, base, prior, cum


def np32(t):
    return None if t is None else t.float().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_seq,beams,select,V,mix", [
    (1, 1, 1, 1, False),       # one candidate
    (1, 1, 3, 3, False),       # the whole vocabulary
    (2, 4, 2, 2, True),
    (3, 2, 7, 255, True),
    (1, 4, 4, 257, False),     # a last group of one
    (2, 3, 6, 1000, True),
    (1, 1, 64, 4096, False),   # the widest selection
    (2, 64, 64, 1537, True),   # the most beams
    (4, 8, 8, 20000, True),
    (1, 5, 10, 50021, False),  # odd rows: element-wise loads
    (2, 4, 4, 151936, True),
])
def test_select_matches_definition(cuda_device, dtype, n_seq, beams, select, V, mix):
    from dels_b200 import ops

    dev = cuda_device
    _, logits, base, prior, cum = make(V + beams, n_seq, beams, V, dtype, mix, dev)
    beta = torch.full((1,), 0.2, device=dev)
    out = ops.beam_select(logits.to(dev), cum.to(dev), select=select, base=None if base is None else base.to(dev),
                          prior=None if prior is None else prior.to(dev), beta=beta if mix else None)
    ref = reference_select(np32(logits), cum.numpy(), select, np32(base), np32(prior), 0.2)
    check_select(out, ref)


@pytest.mark.parametrize("lowest", [-INF, torch.finfo(torch.bfloat16).min, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("kept", [0, 1, 3, 40])
def test_select_masked_rows(cuda_device, lowest, kept):
    """Rows with no, fewer and more allowed tokens than are selected; a mask of the type's
    lowest value is an ordinary logit, so a row masked whole by it is uniform."""
    from dels_b200 import ops

    dev = cuda_device
    dtype = torch.float32 if lowest == torch.finfo(torch.float32).min else torch.bfloat16
    rng, logits, _, _, cum = make(kept + 5, 3, 4, 3001, dtype, False, dev)
    full = logits.clone()
    logits.fill_(lowest)
    for r in range(12):
        at = torch.from_numpy(rng.permutation(3001)[:kept])
        logits[r, at] = full[r, at]
    logits[5] = full[5]  # one row without a mask
    out = ops.beam_select(logits.to(dev), cum.to(dev), select=8)
    check_select(out, reference_select(np32(logits), cum.numpy(), 8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_seq,beams,select,V", [
    (20, 1, 14, 1255), (31, 1, 27, 3920), (9, 2, 29, 1064), (2, 3, 64, 1100), (200, 2, 2, 1689), (3, 5, 40, 530),
    (2, 1, 64, 16384), (2, 1, 64, 16392),
])
def test_select_many_of_a_small_vocabulary(cuda_device, dtype, n_seq, beams, select, V):
    """More candidates than there are groups of logits, half of the vocabulary masked, some beams
    finished."""
    from dels_b200 import ops

    dev = cuda_device
    rng, logits, base, prior, cum = make(V + select, n_seq, beams, V, dtype, True, dev)
    logits[:, torch.from_numpy(rng.permutation(V)[: V // 2])] = -INF
    finished = torch.from_numpy(rng.random((n_seq, beams)) < 0.3)
    beta = torch.tensor([0.2], device=dev)
    out = ops.beam_select(logits.to(dev), cum.to(dev), select=select, base=base.to(dev), prior=prior.to(dev),
                          beta=beta, finished=finished.to(dev), pad_token=2)
    check_select(out, reference_select(np32(logits), cum.numpy(), select, np32(base), prior.numpy(), 0.2,
                                       finished.numpy(), 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [600, 5003, 20000])
def test_select_many_equal_logits(cuda_device, dtype, V):
    """More logits at one value than any list holds, few above it: everywhere, in the last tokens
    only, mixed with lower ones, or at the type's lowest value."""
    from dels_b200 import ops

    dev = cuda_device
    rng = np.random.default_rng(V)
    x = torch.zeros(8, V)
    x[1, : V - 400] = -3.0
    x[2, ::2] = -1.0
    x[3] = torch.finfo(dtype).min
    x[4] = torch.from_numpy(np.sort(rng.integers(0, 3, V))).float()
    x[5] = -0.0
    x[6, : V - 300] = -INF
    x[7] = float(torch.tensor(-1.17e-38).to(dtype))
    for r in range(8):
        x[r, torch.from_numpy(rng.permutation(V)[: 3 * (r % 4)])] = 2.0 + r
    x = x.to(dtype)
    cum = torch.from_numpy(rng.standard_normal((8, 1)).astype(np.float32))
    for select in (1, 16, 64):
        out = ops.beam_select(x.to(dev), cum.to(dev), select=select)
        check_select(out, reference_select(np32(x), cum.numpy(), select))
        both = ops.beam_select(x.to(dev), cum.view(4, 2).to(dev), select=select)
        ref = reference_select(np32(x), cum.view(4, 2).numpy(), select)
        np.testing.assert_allclose(both.scores.cpu().numpy(), ref[2], rtol=2e-7, atol=SCORE_TOL)


@pytest.mark.parametrize("V", [1000, 1003])
def test_select_scores_below_fp32(cuda_device, V):
    """Logits so far below the row's maximum that their scores fall to -inf: still the larger x
    first, before masked tokens."""
    from dels_b200 import ops

    dev = cuda_device
    x = torch.full((2, V), -INF)
    x[0, 5], x[0, 7], x[0, 900], x[0, 901] = 3e38, -3e38, -3e38, -2e38
    x[1, 6] = 1.0
    out = ops.beam_select(x.to(dev), torch.tensor([[-1.0, -2.0]], device=dev), select=6)
    assert out.tokens.tolist() == [[5, 6, 901, 7, 900, 0]]
    assert out.parents.tolist() == [[0, 1, 0, 0, 0, 0]]
    assert out.scores.tolist() == [[-1.0, -2.0] + [-INF] * 4]


def test_select_constant_and_sorted_rows(cuda_device):
    """Equal logits go to the lowest tokens; sorted rows put every candidate in one group."""
    from dels_b200 import ops

    dev = cuda_device
    V = 9001
    x = torch.stack([torch.zeros(V), torch.arange(V) / 64.0, -torch.arange(V) / 64.0, (torch.arange(V) % 256) / 8.0])
    cum = torch.tensor([[0.0, -1.0, -2.5, -0.25]])
    for n in (1, 5, 64):
        out = ops.beam_select(x.to(dev), cum.to(dev), select=n)
        check_select(out, reference_select(x.numpy(), cum.numpy(), n))


def test_select_equal_beams_take_the_lowest(cuda_device):
    """Identical beams give identical scores whatever their rows' alignment: the lower beam
    comes first, token by token."""
    from dels_b200 import ops

    dev = cuda_device
    for V in (1024, 1003):
        row = torch.from_numpy(np.random.default_rng(V).permutation(V).astype(np.float32) / 32)
        out = ops.beam_select(row.expand(4, V).contiguous().to(dev), torch.full((1, 4), -3.0, device=dev), select=8)
        assert out.parents.tolist() == [[0, 1, 2, 3, 0, 1, 2, 3]]
        top = row.argsort(descending=True)
        assert out.tokens.tolist() == [[int(top[0])] * 4 + [int(top[1])] * 4]
        assert out.scores[0, 0] == out.scores[0, 3] and out.scores[0, 4] == out.scores[0, 7]


def test_select_finished_beams(cuda_device):
    from dels_b200 import ops

    dev = cuda_device
    _, logits, _, _, cum = make(3, 3, 3, 700, torch.bfloat16, False, dev)
    finished = torch.tensor([[True, False, False], [False, False, False], [True, True, True]])
    # a finished beam's logits are not read: NaN there changes nothing
    dirty = logits.clone()
    for b in range(3):
        for k in range(3):
            if finished[b, k]:
                dirty[b * 3 + k] = float("nan")
    for pad in (0, 2, 699):
        out = ops.beam_select(dirty.to(dev), cum.to(dev), select=5, finished=finished.to(dev), pad_token=pad)
        check_select(out, reference_select(np32(logits), cum.numpy(), 5, finished=finished.numpy(), pad=pad))


def test_select_dead_beams_and_nan(cuda_device):
    """Beams at -1e9 and -inf lose to live ones; a NaN or +inf logit makes its row's scores
    NaN, which rank above all others."""
    from dels_b200 import ops

    dev = cuda_device
    _, logits, _, _, _ = make(9, 1, 4, 500, torch.float32, False, dev)
    cum = torch.tensor([[-1e9, -1.0, -INF, -1e9]])
    out = ops.beam_select(logits.to(dev), cum.to(dev), select=4)
    assert out.parents.tolist() == [[1, 1, 1, 1]]
    assert out.tokens.tolist() == [logits[1].argsort(descending=True)[:4].tolist()]
    for bad in (float("nan"), INF):
        x = logits.clone()
        x[2, 77] = bad
        out = ops.beam_select(x.to(dev), torch.zeros(1, 4, device=dev), select=4)
        assert out.parents.tolist() == [[2, 2, 2, 2]]
        assert torch.isnan(out.scores).all() and int(out.tokens[0, 0]) == 77


def test_select_strides_and_reuse(cuda_device):
    """Sliced logits and a base slice of [n_seq, steps, V] (rows at odd distances), outputs
    passed in, scores written over the input, a workspace holding another call's leavings,
    another stream."""
    from dels_b200 import ops

    dev = cuda_device
    n_seq, beams, V = 3, 4, 1003
    _, logits, base, prior, cum = make(21, n_seq, beams, V, torch.bfloat16, True, dev)
    wide = torch.full((n_seq * beams, V + 5), 99.0, dtype=torch.bfloat16, device=dev)
    wide[:, 3 : 3 + V] = logits.to(dev)
    steps = torch.full((n_seq, 3, V), 99.0, dtype=torch.bfloat16, device=dev)
    steps[:, 1] = base.to(dev)
    beta = torch.full((1,), 0.2, device=dev)
    ws = ops.Workspace(ops.beam_select_workspace_bytes(n_seq, beams, beams, V), dev)
    ws.buf[8:].fill_(0x5A)
    scores = cum.to(dev)
    out = ops.BeamOut(torch.empty(n_seq, beams, dtype=torch.int32, device=dev),
                      torch.empty(n_seq, beams, dtype=torch.int64, device=dev), scores)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.beam_select(wide[:, 3 : 3 + V], scores, base=steps[:, 1], prior=prior.to(dev), beta=beta, out=out, ws=ws)
    side.synchronize()
    check_select(out, reference_select(np32(logits), cum.numpy(), beams, np32(base), np32(prior), 0.2))


def test_select_empty_and_refusals(cuda_device):
    from dels_b200 import _lib, ops

    dev = cuda_device
    x = torch.zeros(0, 10, device=dev)
    assert ops.beam_select(x, torch.zeros(0, 4, device=dev)).tokens.shape == (0, 4)
    x, cum = torch.zeros(4, 10, device=dev), torch.zeros(2, 2, device=dev)
    with pytest.raises(_lib.DelsArgumentError, match="select"):
        ops.beam_select(x, cum, select=11)  # more than the vocabulary
    with pytest.raises(_lib.DelsArgumentError, match="1..64"):
        ops.beam_select(x, cum, select=0)
    with pytest.raises(_lib.DelsArgumentError, match="1..64"):
        ops.beam_select(torch.zeros(65, 99, device=dev), torch.zeros(1, 65, device=dev))
    with pytest.raises(_lib.DelsArgumentError, match="pad_token"):
        ops.beam_select(x, cum, finished=torch.zeros(2, 2, dtype=torch.bool, device=dev), pad_token=10)
    for bad in (
        dict(logits=x.half()), dict(logits=x.cpu()), dict(logits=x[:3]), dict(scores=cum.view(-1)),
        dict(scores=cum.double()), dict(base=torch.zeros(2, 10, dtype=torch.bfloat16, device=dev)),
        dict(base=torch.zeros(4, 10, device=dev)), dict(prior=torch.zeros(10, device=dev)),
        dict(prior=torch.zeros(9, device=dev), beta=torch.ones(1, device=dev)),
        dict(finished=torch.zeros(2, 2, device=dev)), dict(logits=torch.zeros(10, 4, device=dev).t()),
        dict(scores=torch.zeros(2, 4, device=dev)[:, ::2]),
    ):
        args = {"logits": x, "scores": cum, **bad}
        with pytest.raises(ValueError):
            ops.beam_select(args.pop("logits"), args.pop("scores"), **args)


# ----------------------------------------------------------------------------- reordering
def gather(src, parents, beams):
    n_seq = parents.shape[0]
    at = parents.long() + torch.arange(n_seq, device=parents.device)[:, None] * beams
    return src[at.view(-1)]


@pytest.mark.parametrize("n_seq,beams,select", [(1, 1, 1), (1, 4, 4), (3, 2, 7), (5, 8, 3), (2, 64, 64), (65, 3, 3)])
def test_reorder_moves_rows(cuda_device, n_seq, beams, select):
    """Rows of every width and alignment, several states in a call."""
    from dels_b200 import ops

    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(n_seq)
    parents = torch.randint(0, beams, (n_seq, select), generator=g, device=dev, dtype=torch.int32)
    rows = n_seq * beams
    states = [torch.randint(0, 256, (rows, w), generator=g, device=dev).to(torch.uint8)
              for w in (1, 2, 3, 15, 16, 17, 100, 1000, 4099, 20000)]
    states += [torch.randn(rows, 77, generator=g, device=dev), torch.randn(rows, 3, 5, 8, generator=g, device=dev).bfloat16(),
               torch.randint(0, 99, (rows, 14), generator=g, device=dev), torch.randn(rows, generator=g, device=dev),
               torch.randn(rows, 0, device=dev), torch.randn(rows, 6, 9, 16, generator=g, device=dev)[:, :, :7],
               torch.randn(rows, 33, generator=g, device=dev)[:, 1:]]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = ops.beam_reorder(states, parents, beams=beams, status=status)
    for src, dst in zip(states, out):
        assert torch.equal(dst, gather(src, parents, beams))
    assert int(status) == 0


@pytest.mark.parametrize("beams", [1, 2, 8, 64])
def test_reorder_in_place(cuda_device, beams):
    """Cycles, copies and rows that stay, with nothing outside the used part touched."""
    from dels_b200 import ops

    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(beams)
    parents = torch.stack([torch.roll(torch.arange(beams), 1), torch.zeros(beams, dtype=torch.long),
                           torch.arange(beams), torch.randint(0, beams, (beams,))]).int().to(dev)
    caches = [torch.randn(4 * beams, 3, 40, 16, generator=g, device=dev) for _ in range(2)]
    gru = torch.randn(4 * beams, 1021, generator=g, device=dev).bfloat16()
    want = [c.clone() for c in caches]
    for w, c in zip(want, caches):
        w[:, :, :29] = gather(c[:, :, :29], parents, beams)
    want_gru = gather(gru, parents, beams)
    states = [c[:, :, :29] for c in caches] + [gru]
    ops.beam_reorder(states, parents, beams=beams, out=states)
    for w, c in zip(want, caches):
        assert torch.equal(w, c)
    assert torch.equal(gru, want_gru)


def test_reorder_many_states_and_transposed_rows(cuda_device):
    """More states than one launch takes; a cache whose rows are not its outermost dimension."""
    from dels_b200 import ops

    dev = cuda_device
    parents = torch.tensor([[1, 0, 1], [2, 2, 0]], dtype=torch.int32, device=dev)
    states = [torch.randn(6, 5 + i, device=dev) for i in range(70)]
    layered = torch.randn(4, 6, 10, 8, device=dev)  # [layers, rows, ...]
    states += [layered[i] for i in range(4)] + [layered.transpose(0, 1)]
    out = ops.beam_reorder(states, parents, beams=3)
    for src, dst in zip(states, out):
        assert torch.equal(dst, gather(src, parents, 3))
    # in place over the transposed view: the layers are the runs of a row
    want = gather(layered.transpose(0, 1), parents, 3).transpose(0, 1)
    view = layered.transpose(0, 1)
    ops.beam_reorder([view], parents, beams=3, out=[view])
    assert torch.equal(layered, want)


def test_reorder_single_rows_of_wider_tensors(cuda_device):
    """One sequence with one beam: the row stride of such a slice says nothing of its length."""
    from dels_b200 import ops

    dev = cuda_device
    p = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    wide = torch.randn(3, 50, device=dev)
    assert ops._beam_state(0, wide[1:2, :7], wide[2:3, :7])[-1] == 28
    out = torch.full((3, 50), 7.0, device=dev)
    ops.beam_reorder([wide[1:2, :7]], p, beams=1, out=[out[1:2, 3:10]])
    assert torch.equal(out[1, 3:10], wide[1, :7]) and (out[[0, 2]] == 7).all() and (out[1, 10:] == 7).all()


def test_reorder_bad_parent_is_reported(cuda_device):
    from dels_b200 import _lib, ops

    dev = cuda_device
    src = torch.arange(8.0, device=dev).view(4, 2)
    out = torch.full((4, 2), -1.0, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    parents = torch.tensor([[1, 2], [-1, 0]], dtype=torch.int32, device=dev)
    ops.beam_reorder([src], parents, beams=2, out=[out], status=status)
    assert int(status) == _lib.DELS_ERR_INVALID_ARG
    assert out.tolist() == [[2.0, 3.0], [-1.0, -1.0], [-1.0, -1.0], [4.0, 5.0]]


def test_reorder_refusals(cuda_device):
    from dels_b200 import _lib, ops

    dev = cuda_device
    p = torch.zeros(2, 2, dtype=torch.int32, device=dev)
    x = torch.zeros(4, 8, device=dev)
    assert ops.beam_reorder([], p, beams=2) == []
    assert ops.beam_reorder([x[:0]], p[:0], beams=2)[0].shape == (0, 8)
    with pytest.raises(_lib.DelsArgumentError, match="overlap"):
        big = torch.zeros(6, 8, device=dev)
        ops.beam_reorder([big[:4]], p, beams=2, out=[big[2:]])
    with pytest.raises(_lib.DelsArgumentError, match="overlap"):
        ops.beam_reorder([x], p, beams=2, out=[torch.zeros(1, 8, device=dev).expand(4, 8)])
    with pytest.raises(_lib.DelsArgumentError, match="1..64"):
        ops.beam_reorder([torch.zeros(130, 1, device=dev)], p, beams=65)
    for bad in (
        lambda: ops.beam_reorder([x], p.long(), beams=2),
        lambda: ops.beam_reorder([x], p, beams=3),
        lambda: ops.beam_reorder([x], p, beams=2, out=[]),
        lambda: ops.beam_reorder([x], p, beams=2, out=[torch.zeros(4, 7, device=dev)]),
        lambda: ops.beam_reorder([x], p, beams=2, out=[x.double()]),
        lambda: ops.beam_reorder([x.cpu()], p, beams=2),
        # runs at two distances
        lambda: ops.beam_reorder([torch.zeros(4, 3, 4, 5, device=dev).permute(0, 2, 1, 3)[:, :, :2, :3]], p, beams=2),
    ):
        with pytest.raises(ValueError):
            bad()
