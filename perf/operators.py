"""Cases of the beam-drafting operators: the 8-bit integer product behind the long logits,
the selection over beams and vocabulary, and the reordering of the beams' states.

``run`` computes an operator in its plain form (elementary torch operations, 32 bits) or,
with ``own`` set, through ``dels_b200.ops``.  ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dels-spec_b200")
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_VOCAB = 151936


def _ops():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from dels_b200 import ops

    return ops


# ---------------------------------------------------------------------------- cases
def _linear(rows, K, N, dtype, bias, name=None):
    case = {"op": "linear_w8a8", "rows": rows, "K": K, "N": N, "dtype": dtype, "bias": bias}
    return case if name is None else {"name": name, **case}


def _select(B, beams, select, V, dtype, mix, mask, finished, name=None):
    case = {"op": "beam_select", "B": B, "beams": beams, "select": select, "V": V, "dtype": dtype, "mix": mix,
            "mask": mask, "finished": finished}
    return case if name is None else {"name": name, **case}


def _reorder(kind, B, beams, select, width, length, heads, layers, inplace, name=None):
    case = {"op": "beam_reorder", "kind": kind, "B": B, "beams": beams, "select": select, "width": width,
            "length": length, "heads": heads, "layers": layers, "inplace": inplace}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # the rank projection [256, 4096] of one hidden row: the smallest product of a draft step
        _linear(1, 4096, 256, "bf16", False, "rank projection, 1 row"),
        # the long logits of one sequence's draft block: streams the whole LM head
        _linear(16, 4096, _VOCAB, "bf16", False, "lm head, 16 rows"),
        # the long logits of 32 sequences x 16 positions: bound by the tensor cores
        _linear(512, 4096, _VOCAB, "bf16", False, "lm head, 512 rows"),
        # a biased fp32 layer whose sizes divide nothing
        _linear(77, 2561, 1003, "f32", True, "odd sizes, fp32"),
        # one sequence, four beams, one draft step: latency counts
        _select(1, 4, 4, _VOCAB, "bf16", True, "none", False, "select, 1 x 4 beams"),
        # a full serving batch of the same step
        _select(64, 8, 8, _VOCAB, "bf16", True, "none", False, "select, 64 x 8 beams"),
        # constrained decoding in fp32: a few allowed tokens, rows without any, finished beams, odd vocabulary
        _select(5, 3, 6, 32003, "f32", False, "few", True, "select, masked fp32"),
        # the first step: one root per sequence opens 16 beams, half of the vocabulary masked
        _select(64, 1, 16, _VOCAB, "bf16", False, "half", False, "select, first step"),
        # one sequence's GRU state and token history
        _reorder("gru", 1, 4, 4, 1024, 14, 1, 1, False, "reorder, 1 x 4 beams"),
        # the same for a full serving batch
        _reorder("gru", 64, 8, 8, 1024, 14, 1, 1, False, "reorder, 64 x 8 beams"),
        # two layers of a key and value cache, the used part of a longer allocation, in place
        _reorder("cache", 4, 8, 8, 128, 1537, 8, 2, True, "reorder, kv cache"),
        # beams opening from three to five, rows of an odd number of bytes
        _reorder("bytes", 7, 3, 5, 4099, 1, 1, 1, False, "reorder, odd bytes"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_w8a8", "beam_select", "beam_reorder"])
    if op == "linear_w8a8":
        K, N = _log_int(rng, 64, 6000), _log_int(rng, 64, _VOCAB)
        rows = _log_int(rng, 1, 512)
        if rng.random() < 0.5:
            K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
        N = min(N, 4096 * _VOCAB // K)
        return _linear(rows, K, N, rng.choice(["bf16", "f32"]), rng.random() < 0.5)
    if op == "beam_select":
        beams = _log_int(rng, 1, 16)
        select = min(32, beams * rng.choice([1, 1, 2]) if beams > 1 else rng.randint(1, 32))
        V = _log_int(rng, 1000, _VOCAB)
        if rng.random() < 0.5:
            V = V // 64 * 64
        dtype = rng.choice(["bf16", "bf16", "f32"])
        most = max(1, (512 if dtype == "bf16" else 256) // beams)
        return _select(_log_int(rng, 1, most), beams, select, V, dtype, rng.random() < 0.6,
                       rng.choice(["none", "none", "half", "few"]), rng.random() < 0.3)
    kind = rng.choice(["gru", "cache", "bytes"])
    beams = _log_int(rng, 1, 16)
    inplace = beams > 1 and rng.random() < 0.4
    select = beams if inplace else max(1, min(32, beams + rng.randint(-beams // 2, beams)))
    if kind == "cache":
        B = _log_int(rng, 1, max(1, 32 // max(beams, select)))
        return _reorder(kind, B, beams, select, rng.choice([64, 96, 128]), _log_int(rng, 1, 1500), rng.choice([1, 4, 8]),
                        rng.randint(1, 2), inplace)
    B = _log_int(rng, 1, max(1, 512 // max(beams, select)))
    width = _log_int(rng, 64, 4096) if kind == "gru" else _log_int(rng, 1, 9000)
    return _reorder(kind, B, beams, select, width, rng.randint(1, 16), 1, 1, inplace)


# ---------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _padded(rows, cols, step, dtype):
    """A [rows, cols] matrix whose row stride is a multiple of `step`."""
    return torch.zeros(rows, -(-cols // step) * step, dtype=dtype, device="cuda")[:, :cols]


def _prepare_linear(case, g):
    rows, K, N, dtype = case["rows"], case["K"], case["N"], _DTYPES[case["dtype"]]
    x = torch.randn(rows, K, generator=g, device="cuda").to(dtype)
    # channels quantised at load time: about N(0, 0.02) weights, 127 at four deviations
    wq = _padded(N, K, 16, torch.int8)
    for n in range(0, N, 16384):
        part = torch.randn(min(16384, N - n), K, generator=g, device="cuda").mul_(32)
        wq[n : n + 16384] = part.round_().clamp_(-127, 127).to(torch.int8)
    w_scale = (0.5 + torch.rand(N, generator=g, device="cuda")) * (0.02 / 32)
    bias = torch.randn(N, generator=g, device="cuda").to(dtype) if case["bias"] else None
    return {"op": case["op"], "x": x, "wq": wq, "w_scale": w_scale, "bias": bias, "dtype": dtype}


def _prepare_select(case, g):
    B, beams, V, dtype = case["B"], case["beams"], case["V"], _DTYPES[case["dtype"]]
    rows = B * beams
    spread = 1.0 if case["mix"] else 3.0  # local-head logits beside draft logits, or whole logits
    logits = torch.empty(rows, V, dtype=dtype, device="cuda")
    for r in range(0, rows, 64):
        logits[r : r + 64] = torch.randn(min(64, rows - r), V, generator=g, device="cuda").mul_(spread).to(dtype)
    if case["mask"] == "half":
        keep = torch.rand(V, generator=g, device="cuda") < 0.5
        logits[:, ~keep] = -math.inf
    elif case["mask"] == "few":  # three allowed tokens a row, none in the last row
        allowed = torch.randint(0, V, (rows, 3), generator=g, device="cuda")
        kept = logits.gather(1, allowed)
        logits.fill_(-math.inf)
        logits.scatter_(1, allowed, kept)
        logits[rows - 1] = -math.inf
    base = prior = beta = None
    if case["mix"]:
        base = torch.randn(B, V, generator=g, device="cuda").mul_(3.0).to(dtype)
        p = torch.arange(1, V + 1, dtype=torch.float64, device="cuda").pow(-1.1)
        prior = torch.log(p / p.sum()).to(torch.bfloat16).to(torch.float32)
        beta = torch.full((1,), 0.2, dtype=torch.float32, device="cuda")
    scores = torch.randn(B, beams, generator=g, device="cuda").mul_(1.5).sub_(6.0)
    finished = None
    if case["finished"]:
        finished = torch.rand(B, beams, generator=g, device="cuda") < 0.3
    return {"op": case["op"], "logits": logits, "scores": scores, "base": base, "prior": prior, "beta": beta,
            "finished": finished, "beams": beams, "select": case["select"], "pad": 2}


def _prepare_reorder(case, g):
    B, beams, select = case["B"], case["beams"], case["select"]
    src, out = [], []
    if case["kind"] == "gru":
        src = [torch.randn(B * beams, case["width"], generator=g, device="cuda").to(torch.bfloat16),
               torch.randint(0, _VOCAB, (B * beams, case["length"]), generator=g, device="cuda")]
        out = [torch.zeros(B * select, *t.shape[1:], dtype=t.dtype, device="cuda") for t in src]
    elif case["kind"] == "cache":
        used = case["length"]
        room = used + max(1, used // 3)
        for _ in range(2 * case["layers"]):
            t = torch.empty(B * beams, case["heads"], room, case["width"], dtype=torch.bfloat16, device="cuda")
            t.normal_(generator=g)
            src.append(t[:, :, :used])
            out.append(torch.zeros(B * select, case["heads"], room, case["width"], dtype=torch.bfloat16,
                                   device="cuda")[:, :, :used] if not case["inplace"] else None)
    else:
        src = [torch.randint(0, 256, (B * beams, case["width"]), generator=g, device="cuda").to(torch.uint8)]
        out = [torch.zeros(B * select, case["width"], dtype=torch.uint8, device="cuda")]
    parents = torch.randint(0, beams, (B, select), generator=g, device="cuda", dtype=torch.int32)
    return {"op": case["op"], "src": src, "out": src if case["inplace"] else out, "parents": parents, "beams": beams,
            "inplace": case["inplace"]}


def prepare(case, seed):
    make = {"linear_w8a8": _prepare_linear, "beam_select": _prepare_select, "beam_reorder": _prepare_reorder}
    return make[case["op"]](case, _generator(seed))


# ---------------------------------------------------------------------------- plain forms
def _plain_linear(s):
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    scale = top / 127
    q = (x * torch.where(top > 0, 127 / top, 0.0)).round().clamp(-127, 127)
    y = (q @ s["wq"].float().t()) * scale * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["dtype"])


def _descending(x, n):
    """Values and positions of the n largest of each row; the lowest position among equals."""
    i = (x + 0.0).view(torch.int32).long()
    i = torch.where(i < 0, i ^ 0x7FFFFFFF, i)
    place = torch.arange(x.shape[-1], device=x.device)
    at = 0xFFFFFFFF - (torch.topk((i << 32) | (0xFFFFFFFF - place), n, dim=-1).values & 0xFFFFFFFF)
    return x.gather(-1, at), at


def _plain_select(s):
    B, beams = s["scores"].shape
    n = s["select"]
    x = s["logits"].float()
    if s["base"] is not None:
        x = ((s["base"].float()[:, None] + x.view(B, beams, -1)) - s["beta"] * s["prior"]).view(B * beams, -1)
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    shift = s["scores"].reshape(-1, 1) - torch.log(torch.exp(x - m).sum(1, keepdim=True))
    if s["finished"] is not None:
        done = s["finished"].reshape(-1, 1)
        pad = torch.arange(x.shape[1], device=x.device) == s["pad"]
        x = torch.where(done, torch.where(pad, 0.0, -math.inf), x)
        m = torch.where(done, 0.0, m)
        shift = torch.where(done, s["scores"].reshape(-1, 1), shift)
    value, token = _descending(x, n)
    score = torch.where(value == -math.inf, -math.inf, (value - m) + shift).view(B, beams * n)
    score, at = _descending(score, n)
    return {"parents": (at // n).to(torch.int32), "tokens": token.view(B, beams * n).gather(1, at), "scores": score}


def _plain_reorder(s):
    B = s["parents"].shape[0]
    rows = (s["parents"].long() + torch.arange(B, device="cuda")[:, None] * s["beams"]).view(-1)
    if s["inplace"]:
        return [t.copy_(t.index_select(0, rows)) for t in s["out"]]
    return [torch.index_select(t, 0, rows, out=o) if o.is_contiguous() else o.copy_(t.index_select(0, rows))
            for t, o in zip(s["src"], s["out"])]


# ---------------------------------------------------------------------------- the framework's calls
def _own_linear(s):
    return _ops().linear_w8a8(s["x"], s["wq"], s["w_scale"], s["bias"], out_dtype=s["dtype"])


def _own_select(s):
    r = _ops().beam_select(s["logits"], s["scores"], select=s["select"], base=s["base"], prior=s["prior"],
                           beta=s["beta"], finished=s["finished"], pad_token=s["pad"])
    return {"parents": r.parents, "tokens": r.tokens, "scores": r.scores}


def _own_reorder(s):
    return _ops().beam_reorder(s["src"], s["parents"], beams=s["beams"], out=s["out"])


def run(state):
    plain = {"linear_w8a8": _plain_linear, "beam_select": _plain_select, "beam_reorder": _plain_reorder}
    ours = {"linear_w8a8": _own_linear, "beam_select": _own_select, "beam_reorder": _own_reorder}
    return (ours if own else plain)[state["op"]](state)


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {"bf16": 2, "f32": 4}[case["dtype"]] if "dtype" in case else 1
    if case["op"] == "linear_w8a8":
        rows, K, N = case["rows"], case["K"], case["N"]
        moved = rows * K * size + N * K + 4 * N + rows * N * size + (N * size if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * rows * N * K}
    if case["op"] == "beam_select":
        rows, V = case["B"] * case["beams"], case["V"]
        if case["finished"]:  # their logits need not be read
            rows = 0.7 * rows
        moved = rows * V * size + 4 * rows + 16 * case["B"] * case["select"]
        if case["mix"]:
            moved += case["B"] * V * size + 4 * V
        return {"bytes": moved, "flops": (5 if case["mix"] else 3) * rows * V}
    if case["kind"] == "gru":
        row = case["width"] * 2 + case["length"] * 8
    elif case["kind"] == "cache":
        row = 2 * case["layers"] * case["heads"] * case["length"] * case["width"] * 2
    else:
        row = case["width"]
    # parents are drawn at random: the share of a sequence's rows that some child reads, and
    # (in place) the share of the rows that change
    beams, select = case["beams"], case["select"]
    read = beams * (1 - (1 - 1 / beams) ** select)
    write = select * (1 - 1 / beams) if case["inplace"] else select
    return {"bytes": case["B"] * (read + write) * row + 4 * case["B"] * select, "flops": 0}


# ---------------------------------------------------------------------------- 64 bits
def _exact_linear(case, s):
    x = s["x"].double()
    top = x.abs().max(dim=1).values[:, None]
    q = torch.clamp(torch.round(x * (127.0 / top)), -127, 127)
    left = q * (top / 127.0)
    y = torch.empty(case["rows"], case["N"], dtype=torch.float64, device="cuda")
    for n in range(0, case["N"], 16384):
        w = s["wq"][n : n + 16384].double() * s["w_scale"][n : n + 16384, None].double()
        y[:, n : n + 16384] = left @ w.t()
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_select(case, s):
    """Only the scores: their n largest, over every beam's log-softmax at once."""
    B, beams, V = case["B"], case["beams"], case["V"]
    best = torch.empty(B, case["select"], dtype=torch.float64, device="cuda")
    for b in range(B):
        x = s["logits"][b * beams : (b + 1) * beams].double()
        if s["base"] is not None:
            x = s["base"][b].double() + x - s["beta"].double() * s["prior"].double()
        total = torch.logsumexp(x, dim=1, keepdim=True)
        p = torch.where(x == -math.inf, x, x - total) + s["scores"][b].double()[:, None]
        if s["finished"] is not None:
            for k in torch.nonzero(s["finished"][b]).view(-1).tolist():
                p[k] = -math.inf
                p[k, s["pad"]] = s["scores"][b, k].double()
        best[b] = torch.sort(p.reshape(-1), descending=True).values[: case["select"]] if beams * V < 1 << 16 else \
            torch.topk(p.reshape(-1), case["select"]).values
    return {"parents": None, "tokens": None, "scores": best}


def exact(case, seed):
    if case["op"] == "beam_reorder":
        return None  # moves bytes: compared bit by bit with the plain form
    s = prepare(case, seed)
    return (_exact_linear if case["op"] == "linear_w8a8" else _exact_select)(case, s)
