"""Torch-facing wrappers of the C ABI (``include/dels_b200.h``).

Every function takes CUDA tensors, checks dtypes and shapes, and enqueues the CUDA
kernels on the current stream through :mod:`dels_b200._lib`.  Outputs can be passed in
(``out=`` arguments) so that callers which capture CUDA graphs allocate nothing per
call.  There is deliberately no CPU or PyTorch fallback.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass

import torch

from . import _lib

ACTIVATIONS = {"identity": _lib.DELS_ACT_IDENTITY, "silu": _lib.DELS_ACT_SILU}


def _ptr(t: torch.Tensor | None) -> ctypes.c_void_p | None:
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _require_cuda(name: str, t: torch.Tensor, dtype: torch.dtype, ndim: int | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device}); there is no CPU path")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} (got {t.dtype})")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D (got shape {tuple(t.shape)})")


def _row_major(name: str, t: torch.Tensor) -> int:
    """Leading dimension (elements) of a 2-D tensor with unit column stride."""
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D (got shape {tuple(t.shape)})")
    if t.numel() == 0:
        return max(int(t.shape[1]), 1)
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name} must have contiguous rows (stride {tuple(t.stride())})")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), int(t.shape[1]))


def _f32_vec(name: str, t: torch.Tensor | None, device: torch.device) -> torch.Tensor | None:
    if t is None:
        return None
    _require_cuda(name, t, torch.float32, 1)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _i32_vec(name: str, t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None:
        return None
    _require_cuda(name, t, torch.int32, 1)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def init(device: torch.device | int | None = None) -> None:
    """Load the kernels on ``device`` (do this before capturing a CUDA graph)."""
    if device is None:
        index = torch.cuda.current_device()
    elif isinstance(device, int):
        index = device
    else:
        index = torch.device(device).index
        index = torch.cuda.current_device() if index is None else index
    _lib.call("dels_init", int(index))


class Workspace:
    """Zero-initialised, 256-byte-aligned device scratch owned by the caller.

    The first 8 bytes hold the completion counter and the device status word that the
    kernels use; :meth:`status` reads the latter (one device-to-host copy)."""

    def __init__(self, nbytes: int, device: torch.device):
        nbytes = max(int(nbytes), _lib.DELS_WS_HEADER_BYTES)
        self._raw = torch.zeros(nbytes + 256, dtype=torch.uint8, device=device)
        off = (-self._raw.data_ptr()) % 256
        self.buf = self._raw[off : off + nbytes]
        self.nbytes = nbytes
        self.device = device

    def ensure(self, nbytes: int) -> "Workspace":
        return self if nbytes <= self.nbytes else Workspace(nbytes, self.device)

    @property
    def ptr(self) -> ctypes.c_void_p:
        return ctypes.c_void_p(self.buf.data_ptr())

    def status(self) -> int:
        return int(self.buf[4:8].view(torch.int32).item())

    def clear_status(self) -> None:
        self.buf[4:8].zero_()

    def check(self) -> None:
        """Raise if a kernel recorded a device-side failure (synchronises)."""
        st = self.status()
        if st != 0:
            self.clear_status()
            raise _lib.DelsError("device", st, _lib.load().dels_status_string(st).decode())


_ws_cache: dict[tuple[int, int], Workspace] = {}
_capture_ws: dict[tuple[int, int], tuple[int, Workspace]] = {}


def _capture_id(stream: int) -> int:
    """The number of the graph capture that the current stream, ``stream``, is part of; 0 outside one."""
    if not torch._C._cuda_isCurrentStreamCapturing():
        return 0
    return int(_lib.query("dels_stream_capture_id", stream))


def workspace(nbytes: int, device: torch.device) -> Workspace:
    """A cached workspace per (device, stream) large enough for ``nbytes``.

    A graph keeps the addresses that its capture saw, so a capture shares no workspace with
    calls outside it or with another capture (``torch.cuda.graph`` captures on one stream by
    default): it gets one of its own, in the graph's memory pool."""
    return _stream_workspace(nbytes, device, torch.cuda.current_stream(device).cuda_stream)


def _stream_workspace(nbytes: int, device: torch.device, stream: int) -> Workspace:
    """workspace() for a stream that is known already."""
    key = (device.index or 0, stream)
    capture = _capture_id(stream)
    if capture:
        # a larger one for a later call of the same capture: the pool gives the smaller one's memory
        # to what the capture allocates after it, which runs after it
        last, ws = _capture_ws.get(key, (0, None))
        if last != capture or ws.nbytes < nbytes:
            ws = Workspace(max(nbytes, 1 << 20), device)
            _capture_ws[key] = (capture, ws)
        return ws
    ws = _ws_cache.get(key)
    if ws is None or ws.nbytes < nbytes:
        ws = Workspace(max(nbytes, 1 << 20), device)
        _ws_cache[key] = ws
    return ws


def _positions(n_pos: int | None, alpha: torch.Tensor | None, beta: torch.Tensor | None) -> int:
    if n_pos is not None:
        return int(n_pos)
    for t in (alpha, beta):
        if t is not None:
            return int(t.numel())
    return 1


# --------------------------------------------------------------------------- scorer
@dataclass
class ScoreOut:
    tokens: torch.Tensor  # int64 [rows]
    scores: torch.Tensor | None  # fp32 [rows]
    keys: torch.Tensor  # int64 [rows] packed (score, index) keys


def draft_score_bf16(
    h: torch.Tensor,
    W: torch.Tensor,
    w_rank: torch.Tensor,
    Vr: torch.Tensor,
    prior: torch.Tensor | None,
    alpha: torch.Tensor,
    beta: torch.Tensor,
    *,
    n_pos: int | None = None,
    row_pos: torch.Tensor | None = None,
    rows_dev: torch.Tensor | None = None,
    v_begin: int = 0,
    activation: str = "identity",
    keys_only: bool = False,
    with_scores: bool = False,
    out: ScoreOut | None = None,
    ws: Workspace | None = None,
) -> ScoreOut:
    """argmax_v (h.W[v] + alpha_p * act(h.w_rank^T).Vr[v] - beta_p * prior[v]) per row.

    ``W``/``Vr``/``prior`` may be one rank's contiguous vocabulary slice starting at
    global index ``v_begin``; with ``keys_only=True`` the packed keys are returned
    undecoded for a cross-rank all-reduce(MAX) (then :func:`keys_decode`)."""
    dev = h.device
    for name, t in (("h", h), ("W", W), ("w_rank", w_rank), ("Vr", Vr)):
        _require_cuda(name, t, torch.bfloat16, 2)
    rows, H = h.shape
    V = W.shape[0]
    r = w_rank.shape[0]
    if W.shape[1] != H or w_rank.shape[1] != H or Vr.shape != (V, r):
        raise ValueError(f"shape mismatch: h {tuple(h.shape)}, W {tuple(W.shape)}, w_rank {tuple(w_rank.shape)}, "
                         f"Vr {tuple(Vr.shape)}")
    prior = _f32_vec("prior", prior, dev)
    alpha = _f32_vec("alpha", alpha, dev)
    beta = _f32_vec("beta", beta, dev)
    row_pos = _i32_vec("row_pos", row_pos)
    rows_dev = _i32_vec("rows_dev", rows_dev)
    if prior is not None and prior.numel() != V:
        raise ValueError(f"prior has {prior.numel()} entries, expected {V}")
    npos = _positions(n_pos, alpha, beta)
    if out is None:
        out = ScoreOut(
            tokens=torch.empty(rows, dtype=torch.int64, device=dev),
            scores=torch.empty(rows, dtype=torch.float32, device=dev) if with_scores else None,
            keys=torch.empty(rows, dtype=torch.int64, device=dev),
        )
    need = _lib.query("dels_score_workspace_bytes", rows, H, r)
    ws = workspace(need, dev) if ws is None else ws.ensure(need)
    _lib.call(
        "dels_draft_score_bf16",
        _ptr(h), _row_major("h", h),
        _ptr(W), _row_major("W", W), _ptr(w_rank), _row_major("w_rank", w_rank), _ptr(Vr), _row_major("Vr", Vr),
        _ptr(prior), _ptr(alpha), _ptr(beta), npos, _ptr(row_pos), rows, _ptr(rows_dev), H, r, V, int(v_begin),
        ACTIVATIONS[activation], _ptr(out.keys), None if keys_only else _ptr(out.tokens),
        None if (keys_only or out.scores is None) else _ptr(out.scores), ws.ptr, ws.nbytes, _stream(dev),
    )
    return out


def rank_project_bf16(
    x: torch.Tensor,
    w_rank: torch.Tensor,
    alpha: torch.Tensor | None,
    *,
    n_pos: int | None = None,
    row_pos: torch.Tensor | None = None,
    activation: str = "identity",
    s_out: torch.Tensor | None = None,
    s_scaled: torch.Tensor | None = None,
    keys: torch.Tensor | None = None,
    want_state: bool = True,
    ws: Workspace | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor]:
    """(s, alpha_p * s) with s = bf16(act(bf16(x . w_rank^T))); optionally resets keys."""
    dev = x.device
    _require_cuda("x", x, torch.bfloat16, 2)
    _require_cuda("w_rank", w_rank, torch.bfloat16, 2)
    rows, K = x.shape
    r = w_rank.shape[0]
    if w_rank.shape[1] != K:
        raise ValueError(f"w_rank {tuple(w_rank.shape)} does not match x {tuple(x.shape)}")
    alpha = _f32_vec("alpha", alpha, dev)
    row_pos = _i32_vec("row_pos", row_pos)
    if s_scaled is None:
        s_scaled = torch.empty(rows, r, dtype=torch.bfloat16, device=dev)
    if want_state and s_out is None:
        s_out = torch.empty(rows, r, dtype=torch.bfloat16, device=dev)
    need = _lib.query("dels_rank_workspace_bytes", rows, K, r)
    ws = workspace(need, dev) if ws is None else ws.ensure(need)
    _lib.call(
        "dels_rank_project_bf16",
        _ptr(x), _row_major("x", x), _ptr(w_rank), _row_major("w_rank", w_rank), rows, K, r, ACTIVATIONS[activation],
        _ptr(alpha), _positions(n_pos, alpha, None), _ptr(row_pos), _ptr(s_out), _ptr(s_scaled), _ptr(keys),
        ws.ptr, ws.nbytes, _stream(dev),
    )
    return s_out, s_scaled


def fused_argmax_bf16(
    h: torch.Tensor,
    W: torch.Tensor,
    s_scaled: torch.Tensor,
    Vr: torch.Tensor,
    prior: torch.Tensor | None,
    beta: torch.Tensor,
    *,
    n_pos: int | None = None,
    row_pos: torch.Tensor | None = None,
    rows_dev: torch.Tensor | None = None,
    v_begin: int = 0,
    keys_ready: bool = False,
    keys_only: bool = False,
    with_scores: bool = False,
    out: ScoreOut | None = None,
    ws: Workspace | None = None,
) -> ScoreOut:
    """Scorer with a precomputed bf16 operand ``s_scaled`` = alpha_p * rank state."""
    dev = h.device
    for name, t in (("h", h), ("W", W), ("s_scaled", s_scaled), ("Vr", Vr)):
        _require_cuda(name, t, torch.bfloat16, 2)
    rows, H = h.shape
    V, r = Vr.shape
    if W.shape != (V, H) or s_scaled.shape != (rows, r):
        raise ValueError("shape mismatch between h, W, s_scaled and Vr")
    prior = _f32_vec("prior", prior, dev)
    beta = _f32_vec("beta", beta, dev)
    if out is None:
        out = ScoreOut(
            tokens=torch.empty(rows, dtype=torch.int64, device=dev),
            scores=torch.empty(rows, dtype=torch.float32, device=dev) if with_scores else None,
            keys=torch.empty(rows, dtype=torch.int64, device=dev),
        )
    ws = workspace(_lib.DELS_WS_HEADER_BYTES, dev) if ws is None else ws
    _lib.call(
        "dels_fused_argmax_bf16",
        _ptr(h), _row_major("h", h), _ptr(W), _row_major("W", W), _ptr(s_scaled), _row_major("s_scaled", s_scaled),
        _ptr(Vr), _row_major("Vr", Vr), _ptr(prior), _ptr(beta), _positions(n_pos, None, beta),
        _ptr(_i32_vec("row_pos", row_pos)), rows, _ptr(_i32_vec("rows_dev", rows_dev)), H, r, V, int(v_begin),
        _lib.DELS_FLAG_KEYS_READY if keys_ready else 0, _ptr(out.keys), None if keys_only else _ptr(out.tokens),
        None if (keys_only or out.scores is None) else _ptr(out.scores), ws.ptr, ws.nbytes, _stream(dev),
    )
    return out


def fused_argmax_base_bf16(
    base: torch.Tensor,
    s_scaled: torch.Tensor,
    Vr: torch.Tensor,
    prior: torch.Tensor | None,
    beta: torch.Tensor,
    *,
    n_pos: int | None = None,
    row_pos: torch.Tensor | None = None,
    v_begin: int = 0,
    keys_ready: bool = False,
    with_scores: bool = False,
    out: ScoreOut | None = None,
    ws: Workspace | None = None,
) -> ScoreOut:
    """Runner step: argmax_v(base[i, v] + s_scaled[i].Vr[v] - beta_p prior[v])."""
    dev = base.device
    for name, t in (("base", base), ("s_scaled", s_scaled), ("Vr", Vr)):
        _require_cuda(name, t, torch.bfloat16, 2)
    rows, V = base.shape
    r = Vr.shape[1]
    if Vr.shape[0] != V or s_scaled.shape != (rows, r):
        raise ValueError("shape mismatch between base, s_scaled and Vr")
    prior = _f32_vec("prior", prior, dev)
    beta = _f32_vec("beta", beta, dev)
    if out is None:
        out = ScoreOut(
            tokens=torch.empty(rows, dtype=torch.int64, device=dev),
            scores=torch.empty(rows, dtype=torch.float32, device=dev) if with_scores else None,
            keys=torch.empty(rows, dtype=torch.int64, device=dev),
        )
    ws = workspace(_lib.DELS_WS_HEADER_BYTES, dev) if ws is None else ws
    _lib.call(
        "dels_fused_argmax_base_bf16",
        _ptr(base), _row_major("base", base), _ptr(s_scaled), _row_major("s_scaled", s_scaled), _ptr(Vr),
        _row_major("Vr", Vr), _ptr(prior), _ptr(beta), _positions(n_pos, None, beta),
        _ptr(_i32_vec("row_pos", row_pos)), rows, None, r, V, int(v_begin),
        _lib.DELS_FLAG_KEYS_READY if keys_ready else 0, _ptr(out.keys), _ptr(out.tokens),
        None if out.scores is None else _ptr(out.scores), ws.ptr, ws.nbytes, _stream(dev),
    )
    return out


def fused_argmax_base_gru_bf16(
    base: torch.Tensor,
    s_scaled: torch.Tensor,
    Vr: torch.Tensor,
    prior: torch.Tensor | None,
    beta: torch.Tensor,
    w_hh: torch.Tensor,
    b_hh: torch.Tensor | None,
    h: torch.Tensor,
    gh_out: torch.Tensor,
    *,
    keys_ready: bool = False,
    out: ScoreOut,
    ws: Workspace,
) -> ScoreOut:
    """fused_argmax_base_bf16 for a rollout step of at most 4 rows that also computes the
    next step's gh_out = bf16(w_hh . h + b_hh) in the same launch."""
    dev = base.device
    for name, t in (("base", base), ("s_scaled", s_scaled), ("Vr", Vr), ("w_hh", w_hh), ("h", h), ("gh_out", gh_out)):
        _require_cuda(name, t, torch.bfloat16, 2)
    rows, V = base.shape
    r = Vr.shape[1]
    G = h.shape[1]
    if Vr.shape[0] != V or s_scaled.shape != (rows, r):
        raise ValueError("shape mismatch between base, s_scaled and Vr")
    if w_hh.shape != (3 * G, G) or not w_hh.is_contiguous() or h.shape != (rows, G) or not h.is_contiguous() \
            or gh_out.shape != (rows, 3 * G) or not gh_out.is_contiguous():
        raise ValueError("GRU operands do not match")
    _lib.call(
        "dels_fused_argmax_base_gru_bf16",
        _ptr(base), _row_major("base", base), _ptr(s_scaled), _row_major("s_scaled", s_scaled), _ptr(Vr),
        _row_major("Vr", Vr), _ptr(_f32_vec("prior", prior, dev)), _ptr(_f32_vec("beta", beta, dev)),
        _positions(None, None, beta), rows, r, V, _lib.DELS_FLAG_KEYS_READY if keys_ready else 0, _ptr(out.keys),
        _ptr(out.tokens), ws.ptr, ws.nbytes, _ptr(w_hh), _ptr(b_hh), _ptr(h), G, _ptr(gh_out), _stream(dev),
    )
    return out


def draft_score_f32(
    h: torch.Tensor,
    W: torch.Tensor,
    w_rank: torch.Tensor,
    Vr: torch.Tensor,
    prior: torch.Tensor | None,
    alpha: torch.Tensor,
    beta: torch.Tensor,
    *,
    n_pos: int | None = None,
    row_pos: torch.Tensor | None = None,
    v_begin: int = 0,
    keys_only: bool = False,
    with_scores: bool = False,
    out: ScoreOut | None = None,
    ws: Workspace | None = None,
) -> ScoreOut:
    """fp32 scorer (CUDA cores): argmax_v(h.W[v] + (alpha_p h.w_rank^T).Vr[v] - beta_p prior[v])."""
    dev = h.device
    for name, t in (("h", h), ("W", W), ("w_rank", w_rank), ("Vr", Vr)):
        _require_cuda(name, t, torch.float32, 2)
    rows, H = h.shape
    V = W.shape[0]
    r = w_rank.shape[0]
    if W.shape[1] != H or w_rank.shape[1] != H or Vr.shape != (V, r):
        raise ValueError("shape mismatch between h, W, w_rank and Vr")
    prior = _f32_vec("prior", prior, dev)
    alpha = _f32_vec("alpha", alpha, dev)
    beta = _f32_vec("beta", beta, dev)
    if out is None:
        out = ScoreOut(
            tokens=torch.empty(rows, dtype=torch.int64, device=dev),
            scores=torch.empty(rows, dtype=torch.float32, device=dev) if with_scores else None,
            keys=torch.empty(rows, dtype=torch.int64, device=dev),
        )
    need = _lib.query("dels_score_f32_workspace_bytes", rows, H, r)
    ws = workspace(need, dev) if ws is None else ws.ensure(need)
    _lib.call(
        "dels_draft_score_f32",
        _ptr(h), _row_major("h", h), _ptr(W), _row_major("W", W), _ptr(w_rank), _row_major("w_rank", w_rank),
        _ptr(Vr), _row_major("Vr", Vr), _ptr(prior), _ptr(alpha), _ptr(beta), _positions(n_pos, alpha, beta),
        _ptr(_i32_vec("row_pos", row_pos)), rows, H, r, V, int(v_begin), _ptr(out.keys),
        None if keys_only else _ptr(out.tokens), None if (keys_only or out.scores is None) else _ptr(out.scores),
        ws.ptr, ws.nbytes, _stream(dev),
    )
    return out


def keys_init(keys: torch.Tensor, ws: Workspace | None = None) -> None:
    _require_cuda("keys", keys, torch.int64, 1)
    _lib.call("dels_keys_init", _ptr(keys), keys.numel(), None if ws is None else ws.ptr, _stream(keys.device))


def keys_decode(
    keys: torch.Tensor,
    *,
    rows_dev: torch.Tensor | None = None,
    tokens: torch.Tensor | None = None,
    scores: torch.Tensor | None = None,
    with_scores: bool = True,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Token ids (int64) and scores (fp32) from packed keys."""
    _require_cuda("keys", keys, torch.int64, 1)
    n = keys.numel()
    if tokens is None:
        tokens = torch.empty(n, dtype=torch.int64, device=keys.device)
    if with_scores and scores is None:
        scores = torch.empty(n, dtype=torch.float32, device=keys.device)
    _lib.call("dels_keys_decode", _ptr(keys), n, _ptr(_i32_vec("rows_dev", rows_dev)), _ptr(tokens), _ptr(scores),
              _stream(keys.device))
    return tokens, scores


# --------------------------------------------------------------------------- acceptance
def accept_offsets(
    draft: torch.Tensor,
    target: torch.Tensor,
    *,
    commit_extra: int = 0,
    accept: torch.Tensor | None = None,
    offsets: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-sequence accepted prefix lengths (int32) and packed row offsets (int32, n+1)."""
    _require_cuda("draft", draft, torch.int64, 2)
    _require_cuda("target", target, torch.int64, 2)
    n_seq, n_draft = draft.shape
    if target.shape[0] != n_seq or target.shape[1] < n_draft:
        raise ValueError(f"target {tuple(target.shape)} must be [n_seq, >= {n_draft}]")
    dev = draft.device
    if accept is None:
        accept = torch.empty(n_seq, dtype=torch.int32, device=dev)
    if offsets is None:
        offsets = torch.empty(n_seq + 1, dtype=torch.int32, device=dev)
    _lib.call("dels_accept_offsets", _ptr(draft), _row_major("draft", draft), _ptr(target),
              _row_major("target", target), n_seq, n_draft, int(commit_extra), _ptr(accept), _ptr(offsets),
              _stream(dev))
    return accept, offsets


def pack_rows(
    hidden: torch.Tensor,
    accept: torch.Tensor,
    offsets: torch.Tensor,
    *,
    packed: torch.Tensor | None = None,
    row_pos: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Gather hidden[b, j] for j < accept[b] into rows offsets[b] + j (capacity n_seq*P)."""
    _require_cuda("hidden", hidden, torch.bfloat16, 3)
    n_seq, P, H = hidden.shape
    if hidden.stride(2) != 1:
        raise ValueError("hidden must have contiguous rows")
    dev = hidden.device
    if packed is None:
        packed = torch.empty(n_seq * P, H, dtype=torch.bfloat16, device=dev)
    if row_pos is None:
        row_pos = torch.zeros(n_seq * P, dtype=torch.int32, device=dev)
    _lib.call("dels_pack_rows_bf16", _ptr(hidden), hidden.stride(0), hidden.stride(1), n_seq, P, H,
              _ptr(_i32_vec("accept", accept)), _ptr(_i32_vec("offsets", offsets)), _ptr(packed),
              _row_major("packed", packed), _ptr(row_pos), _stream(dev))
    return packed, row_pos


# --------------------------------------------------------------------------- RNN head
def rnn_rank_states(
    x: torch.Tensor,
    w_in: torch.Tensor,
    w_s: torch.Tensor,
    bias: torch.Tensor | None,
    alpha: torch.Tensor,
    *,
    n_seq: int,
    T: int,
    s_scaled: torch.Tensor | None = None,
    s_out: torch.Tensor | None = None,
    want_state: bool = False,
    keys: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """alpha_t * s_t (bf16) for s_t = tanh(W_in x_t + W_s s_{t-1} + b), s_0 = 0."""
    dev = x.device
    _require_cuda("x", x, torch.bfloat16, 2)
    _require_cuda("w_in", w_in, torch.bfloat16, 2)
    _require_cuda("w_s", w_s, torch.bfloat16, 2)
    rows, H = x.shape
    r = w_in.shape[0]
    if rows != n_seq * T or w_in.shape[1] != H or w_s.shape != (r, r) or not w_s.is_contiguous():
        raise ValueError("shape mismatch between x, w_in and w_s")
    bias = _f32_vec("bias", bias, dev)
    alpha = _f32_vec("alpha", alpha, dev)
    if s_scaled is None:
        s_scaled = torch.empty(rows, r, dtype=torch.bfloat16, device=dev)
    if want_state and s_out is None:
        s_out = torch.empty(rows, r, dtype=torch.bfloat16, device=dev)
    need = _lib.query("dels_rnn_workspace_bytes", n_seq, T, H, r)
    ws = workspace(need, dev) if ws is None else ws.ensure(need)
    _lib.call("dels_rnn_rank_states_bf16", _ptr(x), _row_major("x", x), _ptr(w_in), _row_major("w_in", w_in),
              _ptr(w_s), _ptr(bias), _ptr(alpha), n_seq, T, H, r, _ptr(s_scaled), _ptr(s_out), _ptr(keys), ws.ptr,
              ws.nbytes, _stream(dev))
    return s_scaled, s_out


# --------------------------------------------------------------------------- rollout kernels
def gru_step(
    tokens: torch.Tensor,
    gi_table: torch.Tensor,
    w_hh: torch.Tensor,
    h_in: torch.Tensor | None,
    h_out: torch.Tensor,
    *,
    b_hh: torch.Tensor | None = None,
    ws: Workspace | None = None,
    tokens_are_keys: bool = False,
) -> torch.Tensor:
    """h_out = GRU(gi_table[tokens], h_in) with gh = W_hh h_in (+ b_hh); h_in None = zeros.
    With ``tokens_are_keys`` the tokens are the previous step's packed (score, index) keys."""
    _require_cuda("tokens", tokens, torch.int64)
    _require_cuda("gi_table", gi_table, torch.bfloat16, 2)
    _require_cuda("w_hh", w_hh, torch.bfloat16, 2)
    _require_cuda("h_out", h_out, torch.bfloat16, 2)
    B, G = h_out.shape
    V = gi_table.shape[0]
    if w_hh.shape != (3 * G, G) or not w_hh.is_contiguous() or gi_table.shape[1] != 3 * G:
        raise ValueError("GRU weights do not match the hidden size")
    if h_in is not None and (h_in.shape != (B, G) or not h_in.is_contiguous()):
        raise ValueError("h_in must be a contiguous [B, G] tensor")
    if not h_out.is_contiguous():
        raise ValueError("h_out must be contiguous")
    tok_stride = tokens.stride(0) if tokens.dim() >= 1 and tokens.numel() > 1 else 1
    _lib.call("dels_gru_step_bf16", _ptr(tokens), tok_stride, int(bool(tokens_are_keys)), _ptr(gi_table),
              _row_major("gi_table", gi_table),
              _ptr(w_hh), _ptr(b_hh), _ptr(h_in), _ptr(h_out), B, G, V, None if ws is None else ws.ptr,
              _stream(h_out.device))
    return h_out


def gru_gates(
    tokens: torch.Tensor,
    gi_table: torch.Tensor,
    gh: torch.Tensor,
    h_in: torch.Tensor | None,
    h_out: torch.Tensor,
    *,
    ws: Workspace | None = None,
    tokens_are_keys: bool = False,
) -> torch.Tensor:
    """h_out = GRU gates(gi_table[tokens], gh, h_in) for a precomputed gh = bf16(W_hh h + b_hh).
    With ``tokens_are_keys`` the tokens are the previous step's packed (score, index) keys."""
    _require_cuda("tokens", tokens, torch.int64)
    _require_cuda("gi_table", gi_table, torch.bfloat16, 2)
    _require_cuda("gh", gh, torch.bfloat16, 2)
    _require_cuda("h_out", h_out, torch.bfloat16, 2)
    B, G = h_out.shape
    V = gi_table.shape[0]
    if gh.shape != (B, 3 * G) or gh.stride(1) != 1 or gi_table.shape[1] != 3 * G or not h_out.is_contiguous():
        raise ValueError("GRU gate operands do not match the hidden size")
    if h_in is not None and (h_in.shape != (B, G) or not h_in.is_contiguous()):
        raise ValueError("h_in must be a contiguous [B, G] tensor")
    tok_stride = tokens.stride(0) if tokens.dim() >= 1 and tokens.numel() > 1 else 1
    _lib.call("dels_gru_gates_bf16", _ptr(tokens), tok_stride, int(bool(tokens_are_keys)), _ptr(gi_table),
              _row_major("gi_table", gi_table),
              _ptr(gh), gh.stride(0), _ptr(h_in), _ptr(h_out), B, G, V, None if ws is None else ws.ptr,
              _stream(h_out.device))
    return h_out


def gru_step_tc(
    tokens: torch.Tensor,
    gi_table: torch.Tensor,
    w_hh: torch.Tensor,
    h_in: torch.Tensor,
    h_out: torch.Tensor,
    *,
    b_hh: torch.Tensor | None = None,
    ws: Workspace | None = None,
    tokens_are_keys: bool = False,
) -> torch.Tensor:
    """h_out = GRU(gi_table[tokens], h_in) with gh = bf16(W_hh h_in + b_hh) from a tensor-core
    split-K GEMM whose finalisation evaluates the gates (bit-identical to linear_bf16 followed
    by gru_gates).  With ``tokens_are_keys`` the tokens are packed (score, index) keys."""
    _require_cuda("tokens", tokens, torch.int64)
    _require_cuda("gi_table", gi_table, torch.bfloat16, 2)
    _require_cuda("w_hh", w_hh, torch.bfloat16, 2)
    _require_cuda("h_in", h_in, torch.bfloat16, 2)
    _require_cuda("h_out", h_out, torch.bfloat16, 2)
    B, G = h_out.shape
    V = gi_table.shape[0]
    if w_hh.shape != (3 * G, G) or not w_hh.is_contiguous() or gi_table.shape[1] != 3 * G:
        raise ValueError("GRU weights do not match the hidden size")
    if h_in.shape != (B, G) or not h_in.is_contiguous() or not h_out.is_contiguous():
        raise ValueError("h_in / h_out must be contiguous [B, G] tensors")
    need = _lib.query("dels_gru_step_tc_workspace_bytes", B, G)
    ws = workspace(need, h_out.device) if ws is None else ws.ensure(need)
    tok_stride = tokens.stride(0) if tokens.dim() >= 1 and tokens.numel() > 1 else 1
    _lib.call("dels_gru_step_tc_bf16", _ptr(tokens), tok_stride, int(bool(tokens_are_keys)), _ptr(gi_table),
              _row_major("gi_table", gi_table),
              _ptr(w_hh), _ptr(b_hh), _ptr(h_in), _ptr(h_out), B, G, V, ws.ptr, ws.nbytes, _stream(h_out.device))
    return h_out


def gru_rank_gemv(
    tokens: torch.Tensor,
    gi_table: torch.Tensor,
    gh: torch.Tensor,
    h_in: torch.Tensor | None,
    h_out: torch.Tensor,
    w_rank: torch.Tensor,
    alpha: torch.Tensor | None,
    s_scaled: torch.Tensor,
    *,
    bias: torch.Tensor | None = None,
    activation: str = "identity",
    keys: torch.Tensor | None = None,
    ws: Workspace | None = None,
    tokens_are_keys: bool = False,
) -> torch.Tensor:
    """One small-batch rollout step: h_out = GRU gates(gi_table[tokens], gh, h_in) (gh =
    bf16(W_hh h_in + b_hh) from an earlier rank_gemv), then s_scaled = bf16(alpha[0] *
    act(w_rank . h_out + bias)) in the same launch.  ``tokens_are_keys``: ``tokens`` holds
    the previous step's packed argmax keys (a keys-only scorer call), decoded here."""
    _require_cuda("tokens", tokens, torch.int64)
    _require_cuda("gi_table", gi_table, torch.bfloat16, 2)
    _require_cuda("gh", gh, torch.bfloat16, 2)
    _require_cuda("h_out", h_out, torch.bfloat16, 2)
    _require_cuda("w_rank", w_rank, torch.bfloat16, 2)
    B, G = h_out.shape
    V = gi_table.shape[0]
    r = w_rank.shape[0]
    if gh.shape != (B, 3 * G) or gh.stride(1) != 1 or gi_table.shape[1] != 3 * G or not h_out.is_contiguous():
        raise ValueError("GRU gate operands do not match the hidden size")
    if h_in is not None and (h_in.shape != (B, G) or not h_in.is_contiguous()):
        raise ValueError("h_in must be a contiguous [B, G] tensor")
    if w_rank.shape[1] != G or s_scaled.shape != (B, r) or not s_scaled.is_contiguous():
        raise ValueError("rank projection shapes do not match")
    tok_stride = tokens.stride(0) if tokens.dim() >= 1 and tokens.numel() > 1 else 1
    _lib.call("dels_gru_rank_gemv_bf16", _ptr(tokens), tok_stride, int(tokens_are_keys), _ptr(gi_table),
              _row_major("gi_table", gi_table),
              _ptr(gh), gh.stride(0), _ptr(h_in), _ptr(h_out), B, G, V, _ptr(w_rank), _row_major("w_rank", w_rank),
              _ptr(bias), r, ACTIVATIONS[activation], _ptr(alpha), _ptr(s_scaled), _ptr(keys),
              None if ws is None else ws.ptr, _stream(h_out.device))
    return s_scaled


def gru_correction_mid(
    tokens: torch.Tensor,
    gi_table: torch.Tensor,
    gh: torch.Tensor,
    h_in: torch.Tensor | None,
    h_out: torch.Tensor,
    w_s: torch.Tensor,
    z: torch.Tensor,
    alpha: torch.Tensor,
    s_scaled: torch.Tensor,
    *,
    keys: torch.Tensor | None = None,
    ws: Workspace | None = None,
    tokens_are_keys: bool = False,
) -> torch.Tensor:
    """One small-batch Domino step: h_out = GRU gates(gi_table[tokens], gh, h_in), then
    s_scaled = bf16(alpha[0] * SiLU(z + bf16(w_s . h_out))) in the same launch
    (``tokens_are_keys`` as in :func:`gru_rank_gemv`)."""
    _require_cuda("tokens", tokens, torch.int64)
    for name, t in (("gi_table", gi_table), ("gh", gh), ("h_out", h_out), ("w_s", w_s), ("z", z)):
        _require_cuda(name, t, torch.bfloat16, 2)
    B, G = h_out.shape
    V = gi_table.shape[0]
    M = w_s.shape[0]
    if gh.shape != (B, 3 * G) or gh.stride(1) != 1 or gi_table.shape[1] != 3 * G or not h_out.is_contiguous():
        raise ValueError("GRU gate operands do not match the hidden size")
    if h_in is not None and (h_in.shape != (B, G) or not h_in.is_contiguous()):
        raise ValueError("h_in must be a contiguous [B, G] tensor")
    if w_s.shape[1] != G or z.shape != (B, M) or z.stride(1) != 1 or s_scaled.shape != (B, M) \
            or not s_scaled.is_contiguous():
        raise ValueError("correction MLP shapes do not match")
    tok_stride = tokens.stride(0) if tokens.dim() >= 1 and tokens.numel() > 1 else 1
    _lib.call("dels_gru_correction_mid_bf16", _ptr(tokens), tok_stride, int(tokens_are_keys), _ptr(gi_table),
              _row_major("gi_table", gi_table), _ptr(gh), gh.stride(0), _ptr(h_in), _ptr(h_out), B, G, V, _ptr(w_s),
              _row_major("w_s", w_s), _ptr(z), _row_major("z", z), M, _ptr(_f32_vec("alpha", alpha, h_out.device)),
              _ptr(s_scaled), _ptr(keys), None if ws is None else ws.ptr, _stream(h_out.device))
    return s_scaled


def rank_gemv(
    x: torch.Tensor,
    w: torch.Tensor,
    alpha: torch.Tensor | None,
    s_scaled: torch.Tensor,
    *,
    bias: torch.Tensor | None = None,
    n_pos: int = 1,
    row_pos: torch.Tensor | None = None,
    activation: str = "identity",
    s_out: torch.Tensor | None = None,
    keys: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> torch.Tensor:
    """Small-batch rank projection: s_scaled = bf16(alpha * act(x . w^T + bias))."""
    _require_cuda("x", x, torch.bfloat16, 2)
    _require_cuda("w", w, torch.bfloat16, 2)
    B, K = x.shape
    r = w.shape[0]
    if w.shape[1] != K or s_scaled.shape != (B, r) or not s_scaled.is_contiguous():
        raise ValueError("rank projection shapes do not match")
    _lib.call("dels_rank_gemv_bf16", _ptr(x), _row_major("x", x), _ptr(w), _row_major("w", w), _ptr(bias), B, K, r,
              ACTIVATIONS[activation], _ptr(alpha), int(n_pos), _ptr(_i32_vec("row_pos", row_pos)), _ptr(s_out),
              _ptr(s_scaled), _ptr(keys), None if ws is None else ws.ptr, _stream(x.device))
    return s_scaled


def gather_scaled_rows(
    tokens: torch.Tensor,
    emb: torch.Tensor,
    alpha: torch.Tensor | None,
    s_scaled: torch.Tensor,
    *,
    n_pos: int = 1,
    keys: torch.Tensor | None = None,
    ws: Workspace | None = None,
    tokens_are_keys: bool = False,
) -> torch.Tensor:
    """s_scaled[b] = bf16(alpha * emb[tokens[b]]) (Markov rank state).  With
    ``tokens_are_keys`` the tokens are the previous step's packed (score, index) keys."""
    _require_cuda("tokens", tokens, torch.int64)
    _require_cuda("emb", emb, torch.bfloat16, 2)
    B, r = s_scaled.shape
    if emb.shape[1] != r or not s_scaled.is_contiguous():
        raise ValueError("embedding / output shapes do not match")
    tok_stride = tokens.stride(0) if tokens.numel() > 1 else 1
    _lib.call("dels_gather_scaled_rows_bf16", _ptr(tokens), tok_stride, int(bool(tokens_are_keys)), _ptr(emb),
              _row_major("emb", emb),
              _ptr(alpha), int(n_pos), B, r, emb.shape[0], _ptr(s_scaled), _ptr(keys),
              None if ws is None else ws.ptr, _stream(s_scaled.device))
    return s_scaled


def linear_workspace_bytes(rows: int, K: int, N: int) -> int:
    return int(_lib.query("dels_linear_workspace_bytes", rows, K, N))


def correction_mid_tc_workspace_bytes(B: int, G: int, M: int) -> int:
    return int(_lib.query("dels_correction_mid_tc_workspace_bytes", B, G, M))


def rank_workspace_bytes(rows: int, K: int, r: int) -> int:
    return int(_lib.query("dels_rank_workspace_bytes", rows, K, r))


def linear_bf16(
    x: torch.Tensor,
    w: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    out: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> torch.Tensor:
    """F.linear(x, w, bias) for bf16 operands: out = bf16(x . w^T + bias), one rounding."""
    _require_cuda("x", x, torch.bfloat16, 2)
    _require_cuda("w", w, torch.bfloat16, 2)
    rows, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"w {tuple(w.shape)} does not match x {tuple(x.shape)}")
    if bias is not None:
        _require_cuda("bias", bias, torch.bfloat16, 1)
        if bias.shape[0] != N or not bias.is_contiguous():
            raise ValueError("bias must be a contiguous [N] tensor")
    if out is None:
        out = torch.empty(rows, N, dtype=torch.bfloat16, device=x.device)
    elif out.shape != (rows, N) or out.dtype != torch.bfloat16 or out.stride(1) != 1:
        raise ValueError("out must be a row-major bf16 [rows, N] tensor")
    need = _lib.query("dels_linear_workspace_bytes", rows, K, N)
    ws = workspace(need, x.device) if ws is None else ws.ensure(need)
    _lib.call("dels_linear_bf16", _ptr(x), _row_major("x", x), _ptr(w), _row_major("w", w), _ptr(bias), rows, K, N,
              _ptr(out), _row_major("out", out), ws.ptr, ws.nbytes, _stream(x.device))
    return out


def correction_mid(
    h: torch.Tensor,
    w_s: torch.Tensor,
    z: torch.Tensor,
    alpha: torch.Tensor,
    s_scaled: torch.Tensor,
    *,
    keys: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> torch.Tensor:
    """Domino correction MLP hidden layer: s_scaled = bf16(alpha * SiLU(z + bf16(W_s h))), SiLU in fp32."""
    _require_cuda("h", h, torch.bfloat16, 2)
    _require_cuda("w_s", w_s, torch.bfloat16, 2)
    _require_cuda("z", z, torch.bfloat16, 2)
    B, G = h.shape
    M = w_s.shape[0]
    if w_s.shape[1] != G or z.shape != (B, M) or z.stride(1) != 1 or s_scaled.shape != (B, M) \
            or not s_scaled.is_contiguous():
        raise ValueError("correction MLP shapes do not match")
    _lib.call("dels_correction_mid_bf16", _ptr(h), _row_major("h", h), _ptr(w_s), _row_major("w_s", w_s), _ptr(z),
              _row_major("z", z), B, G, M, _ptr(alpha), _ptr(s_scaled), _ptr(keys),
              None if ws is None else ws.ptr, _stream(h.device))
    return s_scaled


def correction_mid_tc(
    h: torch.Tensor,
    w_s: torch.Tensor,
    z: torch.Tensor,
    alpha: torch.Tensor,
    s_scaled: torch.Tensor,
    *,
    keys: torch.Tensor | None = None,
    ws: Workspace,
) -> torch.Tensor:
    """correction_mid with W_s h on the tensor-core split-K GEMM (larger batches);
    ``ws`` needs correction_mid_tc_workspace_bytes(B, G, M)."""
    _require_cuda("h", h, torch.bfloat16, 2)
    _require_cuda("w_s", w_s, torch.bfloat16, 2)
    _require_cuda("z", z, torch.bfloat16, 2)
    B, G = h.shape
    M = w_s.shape[0]
    if w_s.shape[1] != G or z.shape != (B, M) or z.stride(1) != 1 or s_scaled.shape != (B, M) \
            or not s_scaled.is_contiguous():
        raise ValueError("correction MLP shapes do not match")
    _lib.call("dels_correction_mid_tc_bf16", _ptr(h), _row_major("h", h), _ptr(w_s), _row_major("w_s", w_s),
              _ptr(z), _row_major("z", z), B, G, M, _ptr(_f32_vec("alpha", alpha, h.device)), _ptr(s_scaled),
              _ptr(keys), ws.ptr, ws.nbytes, _stream(h.device))
    return s_scaled


# --------------------------------------------------------------------------- 8-bit product
_FLOATS = {torch.bfloat16: _lib.DELS_DTYPE_BF16, torch.float32: _lib.DELS_DTYPE_F32}


def _require_float(name: str, t: torch.Tensor, ndim: int) -> int:
    """The DELS_DTYPE_* code of a bf16 or fp32 CUDA tensor."""
    code = _FLOATS.get(t.dtype) if isinstance(t, torch.Tensor) and t.is_cuda else None
    if code is None or t.dim() != ndim:
        raise ValueError(f"{name} must be a {ndim}-D bf16 or fp32 CUDA tensor; there is no CPU path")
    return code


def _require_dense(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {device} "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device}, stride {t.stride()})")


def _leading(name: str, t: torch.Tensor) -> int:
    """_row_major() of a tensor that is known to have two dimensions."""
    (rows, cols), (ld, step) = t.shape, t.stride()
    if step != 1 and cols > 1 and rows > 0:
        raise ValueError(f"{name} must have contiguous rows (stride {(ld, step)})")
    return ld if rows > 1 and cols > 0 else max(ld, cols, 1)


# A draft step calls these operators on small tensors, where the host's part of a call is what
# counts: addresses go to ctypes as plain integers, sizes of workspaces are asked for once.
def _addr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _raw_stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


@functools.lru_cache(maxsize=4096)
def _bytes(query: str, *args: int) -> int:
    return int(_lib.query(query, *args))


def quantize_rows_i8(
    x: torch.Tensor,
    *,
    q: torch.Tensor | None = None,
    scale: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of ``x`` [rows, K] (bf16 or fp32): int8 values and fp32 [rows] scales with
    x ~ q * scale, scale = max|row| / 127.  The rows of a ``q`` made here start on 16-byte
    boundaries (its row stride is K rounded up to 16), as the product needs them."""
    code = _require_float("x", x, 2)
    dev = x.device
    rows, K = x.shape
    if q is None:
        q = torch.empty(rows, -(-K // 16) * 16, dtype=torch.int8, device=dev)[:, :K]
    elif q.dtype != torch.int8 or q.shape != (rows, K) or q.device != dev:
        raise ValueError(f"q must be int8 {(rows, K)} on {dev} (got {q.dtype} {tuple(q.shape)} on {q.device})")
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=dev)
    else:
        _require_dense("scale", scale, torch.float32, (rows,), dev)
    _lib.call("dels_quantize_rows_i8", _addr(x), code, _leading("x", x), rows, K, _addr(q), _leading("q", q),
              _addr(scale), _raw_stream(dev))
    return q, scale


def _i8_operands(rows: int, K: int, dev: torch.device, wq, w_scale, bias, out, out_dtype):
    _require_cuda("wq", wq, torch.int8, 2)
    N = wq.shape[0]
    if wq.shape[1] != K or wq.device != dev:
        raise ValueError(f"wq {tuple(wq.shape)} on {wq.device} does not match inputs of width {K} on {dev}")
    _require_dense("w_scale", w_scale, torch.float32, (N,), dev)
    if out is None:
        if out_dtype not in _FLOATS:
            raise ValueError(f"out_dtype must be bf16 or fp32 (got {out_dtype})")
        out = torch.empty(rows, N, dtype=out_dtype, device=dev)
    else:
        _require_float("out", out, 2)
        if out.shape != (rows, N) or out.device != dev:
            raise ValueError(f"out must be {(rows, N)} on {dev} (got {tuple(out.shape)} on {out.device})")
    if bias is not None:
        _require_dense("bias", bias, out.dtype, (N,), dev)
    return N, out


def linear_i8(
    xq: torch.Tensor,
    x_scale: torch.Tensor,
    wq: torch.Tensor,
    w_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    ws: Workspace | None = None,
) -> torch.Tensor:
    """(xq . wq^T) * x_scale[row] * w_scale[channel] (+ bias): int8 operands [rows, K] and
    [N, K] with 16-byte aligned rows, an exact integer sum, a bf16 or fp32 result (``bias``
    has its type)."""
    _require_cuda("xq", xq, torch.int8, 2)
    dev = xq.device
    rows, K = xq.shape
    _require_dense("x_scale", x_scale, torch.float32, (rows,), dev)
    N, out = _i8_operands(rows, K, dev, wq, w_scale, bias, out, out_dtype)
    stream = _raw_stream(dev)
    ws = _stream_workspace(_lib.DELS_WS_HEADER_BYTES, dev, stream) if ws is None else ws
    _lib.call("dels_linear_i8", _addr(xq), _leading("xq", xq), _addr(x_scale), _addr(wq), _leading("wq", wq),
              _addr(w_scale), _addr(bias), rows, K, N, _addr(out), _FLOATS[out.dtype], _leading("out", out), ws.ptr,
              ws.nbytes, stream)
    return out


def linear_w8a8_workspace_bytes(rows: int, K: int) -> int:
    return _bytes("dels_linear_w8a8_workspace_bytes", rows, K)


def linear_w8a8(
    x: torch.Tensor,
    wq: torch.Tensor,
    w_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    ws: Workspace | None = None,
) -> torch.Tensor:
    """F.linear(x, W, bias) with W = wq * w_scale[:, None] and every row of ``x`` (bf16 or
    fp32) quantised on the way: quantize_rows_i8 and linear_i8 in one call, the weights
    loading while the rows are quantised.  The result has x's type unless ``out`` or
    ``out_dtype`` says otherwise.  ``x`` [..., K] gives [..., N]; rows that are not evenly
    spaced (a slice of [B, S, K] along S) are copied first."""
    if isinstance(x, torch.Tensor) and x.dim() != 2 and x.dim() > 0:
        *lead, K = x.shape
        rows, flat = math.prod(lead), None
        if out is not None:
            _require_float("out", out, x.dim())
            if list(out.shape[:-1]) != lead:
                raise ValueError(f"out {tuple(out.shape)} does not match x {tuple(x.shape)}")
            try:
                flat = out.view(rows, out.shape[-1])
            except RuntimeError:
                raise ValueError(f"out's rows must be evenly spaced (stride {out.stride()})") from None
        y = linear_w8a8(x.reshape(rows, K), wq, w_scale, bias, out=flat, out_dtype=out_dtype, ws=ws)
        return y.view(*lead, y.shape[1]) if out is None else out
    code = _require_float("x", x, 2)
    dev = x.device
    rows, K = x.shape
    N, out = _i8_operands(rows, K, dev, wq, w_scale, bias, out, x.dtype if out_dtype is None else out_dtype)
    need = linear_w8a8_workspace_bytes(rows, K)
    stream = _raw_stream(dev)
    ws = _stream_workspace(need, dev, stream) if ws is None else ws.ensure(need)
    _lib.call("dels_linear_w8a8", _addr(x), code, _leading("x", x), _addr(wq), _leading("wq", wq), _addr(w_scale),
              _addr(bias), rows, K, N, _addr(out), _FLOATS[out.dtype], _leading("out", out), ws.ptr, ws.nbytes,
              stream)
    return out


# --------------------------------------------------------------------------- beam drafting
@dataclass
class BeamOut:
    parents: torch.Tensor  # int32 [n_seq, select], the beam (0..beams-1) each child extends
    tokens: torch.Tensor  # int64 [n_seq, select]
    scores: torch.Tensor  # fp32 [n_seq, select], best first


def beam_select(
    logits: torch.Tensor,
    scores: torch.Tensor,
    *,
    select: int | None = None,
    base: torch.Tensor | None = None,
    prior: torch.Tensor | None = None,
    beta: torch.Tensor | None = None,
    finished: torch.Tensor | None = None,
    pad_token: int = 0,
    out: BeamOut | None = None,
    ws: Workspace | None = None,
) -> BeamOut:
    """The ``select`` best extensions (default: as many as there are beams) of every
    sequence's beams by one token, best first.

    ``logits`` [n_seq * beams, V] (bf16 or fp32) and ``scores`` [n_seq, beams] (fp32, the
    beams' accumulated log-probabilities); a candidate scores its beam's score plus
    log_softmax(x)[token] of x = logits, or, with ``base`` [n_seq, V] (draft logits the
    beams of a sequence share) and ``prior`` [V] with ``beta`` [1],
    x = (base + logits) - beta * prior.  Equal scores: the lower beam, then the larger x,
    then the lower token.  A beam whose ``finished`` [n_seq, beams] (bool) is set goes on
    only with ``pad_token`` at its score, and its logits are not read.  Masked tokens hold
    -inf or the type's lowest value; a row may be masked whole.  ``out.scores`` may be
    ``scores`` itself when ``select`` equals the beams."""
    code = _require_float("logits", logits, 2)
    dev, dtype = logits.device, logits.dtype
    rows, V = logits.shape
    if scores.dim() != 2:
        raise ValueError(f"scores must be [n_seq, beams] (got {tuple(scores.shape)})")
    n_seq, beams = scores.shape
    n = beams if select is None else int(select)
    if rows != n_seq * beams:
        raise ValueError(f"logits {tuple(logits.shape)} do not match scores {tuple(scores.shape)}")
    _require_dense("scores", scores, torch.float32, (n_seq, beams), dev)
    if base is not None and (base.dtype != dtype or base.shape != (n_seq, V) or base.device != dev):
        raise ValueError(f"base must be {dtype} {(n_seq, V)} on {dev} (got {base.dtype} {tuple(base.shape)})")
    if prior is not None:
        _require_dense("prior", prior, torch.float32, (V,), dev)
        if beta is None:
            raise ValueError("prior needs beta")
        _require_dense("beta", beta, torch.float32, (1,), dev)
    if finished is not None:
        if finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"finished must be bool or uint8 (got {finished.dtype})")
        _require_dense("finished", finished, finished.dtype, (n_seq, beams), dev)
    if out is None:
        out = BeamOut(torch.empty(n_seq, n, dtype=torch.int32, device=dev),
                      torch.empty(n_seq, n, dtype=torch.int64, device=dev),
                      torch.empty(n_seq, n, dtype=torch.float32, device=dev))
    else:
        _require_dense("out.parents", out.parents, torch.int32, (n_seq, n), dev)
        _require_dense("out.tokens", out.tokens, torch.int64, (n_seq, n), dev)
        _require_dense("out.scores", out.scores, torch.float32, (n_seq, n), dev)
    need = beam_select_workspace_bytes(n_seq, beams, n, V)
    stream = _raw_stream(dev)
    ws = _stream_workspace(need, dev, stream) if ws is None else ws.ensure(need)
    _lib.call(
        "dels_beam_select", _addr(logits), code, _leading("logits", logits), _addr(base),
        0 if base is None else _leading("base", base), _addr(prior), _addr(beta), _addr(scores), _addr(finished),
        int(pad_token), n_seq, beams, n, V, _addr(out.parents), _addr(out.tokens), _addr(out.scores), ws.ptr,
        ws.nbytes, stream,
    )
    return out


def beam_select_workspace_bytes(n_seq: int, beams: int, select: int, V: int) -> int:
    return _bytes("dels_beam_select_workspace_bytes", n_seq, beams, select, V)


@functools.lru_cache(maxsize=None)
def _int64_array(n: int):
    return ctypes.c_int64 * n


def _beam_state(i: int, src: torch.Tensor, dst: torch.Tensor) -> tuple:
    """The dels_beam_state of one (src, dst) pair: rows of ``outer`` runs of contiguous bytes."""
    shape = src.shape
    if src.is_contiguous() and dst.is_contiguous():
        # (by its size: the stride of a dimension of one row may be anything)
        row = src.nbytes // shape[0] if shape[0] else 0
        return src.data_ptr(), dst.data_ptr(), row, row, 0, 0, 1, row
    item, ss, ds = src.element_size(), src.stride(), dst.stride()
    inner, k = 1, src.dim() - 1
    while k >= 1 and (shape[k] == 1 or (ss[k] == inner and ds[k] == inner)):
        inner *= shape[k]
        k -= 1
    outer, so, do = 1, 0, 0
    for j in range(k, 0, -1):
        if shape[j] == 1:
            continue
        if outer == 1:
            so, do = ss[j], ds[j]
        elif ss[j] != so * outer or ds[j] != do * outer:
            raise ValueError(f"state {i}: rows of shape {tuple(shape[1:])} must be evenly spaced runs of contiguous "
                             f"elements (strides {ss}, {ds})")
        outer *= shape[j]
    return (src.data_ptr(), dst.data_ptr(), ss[0] * item, ds[0] * item, so * item, do * item, outer, inner * item)


def beam_reorder(
    states: list[torch.Tensor],
    parents: torch.Tensor,
    *,
    beams: int,
    out: list[torch.Tensor] | None = None,
    status: torch.Tensor | None = None,
) -> list[torch.Tensor]:
    """Move every state's rows after a selection: out[b * select + j] =
    state[b * beams + parents[b, j]].

    ``states`` are CUDA tensors of any type whose first dimension is n_seq * beams (GRU
    states, token histories, caches cut to their used length); ``parents`` is
    ``beam_select``'s int32 [n_seq, select].  ``out`` gives the destinations ([n_seq *
    select, ...]); ``out=states`` reorders in place (select == beams).  The tensors must not
    overlap otherwise.  A parent outside 0..beams-1 leaves its child's row as it was and
    stores an error code in ``status`` (int32 [1], zero before)."""
    _require_cuda("parents", parents, torch.int32, 2)
    if not parents.is_contiguous():
        raise ValueError(f"parents must be contiguous (stride {parents.stride()})")
    dev, index = parents.device, parents.get_device()
    n_seq, n = parents.shape
    if status is not None:
        _require_dense("status", status, torch.int32, (1,), dev)
    rows, out_rows = n_seq * int(beams), n_seq * n
    if out is None:
        out = [torch.empty((out_rows, *t.shape[1:]), dtype=t.dtype, device=dev) for t in states]
    if len(out) != len(states):
        raise ValueError(f"{len(states)} states, but {len(out)} outputs")
    table: list[int] = []
    for i, (src, dst) in enumerate(zip(states, out)):
        have, want = src.shape, dst.shape
        if src.get_device() != index or dst.get_device() != index:
            raise ValueError(f"state {i}: {src.device} -> {dst.device}, but parents are on {dev}")
        if not have or have[0] != rows or want != (have if n == beams else (out_rows, *have[1:])) \
                or src.dtype != dst.dtype:
            raise ValueError(f"state {i}: {src.dtype} {tuple(have)} -> {dst.dtype} {tuple(want)} does not match "
                             f"{n_seq} sequences of {beams} -> {n} beams")
        table += _beam_state(i, src, dst)
    _lib.call("dels_beam_reorder", _int64_array(len(table))(*table), len(states), _addr(parents), n_seq, int(beams), n,
              _addr(status), _raw_stream(dev))
    return out


def zero_pad(t: torch.Tensor | None, rows: int | None = None, cols: int | None = None) -> torch.Tensor | None:
    """``t`` zero-padded to ``rows`` (dim 0) x ``cols`` (dim 1).  The runners carry weight
    widths as multiples of 8 because TMA tiles need 16-byte row pitches; the zero entries
    contribute nothing to any contraction."""
    if t is None:
        return None
    shape = list(t.shape)
    if rows is not None:
        shape[0] = rows
    if cols is not None:
        shape[1] = cols
    if list(t.shape) == shape:
        return t
    out = torch.zeros(shape, dtype=t.dtype, device=t.device)
    out[tuple(slice(0, n) for n in t.shape)] = t
    return out


def round8(n: int) -> int:
    return -(-int(n) // 8) * 8
