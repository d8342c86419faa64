"""CUDA-graph runner for beam drafting with the DeLS local head, on the B200 kernels.

Where ``kernel.dels`` drafts one greedy chain per sequence, ``DeLSBeamGraphRunner`` keeps the
``beams`` best chains: multi-candidate drafts for a verifier that scores several chains of a
sequence at once.  The reference has no such runner; the local head, its weights and the
schedules are those of ``DeLSGraphRunner`` (code/kernel/dels.py:214-478).

One call is one graph replay:

  1. the long logits of all B x steps hidden rows from an 8-bit LM head
     (``dels_linear_w8a8``: half the bytes of the bf16 head, quantised once at construction
     with a scale per token);
  2. per step, for all B x beams rows: the GRU update of the previous token, the rank
     projection with alpha folded in, the local logits (``dels_linear_bf16``), then the
     selection over beams and vocabulary of
         score(beam) + log_softmax(base_t + local - beta_t * prior)
     (``dels_beam_select``; the sequence's beams share base_t), and the reordering of GRU
     states and token histories after the chosen parents (``dels_beam_reorder``).

At the first step all beams of a sequence are the same, so only the first one's candidates
count.  Local logits are bf16-rounded between the two kernels.
"""

from __future__ import annotations

import torch

from dels_b200 import ops

from .dels import DeLSGraphRunner


class DeLSBeamGraphRunner(DeLSGraphRunner):
    """``__call__(prefix_ids [B, 1], parallel_hiddens [B, steps, H])`` returns
    ``(tokens [B, beams, steps], scores [B, beams])``, the best chain first; a score is the
    sum of its tokens' log-probabilities.  Keywords as ``DeLSGraphRunner``, and ``beams`` and
    the target LM head's weight [V, H]."""

    def __init__(self, *, target_lm_head_weight: torch.Tensor, beams: int, batch_size: int, **kwargs):
        w = target_lm_head_weight.detach()
        if w.dim() != 2 or int(w.shape[0]) != int(kwargs["vocab_size"]):
            raise ValueError(
                f"target LM head weight {tuple(w.shape)} does not match vocab_size={kwargs['vocab_size']}."
            )
        if not 1 <= int(beams) <= min(ops._lib.DELS_BEAM_MAX, int(kwargs["vocab_size"])):
            raise ValueError(f"DeLSBeamGraphRunner needs 1 to {ops._lib.DELS_BEAM_MAX} beams, no more than the "
                             f"vocabulary (got {beams}).")
        self.n_seq, self.beams = int(batch_size), int(beams)
        self.hidden_size = int(w.shape[1])
        self._lm_q, self._lm_scale = ops.quantize_rows_i8(
            w.to(device=kwargs["device"], dtype=torch.bfloat16).contiguous())
        super().__init__(batch_size=self.n_seq * self.beams, **kwargs)

    def _scorer_computes_next_gh(self) -> bool:
        return False  # the selection has no helper warps

    def _alloc_step_inputs(self, dtype, device):
        B, K, S, V = self.n_seq, self.beams, self.steps, self.vocab_size
        rows = B * K
        self.static_parallel_hiddens = torch.zeros(B, S, self.hidden_size, dtype=dtype, device=device)
        self.static_base_logits = torch.zeros(B, S, V, dtype=dtype, device=device)
        self.static_scores = torch.zeros(B, K, dtype=torch.float32, device=device)
        self._root_scores = torch.zeros(B, 1, dtype=torch.float32, device=device)
        self._local = torch.zeros(rows, V, dtype=dtype, device=device)
        self._history = [torch.zeros(rows, S, dtype=torch.long, device=device) for _ in range(2)]
        self._beam_out = ops.BeamOut(torch.zeros(B, K, dtype=torch.int32, device=device),
                                     torch.zeros(B, K, dtype=torch.long, device=device), self.static_scores)
        self._moved = torch.zeros(rows, self.gru_hidden_dim, dtype=dtype, device=device)
        self._beam_ws = ops.Workspace(
            max(ops.linear_w8a8_workspace_bytes(B * S, self.hidden_size), ops.linear_workspace_bytes(rows, self._r, V),
                ops.beam_select_workspace_bytes(B, K, K, V), ops.beam_select_workspace_bytes(B, 1, K, V)), device)

    def _select(self, step: int):
        first = step == 0
        # the first step's beams are alike: the first one's rows stand for their sequence
        logits = self._local[:: self.beams] if first else self._local
        return ops.beam_select(logits, self._root_scores if first else self.static_scores, select=self.beams,
                               base=self.static_base_logits[:, step], prior=self._prior_f32,
                               beta=None if self._prior_f32 is None else self._beta[step : step + 1],
                               out=self._beam_out, ws=self._beam_ws)

    def _forward_impl(self):
        B, S, V = self.n_seq, self.steps, self.vocab_size
        ops.linear_w8a8(self.static_parallel_hiddens.view(B * S, self.hidden_size), self._lm_q, self._lm_scale,
                        out=self.static_base_logits.view(B * S, V), ws=self._beam_ws)
        h = self._gru(self.static_prefix_ids[:, 0], None, self._h[0])
        for step in range(S):
            self._rank(h, step)
            ops.linear_bf16(self._s_scaled, self.lm_head_weight, out=self._local, ws=self._beam_ws)
            out = self._select(step)
            old, new = self._history[step % 2], self._history[(step + 1) % 2]
            last = step + 1 == S
            ops.beam_reorder([old] if last else [old, h], out.parents, beams=self.beams,
                             out=[new] if last else [new, self._moved])
            new[:, step].copy_(out.tokens.view(-1))
            if not last:
                h = self._gru(out.tokens.view(-1), self._moved, self._h[(step + 1) % 2])
        self.static_out.copy_(self._history[S % 2])

    @torch.inference_mode()
    def __call__(self, prefix_ids: torch.Tensor, parallel_hiddens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        self.static_prefix_ids.copy_(prefix_ids.view(self.n_seq, 1).repeat_interleave(self.beams, dim=0))
        self.static_parallel_hiddens.copy_(parallel_hiddens)
        self.graph.replay()
        return self.static_out.view(self.n_seq, self.beams, self.steps).clone(), self.static_scores.clone()
