"""Verification of drafted tokens against the target's probabilities."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ..kernels.ops import _nb, draft_call


def verify_drafts(target_probs: torch.Tensor, q_start: torch.Tensor, draft_tokens: torch.Tensor, draft_len: Optional[torch.Tensor],
                  draft_probs: Optional[torch.Tensor], accept_draws: torch.Tensor, token_draws: torch.Tensor,
                  err: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens are kept, and the token behind them, distributed as the target alone would draw them (to the resolution of the
    draws: 2^-24 where they are multiples of that, as torch.rand makes them).

    Request r drafted n = draft_len[r] of the N tokens draft_tokens[r] (None: all N; negative: the request is idle and gets
    nothing) from the distributions draft_probs[r, :n] (None: drafts without probabilities, each taken as certain).  Rows
    q_start[r] .. q_start[r] + n of target_probs [T, V] are the target's distributions at the same places and at the one behind
    them.  Draft i is kept while accept_draws[r, i] * q_i(x_i) < p_i(x_i), and behind the k kept ones token_draws[r] picks from
    max(p_k - q_k, 0), or from p_n where all were kept: the first token whose cumulative weight is above that share of the whole.
    Weights are summed as integers of 2^-48, so a result does not depend on the order of the sums.  A greedy request passes
    rows that are 1 at the largest logit.

    Probabilities and draws are float32, draws in [0, 1); rows may be any distance apart.  Returns int32 tokens [R, N + 1] (the kept
    ones, the new one, -1) and emitted [R] = k + 1 (0 for an idle request): by how many tokens the request has grown.  Rows that are
    not there (the request is left idle), a drafted token outside the vocabulary (refused, and the one
    behind it comes from the target's whole row) and a row without mass or with that of
    thousands (token 0: logits, say, are no probabilities) set the error word."""
    return draft_call("verify_drafts", _nb(token_draws) and _nb(token_draws) * target_probs.shape[-1], target_probs, q_start, draft_tokens, draft_len,
                      draft_probs, accept_draws, token_draws, err)
