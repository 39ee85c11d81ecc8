"""Verification of drafted tokens against the target's probabilities."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ..kernels.loader import KernelError, check
from ..kernels.ops import int_rows, launcher, on_current_device
from ..kernels.profile import region

MAX_VOCAB = 1 << 20


def verify_drafts(target_probs: torch.Tensor, q_start: torch.Tensor, draft_tokens: torch.Tensor, draft_len: Optional[torch.Tensor],
                  draft_probs: Optional[torch.Tensor], accept_draws: torch.Tensor, token_draws: torch.Tensor,
                  err: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens are kept, and the token behind them, distributed as the target alone would draw them.

    Request r drafted n = draft_len[r] of the N tokens draft_tokens[r] (None: all N; negative: the request is idle and gets
    nothing) from the distributions draft_probs[r, :n] (None: drafts without probabilities, each taken as certain).  Rows
    q_start[r] .. q_start[r] + n of target_probs [T, V] are the target's distributions at the same places and at the one behind
    them.  Draft i is kept while accept_draws[r, i] * q_i(x_i) < p_i(x_i), and behind the k kept ones token_draws[r] picks from
    max(p_k - q_k, 0), or from p_n where all were kept: the first token whose cumulative weight is above that share of the whole.
    Weights are summed as integers of 2^-48, so a result does not depend on the order of the sums.  A greedy request passes
    rows that are 1 at the largest logit.

    Probabilities and draws are float32, draws in [0, 1); rows may be any distance apart.  Returns int32 tokens [R, N + 1] (the kept
    ones, the new one, -1) and emitted [R] = k + 1 (0 for an idle request): by how many tokens the request has grown.  Rows that are
    not there (the request is left idle), a drafted token outside the vocabulary (refused) and a row without mass (token 0) set the
    error word."""
    if target_probs.dim() != 2 or draft_tokens.dim() != 2:
        raise KernelError("verify_drafts: target_probs must be [T, V] and draft_tokens [R, N]")
    (T, V), (R, N) = target_probs.shape, draft_tokens.shape
    if not 0 < V <= MAX_VOCAB:
        raise KernelError(f"verify_drafts: a vocabulary of {V} (1 to {MAX_VOCAB} are taken)")
    int_rows("verify_drafts", q_start=(q_start, (R,)), draft_tokens=(draft_tokens, (R, N)), err=(err, (1,)))
    if draft_len is not None:
        int_rows("verify_drafts", draft_len=(draft_len, (R,)))
    for name, t, shape in (("target_probs", target_probs, (T, V)), ("draft_probs", draft_probs, (R, N, V)),
                           ("accept_draws", accept_draws, (R, N)), ("token_draws", token_draws, (R,))):
        if t is not None and (t.dtype != torch.float32 or t.shape != shape):
            raise KernelError(f"verify_drafts: {name} must be float32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    if V > 1 and (target_probs.stride(1) != 1 or (draft_probs is not None and draft_probs.stride(2) != 1)):
        raise KernelError("verify_drafts: the probabilities of a row must be contiguous")
    if not (accept_draws.is_contiguous() and token_draws.is_contiguous()):
        raise KernelError("verify_drafts: draws must be contiguous")
    stream = on_current_device("verify_drafts", target_probs, q_start, draft_tokens, draft_len, draft_probs, accept_draws, token_draws, err)
    tokens = torch.empty((R, N + 1), dtype=torch.int32, device=target_probs.device)
    emitted = torch.empty(R, dtype=torch.int32, device=target_probs.device)
    if R == 0:
        return tokens, emitted
    guess, by_req, by_place = (draft_probs.data_ptr(), draft_probs.stride(0), draft_probs.stride(1)) if draft_probs is not None else (None, 0, 0)
    fn = launcher("verify_drafts.cu", "aie_verify_drafts", "pliippppll" + "iipppppp")
    with region("verify_drafts", 4 * R * V * (2 if draft_probs is not None else 1)):
        check(fn(target_probs.data_ptr(), target_probs.stride(0), T, V, q_start.data_ptr(), draft_tokens.data_ptr(),
                 draft_len.data_ptr() if draft_len is not None else None, guess, by_req, by_place, R, N, accept_draws.data_ptr(),
                 token_draws.data_ptr(), tokens.data_ptr(), emitted.data_ptr(), err.data_ptr(), stream), "verify_drafts")
    return tokens, emitted
