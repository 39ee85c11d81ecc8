"""Verification of drafted tokens against the target's probabilities."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ..kernels.loader import KernelError
from ..kernels.ops import Launcher, check_operands
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
    for name, t, shape in (("target_probs", target_probs, (T, V)), ("draft_probs", draft_probs, (R, N, V)),
                           ("accept_draws", accept_draws, (R, N)), ("token_draws", token_draws, (R,))):
        if t is not None and (t.dtype != torch.float32 or t.shape != shape):
            raise KernelError(f"verify_drafts: {name} must be float32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    row, element = target_probs.stride()
    guess, by_req, by_place = None, 0, 0
    if draft_probs is not None:
        guess, (by_req, by_place, last) = draft_probs.data_ptr(), draft_probs.stride()
        element = element if last == 1 else last
    if element != 1 and V > 1:
        raise KernelError("verify_drafts: the probabilities of a row must be contiguous")
    if not (accept_draws.is_contiguous() and token_draws.is_contiguous()):
        raise KernelError("verify_drafts: draws must be contiguous")
    stream = check_operands("verify_drafts", (("q_start", q_start, (R,)), ("draft_tokens", draft_tokens, (R, N)), ("draft_len", draft_len, (R,)),
                                              ("err", err, (1,))), (target_probs, draft_probs, accept_draws, token_draws))
    tokens, emitted = torch.empty(R * (N + 2), dtype=torch.int32, device=target_probs.device).split_with_sizes((R * (N + 1), R))
    tokens = tokens.view(R, N + 1)
    if R == 0:
        return tokens, emitted
    with region("verify_drafts", 4 * R * V * (2 if guess else 1)):
        _VERIFY((target_probs.data_ptr(), q_start.data_ptr(), draft_tokens.data_ptr(), draft_len.data_ptr() if draft_len is not None else 0,
                 guess or 0, accept_draws.data_ptr(), token_draws.data_ptr(), tokens.data_ptr(), emitted.data_ptr(), err.data_ptr(), row,
                 by_req, by_place, T, V, R, N), stream)
    return tokens, emitted


_VERIFY = Launcher("verify_drafts.cu", "aie_verify_drafts", "10P3q4i")
