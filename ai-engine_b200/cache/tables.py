"""A step's pages, block tables and cache slots, made on the device from the requests' lengths.

The host's bookkeeping (`PagedCache`) knows every length when it packs a step.  A program that verifies drafted tokens does not: how
many tokens a request kept is known on the device alone until somebody waits for it.  `step_tables` makes from device lengths what
a step needs, without a word from the host."""
from __future__ import annotations

from typing import NamedTuple

import torch

from ..kernels.ops import _nb, draft_call


class StepTables(NamedTuple):
    """What `step_tables` makes; all int32, in one buffer."""
    tables: torch.Tensor        # [R, W] page ids: what a request held, what it took, -1
    held: torch.Tensor          # [R] pages of each request
    free_count: torch.Tensor    # [1] pages left in the free list
    q_start: torch.Tensor       # [R] first token of each request
    q_len: torch.Tensor         # [R] tokens that go ahead: counts, or 0 for a request that has to wait
    positions: torch.Tensor     # [max_tokens] place of each token in its request; -1 behind the last token
    token_req: torch.Tensor     # [max_tokens] row of its request; -1 behind the last token
    slots: torch.Tensor         # [max_tokens] page * page_size + place in the page; -1 where nothing is to be written


def step_tables(cached: torch.Tensor, counts: torch.Tensor, held: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor,
                free_count: torch.Tensor, page_size: int, num_pages: int, max_tokens: int, err: torch.Tensor) -> StepTables:
    """Request r holds cached[r] tokens in the first held[r] pages of tables[r] and brings counts[r] more; free_pages[:free_count] are
    free.  In the order of the requests, each takes the pages it is short of from the end of the free list; one that cannot have
    all of them has to wait (it takes none, its tokens' slots are -1, its q_len is 0), and so has every later one that is
    short of pages.  Pages held beyond the tokens (drafts that were refused) are used first.  Nothing that is given is changed: the
    next step passes the outputs on.  Sizes: R up to 4,096; max_tokens bounds the sum of the counts.

    A request whose lengths are negative, do not fit the table's width or bring tokens past max_tokens waits and sets the error
    word; a page outside the pool sets it too and makes no slot."""
    return StepTables(*draft_call("step_tables", 2 * _nb(tables), cached, counts, held, tables, free_pages, free_count, page_size,
                                  num_pages, max_tokens, err))
