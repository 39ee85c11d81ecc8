"""Pages, block tables and cache slots made on the device, against the same request by request."""
import random

import pytest
import torch

from draft_helpers import plain_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)


def call(cached, counts, held, table, free, free_count, P, n_pages, max_tokens, err=None):
    from ai_engine_b200.cache import step_tables

    e = ints([0]) if err is None else err
    t = step_tables(ints(cached), ints(counts), ints(held), ints(table), ints(free), ints([free_count]), P, n_pages, max_tokens, e)
    return t, int(e.item())


def batch(R, P, W, seed, most_new=9, kept=2):
    """Lengths, pages and a shuffled free list of requests that may hold up to `kept` pages more than their tokens need."""
    rng = random.Random(seed)
    cached = [rng.randint(0, max(0, W * P - most_new)) for _ in range(R)]
    counts = [rng.choice([0, 1, 1, rng.randint(1, most_new)]) for _ in range(R)]
    held = [min(W, -(-c // P) + rng.randint(0, kept)) for c in cached]
    n_pages = sum(held) + R * most_new
    ids = list(range(n_pages))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (W - h))
        at += h
    return cached, counts, held, table, ids[at:], n_pages


@pytest.mark.parametrize("R,P,W,free_share", [(1, 16, 4, 1.0), (3, 1, 40, 1.0), (8, 16, 256, 0.3), (33, 7, 13, 0.5), (255, 16, 9, 0.2),
                                              (256, 8, 20, 0.0), (257, 16, 8, 0.5), (700, 16, 33, 0.7), (4096, 32, 5, 0.4)])
@pytest.mark.parametrize("spare", [0, 37])
def test_tables_against_request_by_request(R, P, W, free_share, spare):
    cached, counts, held, table, free, n_pages = batch(R, P, W, 100 * R + W)
    need = sum(max(0, -(-(c + n) // P) - h) if n else 0 for c, n, h in zip(cached, counts, held))
    free_count = min(len(free), int(need * free_share) + (3 if free_share == 1.0 else 0))
    max_tokens = sum(counts) + spare
    want = plain_tables(cached, counts, held, table, free, free_count, P, max_tokens)
    got, word = call(cached, counts, held, table, free, free_count, P, n_pages, max_tokens)
    for name, g, w in zip(got._fields, got, want):
        assert g.tolist() == w, name
    assert word == 0


def test_inputs_stay_and_outputs_feed_the_next_step():
    from ai_engine_b200.cache import step_tables

    P, W, R = 4, 8, 5
    held, table, free_count = ints([0] * R), ints([[-1] * W] * R), ints([30])
    free, cached, e = ints(list(range(30))), ints([0] * R), ints([0])
    h_cached, h_held, h_table, h_free = [0] * R, [0] * R, [[-1] * W for _ in range(R)], 30
    rng = random.Random(5)
    for step in range(6):
        counts = [rng.randint(0, 5) for _ in range(R)]
        kept = [rng.randint(1, n) if n else 0 for n in counts]
        before = [t.clone() for t in (cached, held, table, free, free_count)]
        t = step_tables(cached, ints(counts), held, table, free, free_count, P, 30, 25, e)
        assert all(torch.equal(a, b) for a, b in zip(before, (cached, held, table, free, free_count)))
        want = plain_tables(h_cached, counts, h_held, h_table, list(range(30)), h_free, P, 25)
        assert [x.tolist() for x in t] == list(want)
        h_table, h_held, (h_free,), _, lens = want[:5]
        table, held, free_count = t.tables, t.held, t.free_count
        cached = cached + torch.minimum(ints(kept), t.q_len)
        h_cached = [c + min(k, n) for c, k, n in zip(h_cached, kept, lens)]
    assert int(e.item()) == 0


def test_lengths_that_do_not_fit_wait_and_are_flagged():
    W, P = 4, 8
    table = [[0, 1, -1, -1], [2, -1, -1, -1], [3, 4, 5, 6], [7, -1, -1, -1], [8, -1, -1, -1]]
    free = [20, 21, 22, 23, 24, 25]
    good = dict(cached=[16, 8, 31, 8, 3], counts=[1, 1, 1, 1, 2], held=[2, 1, 4, 1, 1])
    # the third brings one token more than its table's row has places for; the others are served as if it were not there
    got, word = call(good["cached"], [1, 1, 2, 1, 2], good["held"], table, free, 6, P, 30, 10)
    assert word == 8 and got.q_len.tolist() == [1, 1, 0, 1, 2] and got.held.tolist() == [3, 2, 4, 2, 1]
    assert got.q_start.tolist() == [0, 1, 2, 4, 5] and got.slots.tolist()[2:4] == [-1, -1] and got.free_count.tolist() == [3]
    # negative lengths
    for key, values in (("cached", [16, 0x7fffffff, 31, 8, 3]), ("cached", [16, -8, 31, 8, 3]), ("held", [2, -1, 4, 1, 1]), ("counts", [1, -1, 1, 1, 2]), ("held", [2, 5, 4, 1, 1])):
        a = dict(good)
        a[key] = values
        got, word = call(a["cached"], a["counts"], a["held"], table, free, 6, P, 30, 10)
        assert word == 8 and got.q_len.tolist() == [1, 0, 1, 1, 2]
    # tokens past max_tokens: the last request waits, and nothing is written behind the arrays
    got, word = call(good["cached"], good["counts"], good["held"], table, free, 6, P, 30, 5)
    assert word == 8 and got.q_len.tolist() == [1, 1, 1, 1, 0] and got.free_count.tolist() == [3]
    # a free count that the list does not have
    got, word = call(good["cached"], good["counts"], good["held"], table, free, 9, P, 30, 10)
    assert word == 8 and got.free_count.tolist() == [3]
    got, word = call(good["cached"], good["counts"], good["held"], table, free, -2, P, 30, 10)
    assert word == 8 and got.q_len.tolist() == [0, 0, 1, 0, 2] and got.free_count.tolist() == [0]
    # pages outside the pool make no slot
    got, word = call(good["cached"], good["counts"], good["held"], table, [20, 21, 22, 23, 24, 30], 6, P, 30, 10)
    assert word == 2 and got.slots.tolist()[0] == -1 and got.slots.tolist()[1] == 24 * P
    got, word = call([3], [1], [1], [[-1, -1]], free, 6, P, 30, 4)
    assert word == 2 and got.slots.tolist() == [-1] * 4 and got.positions.tolist() == [3, -1, -1, -1]
    # sums beyond 32 bits
    got, word = call([0, 0, 0], [0x7fffffff] * 3, [0] * 3, [[-1] * 4] * 3, free, 6, P, 30, 4)
    assert word == 8 and got.q_len.tolist() == [0, 0, 0] and got.free_count.tolist() == [6]


def test_no_free_list_and_no_tokens():
    got, word = call([3, 4], [1, 0], [1, 1], [[0], [1]], [], 0, 8, 2, 1)
    assert word == 0 and got.slots.tolist() == [3] and got.q_len.tolist() == [1, 0]
    got, word = call([3, 4], [0, 0], [1, 1], [[0], [1]], [], 0, 8, 2, 0)
    assert word == 0 and got.tables.tolist() == [[0], [1]] and got.slots.numel() == 0
