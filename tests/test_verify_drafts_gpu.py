"""Verification of drafted tokens against whole-number sums made one by one."""
import pytest
import torch

from draft_helpers import plain_verify

pytestmark = pytest.mark.gpu
DEV = "cuda"


def call(target, q_start, tokens, lens, guess, accept, pick):
    from ai_engine_b200.sampling import verify_drafts

    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)
    move = lambda x: None if x is None else x.to(DEV)
    out, emitted = verify_drafts(move(target), ints(q_start), ints(tokens), ints(lens), move(guess),
                                 torch.tensor(accept, dtype=torch.float32, device=DEV).view(len(tokens), -1),
                                 torch.tensor(pick, dtype=torch.float32, device=DEV), e)
    return out.tolist(), emitted.tolist(), int(e.item())


def batch(R, N, V, seed, near=0.7, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, N + 1, (R,), generator=g).tolist()
    start = [sum(n + 1 for n in lens[:i]) for i in range(R)]
    logits = sharp * torch.randn(sum(lens) + R, V, generator=g)
    rows = torch.tensor([[min(start[r] + i, len(logits) - 1) for i in range(N)] for r in range(R)], dtype=torch.long).view(R, N)
    guess = torch.softmax(logits[rows] + near * torch.randn(R, N, V, generator=g), -1)
    tokens = (guess / torch.empty_like(guess).exponential_(generator=g)).argmax(-1)
    f32 = lambda x: x.float().tolist()
    return (torch.softmax(logits, -1), start, tokens.tolist(), lens, guess, f32(torch.rand(R, N, generator=g)), f32(torch.rand(R, generator=g)))


@pytest.mark.parametrize("R,N,V", [(1, 1, 1), (3, 4, 5), (7, 2, 511), (5, 5, 512), (4, 3, 513), (6, 4, 4099), (2, 33, 700), (9, 1, 32000),
                                   (3, 2, 50257), (130, 3, 64)])
@pytest.mark.parametrize("certain", [False, True])
def test_against_one_by_one(R, N, V, certain):
    target, start, tokens, lens, guess, accept, pick = batch(R, N, V, R * 7 + N + V)
    a = (target, start, tokens, lens, None if certain else guess, accept, pick)
    out, emitted, word = call(*a)
    assert (out, emitted) == plain_verify(*a) and word == 0


def test_the_widest_vocabulary():
    V = 1 << 20
    target, start, tokens, lens, guess, accept, pick = batch(1, 1, V, 3, sharp=1.0)
    for u in (0.0, 0.37, 1 - 2.0 ** -24):
        a = (target, start, tokens, [1], guess, [[1 - 2.0 ** -24]], [u])
        target_rows = torch.cat([target, target])[:2]
        a = (target_rows,) + a[1:]
        assert call(*a)[:2] == plain_verify(*a)


@pytest.mark.parametrize("N", [1, 3])
def test_every_number_of_kept_tokens(N):
    """Draws of 0 keep a draft whose token the target may have at all, draws just below 1 refuse one that the draft model overrates."""
    V = 40
    target, start, tokens, lens, guess, _, pick = batch(8, N, V, 21)
    lens, start = [N] * 8, [(N + 1) * r for r in range(8)]
    target = torch.softmax(torch.randn(8 * (N + 1), V, generator=torch.Generator().manual_seed(1)), -1)
    for kept in range(N + 1):
        accept = [[0.0 if i < kept else 1 - 2.0 ** -24 for i in range(N)] for _ in range(8)]
        for r in range(8):
            for i in range(N):
                guess[r, i, tokens[r][i]] = 0.9
        a = (target, start, tokens, lens, guess, accept, pick)
        out, emitted, _ = call(*a)
        assert (out, emitted) == plain_verify(*a) and emitted == [kept + 1] * 8


def test_greedy_requests_pass_rows_of_one():
    target = torch.zeros(4, 9)
    target[torch.arange(4), torch.tensor([3, 5, 5, 1])] = 1
    out, emitted, word = call(target, [0], [[3, 5, 7]], [3], None, [[0.99, 0.99, 0.99]], [0.5])
    assert out == [[3, 5, 5, -1]] and emitted == [3] and word == 0


def test_idle_requests_and_no_drafts():
    target, start, tokens, lens, guess, accept, pick = batch(4, 2, 100, 9)
    lens = [-1, 0, 2, -5]
    start = [0, 0, 1, 0]
    target = target[:4] if len(target) >= 4 else target.repeat(4, 1)[:4]
    a = (target, start, tokens, lens, guess, accept, pick)
    out, emitted, word = call(*a)
    assert (out, emitted) == plain_verify(*a) and word == 0 and emitted[0] == emitted[3] == 0 and out[0] == [-1, -1, -1]
    # no places for drafts at all: one token a request, drawn from its row
    a = (target, [3, 1, 0, 2], [[], [], [], []], None, None, [], pick)
    out, emitted, word = call(*a)
    assert (out, emitted) == plain_verify(*a) and emitted == [1] * 4


def test_nothing_left_draws_from_the_target():
    """p nowhere above q (the draft's row sums to more), and a refusal all the same."""
    p = torch.tensor([[0.25, 0.25, 0.5, 0.0]])
    a = (torch.cat([p, p]), [0], [[0]], [1], torch.tensor([[[0.5, 0.25, 0.5, 0.0]]]), [[0.75]], [0.6])
    out, emitted, word = call(*a)
    assert (out, emitted) == plain_verify(*a) == ([[2, -1]], [1]) and word == 0


def test_rows_that_are_not_distributions():
    zero, nan = torch.zeros(2, 700), torch.full((2, 700), float("nan"))
    for row in (zero, nan):
        out, emitted, word = call(row, [0], [[5]], [1], None, [[0.5]], [0.5])
        assert out == [[0, -1]] and emitted == [1] and word == 16
    # what is not a number weighs nothing, what is above 1 weighs 1
    row = torch.tensor([[float("nan"), float("inf"), -3.0, 0.5, float("-inf")]])
    assert call(row, [0], [[0]], [0], None, [[0.5]], [0.66])[0] == [[1, -1]]
    assert call(row, [0], [[0]], [0], None, [[0.5]], [0.67])[0] == [[3, -1]]
    # draws outside [0, 1)
    for u, t in ((1.0, 3), (float("inf"), 3), (-1.0, 1), (float("nan"), 1)):
        assert call(row, [0], [[0]], [0], None, [[0.5]], [u])[0] == [[t, -1]]


@pytest.mark.parametrize("R", [1, 20, 40])
def test_rows_whose_sums_do_not_fit(R):
    """Entries that are no probabilities: 70,000 ones weigh more than 64 bits hold; 20,000 still fit and are drawn from."""
    ask = lambda row: call(row.expand(2, -1), [0] * R, [[-1]] * R, [1] * R, None, [[0.5]] * R, [0.5] * R)
    for V, first in ((70000, 0), (100000, 12800), (1048576, 0)):
        row = torch.ones(1, V)
        row[:, :first] = 0
        assert ask(row) == ([[0, -1]] * R, [1] * R, 1 | 16)
    assert ask(torch.ones(1, 20000)) == ([[10000, -1]] * R, [1] * R, 1)


def test_rows_and_tokens_that_are_not_there():
    target = torch.softmax(torch.randn(3, 600, generator=torch.Generator().manual_seed(2)), -1)
    for start, n in ((2, 1), (-1, 0), (3, 0), (0, 3), (2 ** 31 - 1, 1)):
        out, emitted, word = call(target, [start], [[1, 1]], [n], None, [[0.5, 0.5]], [0.5])
        assert out == [[-1, -1, -1]] and emitted == [0] and word == 8
    for x in (-1, 600, -2 ** 31, 2 ** 31 - 1):          # refused; nothing is taken off the target for it
        out, emitted, word = call(target, [0], [[x, 1]], [2], None, [[0.0, 0.0]], [0.5])
        assert out[0] == plain_verify(target, [0], [[]], [0], None, [[]], [0.5])[0][0] + [-1, -1] and emitted == [1] and word == 1


@pytest.mark.parametrize("V", [4096, 4097])
def test_rows_any_distance_apart(V):
    target, start, tokens, lens, guess, accept, pick = batch(5, 3, V, 77)
    from ai_engine_b200.sampling import verify_drafts
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    wide_t = torch.full((len(target), V + 9), float("nan"), device=DEV)
    wide_t[:, 4:4 + V] = target
    wide_g = torch.full((3, 5, V + 2), float("nan"), device=DEV)           # place by place, as a draft model makes them
    wide_g[:, :, :V] = guess.transpose(0, 1)
    e = ints([0])
    out, emitted = verify_drafts(wide_t[:, 4:4 + V], ints(start), ints(tokens), ints(lens), wide_g[:, :, :V].transpose(0, 1),
                                 torch.tensor(accept, device=DEV), torch.tensor(pick, device=DEV), e)
    assert (out.tolist(), emitted.tolist()) == plain_verify(target, start, tokens, lens, guess, accept, pick)


def test_tokens_follow_the_target():
    """The first token of 40,000 requests with the same rows: its shares are the target's, whatever the draft's.  A share's standard
    deviation is at most sqrt(1/4 / 40000) = 0.0025; five of them are allowed."""
    from ai_engine_b200.sampling import verify_drafts
    g = torch.Generator(device=DEV).manual_seed(4)
    R, V = 40000, 6
    p = torch.tensor([0.3, 0.05, 0.2, 0.0, 0.25, 0.2], device=DEV)
    q = torch.tensor([0.1, 0.4, 0.1, 0.3, 0.05, 0.05], device=DEV)
    drafts = torch.multinomial(q, R, replacement=True, generator=g).int()[:, None]
    target = p.repeat(2 * R, 1)
    out, _ = verify_drafts(target, torch.arange(0, 2 * R, 2, device=DEV, dtype=torch.int32), drafts, None, q.expand(R, 1, V),
                           torch.rand(R, 1, device=DEV, generator=g), torch.rand(R, device=DEV, generator=g),
                           torch.zeros(1, dtype=torch.int32, device=DEV))
    share = torch.bincount(out[:, 0].long(), minlength=V).double() / R
    assert (share - p.double()).abs().max() < 5 * 0.0025
