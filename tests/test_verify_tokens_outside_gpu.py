"""Drafted tokens outside the vocabulary, of drafts with and without probabilities: refused, and since they came out of no distribution
nothing is taken off the target's row that the next token is drawn from."""
import pytest
import torch

from draft_helpers import plain_verify
from test_verify_drafts_gpu import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [600, 601])
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("at", [0, 1, 33])
def test_the_next_token_is_drawn_from_the_whole_row(V, certain, at):
    N, g = at + 2, torch.Generator().manual_seed(V + at)
    target = torch.softmax(torch.randn(N + 1, V, generator=g), -1)
    guess = torch.softmax(torch.randn(1, N, V, generator=g), -1)
    good = [[int(row.argmax()) for row in target[:N]]]
    for x in (-1, V, -2 ** 31, 2 ** 31 - 1):
        for pick in (0.0, 0.37, 0.8, 1 - 2.0 ** -24):
            tokens = [good[0][:at] + [x] + good[0][at + 1:]]
            out, emitted, word = call(target, [0], tokens, [N], None if certain else guess, [[0.0] * N], [pick])
            drawn = plain_verify(target, [at], [[]], [0], None, [[]], [pick])[0][0]
            assert out[0] == good[0][:at] + drawn + [-1] * (N - at) and emitted == [at + 1] and word == 1
