"""Keys and values that are not finite, in attention of new tokens: they reach the tokens that see them and no others, whatever the form.
A value that is not finite reaches its own column alone."""
import pytest
import torch

from draft_helpers import paged_batch, plain_attention
from test_attention_chunks_gpu import call

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF, NAN = float("inf"), float("nan")
FORMS = [pytest.param((-1, F32), id="float32"), pytest.param((0, BF16), id="float32 of bfloat16 pools"), pytest.param((16, BF16), id="mma"),
         pytest.param((1, BF16), id="tcgen05"), pytest.param((18, BF16), id="clusters of 2"), pytest.param((20, BF16), id="clusters of 4"), pytest.param((24, BF16), id="clusters of 8")]


@pytest.fixture(params=FORMS)
def dtype(request, monkeypatch):
    from ai_engine_b200.kernels import ops

    form, dtype = request.param
    monkeypatch.setattr(ops, "CHUNK_FORM", form)
    return dtype


def poison(b, what, r, key, head, columns, value):
    """Sets b's key or value row `key` of request r's key head, in its pages and in what the plain form reads; the plain form's rows stay
    finite and the places are noted."""
    P, page = b["k_pages"].shape[2], int(b["table"][r, key // b["k_pages"].shape[2]])
    if page < 0:
        return
    pool = b["k_pages"] if what == "k" else b["v_pages"]
    pool[page, head, key % P, columns] = value
    b["rows"][r][0 if what == "k" else 1][key, head, columns] = 0.0
    b.setdefault("poisoned", []).append((what, r, key, head, columns, value))


def check(b, dtype):
    out, word = call(b)
    assert word == 0
    out = out.double().cpu()
    want, tol = plain_attention(b, dtype)
    G = b["q"].shape[1] // b["k_pages"].shape[1]
    add = torch.zeros_like(want)
    for what, r, key, head, columns, value in b["poisoned"]:
        for i in range(b["new"][r]):
            pos = b["cached"][r] + i
            if key <= pos and (not b["window"] or key > pos - b["window"]):
                row = add[b["start"][r] + i, head * G:(head + 1) * G]
                if what == "k":
                    row[:] = NAN
                else:
                    row[:, columns] += value
    rows = [s + i for s, n in zip(b["start"], b["new"]) for i in range(n)]
    good = torch.isfinite(add)
    assert torch.equal(torch.isfinite(out)[rows], good[rows])
    assert ((out - want).abs() <= tol)[rows][good[rows]].all()
    assert good[rows].any() and not good[rows].all()
    return out, add


CASES = [([300], [5]), ([40, 0, 129], [7, 3, 2]), ([1000, 63], [40, 130]), ([0], [300]), ([20000], [3]), ([700] * 40, [4] * 40)]


@pytest.mark.parametrize("cached,new", CASES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("P", [16, 128])
def test_values_of_new_tokens(dtype, cached, new, d, P):
    """The values of every request's last token, of one in the middle and of its first, each not finite in a few columns."""
    b = paged_batch(cached, new, 8, 2, d, P, dtype, sum(cached) + d + P)
    for r, (c, n) in enumerate(zip(cached, new)):
        poison(b, "v", r, c + n - 1, 0, [0, 5, d - 1], INF)
        poison(b, "v", r, c + n // 2, 1, [3], NAN)
        poison(b, "v", r, c + n // 2, 1, [7, 8], -INF)
        poison(b, "v", r, c, r % 2, [11], INF)
    out, add = check(b, dtype)
    seen = torch.isinf(add)                         # an infinite value stays one, with its sign
    assert torch.equal(out[seen], add[seen])


@pytest.mark.parametrize("cached,new", CASES)
@pytest.mark.parametrize("d", [64, 128])
def test_keys_of_new_tokens(dtype, cached, new, d):
    b = paged_batch(cached, new, 8, 2, d, 16, dtype, sum(cached) + d)
    for r, (c, n) in enumerate(zip(cached, new)):
        poison(b, "k", r, c + n - 1, 0, [2, d - 2], NAN)
        poison(b, "k", r, c + n // 2, 1, [0, 1, 2, 3], NAN)
    check(b, dtype)


@pytest.mark.parametrize("window", [1, 17, 128, 200])
@pytest.mark.parametrize("cached,new", [([300, 700], [5, 1]), ([500], [60]), ([90], [300])])
def test_values_that_some_tokens_have_passed(dtype, window, cached, new):
    """Values that the window of the first tokens holds and that of later ones has passed, and values that all have."""
    b = paged_batch(cached, new, 8, 2, 64, 16, dtype, window, window=window)
    for r, (c, n) in enumerate(zip(cached, new)):
        for key, head, column in ((c + n // 2 - window, 0, 1), (c - window + 1, 1, 2), (c - window, 0, 3), (c + n - 1, 0, 4)):
            if key >= 0:
                poison(b, "v", r, key, head, [column], INF)
        poison(b, "k", r, max(0, c - window), 1, [0], NAN)
    check(b, dtype)


@pytest.mark.parametrize("d", [8, 96, 200, 256])
def test_other_head_sizes(dtype, d):
    if dtype == BF16:
        from ai_engine_b200.kernels import ops
        if ops.CHUNK_FORM != 0:
            pytest.skip("a form of heads of 64 and 128")
    b = paged_batch([130, 3], [9, 40], 6, 2, d, 16, dtype, d)
    for r, (c, n) in enumerate(zip(b["cached"], b["new"])):
        poison(b, "v", r, c + n - 1, 0, [0, d - 1], -INF)
        poison(b, "v", r, c + 4, 1, [d // 2], NAN)
    check(b, dtype)


def test_other_requests_stay_clean(dtype):
    """All keys and values of one request: the others' results are the same bits."""
    b = paged_batch([300, 40, 900], [5, 3, 7], 8, 2, 64, 16, dtype, 4)
    clean, _ = call(b)
    pages = b["table"][1][b["table"][1] >= 0].long()
    for pool in (b["k_pages"], b["v_pages"]):
        pool[pages] = NAN
    out, word = call(b)
    assert word == 0 and torch.isnan(out[5:8]).all()
    assert torch.equal(out[:5], clean[:5]) and torch.equal(out[8:], clean[8:])
