"""Lengths, rows and pages that are not there, in every form of the attention of new tokens: they are flagged, bring nothing, and leave the
other requests' results as they are."""
import pytest
import torch

from draft_helpers import paged_batch, plain_attention
from test_attention_chunks_gpu import call, check

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
FORMS = [pytest.param((-1, F32), id="float32"), pytest.param((0, BF16), id="float32 of bfloat16 pools"), pytest.param((16, BF16), id="mma"),
         pytest.param((1, BF16), id="tcgen05"), pytest.param((18, BF16), id="clusters of 2"), pytest.param((20, BF16), id="clusters of 4"),
         pytest.param((24, BF16), id="clusters of 8")]
FAR = 2 ** 31 - 1


@pytest.fixture(params=FORMS)
def dtype(request, monkeypatch):
    from ai_engine_b200.kernels import ops

    form, dtype = request.param
    monkeypatch.setattr(ops, "CHUNK_FORM", form)
    return dtype


BATCHES = [([40, 100, 20, 7], [2, 3, 1, 2]), ([900, 1500, 260, 3000], [5, 70, 130, 1])]


def others(b, r):
    return [s + i for o, (s, n) in enumerate(zip(b["start"], b["new"])) if o != r for i in range(n)]


@pytest.mark.parametrize("cached,new", BATCHES)
@pytest.mark.parametrize("P", [16, 128])
def test_lengths_that_do_not_fit(dtype, cached, new, P):
    b = paged_batch(cached, new, 8, 2, 64, P, dtype, sum(cached) + P)
    want, tol = plain_attention(b, dtype)
    T = b["q"].shape[0]
    for key, value in (("q_len", -1), ("q_len", T), ("q_len", FAR), ("q_start", -1), ("q_start", T + 1), ("q_start", FAR), ("ctx_len", -3),
                       ("ctx_len", P * b["table"].shape[1]), ("ctx_len", FAR)):
        a = dict(b, **{key: b[key].clone()})
        a[key][1] = value
        out = torch.full_like(b["q"], 7.0)
        _, word = call(a, out=out)
        rows = others(b, 1)
        assert word == 8, (key, value)
        assert ((out.double().cpu() - want).abs() <= tol)[rows].all()
        assert (out[b["start"][1]:b["start"][1] + new[1]] == 7).all()


@pytest.mark.parametrize("cached,new", BATCHES)
@pytest.mark.parametrize("P,window", [(16, 0), (128, 0), (16, 50)])
def test_pages_outside_the_pool(dtype, cached, new, P, window):
    """Their keys and values are zeros: they share in the softmax with weight 2^0."""
    b = paged_batch(cached, new, 8, 2, 64, P, dtype, sum(cached) + P, window=window)
    place = (cached[1] + new[1] - 1) // P            # the page of the last token
    a, zeros = dict(b, table=b["table"].clone()), dict(b, rows=[(k.clone(), v.clone()) for k, v in b["rows"]])
    for x in zeros["rows"][1]:
        x[place * P:] = 0
    want, tol = plain_attention(zeros, dtype)
    named = [s + i for s, n in zip(b["start"], new) for i in range(n)]
    for bad in (-1, b["k_pages"].shape[0], -2 ** 31, FAR):
        a["table"][1, place] = bad
        out, word = call(a)
        assert word == 2 and ((out.double().cpu() - want).abs() <= tol)[named].all()


def test_clusters_of_four(monkeypatch):
    """The choice by size takes them for small batches; edges as in the other forms."""
    from ai_engine_b200.kernels import ops

    monkeypatch.setattr(ops, "CHUNK_FORM", 20)
    for cached, new in (([0], [1]), ([126], [1]), ([127], [1]), ([0], [129]), ([383, 0, 1, 900, 127], [1, 32, 33, 65, 0]), ([20000], [3])):
        for H, K, d in ((8, 2, 64), (6, 2, 128), (7, 1, 64)):
            check(paged_batch(cached, new, H, K, d, 16, BF16, sum(cached) + H + d), BF16)
            check(paged_batch(cached, new, H, K, d, 16, BF16, sum(cached) + H + d, window=40), BF16)
