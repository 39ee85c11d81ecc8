"""Every form of the attention of new tokens at sizes that the choice between them would give to another: items of one row and of
several tiles, rows that end inside a tile, tokens whose heads two items share, keys that end on and beside a tile's edge."""
import pytest
import torch

from draft_helpers import paged_batch
from test_attention_chunks_gpu import check

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


FORMS = {"float32": 0, "tcgen05": 1, "mma": 16, "clusters of 2": 18, "clusters of 3": 19, "clusters of 8": 24}


@pytest.fixture(params=list(FORMS))
def form(request, monkeypatch):
    from ai_engine_b200.kernels import ops

    monkeypatch.setattr(ops, "CHUNK_FORM", FORMS[request.param])
    return request.param


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,K", [(4, 4), (8, 2), (6, 2), (16, 1), (7, 1)])
@pytest.mark.parametrize("cached,new", [([0], [1]), ([1], [1]), ([126], [1]), ([127], [1]), ([128], [1]), ([0], [129]), ([255], [2]),
                                        ([383, 0, 1, 900, 127], [1, 32, 33, 65, 0])])
def test_edges(form, d, H, K, cached, new):
    check(paged_batch(cached, new, H, K, d, 16, BF16, sum(cached) + H + d), BF16)


@pytest.mark.parametrize("P", [8, 32, 128, 256, 384])
def test_page_sizes(form, P):
    check(paged_batch([700, 0, 385, 128], [9, 64, 1, 40], 8, 2, 128, P, BF16, P), BF16)


@pytest.mark.parametrize("window", [1, 40, 128, 129, 600])
@pytest.mark.parametrize("d", [64, 128])
def test_windows(form, window, d):
    check(paged_batch([1500, 0, 300, 127], [1, 90, 40, 2], 8, 2, d, 16, BF16, window, window=window), BF16)


def test_items_over_many_blocks_and_many_items_a_block(form):
    check(paged_batch([20000], [3], 4, 1, 128, 16, BF16, 1), BF16)
    check(paged_batch([200] * 90, [1 + i % 60 for i in range(90)], 8, 2, 64, 16, BF16, 2), BF16)


@pytest.mark.parametrize("scale", [0.0, -0.2, 20.0])
def test_scales(form, scale):
    b = paged_batch([300, 40], [40, 3], 4, 2, 64, 16, BF16, 9)
    b["scale"] = scale
    check(b, BF16)


def test_out_may_be_the_queries(form):
    """In place: the rows that requests name become their results, the others stay.  Items of one block, of several, and of several tiles."""
    from ai_engine_b200.kernels import ops

    for cached, new, H, K, d in (([300, 0, 1500], [9, 70, 3], 8, 2, 64), ([20000], [3], 4, 1, 128), ([40] * 60, [2] * 60, 4, 4, 64)):
        b = paged_batch(cached, new, H, K, d, 16, BF16, sum(new), slack=2)
        e = torch.zeros(1, dtype=torch.int32, device="cuda")
        a = (b["k_pages"], b["v_pages"], b["q_start"], b["q_len"], b["ctx_len"], b["table"], b["scale"], 0, e)
        apart = ops.paged_attention_chunks(b["q"], *a, out=b["q"].clone())
        place = b["q"].clone()
        assert ops.paged_attention_chunks(place, *a, out=place).data_ptr() == place.data_ptr()
        assert torch.equal(place, apart) and int(e) == 0
