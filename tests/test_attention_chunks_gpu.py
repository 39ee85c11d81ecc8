"""Attention of new tokens over a paged cache with the lengths on the device, against softmax in 64 bits."""
import pytest
import torch

from draft_helpers import paged_batch, plain_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def call(b, **more):
    from ai_engine_b200.kernels import ops

    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = ops.paged_attention_chunks(b["q"], b["k_pages"], b["v_pages"], b["q_start"], b["q_len"], b["ctx_len"], b["table"], b["scale"],
                                     b["window"], e, **more)
    return out, int(e.item())


def check(b, dtype, **more):
    out, word = call(b, **more)
    want, tol = plain_attention(b, dtype)
    rows = [s + i for s, n in zip(b["start"], b["new"]) for i in range(n)]
    d = (out.double().cpu() - want).abs()[rows]
    assert word == 0 and not torch.isnan(out[rows]).any()
    assert (d <= tol[rows]).all(), float((d / tol[rows]).max())
    return out


HEADS = [(8, 2, 64), (4, 4, 128), (32, 8, 128), (5, 1, 64), (24, 8, 128), (16, 1, 128), (6, 2, 96), (4, 2, 8), (3, 1, 200), (2, 2, 256)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,K,d", HEADS)
@pytest.mark.parametrize("P", [16, 7])
def test_head_layouts(dtype, H, K, d, P):
    check(paged_batch([130, 0, 37, 1], [5, 3, 1, 9], H, K, d, P, dtype, H * d + P), dtype)


CACHED = [([0], [1]), ([1], [1]), ([63], [1]), ([64], [2]), ([127, 128, 129], [1, 1, 1]), ([0, 0, 0, 0], [1, 2, 17, 64]),
          ([1000], [4]), ([500, 3, 0, 2000, 64], [33, 70, 130, 1, 5]), ([4000], [300]), ([250] * 70, [2, 3] * 35), ([9] * 300, [1] * 300)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cached,new", CACHED)
@pytest.mark.parametrize("d", [64, 128])
def test_lengths(dtype, cached, new, d):
    check(paged_batch(cached, new, 8, 2, d, 16, dtype, sum(cached) + d), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P", [1, 3, 8, 24, 32, 64, 128, 256])
def test_pages(dtype, P):
    check(paged_batch([200, 0, 77, 511], [6, 1, 20, 2], 8, 2, 128, P, dtype, P), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [1, 2, 15, 64, 200, 5000])
@pytest.mark.parametrize("d", [64, 128])
def test_windows(dtype, window, d):
    """Pages that every token's window has passed are gone from the table."""
    check(paged_batch([700, 0, 190, 64], [7, 5, 150, 1], 8, 2, d, 16, dtype, window + d, window=window), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_requests_without_tokens_and_rows_of_nobody(dtype):
    b = paged_batch([40, 100, 0, 7, 0], [0, 3, 0, 2, 0], 8, 2, 64, 16, dtype, 3, slack=6)
    out = torch.full_like(b["q"], 7.0)
    check(b, dtype, out=out)
    assert (out[5:] == 7).all()
    b = paged_batch([40, 100], [0, 0], 8, 2, 64, 16, dtype, 3, slack=6)
    out = torch.full_like(b["q"], 7.0)
    assert call(b, out=out)[1] == 0 and (out == 7).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_of_the_queries(dtype):
    b = paged_batch([300, 12], [5, 3], 8, 2, 64, 16, dtype, 5)
    dense = check(b, dtype)
    fused = torch.full((8, 12 * 64), float("nan"), dtype=dtype, device=DEV)
    fused[:, :512] = b["q"].view(8, 512)
    assert torch.equal(call(dict(b, q=fused[:, :512].view(8, 8, 64)))[0], dense)
    heads = b["q"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(call(dict(b, q=heads))[0], dense)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_requests_in_any_order_of_rows(dtype):
    b = paged_batch([300, 12, 90], [5, 3, 2], 8, 2, 64, 16, dtype, 6)
    dense = check(b, dtype)
    order = [2, 0, 1]
    moved = {k: b[k][order].contiguous() for k in ("q_start", "q_len", "ctx_len", "table")}
    out, word = call(dict(b, **moved))
    want, tol = plain_attention(b, dtype)
    assert word == 0 and ((out.double().cpu() - want).abs() <= tol).all() and out.shape == dense.shape


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lengths_and_pages_that_are_not_there(dtype):
    b = paged_batch([40, 100, 20, 7], [2, 3, 1, 2], 8, 2, 64, 16, dtype, 8)
    want, tol = plain_attention(b, dtype)
    far = 2 ** 31 - 1
    for key, value in (("q_len", -1), ("q_len", 8), ("q_len", far), ("q_start", -1), ("q_start", 9), ("q_start", far), ("ctx_len", -3),
                       ("ctx_len", 16 * b["table"].shape[1]), ("ctx_len", far)):
        a = dict(b, **{key: b[key].clone()})
        a[key][1] = value
        out = torch.full_like(b["q"], 7.0)
        _, word = call(a, out=out)
        rows = [0, 1, 5, 6, 7]
        assert word == 8, (key, value)
        assert ((out.double().cpu() - want).abs() <= tol)[rows].all() and (out[2:5] == 7).all()
    # a page outside the pool: its keys are zeros, so they share in the softmax with weight 2^0
    for bad in (-1, b["k_pages"].shape[0], -2 ** 31, far):
        a = dict(b, table=b["table"].clone())
        a["table"][1, 2] = bad
        out, word = call(a)
        assert word == 2 and ((out.double().cpu() - want).abs() <= tol)[[0, 1, 5, 6, 7]].all() and torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_and_small_scores(dtype):
    """Scores that reach thousands: one key takes all; and a batch whose scores are all alike."""
    b = paged_batch([300], [4], 4, 2, 64, 16, dtype, 9)
    b["scale"] = 30.0
    check(b, dtype)
    b["scale"] = 0.0
    check(b, dtype)


def test_many_requests():
    """More requests than a block has threads, most of them without tokens."""
    new = [0] * 1500
    for i in (0, 7, 255, 256, 257, 900, 1499):
        new[i] = 1 + i % 5
    check(paged_batch([i % 50 for i in range(1500)], new, 4, 2, 64, 16, BF16, 10), BF16)
    check(paged_batch([i % 50 for i in range(1500)], new, 4, 2, 64, 16, F32, 10), F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_same_bits_again_and_on_another_stream(dtype):
    b = paged_batch([3000, 5, 700], [5, 8, 40], 8, 2, 128, 16, dtype, 11)
    first = check(b, dtype)
    assert torch.equal(call(b)[0], first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = call(b)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, first)
    # two calls at once, each with scratch of its own
    b2 = paged_batch([1000, 2500], [7, 3], 8, 2, 128, 16, dtype, 12)
    want = call(b2)[0]
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s):
            x = call(b2)[0]
        y = call(b)[0]
        torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(y, first)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_captured_call_follows_the_lengths(dtype):
    from ai_engine_b200.kernels import ops

    b = paged_batch([3000, 5, 700], [5, 8, 3], 8, 2, 64, 16, dtype, 13)
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = {k: b[k].clone() for k in ("q_start", "q_len", "ctx_len", "table")}
    run = lambda: ops.paged_attention_chunks(b["q"], b["k_pages"], b["v_pages"], args["q_start"], args["q_len"], args["ctx_len"],
                                             args["table"], b["scale"], 0, e)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for order in ([0, 1, 2], [2, 1, 0], [1, 0, 2]):
        for k in args:
            args[k].copy_(b[k][order])
        graph.replay()
        want, tol = plain_attention(b, dtype)
        assert ((out.double().cpu() - want).abs() <= tol).all()
    args["q_len"].zero_()
    out.fill_(7)
    graph.replay()
    assert (out == 7).all() and int(e.item()) == 0


def test_rows_whose_offset_passes_32_bits():
    """Pages in the last part of a pool of more than 2^31 elements."""
    b = paged_batch([900, 40], [5, 3], 8, 4, 128, 16, BF16, 14)
    want = check(b, BF16)
    n, far = b["k_pages"].shape[0], 270000                    # 270,000 pages of 4 x 16 x 128: 2.2e9 elements
    for name in ("k_pages", "v_pages"):
        big = torch.zeros(far + n, 4, 16, 128, dtype=BF16, device=DEV)
        big[far:] = b[name]
        b[name] = big
    b["table"] = torch.where(b["table"] >= 0, b["table"] + far, b["table"]).int()
    assert torch.equal(call(b)[0], want)


def test_rows_named_again_and_again(monkeypatch):
    """Requests may name the same rows.  So many of them that their work does not fit 31 bits bring nothing and are flagged."""
    from ai_engine_b200.kernels import ops

    b = paged_batch([70], [3], 8, 2, 64, 16, BF16, 15)
    want = check(b, BF16)
    twice = dict(b, **{k: torch.cat([b[k], b[k]]) for k in ("q_start", "q_len", "ctx_len", "table")})
    out, word = call(twice)
    assert word == 0 and torch.equal(out, want)
    monkeypatch.setattr(ops, "CHUNK_FORM", 16)
    R, n, W = 12000, 2000, 1024               # 12,000 x 8 key heads x 250 row tiles x 110 key tiles and more: 2.6e9
    ints = lambda x, *s: torch.full(s, x, dtype=torch.int32, device=DEV)
    q = torch.full((n, 32, 64), 2.0, dtype=BF16, device=DEV)
    pool = torch.zeros(4, 8, 16, 64, dtype=BF16, device=DEV)
    out, e = torch.full_like(q, 7.0), ints(0, 1)
    ops.paged_attention_chunks(q, pool, pool, ints(0, R), ints(n, R), ints(14000, R), ints(0, R, W), 0.1, 0, e, out=out)
    assert int(e.item()) == 8 and (out == 7).all()


def test_sizes_whose_work_does_not_fit():
    """A table so wide and so many rows that the work could not be counted: refused before anything runs."""
    from ai_engine_b200.kernels import ops
    from ai_engine_b200.kernels.loader import KernelError

    pool = torch.zeros(1, 1, 128, 64, dtype=F32, device=DEV)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    with pytest.raises(KernelError):
        ops.paged_attention_chunks(torch.zeros(4096, 64, 64, device=DEV), pool, pool, ints(1), ints(1), ints(1), ints(1, 1 << 19), 0.1, 0, ints(1))
