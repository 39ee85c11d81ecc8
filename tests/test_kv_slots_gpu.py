"""Keys and values written to cache slots."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def write(*a):
    from ai_engine_b200.kernels import ops

    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.write_kv_slots(*a, e)
    return int(e.item())


def want(pages, rows, slots):
    """The pool with its rows set one by one (a copy; bit patterns are compared)."""
    out, P = pages.clone(), pages.shape[2]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages.shape[0] * P:
            out[s // P, :, s % P] = rows[t].to(pages.dtype)
    return out


@pytest.mark.parametrize("rows,cache", [(F32, BF16), (BF16, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("T,K,d,P", [(1, 1, 64, 16), (5, 8, 128, 16), (33, 3, 40, 7), (130, 2, 6, 1), (257, 8, 64, 32), (2, 5, 1, 3)])
@pytest.mark.parametrize("layout", ["own", "fused", "odd", "heads first"])
def test_rows_land_in_their_slots(rows, cache, T, K, d, P, layout):
    g = torch.Generator(device=DEV).manual_seed(T * d + K)
    N = (T + P - 1) // P + 2
    if layout == "own":
        kv = torch.randn(2, T, K, d, device=DEV, generator=g).to(rows)
        k, v = kv[0], kv[1]
    elif layout == "fused":
        kv = torch.randn(T, 5 * K * d, device=DEV, generator=g).to(rows)
        k, v = (kv[:, i * K * d:(i + 1) * K * d].view(T, K, d) for i in (3, 4))
    elif layout == "odd":         # rows that do not start on 16 bytes
        kv = torch.randn(T, 2 * K * d + 3, device=DEV, generator=g).to(rows)
        k, v = kv[:, 1:1 + K * d].view(T, K, d), kv[:, 3 + K * d:].view(T, K, d)
    else:
        k, v = (torch.randn(K, T, d, device=DEV, generator=g).to(rows).transpose(0, 1) for _ in range(2))
    pools = [torch.randn(N, K, P, d, device=DEV, generator=g).to(cache) for _ in range(2)]
    slots = torch.randperm(N * P, device=DEV, generator=g)[:T].int()
    slots[::4] = -1 - slots[::4]
    expect = want(pools[0], k, slots), want(pools[1], v, slots)
    assert write(k, v, pools[0], pools[1], slots) == 0
    assert torch.equal(pools[0], expect[0]) and torch.equal(pools[1], expect[1])


def test_slots_past_the_pool_are_left_out_and_flagged():
    k = torch.randn(4, 2, 64, device=DEV)
    pools = [torch.zeros(3, 2, 4, 64, device=DEV) for _ in range(2)]
    slots = torch.tensor([12, 0, 2 ** 31 - 1, 11], dtype=torch.int32, device=DEV)
    expect = want(pools[0], k, slots)
    assert write(k, k, pools[0], pools[1], slots) == 2
    assert torch.equal(pools[0], expect) and torch.equal(pools[1], expect)


def test_no_rows():
    pools = [torch.zeros(3, 2, 4, 64, device=DEV) for _ in range(2)]
    assert write(torch.zeros(0, 2, 64, device=DEV), torch.zeros(0, 2, 64, device=DEV), *pools, torch.zeros(0, dtype=torch.int32, device=DEV)) == 0


def test_slots_whose_offset_passes_32_bits():
    """A pool of 2^31 elements and more: 70,000 pages of 16 x 2 x 1,024 bfloat16."""
    pools = [torch.zeros(70000, 2, 16, 1024, device=DEV, dtype=BF16) for _ in range(2)]
    k = torch.randn(3, 2, 1024, device=DEV, dtype=BF16)
    slots = torch.tensor([70000 * 16 - 1, 5, 69000 * 16], dtype=torch.int32, device=DEV)
    assert write(k, 2 * k, *pools, slots) == 0
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(pools[0][s // 16, :, s % 16], k[t]) and torch.equal(pools[1][s // 16, :, s % 16], 2 * k[t])
    assert int(torch.count_nonzero(pools[0])) == int(torch.count_nonzero(k))
