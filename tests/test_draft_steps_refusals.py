"""What the operators of a step that verifies drafted tokens refuse, before anything is launched (no device is needed)."""
import pytest
import torch

from ai_engine_b200.cache import step_tables
from ai_engine_b200.kernels import ops
from ai_engine_b200.kernels.loader import KernelError, KernelUnavailable
from ai_engine_b200.sampling import verify_drafts

I32, BF16 = torch.int32, torch.bfloat16
ints = lambda *s: torch.zeros(*s, dtype=I32)


def attend(**change):
    a = dict(q=torch.zeros(6, 8, 64, dtype=BF16), k_pages=torch.zeros(5, 2, 16, 64, dtype=BF16),
             v_pages=torch.zeros(5, 2, 16, 64, dtype=BF16), q_start=ints(3), q_len=ints(3), ctx_len=ints(3), block_table=ints(3, 4),
             scale=0.1, window=0, err=ints(1))
    a.update(change)
    return ops.paged_attention_chunks(**a)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(6, 8, 64)),                                               # another dtype than the pools
    dict(q=torch.zeros(6, 7, 64, dtype=BF16)),                                   # heads that are no multiple of the key heads
    dict(q=torch.zeros(6, 8, 32, dtype=BF16)),
    dict(q=torch.zeros(6, 8, 68, dtype=BF16)[:, :, :64]),                        # heads that do not start on 16 bytes
    dict(q=torch.zeros(6 * 8 * 64 + 1, dtype=BF16)[1:].view(6, 8, 64)),
    dict(q=torch.zeros(6, 64, 8, dtype=BF16).transpose(1, 2)),
    dict(q=torch.zeros(6, 8, 12, dtype=BF16), k_pages=torch.zeros(5, 2, 16, 12, dtype=BF16), v_pages=torch.zeros(5, 2, 16, 12, dtype=BF16)),
    dict(q=torch.zeros(6, 8, 264, dtype=BF16), k_pages=torch.zeros(5, 2, 16, 264, dtype=BF16), v_pages=torch.zeros(5, 2, 16, 264, dtype=BF16)),
    dict(v_pages=torch.zeros(5, 2, 8, 64, dtype=BF16)),
    dict(k_pages=torch.zeros(5, 2, 16, 64)),
    dict(k_pages=torch.zeros(0, 2, 16, 64, dtype=BF16), v_pages=torch.zeros(0, 2, 16, 64, dtype=BF16)),
    dict(k_pages=torch.zeros(5, 16, 2, 64, dtype=BF16).transpose(1, 2)),
    dict(q_len=torch.zeros(3, dtype=torch.int64)),
    dict(ctx_len=ints(2)),
    dict(q_start=ints(6)[::2]),
    dict(block_table=ints(3, 0)),
    dict(block_table=ints(4, 3).T),
    dict(window=-1),
    dict(out=torch.zeros(6, 8, 64)),
    dict(out=torch.zeros(6, 8, 128, dtype=BF16)[:, :, :64]),
    dict(err=torch.zeros(1)),
    dict(q=torch.zeros(6, 8, 64, dtype=torch.float16), k_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float16),
         v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float16)),
])
def test_attention_refuses(change):
    with pytest.raises(KernelError):
        attend(**change)


@pytest.mark.parametrize("form", [1, 16, 18, 24])
def test_attention_refuses_forms_of_another_type(form, monkeypatch):
    monkeypatch.setattr(ops, "CHUNK_FORM", form)
    with pytest.raises(ops.KernelError, match="bfloat16 pools only"):
        attend(q=torch.zeros(6, 8, 64), k_pages=torch.zeros(5, 2, 16, 64), v_pages=torch.zeros(5, 2, 16, 64))


def write(**change):
    a = dict(k=torch.zeros(6, 2, 64), v=torch.zeros(6, 2, 64), k_pages=torch.zeros(5, 2, 16, 64, dtype=BF16),
             v_pages=torch.zeros(5, 2, 16, 64, dtype=BF16), slots=ints(6), err=ints(1))
    a.update(change)
    return ops.write_kv_slots(**a)


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(6, 3, 64)), dict(v=torch.zeros(5, 2, 64)), dict(v=torch.zeros(6, 2, 64, dtype=BF16)),
    dict(k=torch.zeros(6, 64, 2).transpose(1, 2)), dict(slots=ints(5)), dict(slots=torch.zeros(6, dtype=torch.int64)),
    dict(k=torch.zeros(6, 2, 64, dtype=torch.float16), v=torch.zeros(6, 2, 64, dtype=torch.float16)),
    dict(k_pages=torch.zeros(5, 2, 64, 16, dtype=BF16).transpose(2, 3)),
])
def test_write_refuses(change):
    with pytest.raises(KernelError):
        write(**change)


def tables(**change):
    a = dict(cached=ints(3), counts=ints(3), held=ints(3), tables=ints(3, 4), free_pages=ints(7), free_count=ints(1), page_size=16,
             num_pages=20, max_tokens=9, err=ints(1))
    a.update(change)
    return step_tables(**a)


@pytest.mark.parametrize("change", [
    dict(cached=ints(2)), dict(counts=torch.zeros(3, dtype=torch.int64)), dict(tables=ints(3, 0)), dict(tables=ints(4, 3).T),
    dict(free_count=ints(2)), dict(page_size=0), dict(num_pages=-1), dict(num_pages=1 << 28), dict(max_tokens=-1), dict(max_tokens=1 << 31),
    dict(held=ints(6)[::2]), dict(free_pages=ints(2, 7)),
    dict(cached=ints(4097), counts=ints(4097), held=ints(4097), tables=ints(4097, 1)),
    dict(cached=ints(0), counts=ints(0), held=ints(0), tables=ints(0, 4)),
])
def test_tables_refuse(change):
    with pytest.raises(KernelError):
        tables(**change)


def verify(**change):
    a = dict(target_probs=torch.zeros(9, 50), q_start=ints(3), draft_tokens=ints(3, 2), draft_len=ints(3), draft_probs=torch.zeros(3, 2, 50),
             accept_draws=torch.zeros(3, 2), token_draws=torch.zeros(3), err=ints(1))
    a.update(change)
    return verify_drafts(**a)


@pytest.mark.parametrize("change", [
    dict(target_probs=torch.zeros(9, 50, dtype=BF16)), dict(draft_probs=torch.zeros(3, 2, 49)), dict(draft_tokens=torch.zeros(3, 2)),
    dict(draft_len=ints(2)), dict(accept_draws=torch.zeros(3, 3)), dict(accept_draws=torch.zeros(3, 4)[:, ::2]), dict(token_draws=torch.zeros(3, 1)),
    dict(target_probs=torch.zeros(50, 9).T), dict(target_probs=torch.zeros(9, 0)), dict(q_start=ints(4)),
    dict(target_probs=torch.zeros(1, 1).expand(9, (1 << 20) + 1), draft_probs=None),
])
def test_verification_refuses(change):
    with pytest.raises(KernelError):
        verify(**change)


@pytest.mark.skipif(torch.cuda.is_available(), reason="without a device")
@pytest.mark.parametrize("call", [attend, write, tables, verify])
def test_without_a_device_nothing_runs(call):
    with pytest.raises(KernelUnavailable):
        call()


@pytest.mark.gpu
@pytest.mark.parametrize("call", [attend, write, tables, verify])
def test_operands_of_the_host_are_refused(call):
    with pytest.raises(KernelError):
        call()
