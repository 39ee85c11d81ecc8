"""Outputs and scratch that do not fit raise what torch's own operators raise, so that a program which makes room and tries again can."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)


def tables():
    from ai_engine_b200.cache import step_tables

    a = ints(3), ints(3), ints(3), ints(3, 4), ints(7), ints(1)
    return lambda: step_tables(*a, 16, 20, 1 << 28, ints_ready)


def attention():
    from ai_engine_b200.kernels import ops

    q = torch.zeros(1 << 17, 32, 128, dtype=torch.bfloat16, device=DEV)
    pool = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16, device=DEV)
    a = ints(2), ints(2), ints(2), ints(2, 4)
    return lambda: ops.paged_attention_chunks(q, pool, pool, *a, 0.1, 0, ints_ready)


@pytest.mark.parametrize("make", [tables, attention])
def test_what_does_not_fit_is_out_of_memory(make):
    global ints_ready
    torch.cuda.empty_cache()                  # (no segment with room left over from before)
    ints_ready = ints(1)
    call = make()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    call()
    assert int(ints_ready) == 0
