"""The count of the package's own launches, which a benchmark reports, and the timers' bytes: what ran, in every form and in calls that
have nothing to do."""
import pytest
import torch

from draft_helpers import paged_batch
from test_attention_chunks_gpu import call as attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)


def launches(f):
    """(counted, kernels that the device ran)"""
    from ai_engine_b200.kernels.loader import LAUNCHES

    f()                                          # libraries are there
    torch.cuda.synchronize()
    before = LAUNCHES[0]
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        f()
    from cuda.bindings import runtime as rt
    err, _, n = rt.cudaGraphGetNodes(graph.raw_cuda_graph(), 0)
    assert int(err) == 0
    return LAUNCHES[0] - before, n


@pytest.mark.parametrize("form,dtype,count", [(0, torch.float32, 2), (0, torch.bfloat16, 2), (1, torch.bfloat16, 2), (16, torch.bfloat16, 2),
                                              (18, torch.bfloat16, 1), (20, torch.bfloat16, 1), (24, torch.bfloat16, 1)])
def test_attention(form, dtype, count, monkeypatch):
    from ai_engine_b200.kernels import ops

    monkeypatch.setattr(ops, "CHUNK_FORM", form)
    b = paged_batch([100, 30], [3, 2], 8, 2, 64, 16, dtype, 1)
    e = ints(1)
    run = lambda **more: ops.paged_attention_chunks(*(dict(b, **more)[k] for k in ("q", "k_pages", "v_pages", "q_start", "q_len", "ctx_len", "table")),
                                                    b["scale"], 0, e)
    assert launches(run) == (count, count)
    assert launches(lambda: run(q=b["q"][:0])) == (0, 0)
    assert launches(lambda: run(q_start=ints(0), q_len=ints(0), ctx_len=ints(0), table=ints(0, 7))) == (0, 0)


def test_the_others():
    from ai_engine_b200.cache import step_tables
    from ai_engine_b200.kernels import ops
    from ai_engine_b200.sampling import verify_drafts

    e, pool, p = ints(1), torch.zeros(3, 2, 4, 64, device=DEV), torch.full((4, 50), 0.02, device=DEV)
    rows, pick = torch.zeros(5, 2, 64, device=DEV), torch.zeros(2, device=DEV)
    slots, a, v = ints(5), (ints(2), ints(2), ints(2), ints(2, 4), ints(7), ints(1)), (ints(2), ints(2, 1), ints(2), torch.zeros(2, 1, device=DEV))
    assert launches(lambda: ops.write_kv_slots(rows, rows, pool, pool, slots, e)) == (1, 1)
    assert launches(lambda: ops.write_kv_slots(rows[:0], rows[:0], pool, pool, slots[:0], e)) == (0, 0)
    assert launches(lambda: step_tables(*a, 16, 20, 9, e)) == (1, 1)
    assert launches(lambda: verify_drafts(p, v[0], v[1], v[2], None, v[3], pick, e)) == (1, 1)
    assert launches(lambda: verify_drafts(p, v[0][:0], v[1][:0], v[2][:0], None, v[3][:0], pick[:0], e)) == (0, 0)


def test_the_timers_name_no_bytes_that_only_the_device_knows():
    from ai_engine_b200.kernels import profile

    profile.start()
    try:
        attend(paged_batch([100, 30], [3, 2], 8, 2, 64, 16, torch.bfloat16, 1))
    finally:
        rows = profile.stop(6000.0, 1600.0)
    row, = (r for r in rows if r["kernel"] == "paged_attention_chunks")
    assert row["gb"] == row["frac"] == 0
