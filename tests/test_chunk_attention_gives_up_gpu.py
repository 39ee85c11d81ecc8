"""Attention of new tokens on tcgen05 when a copy never completes: every role's bounded wait runs out, the kernel returns with its error
bit, and the next call is as any other."""
import ctypes
import hashlib
import os

import pytest
import torch

from draft_helpers import paged_batch
from test_attention_chunks_gpu import call, check

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
NAME = "aie_attention_chunks_tc"


@pytest.mark.parametrize("stray", [0, 1, 5])
@pytest.mark.parametrize("cached,new,d", [([6000] * 8, [70] * 8, 128), ([3000, 2500] * 8, [4] * 16, 64), ([9000, 900, 20000, 0], [70, 3, 40, 130], 128)])
def test_a_tile_that_never_comes(stray, cached, new, d, monkeypatch):
    from ai_engine_b200.csrc.build import CSRC, cuda_library
    from ai_engine_b200.kernels import ops

    monkeypatch.setattr(ops, "CHUNK_FORM", 1)
    b = paged_batch(cached, new, 16, 4, d, 16, torch.bfloat16, stray + d)
    want = check(b, torch.bfloat16)
    with open(os.path.join(CSRC, "attention_chunks_tc.cu"), "rb") as f:      # (a source that another includes is not in its key)
        key = hashlib.sha256(f.read()).hexdigest()[:8]
    lib = ctypes.CDLL(cuda_library(os.path.join(HERE, "chunk_attention_gives_up.cu"), [f"-DSOURCE_KEY=0x{key}", f"-DCT_STRAY={stray}"]))
    address = lambda x: ctypes.cast(getattr(x, NAME), ctypes.c_void_p).value
    ops.draft_ops().set_launcher(NAME, address(lib))
    try:
        _, word = call(b)
    finally:
        ops.draft_ops().set_launcher(NAME, address(ops.library("attention_chunks_tc.cu")))
    assert word == 4
    out, word = call(b)
    assert word == 0 and torch.equal(out, want)
