"""Outputs and scratch that do not fit raise what torch's own operators raise, so that a program which makes room and tries again can.  In a
process of its own, whose memory holds nothing else."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

PROGRAM = """
import sys
sys.path.insert(0, {root!r})
import torch
from ai_engine_b200.cache import step_tables
from ai_engine_b200.kernels import ops
ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
e = ints(1)

def tables():
    a = ints(3), ints(3), ints(3), ints(3, 4), ints(7), ints(1)
    return lambda: step_tables(*a, 16, 20, 1 << 28, e)

def attention():
    q = torch.zeros(1 << 17, 32, 128, dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16, device="cuda")
    a = ints(2), ints(2), ints(2), ints(2, 4)
    return lambda: ops.paged_attention_chunks(q, pool, pool, *a, 0.1, 0, e)

call = {which}()
total = torch.cuda.get_device_properties(0).total_memory
torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / total)
try:
    call()
except torch.OutOfMemoryError:
    torch.cuda.set_per_process_memory_fraction(1.0)
    call()
    assert int(e) == 0
else:
    raise AssertionError("it fits")
"""


@pytest.mark.parametrize("which", ["tables", "attention"])
def test_what_does_not_fit_is_out_of_memory(which):
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(root=os.path.dirname(HERE), which=which)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
