"""Batches whose rows (16 bytes a request) take about as much shared memory as a kernel gets without asking for more, 48 KB with what the
kernel has besides, in a process of their own: what a kernel was once told about its shared memory stays."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

PROGRAM = """
import sys
sys.path[:0] = [{here!r}, {root!r}]
from draft_helpers import plain_tables
from test_step_tables_gpu import batch, call
for W in {widths}:
    for R in (3055, 3056, 3064, 3071, 3100, 4096):
        cached, counts, held, table, free, n_pages = batch(R, 16, W, R + W)
        want = plain_tables(cached, counts, held, table, free, len(free) // 20, 16, sum(counts))
        got, word = call(cached, counts, held, table, free, len(free) // 20, 16, n_pages, sum(counts))
        assert word == 0 and [x.tolist() for x in got] == list(want), (R, W)
"""


@pytest.mark.parametrize("widths", [(4,), (5,), (8, 7)])
def test_batches_around_the_shared_memory_that_needs_no_asking(widths):
    text = PROGRAM.format(here=HERE, root=os.path.dirname(HERE), widths=widths)
    r = subprocess.run([sys.executable, "-c", text], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
