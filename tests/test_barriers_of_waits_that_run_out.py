"""Softmax warps and the warp that issues their products meet at named barriers without a limit.  A hardware barrier counts arrivals, not
who comes: a warp that gave up its bounded wait and then arrives for step after step without waiting fills barriers for the others, and
the issuing warp waits for ever at a later one.  The protocol is searched through on the CPU, every order of moves with every warp
giving up wherever it may, and the sources are read for the form of it that they use."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ai-engine_b200", "csrc")


def stuck_or_mixed(bars, ahead, gave_up_waits, warps=3, steps=5):
    """Whether some order of moves ends with a warp that waits for ever, or with a barrier filled by arrivals that are not one of each warp
    for one step.  Step j is handed over at barrier j % bars; its scores are announced behind the barrier of step j - ahead (ahead 1), or
    one earlier (ahead 2).  A softmax warp: (next step, may still wait for scores, waits at a barrier); the issuing warp: (next step, may
    still announce, announced, waits at its barrier); of each barrier what arrived."""
    everyone = warps + 1
    first = (tuple((0, True, False) for _ in range(warps)), (0, True, min(ahead, steps), False), tuple(() for _ in range(bars)))
    seen, todo = {first}, [first]

    def arrive(barriers, b, who):
        """(barriers, barrier is over, its arrivals are sound)"""
        here = barriers[b] + (who,)
        over = len(here) == everyone
        sound = not over or ({w for w, _ in here} == set(range(everyone)) and len({j for _, j in here}) == 1)
        return barriers[:b] + (() if over else tuple(sorted(here)),) + barriers[b + 1:], over, sound

    def released(soft, issue, b):
        """Everyone who waits at barrier b goes on."""
        soft = tuple((j + 1, ok, False) if waits and j % bars == b else (j, ok, waits) for j, ok, waits in soft)
        j, ok, told, waits = issue
        if waits and j % bars == b:
            issue = (j + 1, ok, min(steps, max(told, j + 1 + ahead)) if ok else told, False)
        return soft, issue

    while todo:
        soft, issue, barriers = todo.pop()
        nexts = []
        j, ok, told, waits = issue
        if not waits and j < steps:
            after, over, sound = arrive(barriers, j % bars, (warps, j))
            if not sound:
                return True
            nexts.append((*(released(soft, (j, ok, told, True), j % bars) if over else (soft, (j, ok, told, True))), after))
            if ok:
                nexts.append((soft, (j, False, told, False), barriers))
        for w, (i, fine, at_barrier) in enumerate(soft):
            if at_barrier or i >= steps:
                continue
            put = lambda x: soft[:w] + (x,) + soft[w + 1:]
            if fine:
                nexts.append((put((i, False, False)), issue, barriers))          # the wait runs out
                if i >= told:
                    continue
            after, over, sound = arrive(barriers, i % bars, (w, i))
            if not sound:
                return True
            new = put((i, fine, True) if not fine and gave_up_waits else (i + 1, fine, False))
            nexts.append((*(released(new, issue, i % bars) if over else (new, issue)), after))
        if not nexts and (issue[0] < steps or any(i < steps for i, _, _ in soft)):
            return True
        for s in nexts:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return False


def test_the_search_finds_what_is_wrong_with_arriving_without_waiting():
    assert stuck_or_mixed(1, 1, False) and stuck_or_mixed(2, 1, False) and stuck_or_mixed(2, 2, False)
    assert stuck_or_mixed(1, 1, True)               # waiting alone does not do: it may have arrived for the step before
    assert stuck_or_mixed(2, 2, True)
    assert not stuck_or_mixed(2, 1, True) and not stuck_or_mixed(3, 2, True)


# source, constant with the number of barriers that a stream's steps take turns at, how many steps ahead scores are announced
KERNELS = [("attention_chunks_tc.cu", "CT_BARS", 1), ("attention_prefill_tc.cu", "AT_BARS", 2), ("attention_prefill_tc.cu", "AT2_BARS", 1)]


@pytest.mark.parametrize("name,constant,ahead", KERNELS)
def test_kernels_hand_over_in_a_way_that_always_ends(name, constant, ahead):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    with open(os.path.join(CSRC, "tc_rows.cuh")) as f:
        helper = re.search(r"void tc_hand_over\(.*?\n}", f.read(), re.S)
    waits = "bar.arrive" not in text and 'else asm volatile("bar.sync' in helper.group(0)
    bars = re.search(rf"#define {constant} (\d)", text)
    assert not stuck_or_mixed(int(bars.group(1)) if bars else 1, ahead, waits)
