"""What the host side packs for a launcher and what the launcher reads are one declaration, and the scratch that the host makes is for the
grid that the launcher starts."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ai-engine_b200", "csrc")


def sources():
    for folder in (CSRC, os.path.join(CSRC, "host")):
        for name in sorted(os.listdir(folder)):
            if name.endswith((".cu", ".cuh", ".cpp", ".h", ".hpp")):
                with open(os.path.join(folder, name)) as f:
                    yield name, f.read()


def test_each_structure_is_declared_once():
    for struct in ("StArgs", "CwArgs", "VdArgs", "ChCall"):
        assert [name for name, text in sources() if re.search(rf"\bstruct {struct}\b", text)] == ["draft_args.h"]


def test_the_grid_is_the_one_that_the_scratch_was_made_for():
    for name, text in sources():
        if name.startswith("attention_chunks"):
            assert "aie_sm_count" not in text, name


def test_the_division_by_multiplication_stands_once():
    assert [name for name, text in sources() if "Granlund" in text] == ["division.cuh"]


def test_the_division_by_multiplication_is_exact():
    """(n + high half of n * mul) >> shift for n below 2^31, at the multiples of d and beside them, where a quotient changes."""
    for d in [1, 2, 3, 5, 6, 7, 10, 16, 24, 100, 127, 128, 129, 641, 1000, 65535, 65537, 2 ** 20 - 1, 2 ** 30 + 1, 2 ** 31 - 1]:
        shift = (d - 1).bit_length()
        mul = ((1 << 32) * ((1 << shift) - d) // d + 1) & 0xffffffff
        top = (2 ** 31 - 1) // d
        for q in {0, 1, 2, 3, 1000, top // 3, top // 2, top - 1, top}:
            for n in (q * d - 1, q * d, q * d + 1):
                if 0 <= n < 2 ** 31:
                    assert (n + (n * mul >> 32)) >> shift == n // d and n + (n * mul >> 32) < 2 ** 32, (n, d)
