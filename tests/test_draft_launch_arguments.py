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
