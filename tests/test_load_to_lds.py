"""Loads to LDS take their place from M0, which they may read one wait state behind its write at the earliest (the compiler puts an s_nop between the two; within
an asm block nobody does). Read from the sources, without a device."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "metaltile_amd", "csrc")


def _blocks(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    for m in re.finditer(r'\basm\b\s*(?:volatile)?\s*\(\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', text):
        code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', m.group(1)))
        yield [i.strip() for i in re.split(r"\\n|\\t|;", code) if i.strip()]


FILES = sorted(f for f in os.listdir(CSRC) if f.endswith((".hip", ".h")) and any("m0" in i for b in _blocks(f) for i in b))


def test_some_are_there():
    assert {"fp8_tiles.hip", "gated_delta_chunks.hip"} <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_a_wait_state_behind_m0(name):
    for block in _blocks(name):
        for i, instruction in enumerate(block):
            if re.match(r"s_\w+\s+m0\b", instruction):
                assert i + 1 == len(block) or block[i + 1].startswith("s_nop"), block
