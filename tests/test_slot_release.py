"""Shared-memory slots are given back through mbar_arrive_loaded, whose arrive depends on the loads: an asm statement
without an instruction, the other way this was once tried, orders nothing in the machine code.  Read from the sources."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "blackwell-inference-server_b200" / "csrc"


@pytest.mark.parametrize("path", sorted(CSRC.glob("*.cu*")), ids=lambda p: p.name)
def test_no_empty_asm(path):
    assert not re.findall(r'asm\s+(?:volatile\s*)?\(\s*""', path.read_text())


@pytest.mark.parametrize("file,barriers", [("gemm.cu", ["empty"]), ("lora.cu", ["empty"]),
                                           ("tree_attention.cu", ["kempty", "vempty"])])
def test_slots_that_are_read_into_registers(file, barriers):
    text = (CSRC / file).read_text()
    for b in barriers:
        assert re.search(rf"mbar_arrive_loaded\(&{b}\[\w+\],", text) and not re.search(rf"mbar_arrive\(&{b}\[", text), b
