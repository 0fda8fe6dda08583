"""The kernels on 8-bit floating point weights load LDS stages by DMA, which the compiler's own waits do not see: a
barrier after which a stage is loaded again has to wait for this wave's loads (vmcnt) and for its reads of that stage
(lgkmcnt(0)) in the same statement, since nothing else keeps the reads' waits before it."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "decisive_amd" / "csrc"


@pytest.mark.parametrize("name,barriers", [("fp8.hip", 1), ("moe.hip", 2)])
def test_barriers_between_stages_wait_for_loads_and_reads(name, barriers):
    source = (CSRC / name).read_text()
    found = [a for a in re.findall(r"asm volatile\(\s*((?:\"[^\"]*\"\s*)+)", source) if "s_barrier" in a]
    assert len(found) >= barriers
    for text in found:
        wait = text.split("s_barrier")[0]
        assert re.search(r"vmcnt\((%0|0)\)", wait) and "lgkmcnt(0)" in wait, text
