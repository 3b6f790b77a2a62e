"""How wide the kernels' loads and stores of global memory are, read from their sources: the interfaces ask for tensors, caches and pages that
begin at multiples of 16 bytes, and an access of 32 bytes needs a multiple of 32.  No GPU needed."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlsys-contest-syfi-agent-assisted_b200", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")))


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_no_access_of_global_memory_is_wider_than_its_alignment(path):
    text = open(path).read()
    for kind, count, bits in re.findall(r"\b((?:ld|st|red|atom)\.[a-z0-9_.:]*?)\.v(\d)\.[busf](\d+)", text, flags=re.I):
        assert int(count) * int(bits) <= 128, f"{kind}.v{count} of {bits} bits"
    assert not re.search(r"\b(?:double4|u?long(?:long)?4)\b", text)


def test_the_widest_access_is_found():
    """The pattern sees the loads that the chunk kernel of the 4-bit cache makes."""
    text = open(os.path.join(CSRC, "kv4_attention_chunk.cu")).read()
    assert re.findall(r"\b((?:ld|st|red|atom)\.[a-z0-9_.:]*?)\.v(\d)\.[busf](\d+)", text, flags=re.I).count(("ld.global.nc.L1::no_allocate", "4", "32")) == 2
