"""Static checks of the routing and MXFP4 sources (CPU).  Their launches name kernels through variables and
templates, so every kernel they define is looked at: each starts with pdl_wait(), since all are launched
with programmatic stream serialisation, and none waits for a barrier without a time limit."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "magi-2-preview_b200" / "csrc"


def _kernels(text):
    """(name, first statement) of every __global__ definition."""
    text = re.sub(r"//[^\n]*", "", text)
    for part in text.split("__global__")[1:]:
        head, body = part.split(") {", 1)
        yield re.findall(r"\b(\w+_kernel)\s*\(", head)[0], body.strip().split(";")[0]


@pytest.mark.parametrize("source,count", [("mxfp4.cu", 2), ("mxfp4_gemm.cu", 4), ("route_experts.cu", 2)])
def test_every_kernel_waits_first(source, count):
    found = list(_kernels((CSRC / source).read_text()))
    assert len(found) == count, found
    for name, first in found:
        assert first == "pdl_wait()", (name, first)


def test_products_waits_are_bounded():
    text = re.sub(r"//[^\n]*", "", (CSRC / "mxfp4_gemm.cu").read_text())
    assert "mbarrier.try_wait" not in text and "while (true)" not in text
    for call in re.findall(r"mbar_wait\((?:[^()]|\([^()]*\))*\)", text):
        assert call.endswith("MHMOE_DRAIN_NS)"), call
