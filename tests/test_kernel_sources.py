"""What the sources of kernels that start beside the one before them may not do, as no run can show it."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "hive-limited_b200" / "csrc"
CALL_WRITES = r"\b(part|ml|stretches|stat|scores|terms|facs)\b"     # in a call's scratch


def arguments(text, name):
    """Of every call of `name` in the text, what stands between its parentheses."""
    for m in re.finditer(rf"\b{name}\(", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        yield text[m.end():i - 1]


@pytest.mark.parametrize("name", ["k_shared.cu", "k_span_tile.cu", "k_mass_tile.cu"])
def test_results_of_the_kernel_before_are_not_read_as_constants(name):
    found = list(arguments((CSRC / name).read_text(), "__ldg"))
    assert found
    for arg in found:
        assert not re.search(CALL_WRITES, arg), arg


def test_bounded_waits_begin_after_the_kernel_before():
    """The limit of a wait on a barrier is for this kernel's work: no role counts the time that the
    kernel before it still takes."""
    text = (CSRC / "k_mass_tile.cu").read_text()
    starts = [text.index(x) for x in ("if (warp < 16) {", "} else if (warp == 16) {", "} else if (lane == 0) {")]
    for lo, hi in zip(starts, starts[1:] + [text.index("tcgen05.dealloc")]):
        role = text[lo:hi]
        assert "bar_wait" in role and 0 < role.find("prior_done();") < role.index("bar_wait")
