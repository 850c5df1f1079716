"""Properties of the kernel sources that no run shows reliably."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "visionhope_b200" / "csrc"
# What starts, groups or awaits copies that run behind the thread's own accesses, and the waits of
# dependent launches.
ORDERED = re.compile(r"cp\.async|griddepcontrol\.wait|mbarrier\.try_wait")


def _statements():
    for path in sorted(CSRC.glob("*.cu*")):
        for m in re.finditer(r"\basm\b[^;]*?\((?:[^;\"]|\"(?:[^\"\\]|\\.)*\")*\)\s*;", path.read_text()):
            if ORDERED.search(m.group(0)):
                yield pytest.param(m.group(0), id=f"{path.name}:{path.read_text()[:m.start()].count(chr(10)) + 1}")


@pytest.mark.parametrize("statement", list(_statements()))
def test_asynchronous_copies_and_waits_order_memory(statement):
    """Without the clobber the compiler may move a plain shared-memory load above the wait for the
    copy that it reads, or below the copy that overwrites what it reads."""
    assert re.search(r'volatile\b', statement) and re.search(r':[^:"]*"memory"', statement), statement
