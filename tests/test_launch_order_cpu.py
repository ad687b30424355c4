"""Kernels that may start while the one before them still runs, as their sources stand."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "csrc"
WAIT, KERNEL = "wait_for_launch_before();", re.compile(r"__global__ void (?:__launch_bounds__\([^{;]*?\) )?(\w+)\(")


def _kernels():
    """(file, name, body) of the kernels that are launched behind others."""
    for f in sorted(CSRC.glob("*.cu*")):
        text = f.read_text()
        for m in KERNEL.finditer(text):
            start = text.index("{\n", m.end())
            body = text[start:text.index("\n}\n", start)]
            if WAIT in body:
                yield pytest.param(body, id=f"{f.name}:{m.group(1)}")


KERNELS = list(_kernels())


def test_they_are_found():
    assert len(KERNELS) >= 10


@pytest.mark.parametrize("body", KERNELS)
def test_no_way_out_without_the_wait(body):
    """A block that returns before it has waited lets its kernel end before the one before it, and so lets the next kernel
    run beside that one."""
    assert not re.search(r"\breturn;", body[:body.index(WAIT)])
