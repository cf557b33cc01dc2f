"""Kernels that start while their predecessor ends, read as source: a kernel lets its successor start only
once it holds its own TMEM. An allocation waits without a limit; a successor that takes TMEM before it waits
for its predecessor could otherwise keep the columns that the predecessor still has to get."""

import re

import pytest

from conftest import REPO

CSRC = REPO / "iris-3b-metal_b200" / "csrc"
ALLOCATES = re.compile(r"\btmem_alloc(?:_pair)?\([^;]*\);")


def functions(text):
    """Bodies of the functions of a source file (blocks behind a parameter list, outside of any other)."""
    text = re.sub(r"//[^\n]*", "", text)
    at = 0
    while (found := re.compile(r"\)\s*\{").search(text, at)) is not None:
        depth, end = 1, found.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield text[found.end() : end]
        at = end


def kernels():
    for path in sorted(CSRC.glob("*.cu")):
        for i, body in enumerate(functions(path.read_text())):
            if ALLOCATES.search(body):
                yield pytest.param(body, id=f"{path.stem}-{i}")


def test_there_are_such_kernels():
    assert sum("grid_wait()" in p.values[0] for p in kernels()) >= 5


@pytest.mark.parametrize("body", list(kernels()))
def test_tmem_is_held_before_a_successor_may_start(body):
    triggers = [m.start() for m in re.finditer(r"\bgrid_trigger\(\);", body)]
    waits = [m.start() for m in re.finditer(r"\bgrid_wait\(\);", body)]
    if not triggers:
        return  # its successor starts when it has ended
    allocations = list(ALLOCATES.finditer(body))
    assert len(triggers) == len(waits) == len(allocations) == 1
    # the wait, the allocation, and directly behind it, so by the same warp alone, the trigger
    allocation = allocations[0]
    assert waits[0] < allocation.start() < triggers[0]
    assert body[allocation.end() : triggers[0]].strip() == ""
    if re.search(r"if \([^()]*\) $", body[: allocation.start()]):
        raise AssertionError("the condition of the allocation does not hold for the trigger")
