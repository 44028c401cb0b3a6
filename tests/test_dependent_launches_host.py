"""Kernels that may start while the launch before them drains (``launch_dependent``): what
their sources must keep to, read without a GPU.

Such a kernel's lifetime begins before the earlier launch has written its results. A
non-coherent load (``__ldg``) promises that the data is read-only for that whole lifetime and
is not ordered by the wait, so nothing that follows ``grid_dependency_wait()`` in the kernel's
body may use one.

A launch after it waits for its end alone, so that end must not come before the earlier
launch's: every block waits, and none returns before.
"""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "ascendc_kernel_b200", "csrc")


def dependent_kernels():
    """(name, body) of every kernel that waits for the launch before it."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__[^;{]*?(\w+_kernel)\s*\(", text):
            at = text.index("{", m.end())
            depth, end = 1, at + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            body = text[at:end]
            if "grid_dependency_wait()" in body:
                found.append((m.group(1), body))
    return found


def test_the_dependent_kernels_are_found():
    assert {n for n, _ in dependent_kernels()} == {"paged_join_kernel", "paged_weights_kernel",
                                                   "evict_copy_kernel"}


@pytest.mark.parametrize("name,body", dependent_kernels(), ids=lambda x: x if len(x) < 40 else "")
def test_no_read_only_loads_after_the_wait(name, body):
    assert "__ldg" not in body.split("grid_dependency_wait()", 1)[1], name


@pytest.mark.parametrize("name,body", dependent_kernels(), ids=lambda x: x if len(x) < 40 else "")
def test_no_block_leaves_before_the_wait(name, body):
    # returns of lambdas (`-> type {`) belong to the lambda
    before = re.sub(r"->[^{;]*\{[^}]*\}", "", body.split("grid_dependency_wait()", 1)[0])
    assert not re.search(r"\breturn\b", before), name
