"""What a kernel that starts while its predecessor still runs has to keep to beyond waiting for it, looked up in the sources."""

import re

import pytest

from test_kernel_launches_cpu import CSRC, KERNEL, _body

SOURCES = sorted(path.name for path in CSRC.glob("kernels_*.cu"))


def dependent_kernels(source):
    """(name, parameters, body) of every kernel that holds the dependency wait."""
    text = (CSRC / source).read_text()
    for match in KERNEL.finditer(text):
        body = _body(text, match.end())
        if "grid_dependency_wait()" in body:
            yield match.group(1), text[match.end() : text.index("{", match.end())], body


@pytest.mark.parametrize("source", SOURCES)
def test_tensor_memory_is_held_before_the_next_kernel_may_start(source):
    """The next kernel's CTA on the same multiprocessor may allocate tensor memory, too, and keeps it while it waits for this kernel: if that
    came first, either would wait for the other for good."""
    for name, _, body in dependent_kernels(source):
        if "tcgen05.alloc" in body:
            assert body.index("grid_launch_dependents()") > body.index("tcgen05.alloc"), f"{source}: {name}"
