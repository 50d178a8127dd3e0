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


# what no kernel of the library writes once a package is mounted or a caller has laid it out: weights and tables, the layers' descriptions,
# the ranks' addresses, lists that the host has filled before the launch
CONSTANT = {"table", "weight", "norm_weight", "w", "wg", "wu", "cos_sin", "layers", "tp_pointer", "pools", "pages"}
CONSTANT_ADDRESS = re.compile(r"\b(?:weight|w|wrow|source|scales_[ab]|row_scales|embedding|rope_table)\b")


@pytest.mark.parametrize("source", SOURCES)
def test_nothing_promises_that_the_kernel_in_front_writes_nothing(source):
    """__restrict__ and __ldg say that what a pointer reads is written by nobody else while the kernel runs.  The kernel in front still does, and
    the compiler may move such an access in front of the wait for it (routes of a replayed graph were read before they were there)."""
    for name, parameters, body in dependent_kernels(source):
        promised = set(re.findall(r"__restrict__\s+(\w+)", parameters + body))
        assert promised <= CONSTANT, f"{source}: {name}: {promised - CONSTANT}"
        for address in re.findall(r"__ldg\(([^;]*)", body):
            assert CONSTANT_ADDRESS.search(address), f"{source}: {name}: __ldg({address}"
