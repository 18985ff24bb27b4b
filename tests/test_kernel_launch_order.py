"""Tensor memory and programmatic launches, read from the kernels' source."""
import re

import pytest

from test_kernel_sources import KERNELS

TENSOR_MEMORY = sorted(k for k, (_, body) in KERNELS.items() if re.search(r"\btmem_alloc\w*\(", body))


def test_the_kernels_are_found():
    assert "kv4_prefill_kernel" in TENSOR_MEMORY and len(TENSOR_MEMORY) >= 4


@pytest.mark.parametrize("kernel", TENSOR_MEMORY)
def test_tensor_memory_is_taken_before_the_next_kernel_may_start(kernel):
    """A kernel that starts early and takes tensor memory holds it until the kernels before it are done: had it come first on an
    SM, those could not take theirs.  So a kernel asks for its own before it lets others start."""
    body = KERNELS[kernel][1]
    starts = body.find("grid_dep_launch_dependents")
    assert starts < 0 or re.search(r"\btmem_alloc\w*\(", body).start() < starts
