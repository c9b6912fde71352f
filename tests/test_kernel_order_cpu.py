"""An order that the kernels' sources have to keep: what cannot be shown by a run, since breaking it ends in a hang."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "ezops_b200" / "csrc"


def test_tensor_memory_is_taken_before_the_next_kernel_may_start():
    """A kernel that releases its dependent launch first can find the dependent's CTA on its SM, holding tensor memory while it waits
    for this kernel, which waits for the tensor memory."""
    kernels = 0
    for path in sorted(CSRC.glob("*.cu")):
        for body in path.read_text().split("__global__")[1:]:
            taken = re.search(r"\btmem_alloc(_pair)?\(", body)
            if taken is None:
                continue
            kernels += 1
            released = re.search(r"\bpdl_(open|trigger)\(", body)
            assert released is None or taken.start() < released.start(), path.name
    assert kernels >= 3
