"""8-bit operators and the distillation loss: what can be said of their calls without a GPU."""
import pytest
import torch

from geo_b200 import functional as F, layers, train


def i8(*shape):
    return torch.zeros(*shape, dtype=torch.int8)


def test_kernels_launched_ahead_read_by_plain_loads():
    """A kernel that is launched while the one in front of it still writes reads nothing through the read-only path, which is
    promised only for memory that nobody writes as long as the kernel lives (nor may such a load be kept behind the wait)."""
    import os
    import re

    csrc = os.path.join(os.path.dirname(os.path.abspath(layers.__file__)), "csrc")
    ahead = []
    for name in sorted(os.listdir(csrc)):
        with open(os.path.join(csrc, name)) as f:
            code = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
        if "launch_behind(" in code:
            ahead.append(name)
            assert not re.search(r"\b__ldg\b|ld\.global\.nc|\b__restrict__\b", code), name
    assert {"sc_norm_int8.cu", "sc_linear_int8.cu", "sc_linear_int8_tc.cu", "sc_distill.cu"} <= set(ahead)
