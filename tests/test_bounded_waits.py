"""Waits inside the kernels: each goes through the one loop that is bounded and reports where it gave up (tests/test_gpu_status.py
lets that loop run out)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "simplical_attn_b200", "csrc")


@pytest.mark.parametrize("name", sorted(os.listdir(CSRC)))
def test_no_wait_of_its_own(name):
    """Only the shared loop looks at the clock and at the limit of a wait: a loop beside it could give up without a report."""
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    used = re.findall(r"globaltimer_ns\(\)|ctx\.limit_ns", text)
    assert not used or name == "sa_ptx.cuh", used
