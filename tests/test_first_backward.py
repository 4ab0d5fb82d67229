"""The first backward pass of a process runs on a thread of autograd's that has made no CUDA call: it takes the kernels that every
later one takes."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
import torch
import simplical_attn_b200 as sab
g = torch.Generator().manual_seed(0)
t = lambda h: torch.randn(1, 200, h, 64, generator=g).cuda().bfloat16().requires_grad_()
ts, d = {tensors}, t(4).detach()
small = [torch.empty(64, device="cuda") for _ in range(8)]          # (the allocator has memory at hand)
large = [torch.empty(8 << 20, device="cuda") for _ in range(8)]
del small, large
o = {call}
torch.cuda.synchronize()
grads = [torch.autograd.grad(o, ts, d, retain_graph=True) for _ in range(3)]
for i in (0, 1):
    for a, b in zip(grads[i], grads[2]):
        assert torch.equal(a, b), ("a later pass differs from number", i, float((a.float() - b.float()).abs().max()))
"""
CALLS = {"causal": ("[t(4), t(2), t(2)]", "sab.causal_attention(*ts)"),
         "simplicial": ("[t(4), t(2), t(2), t(2), t(2)]", "sab.two_simplicial_attention(*ts, 32, 16)")}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CALLS))
def test_first_backward_of_a_process(name):
    tensors, call = CALLS[name]
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(tensors=tensors, call=call)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
