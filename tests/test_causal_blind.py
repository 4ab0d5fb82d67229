"""Causal attention with more queries than keys: the rows that see no key."""
import math

import pytest
import torch

from tests.test_causal import algo, make, step  # noqa: F401 (algo: fixture)

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "fp16"), (128, "bf16"), (64, "fp16"), (40, "fp32")])
def test_queries_that_see_nothing_take_part_in_no_gradient(D, dtype, algo):  # noqa: F811
    """More queries than keys: whatever lies in the rows of Q and dO that see no key, the other rows' results are what they were, and
    such a row's gradient is zero whatever lies in K and V."""
    lens = [(300, 100), (129, 127), (400, 30)]
    (q, k, v, d_o), (cu_q, cu_k), seqs = make(lens, 4, 2, D, dtype, seed=51)
    want = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    blind = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for q0, n, _, m in seqs:
        blind[q0:q0 + n - m] = True
    rows = blind.nonzero()[:, 0]
    q[rows[::2]], q[rows[1::2]] = math.nan, math.inf
    d_o[rows[::3]], d_o[rows[1::3]] = -math.inf, math.nan
    got = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    assert all(torch.equal(got[n], want[n]) for n in want), [n for n in want if not torch.equal(got[n], want[n])]
    assert not got["dq"][blind].any() and not got["o"][blind].any()
    k[0], v[110] = math.nan, math.inf          # (the first key of the first sequence, the eleventh of the second)
    got = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    assert not got["dq"][blind].any() and not got["o"][blind].any()
