"""The low part of causal attention's output (what the rounding of a 16-bit O took, which the backward sums dO O with)."""
import pytest
import torch

import simplical_attn_b200 as sab
from tests.test_causal import DT, make

gpu = pytest.mark.gpu


# (queries, keys) of the sequences, H, Hkv, D, dtype, bounds of the lengths, kernels
LOW = [
    ([(1500, 1500)] * 3, 16, 8, 64, "bf16", {}, "auto"),              # whole walks of pairs of query tiles
    ([(1500, 1500)] * 2, 16, 16, 128, "fp16", {}, "auto"),
    ([(300, 5000), (130, 700)], 2, 1, 128, "bf16", {}, "auto"),       # shares, joined
    ([(200, 40), (300, 299)], 2, 1, 64, "fp16", {}, "auto"),          # rows that see nothing
    ([(3, 5000), (2, 1), (4, 77)], 4, 1, 64, "bf16", dict(max_q=4, max_k=5000), "auto"),        # a few rows, shares joined by a kernel
    ([(3, 500), (2, 1), (4, 77)], 4, 1, 128, "fp16", dict(max_q=4, max_k=500), "auto"),         # ... in a cluster
    ([(1, 40)], 4, 1, 40, "bf16", dict(max_q=1, max_k=40), "auto"),                             # ... one share
    ([(300, 300)] * 4, 32, 32, 100, "bf16", {}, "auto"),              # the general kernels, whole walks
    ([(70, 3000), (9, 3)], 2, 1, 256, "fp16", {}, "auto"),            # ... shares
]


@gpu
@pytest.mark.parametrize("case", LOW)
def test_low_part_of_the_output(case):
    """O and what its rounding took, together, where nothing else is rounded: with Q = 0 every P is one, and O the mean of the rows of
    V that a query sees; V are multiples of 1/8 of at most 2, whose sums are exact in 32 bits.  Division: 2 x 2^-24.  Joined shares: an
    LSE of at most ln 5000 < 16 is off by half a step of it (2^-21) and 2^-20 of its logarithm, so a weight by less than 2^-18 with its
    own exponential, and the normalised sum by less than 2^-17 of the mean |V|.  Then two roundings, the second (u) of what the first
    one took (u |O|)."""
    lens, H, Hkv, D, dtype, kw, which = case
    (q, k, v, _), (cu_q, cu_k), seqs = make(lens, H, Hkv, D, dtype, seed=43, gap=3)
    v = (1 + (8 * v.float()).round().clamp(-8, 8) / 8).to(v.dtype)
    o, lse, low = sab.causal_attention_fwd(torch.zeros_like(q), k, v, 0.1, cu_q, cu_k, low=True, algo=which, **kw)
    u = torch.finfo(DT[dtype]).eps / 2
    vd = v.double().cpu()
    rounded = 0
    for q0, n, k0, m in seqs:
        sums, sizes = vd[k0:k0 + m].cumsum(0), vd[k0:k0 + m].abs().cumsum(0)
        see = torch.arange(n) + 1 + m - n
        live = see > 0
        at = (see.clamp(min=1) - 1)
        count = see.clamp(min=1).double()[:, None, None]
        want, size = (torch.where(live[:, None, None], x[at] / count, torch.zeros((), dtype=torch.float64)).repeat_interleave(H // Hkv, 1)
                      for x in (sums, sizes))
        got_o, got_low = (t[q0:q0 + n].double().cpu() for t in (o, low))
        bound = 2.0 ** -17 * size + 1.01 * u * u * want.abs() + (2.0 ** -25 if dtype == "fp16" else 1e-30)
        off = (got_o + got_low - want).abs()
        assert (off <= bound).all(), float((off / bound.clamp(min=1e-30)).max())
        assert not got_low[~live].any() and (got_low.abs() <= 1.01 * u * got_o.abs() + 2.0 ** -25).all()
        rounded += int((((got_o - want).abs() > bound)).sum())
    assert rounded > 0          # (O alone is farther off: the low part counts)
