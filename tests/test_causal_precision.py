"""What rounding costs causal attention, as a norm: errors of single roundings are independent and of either sign, so the square of
an error's norm is at most the sum of the squares of what every rounding (half a step, u = eps / 2 relative to the value) does to
the result.  Tolerance: four times the root of that sum, taken over 10^4 elements and more."""
import math

import pytest
import torch

from tests.test_causal import algo, make, step  # noqa: F401 (algo: fixture)

gpu = pytest.mark.gpu


def gradients_and_noise(q, k, v, d_o, scale):
    """One head, fp16 [n, D], [m, D]: the gradients in 64 bits and the squares of what their roundings do to each element.
    P is rounded in the forward (against V: the error of O, which Delta has) and for dV, dS for dQ and dK, and the results; half a
    step of a result below 2^-14 is 2^-25."""
    u = torch.finfo(torch.float16).eps / 2
    q, k, v, d_o = (t.double().cpu() for t in (q, k, v, d_o))
    seen = torch.ones(q.shape[0], k.shape[0], dtype=torch.bool).tril(k.shape[0] - q.shape[0])
    p = torch.softmax((q @ k.T * scale).masked_fill(~seen, -math.inf), -1)
    dp = d_o @ v.T
    ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
    delta2 = ((u * p * dp) ** 2).sum(1, keepdim=True)
    value = dict(dq=ds @ k, dk=ds.T @ q, dv=p.T @ d_o)
    noise = dict(dq=(u * ds) ** 2 @ k ** 2 + delta2 * scale ** 2 * (p @ k) ** 2,
                 dk=((u * ds) ** 2 + delta2 * (scale * p) ** 2).T @ q ** 2,
                 dv=((u * p) ** 2).T @ d_o ** 2)
    return value, {n: x + (u * value[n].abs()).clamp(min=2.0 ** -25) ** 2 for n, x in noise.items()}


@gpu
@pytest.mark.parametrize("d_scale,v_scale", [(1e-3, 1.0), (1e-4, 1.0), (200.0, 20.0), (1e-3, 2e-3), (30.0, 1e-3)])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_gradients_of_any_size(D, d_scale, v_scale, algo):  # noqa: F811
    """P and dS are far below 1 over thousands of keys, and dS has the size of dO times that of V: neither may fall below what fp16
    holds, nor rise above it, where the gradients themselves do not."""
    (q, k, v, d_o), (cu_q, cu_k), _ = make([(700, 4000)], 2, 1, D, "fp16", seed=41)
    v, d_o = (v * v_scale).contiguous(), (d_o * d_scale).contiguous()
    got = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    value, noise = {}, {}
    for h in range(2):
        for d, x in zip((value, noise), gradients_and_noise(q[:, h], k[:, 0], v[:, 0], d_o[:, h], D ** -0.5)):
            for n, t in x.items():
                if n == "dq":
                    d.setdefault(n, []).append(t)
                else:
                    d[n] = d.get(n, 0) + t
    for n in ("dq", "dk", "dv"):
        want = torch.stack(value[n], 1) if n == "dq" else value[n][:, None]
        bound = 4 * math.sqrt(float(sum(noise[n]).sum() if n == "dq" else noise[n].sum()))
        off = float((got[n].double().cpu() - want).norm())
        assert off <= bound, (n, off / float(want.norm()), bound / float(want.norm()))


@gpu
@pytest.mark.parametrize("packed", [True, False])
def test_fp16_gradients_do_not_depend_on_other_sequences(packed, algo):  # noqa: F811
    """... whatever the size of the values of its neighbours in the batch is."""
    ts, (cu_q, cu_k), _ = make([(300, 300)] * 3, 2, 1, 64, "fp16", seed=42)
    q, k, v, d_o = ts if packed else [t.view(3, 300, *t.shape[1:]) for t in ts]
    kw = dict(cu_q=cu_q, cu_k=cu_k) if packed else {}
    middle = lambda t: t[300:600] if packed else t[1]
    one = {n: middle(t).clone() for n, t in step(q, k, v, d_o, **kw).items() if n != "lse"}
    for t in (ts[2], ts[3]):
        t[:300] *= 100
        t[600:] *= 1e-3
    ts[3][700] = math.inf
    ts[2][50] = math.nan
    two = step(q, k, v, d_o, **kw)
    for n in one:
        assert torch.equal(one[n], middle(two[n])), n


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_gradients_at_huge_scores(D, algo):  # noqa: F811
    """Scores of some 10^6, which 32 bits hold to a unit or so: P may come out above 1, and nothing overflows for it."""
    (q, k, v, d_o), (cu_q, cu_k), _ = make([(300, 300)], 2, 1, D, "fp16", seed=44, spread=1.0)
    q, k = q * 700, k * 700
    got = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    assert float((q.float()[:, 0] @ k.float()[:, 0].T).abs().max()) * D ** -0.5 > 1e6
    assert all(torch.isfinite(t).all() for t in got.values())
