"""Causal attention in 64 bits, sequence by sequence, with bounds of what rounding may do to every element.

u = eps / 2 of the tensors' type is the relative error of one rounding.  The kernels round the probabilities P, dS and the
results; everything else is 32-bit arithmetic, whose errors are relative to sums of absolute values:
  * a score is off by 2^-24 (D + 6) sum_d |Q K| scale, so P is off by twice that (numerator and LSE), plus n + 64 roundings for the
    sums over n keys, the approximate exponential (2^-22) and the division: P (1 + r), r = 2^-24 (2 (D + 6) A + n + 64);
  * O: P rounded to the type (u) against |V|, r against |V|, the result rounded once (u);
  * Delta = sum dO O takes O's error, weighted with |dO|;
  * dS = scale P (dP - Delta): r and Delta's error, then u for its rounding; dQ and dK take it against |K| and |Q|, dV takes P's.
fp16 has subnormals: a P below 2^-14 is off by 2^-25 absolutely, against rows whose largest P is at least 1 (the
backward's P is at most 1); a dS likewise.
"""
import math

import torch


def _sequence(q, k, v, d_o, scale, u, tiny):
    """One sequence and query head, fp64 [n, D], [m, D]: dict of values and of bounds of their errors."""
    n, m, D = q.shape[0], k.shape[0], q.shape[1]
    seen = torch.ones(n, m, dtype=torch.bool).tril(m - n)
    s = torch.where(seen, q @ k.T * scale, torch.full((), -math.inf, dtype=torch.float64))
    live = seen.any(1)
    lse = torch.logsumexp(s, 1) if m else torch.full((n,), -math.inf, dtype=torch.float64)
    p = torch.where(seen, torch.exp(s - torch.where(live, lse, torch.zeros_like(lse))[:, None]), torch.zeros((), dtype=torch.float64))
    a = torch.where(seen, q.abs() @ k.abs().T * abs(scale), torch.zeros((), dtype=torch.float64)).amax(1) if m else torch.zeros(n, dtype=torch.float64)
    r = 2.0 ** -24 * (2 * (D + 6) * a + m + 64)
    o = p @ v
    pv = p @ v.abs()
    e_o = (u + r[:, None]) * pv + u * o.abs() + tiny * (seen.double() @ v.abs())
    e_o = e_o * (1 + 2 * u) + 1e-30
    out = dict(o=o, lse=lse, e_o=e_o, e_lse=torch.where(live, r + 2.0 ** -22 * lse.abs(), torch.zeros_like(r)))
    if d_o is None:
        return out
    d_o = torch.where(live[:, None], d_o, torch.zeros((), dtype=torch.float64))
    delta = (d_o * o).sum(1)
    dp = d_o @ v.T
    ds = p * (dp - delta[:, None]) * scale
    # 32-bit sums over D in dP and Delta, and what O's rounding does to Delta
    e_dp = 2.0 ** -24 * (D + 8) * (d_o.abs() @ v.abs().T)
    e_delta = (d_o.abs() * e_o).sum(1) + 2.0 ** -24 * (D + 8) * (d_o.abs() * o.abs()).sum(1)
    e_ds = (u + r[:, None] + 2.0 ** -22) * ds.abs() + p * abs(scale) * (1 + r[:, None]) * (e_dp + e_delta[:, None])
    e_ds = torch.where(seen, e_ds + tiny * (dp - delta[:, None]).abs() * abs(scale) + tiny, torch.zeros((), dtype=torch.float64))
    e_p = torch.where(seen, (u + r[:, None]) * p + tiny, torch.zeros((), dtype=torch.float64))
    sums = 2.0 ** -24 * (n + m)
    out.update(dq=ds @ k, dk=ds.T @ q, dv=p.T @ d_o, e_dq=e_ds @ k.abs() + sums * (ds.abs() @ k.abs()),
               e_dk=e_ds.T @ q.abs() + sums * (ds.abs().T @ q.abs()), e_dv=e_p.T @ d_o.abs() + sums * (p.T @ d_o.abs()))
    return out


def reference(q, k, v, d_o, seqs, scale):
    """Packed q [T, H, D], k, v [Tk, Hkv, D] (d_o like q, or None); seqs: (q0, nq, k0, nk) of every sequence.  Returns (values,
    bounds): o, lse [H, T] and the gradients, on the CPU in fp64; rows outside the sequences are zero (LSE -inf)."""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    d_o = None if d_o is None else d_o.double().cpu()
    T, H, D = q.shape
    G = H // k.shape[1]
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64)
    val = dict(o=z(q), lse=torch.full((H, T), -math.inf, dtype=torch.float64))
    err = dict(o=z(q), lse=torch.zeros(H, T, dtype=torch.float64))
    if d_o is not None:
        for d in (val, err):
            d.update(dq=z(q), dk=z(k), dv=z(v))
    for q0, nq, k0, nk in seqs:
        for h in range(H):
            rq, rk = slice(q0, q0 + nq), slice(k0, k0 + nk)
            x = _sequence(q[rq, h], k[rk, h // G], v[rk, h // G], None if d_o is None else d_o[rq, h], scale, u, tiny)
            val["o"][rq, h], err["o"][rq, h] = x["o"], x["e_o"]
            val["lse"][h, rq], err["lse"][h, rq] = x["lse"], x["e_lse"]
            if d_o is not None:
                val["dq"][rq, h], err["dq"][rq, h] = x["dq"], x["e_dq"]
                for n in ("dk", "dv"):
                    val[n][rk, h // G] += x[n]
                    err[n][rk, h // G] += x["e_" + n]
    if d_o is not None:          # the result's own rounding
        for n in ("dq", "dk", "dv"):
            err[n] = err[n] * (1 + u) + u * val[n].abs() + (2.0 ** -25 if tiny else 1e-30)
    if tiny:
        err["o"] += 2.0 ** -25
    return val, err


def check(got, val, err, name):
    got = got.detach().double().cpu()
    assert got.shape == val.shape, (name, got.shape, val.shape)
    inf = torch.isinf(val)
    assert torch.equal(got[inf], val[inf]), f"{name}: rows that see nothing"
    bad = ~((got - val).abs() <= err) & ~inf
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside the bound; worst by a factor "
                           f"{float(((got - val).abs() / err.clamp(min=1e-300))[bad].max()):.2f}, first at {bad.nonzero()[0].tolist()}: "
                           f"{float(got[bad][0])} for {float(val[bad][0])} within {float(err[bad][0]):.3g}")
