"""Causal attention where a column of V holds several kinds of values that are not finite."""
import math

import pytest
import torch

import simplical_attn_b200 as sab
from tests import causal_ref
from tests.test_causal import algo, make, step  # noqa: F401 (algo: fixture)

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "fp16"), (48, "fp32")])
@pytest.mark.parametrize("B,H,N", [(1, 2, 300), (5, 32, 300)])
def test_several_kinds_in_a_column(D, dtype, B, H, N, algo):  # noqa: F811
    """An infinity does not hide the NaN or the opposite infinity of an earlier key: their sum is NaN, as in the definition."""
    (q, k, v, _), _, _ = make([(N, N)] * B, H, H, D, dtype, seed=52)
    q, k, v = (t.view(B, N, H, D) for t in (q, k, v))
    clean = sab.causal_attention(q, k, v)
    for first, value in ((3, math.nan), (7, -math.inf)):
        for d in (first, first + 20):
            v[:, 10, :, d] = value
            v[:, 270 if d == first else 100, :, d] = math.inf
    got = sab.causal_attention(q, k, v)
    for d, early, late in ((3, math.nan, 270), (23, math.nan, 100), (7, -math.inf, 270), (27, -math.inf, 100)):
        assert torch.equal(got[:, :10, :, d], clean[:, :10, :, d])
        x = got[:, 10:late, :, d]
        assert torch.isnan(x).all() if math.isnan(early) else (x == early).all(), d
        assert torch.isnan(got[:, late:, :, d]).all(), d
    keep = [d for d in range(D) if d not in (3, 23, 7, 27)]
    assert torch.equal(got[..., keep], clean[..., keep])


@gpu
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "fp16")])
def test_a_row_that_is_not_finite_stays_so(D, dtype, algo):  # noqa: F811
    """A NaN in Q makes the whole row NaN, an infinity in a column of V notwithstanding."""
    (q, k, v, _), (cu_q, cu_k), _ = make([(300, 300)], 2, 1, D, dtype, seed=53)
    q[290, :, 0] = math.nan
    v[280, :, 5] = math.inf
    got = sab.causal_attention(q, k, v, cu_q=cu_q, cu_k=cu_k)
    assert torch.isnan(got[290]).all() and (got[280:290, :, 5] == math.inf).all() and (got[291:, :, 5] == math.inf).all()


# B, N, M: whole walks of many units, shares joined by a kernel, a few rows in one share, in a cluster, in many shares
@gpu
@pytest.mark.parametrize("shape", [(5, 300, 300), (1, 130, 3000), (1, 2, 40), (1, 2, 700), (1, 2, 20000)])
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "bf16"), (64, "fp32")])
def test_scores_of_minus_infinity(shape, D, dtype, algo):  # noqa: F811
    """A query all of whose scores overflow to -inf weighs no key, as if it saw none: O = 0, LSE = -inf and no gradient, however the
    keys are cut up.  Beside finite scores such a key has weight zero."""
    B, N, M = shape
    H, Hkv = (32, 32) if B > 1 else (4, 2)
    (q, k, v, d_o), _, _ = make([(N, M)] * B, H, Hkv, D, dtype, seed=54)
    q, k, v, d_o = (t.view(B, -1, *t.shape[1:]) for t in (q, k, v, d_o))
    row = N // 2
    q, k = q.clone(), k.clone()
    k[..., 0], q[..., 0] = -1e20, 0          # (products of zero with the big elements change nothing: the other rows keep their scores)
    base = step(q, k, v, d_o)
    q[:, row, :, 0] = 1e25
    got = step(q, k, v, d_o)
    assert not got["o"][:, row].any() and (got["lse"][:, :, row] == -math.inf).all() and not got["dq"][:, row].any()
    rest = [i for i in range(N) if i != row]
    assert torch.equal(got["o"][:, rest], base["o"][:, rest]) and torch.equal(got["dq"][:, rest], base["dq"][:, rest])
    # the row takes part in no gradient: those of K and V are what they are without its dO
    d_o = d_o.clone()
    d_o[:, row] = 0
    q[:, row] = 0
    without = step(q, k, v, d_o)
    assert torch.equal(got["dv"], without["dv"]) and torch.equal(got["dk"], without["dk"])


@gpu
@pytest.mark.parametrize("N,M", [(300, 300), (130, 3000), (2, 700)])
def test_scores_of_minus_infinity_beside_others(N, M, algo):  # noqa: F811
    """The keys whose scores are -inf have weight zero, whole tiles of them before the first other one included."""
    (q, k, v, d_o), (cu_q, cu_k), _ = make([(N, M)], 2, 1, 64, "bf16", seed=55)
    row, first = N - 1, M - M // 4
    k[:, :, 0], q[:, :, 0] = 0, 0
    k[:first, :, 0] = -1e20
    q[row, :, 0] = 1e25
    got = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    val, err = causal_ref.reference(q[row:row + 1] * (torch.arange(64, device="cuda") > 0), k[first:] * (torch.arange(64, device="cuda") > 0), v[first:], None,
                                    [(0, 1, 0, M - first)], 0.125)
    causal_ref.check(got["o"][row:row + 1], val["o"], err["o"], "o")
    causal_ref.check(got["lse"][:, row:row + 1], val["lse"], err["lse"], "lse")
    assert torch.isfinite(got["dq"][:row]).all() and torch.isfinite(got["dv"]).all()
