"""Causal attention where blocks of the tensor-core kernels take several units: the barriers' phases, the rings and what a unit leaves
behind are handed on from one to the next.  Values against the definition in 64 bits (tests/causal_ref.py has the bounds)."""
import ctypes
import math

import pytest
import torch

import simplical_attn_b200 as sab
from simplical_attn_b200 import _abi
from tests import causal_ref
from tests.test_causal import compare, make, step

gpu = pytest.mark.gpu


def tiles(n):
    return -(-n // 128)


def check_plan(lens, H, Hkv, D, dtype, packed, shares=False, max_q=0, max_k=0):
    """That all three kernels have more units than there are multiprocessors, and whether their walks are cut into shares, by the
    size of the workspaces: shares have partial rows there, and a packed batch a list of 32 bytes for every tile."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    lib = _abi.load()
    p = _abi.CausalParams()
    Tq, Tk = sum(n for n, _ in lens), sum(m for _, m in lens)
    p.B, p.Nq, p.Nk = (1, Tq, Tk) if packed else (len(lens), *lens[0])
    p.H, p.Hkv, p.D, p.scale = H, Hkv, D, 0.1
    p.sequences, p.max_q, p.max_k = len(lens) if packed else 0, max_q, max_k
    p.dtype = _abi.SA_F16 if dtype == "fp16" else _abi.SA_BF16
    for n, h in (("q", H), ("k", Hkv), ("v", Hkv), ("o", H), ("d_o", H), ("dq", H), ("dk", Hkv), ("dv", Hkv)):
        setattr(p, n, _abi.Strides((p.Nq if h == H else p.Nk) * h * D, h * D, D))
    forward, backward = lib.sa_causal_forward_workspace_size(ctypes.byref(p)), lib.sa_causal_backward_workspace_size(ctypes.byref(p))
    # (the least that two shares' partial rows take; without them there are Delta, lists and a few numbers for each sequence)
    part = 2 * min(Tq * H, Tk * Hkv) * 64 * 4
    assert (forward >= part) == shares and (shares or backward < part), (forward, backward, part)
    queries, keys, pairs = (sum(x) for x in zip(*((tiles(n), tiles(m), tiles(-(-n // 2))) for n, m in lens)))
    cut = forward // (Tq * H * (64 if D <= 64 else 128) * 4) if shares else 1
    assert cut * pairs * H > sms and keys * Hkv > sms and (shares or queries * H > sms)
    if packed and not shares:        # pairs of query tiles
        assert forward <= 32 * (Tq // 256 + len(lens) + 1) + 256


# lengths, H, Hkv, D, dtype, packed, shares of the forward's walks, K/V heads that are compared (None: all)
CASES = [
    ([(1500, 1500)] * 3, 16, 8, 64, "bf16", False, False, None),
    ([(1500, 1500), (700, 700), (1300, 1300), (333, 333), (1100, 1100)], 16, 8, 128, "fp16", True, False, None),
    ([(1500, 1500), (700, 900), (1300, 1001), (333, 333), (1100, 1100)], 16, 16, 64, "fp16", True, False, (0, 7, 15)),
    ([(1300, 2000)] * 2, 16, 16, 128, "bf16", False, False, (0, 6, 15)),
    ([(1280, 8192)], 10, 5, 64, "bf16", False, True, (0, 4)),
]


@pytest.mark.parametrize("case", CASES)
def test_cases_have_several_units_for_a_block(case):
    lens, H, Hkv, D, dtype, packed, shares, _ = case
    check_plan(lens, H, Hkv, D, dtype, packed, shares)


@gpu
@pytest.mark.parametrize("case", CASES)
def test_several_units_for_a_block(case):
    lens, H, Hkv, D, dtype, packed, shares, some = case
    check_plan(lens, H, Hkv, D, dtype, packed, shares)
    (q, k, v, d_o), (cu_q, cu_k), seqs = make(lens, H, Hkv, D, dtype, seed=31)
    if packed:
        got = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    else:
        got = step(*(t.view(len(lens), -1, *t.shape[1:]) for t in (q, k, v, d_o)))
        got["lse"] = got["lse"].transpose(0, 1).reshape(H, -1)
        got = {n: t if n == "lse" else t.reshape(-1, *t.shape[2:]) for n, t in got.items()}
    G = H // Hkv
    for hk in range(Hkv) if some is None else some:
        hs, ks = slice(hk * G, hk * G + G), slice(hk, hk + 1)
        ref = causal_ref.reference(q[:, hs], k[:, ks], v[:, ks], d_o[:, hs], seqs, D ** -0.5)
        compare({n: t[hs] if n == "lse" else t[:, ks] if n in ("dk", "dv") else t[:, hs] for n, t in got.items()}, ref)
    sab.check_device_status()


@gpu
@pytest.mark.parametrize("D,dtype,packed", [(64, "bf16", False), (128, "fp16", False), (128, "bf16", True), (64, "fp16", True)])
def test_values_that_are_not_finite_in_several_units_of_a_block(D, dtype, packed):
    """+inf, -inf and NaN in V under the mask of many units, of every head at another place: exactly the rows that see them have them."""
    lens = [(1500, 1500)] * 3
    H, Hkv = 16, 8
    check_plan(lens, H, Hkv, D, dtype, packed)
    (q, k, v, _), (cu_q, cu_k), _ = make(lens, H, Hkv, D, dtype, seed=32)
    shape = (lambda t: t) if packed else (lambda t: t.view(len(lens), -1, *t.shape[1:]))
    kw = dict(cu_q=cu_q, cu_k=cu_k) if packed else {}
    call = lambda: sab.causal_attention(shape(q), shape(k), shape(v), **kw).reshape(-1, H, D)
    want = call().clone()
    for s in range(len(lens)):
        for hk in range(Hkv):
            for x, value in enumerate((math.inf, -math.inf, math.nan, math.inf)):
                j, d = (59 + 173 * s + 401 * x + 37 * hk) % 1500, (5 + 11 * x + 3 * hk + 7 * s) % D
                v[1500 * s + j, hk, d] = value
                rows, heads = slice(1500 * s + j, 1500 * (s + 1)), slice(2 * hk, 2 * hk + 2)
                want[rows, heads, d] = value
    got = call()
    sab.check_device_status()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan])
