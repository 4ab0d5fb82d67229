"""Causal attention against its definition in 64 bits (tests/causal_ref.py has the bounds), its refusals and its uses."""
import ctypes
import math

import pytest
import torch

import simplical_attn_b200 as sab
from simplical_attn_b200 import _abi
from simplical_attn_b200 import simplicial_attn as host
from tests import causal_ref

gpu = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(lens, H, Hkv, D, dtype, seed=0, gap=0, device="cuda", spread=1.0):
    """Packed tensors of sequences with these (queries, keys), `gap` rows before the first and behind the last."""
    g = torch.Generator().manual_seed(seed)
    Tq, Tk = sum(n for n, _ in lens) + 2 * gap, sum(m for _, m in lens) + 2 * gap
    q, d_o = (torch.randn(Tq, H, D, generator=g) * spread for _ in range(2))
    k, v = (torch.randn(Tk, Hkv, D, generator=g) * spread for _ in range(2))
    cu_q, cu_k = [gap], [gap]
    for n, m in lens:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    seqs = [(a, n, b, m) for a, b, (n, m) in zip(cu_q, cu_k, lens)]
    t = [x.to(device=device, dtype=DT[dtype]) for x in (q, k, v, d_o)]
    cu = [torch.tensor(x, dtype=torch.int32, device=device) for x in (cu_q, cu_k)]
    return t, cu, seqs


def step(q, k, v, d_o, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o, lse = sab.causal_attention(*leaves, return_lse=True, **kw)
    return dict(zip(("o", "lse", "dq", "dk", "dv"), (o, lse) + torch.autograd.grad(o, leaves, d_o)))


def compare(got, ref):
    for n in got:
        causal_ref.check(got[n], ref[0][n], ref[1][n], n)


@pytest.fixture(params=["auto", "general"])
def algo(request, monkeypatch):
    monkeypatch.setattr(host, "default_algo", request.param)
    return request.param


# (queries, keys) of the sequences, H, Hkv, D, dtype
PACKED = [
    ([(1, 1)], 1, 1, 64, "bf16"),
    ([(1, 1), (2, 2), (3, 3)], 2, 1, 128, "fp16"),
    ([(130, 130), (1, 1), (0, 0), (64, 64), (257, 257)], 2, 2, 64, "bf16"),
    ([(127, 127), (128, 128), (129, 129)], 2, 1, 128, "bf16"),
    ([(300, 300), (77, 77)], 4, 2, 128, "fp16"),
    ([(5, 200), (64, 300), (1, 129)], 4, 2, 64, "fp16"),             # chunks over earlier keys
    ([(200, 40), (7, 0), (0, 9), (300, 299)], 2, 1, 128, "bf16"),    # more queries than keys: rows that see nothing
    ([(513, 513)], 3, 1, 64, "bf16"),
    ([(1, 2001), (1, 1), (1, 64), (1, 0), (1, 65)], 16, 2, 128, "bf16"),       # single tokens
    ([(3, 500), (7, 100), (4, 4), (2, 1), (0, 30)], 4, 1, 64, "fp16"),         # a few tokens: 28 rows
    ([(2, 900), (1, 63)], 5, 5, 128, "fp16"),
    ([(1, 300), (1, 128)], 24, 1, 64, "bf16"),
    ([(100, 100), (45, 70)], 2, 1, 80, "bf16"),                      # head dims that fill a tile's columns in part
    ([(140, 140), (3, 200)], 2, 1, 32, "fp16"),
    ([(20, 150), (1, 77)], 6, 2, 8, "bf16"),
    ([(130, 257)], 2, 1, 120, "fp16"),
    ([(70, 70), (33, 97)], 2, 2, 256, "fp16"),                       # ... of the general kernels
    ([(40, 90), (1, 500)], 2, 1, 100, "bf16"),
    ([(3, 1500), (40, 700)], 8, 1, 64, "fp32"),                      # few blocks with long walks: shares
    ([(300, 300)], 8, 1, 200, "fp32"),
    ([(1, 900), (0, 3)], 2, 2, 33, "fp32"),
    ([(65, 65), (64, 100), (1, 7)], 4, 1, 64, "fp32"),
    ([(90, 33)], 1, 1, 17, "fp32"),
]


@gpu
@pytest.mark.parametrize("case", PACKED)
def test_packed_against_definition(case, algo):
    lens, H, Hkv, D, dtype = case
    (q, k, v, d_o), (cu_q, cu_k), seqs = make(lens, H, Hkv, D, dtype, seed=1)
    ref = causal_ref.reference(q, k, v, d_o, seqs, D ** -0.5)
    for kw in ({}, dict(max_q=max(n for n, _ in lens), max_k=max(m for _, m in lens))):
        compare(step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k, **kw), ref)


@gpu
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "fp16"), (64, "fp32")])
def test_rows_outside_the_sequences(D, dtype, algo):
    """Rows before the first and behind the last sequence: zeros, LSE -inf, zero gradients, whatever lies there."""
    lens = [(70, 70), (3, 200)]
    (q, k, v, d_o), (cu_q, cu_k), seqs = make(lens, 4, 2, D, dtype, seed=2, gap=9)
    ref = causal_ref.reference(q, k, v, d_o, seqs, D ** -0.5)
    for t in (q, k, v, d_o):
        t[:9] = math.nan
        t[-9:] = math.inf
    compare(step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k), ref)


@gpu
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16"), (32, "bf16")])
def test_other_sequences_do_not_leak(D, dtype, algo):
    """NaN and infinities in one packed sequence leave its neighbours' results as they were."""
    lens = [(100, 100), (61, 61), (140, 140), (1, 90), (30, 30)]
    (q, k, v, d_o), (cu_q, cu_k), seqs = make(lens, 2, 1, D, dtype, seed=3)
    before = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    bad_q, bad_k = slice(161, 301), slice(161, 301)
    for t, rows in ((q, bad_q), (k, bad_k), (v, bad_k), (d_o, bad_q)):
        t[rows][::2] = math.nan
        t[rows][1::2] = math.inf
    after = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    for n in ("o", "dq", "dk", "dv"):
        a, b = before[n].clone(), after[n].clone()
        a[161:301] = b[161:301] = 0
        assert torch.equal(a, b), n


@gpu
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "fp16"), (128, "bf16"), (48, "fp32")])
def test_later_keys_do_not_leak_forward(D, dtype, algo):
    """NaN and infinities in K and V of a sequence reach only the queries that see them."""
    lens = [(150, 150), (140, 260)]
    (q, k, v, _), (cu_q, cu_k), seqs = make(lens, 2, 1, D, dtype, seed=4)
    before = sab.causal_attention(q, k, v, cu_q=cu_q, cu_k=cu_k)
    k[133, :, 3] = math.nan
    v[100, :, 5] = math.inf
    v[150 + 250, :, :] = math.nan
    after = sab.causal_attention(q, k, v, cu_q=cu_q, cu_k=cu_k)
    ok = torch.ones_like(before, dtype=torch.bool)
    ok[100:150, :, 5] = False
    ok[133:150] = False
    ok[150 + 130:] = False
    assert torch.equal(before[ok], after[ok])
    assert not torch.isfinite(after[100:133, :, 5]).any() and torch.isnan(after[133:150]).all() and torch.isnan(after[280:]).all()


@gpu
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "fp16")])
def test_later_keys_do_not_leak_into_a_few_rows(D, dtype, algo):
    lens = [(6, 150), (5, 131), (3, 8)]
    (q, k, v, _), (cu_q, cu_k), _ = make(lens, 4, 1, D, dtype, seed=4)
    call = lambda: sab.causal_attention(q, k, v, cu_q=cu_q, cu_k=cu_k, max_q=6, max_k=150)
    before = call()
    v[147, :, 5] = math.inf            # the last but two: queries 3 to 5 of the first sequence see it
    k[150 + 129] = math.nan            # the last but one of the second
    v[281 + 7] = -math.inf             # the last of the third
    after = call()
    ok = torch.ones_like(before, dtype=torch.bool)
    ok[3:6, :, 5] = False
    ok[9:11] = False
    ok[13] = False
    assert torch.equal(before[ok], after[ok])
    assert not torch.isfinite(after[~ok]).any() and torch.isnan(after[9:11]).all()


# B, N, M, H, Hkv, D, dtype, layout
BATCHED = [
    (2, 100, 100, 4, 2, 64, "bf16", "bnhd"),
    (3, 129, 129, 2, 2, 128, "fp16", "bhnd"),
    (2, 70, 200, 4, 1, 64, "fp16", "fused"),
    (2, 1, 300, 8, 1, 128, "bf16", "bnhd"),
    (2, 3, 65, 6, 2, 64, "fp16", "bhnd"),
    (1, 1, 1, 1, 1, 64, "bf16", "bnhd"),
    (1, 33, 20, 2, 1, 64, "bf16", "odd"),         # rows that are not 16-byte aligned; queries that see nothing
    (2, 50, 50, 3, 3, 128, "bf16", "transposed"), # inner stride that is not 1
    (1, 40, 40, 4, 2, 96, "fp32", "fused"),
]


def layout(t, kind):
    """The same values laid out otherwise."""
    B, N, h, D = t.shape
    if kind == "bhnd":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "fused":
        buf = torch.full((B, N, h + 3, D), math.nan, dtype=t.dtype, device=t.device)
        buf[:, :, 2:2 + h] = t
        return buf[:, :, 2:2 + h]
    if kind == "odd":
        buf = torch.empty(B, N, h, D + 1, dtype=t.dtype, device=t.device)
        buf[..., 1:] = t
        return buf[..., 1:]
    if kind == "transposed":
        return t.transpose(1, 3).contiguous().transpose(1, 3)
    return t


@gpu
@pytest.mark.parametrize("case", BATCHED)
def test_batched_layouts(case, algo):
    B, N, M, H, Hkv, D, dtype, kind = case
    (q, k, v, d_o), _, seqs = make([(N, M)] * B, H, Hkv, D, dtype, seed=5)
    ref = causal_ref.reference(q, k, v, d_o, seqs, 0.3)
    shaped = [layout(t.view(B, -1, *t.shape[1:]), kind) for t in (q, k, v, d_o)]
    got = step(*shaped, scale=0.3)
    assert got["lse"].shape == (B, H, N)
    got["lse"] = got["lse"].transpose(0, 1).reshape(H, B * N)
    compare({n: t if n == "lse" else t.reshape(-1, *t.shape[2:]) for n, t in got.items()}, ref)


@gpu
@pytest.mark.parametrize("scale", [0.0, -0.4, 3.0])
@pytest.mark.parametrize("D", [64, 128])
def test_scales(scale, D, algo):
    (q, k, v, d_o), (cu_q, cu_k), seqs = make([(150, 150), (2, 170)], 2, 1, D, "bf16", seed=6)
    compare(step(q, k, v, d_o, scale=scale, cu_q=cu_q, cu_k=cu_k), causal_ref.reference(q, k, v, d_o, seqs, scale))


@gpu
def test_long_keys_and_rising_maxima(algo):
    """Keys that grow along the sequence (the running maximum keeps moving), and many of them."""
    (q, k, v, d_o), (cu_q, cu_k), seqs = make([(3, 5000), (200, 1500)], 2, 1, 64, "bf16", seed=7)
    k *= torch.linspace(0.1, 4, k.shape[0], device="cuda", dtype=k.dtype)[:, None, None]
    compare(step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k), causal_ref.reference(q, k, v, d_o, seqs, 0.125))


@gpu
def test_gradient_against_differences(algo):
    """fp32: the directional derivative of sum(O * d_o) along random directions, by central differences in 64 bits."""
    lens = [(37, 37), (5, 60)]
    (q, k, v, d_o), (cu_q, cu_k), seqs = make(lens, 2, 1, 64, "fp32", seed=8)
    got = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)

    def f(ts):
        out = 0.0
        for q0, n, k0, m in seqs:
            for h in range(2):
                x = ts[0][q0:q0 + n, h] @ ts[1][k0:k0 + m, 0].T / 8
                x = x.masked_fill(~torch.ones(n, m, dtype=torch.bool).tril(m - n), -math.inf)
                out += float((torch.softmax(x, -1) @ ts[2][k0:k0 + m, 0] * d_o64[q0:q0 + n, h]).sum())
        return out

    d_o64 = d_o.double().cpu()
    base = [t.double().cpu() for t in (q, k, v)]
    g = torch.Generator().manual_seed(9)
    for i, n in enumerate(("dq", "dk", "dv")):
        d = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        slope = (f(up) - f(down)) / 2e-5
        have = float((got[n].double().cpu() * d).sum())
        # differences: 1e-10 of third derivatives and 2^-52 / 1e-5 of f; the kernel: its elements' bounds, against |d|
        err = causal_ref.reference(q, k, v, d_o, seqs, 0.125)[1][n]
        assert abs(have - slope) <= float((err * d.abs()).sum()) + 1e-6 * (1 + abs(slope)), n


@gpu
def test_wrong_bounds_only_cost_time(algo):
    (q, k, v, d_o), (cu_q, cu_k), seqs = make([(140, 140), (9, 300), (1, 40)], 4, 2, 64, "bf16", seed=10)
    ref = causal_ref.reference(q, k, v, d_o, seqs, 0.125)
    for max_q, max_k in ((1, 1), (1, 300), (140, 2), (10 ** 6, 10 ** 6)):
        compare(step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k, max_q=max_q, max_k=max_k), ref)


@gpu
def test_starts_outside_the_tensors_are_clipped(algo):
    (q, k, v, d_o), _, _ = make([(100, 100)], 2, 1, 64, "bf16", seed=11)
    cu = torch.tensor([-5, 60, 400], dtype=torch.int32, device="cuda")
    got = step(q, k, v, d_o, cu_q=cu, cu_k=cu)
    compare(got, causal_ref.reference(q, k, v, d_o, [(0, 60, 0, 60), (60, 40, 60, 40)], 0.125))


@gpu
def test_partial_gradients_and_broadcast_inputs(algo):
    """Only some leaves need a gradient; K and V broadcast over batch and heads get the sum."""
    g = torch.Generator().manual_seed(12)
    q, d_o = (torch.randn(2, 70, 4, 64, generator=g).cuda().bfloat16() for _ in range(2))
    kv = [torch.randn(1, 70, 1, 64, generator=g).cuda().bfloat16().requires_grad_() for _ in range(2)]
    k, v = (t.expand(2, 70, 4, 64) for t in kv)
    o = sab.causal_attention(q, k, v)
    got = torch.autograd.grad(o, kv, d_o)
    full = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
    every = torch.autograd.grad(sab.causal_attention(*full), full, d_o)
    assert torch.equal(o, sab.causal_attention(*full))
    for a, b in zip(got, every[1:]):
        # the sum over the expanded extents is torch's, in the tensors' type or 32 bits, in whatever order: compare with it
        assert torch.equal(a, b.sum((0, 2), keepdim=True))
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate(full)]
        only, = torch.autograd.grad(sab.causal_attention(*leaves), leaves[i], d_o)
        assert torch.equal(only, every[i])


@gpu
def test_equal_calls_give_equal_bits(algo):
    (q, k, v, d_o), (cu_q, cu_k), _ = make([(400, 400), (30, 900)], 8, 2, 64, "bf16", seed=13)
    a, b = (step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)


@gpu
@pytest.mark.parametrize("lens", [[(90, 90), (200, 200)], [(1, 700), (1, 1200)], [(1, 9000), (1, 4000)], [(200, 3000), (30, 700)]])
def test_captured_call_follows_its_inputs(lens, algo):
    """A captured forward and backward replays on new values and new lengths, and beside another graph."""
    first, (cu_q, cu_k), seqs = make(lens, 4, 2, 64, "bf16", seed=14)
    second, (cu_q2, cu_k2), seqs2 = make(lens[::-1], 4, 2, 64, "bf16", seed=15)
    # (the gradients' sums must not run over the capture's end: the leaves are the graph's own)
    static = [t.clone() for t in first]
    run = lambda: step(*static, cu_q=cu_q, cu_k=cu_k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    for tensors, cq, ck, s in ((first, cu_q.clone(), cu_k.clone(), seqs), (second, cu_q2, cu_k2, seqs2)):
        for a, b in zip(static, tensors):
            a.copy_(b)
        cu_q.copy_(cq)
        cu_k.copy_(ck)
        ref = causal_ref.reference(*tensors, s, 0.125)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            compare(out, ref)
    sab.check_device_status()


@gpu
def test_two_streams_at_once(algo):
    cases = [make([(300, 300), (1, 800)], 4, 2, 128, "bf16", seed=20 + i) for i in range(2)]
    alone = [step(*t, cu_q=cu[0], cu_k=cu[1]) for t, cu, _ in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(3):
        for i, (t, cu, _) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i] = step(*t, cu_q=cu[0], cu_k=cu[1])
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(a[n], b[n]) for n in a)


@gpu
@pytest.mark.parametrize("direction,label", [(2, "sa_causal_forward"), (3, "sa_causal_backward")])
def test_report_of_an_earlier_call_is_raised_once(direction, label):
    """What a kernel that gave up on a wait leaves in the pinned word of its kind of call (here: the library's self-test) is raised by
    the next call."""
    lib = _abi.load()
    word = ctypes.c_void_p(_abi.binding().status_word(torch.cuda.current_device(), direction))
    q = torch.randn(1, 70, 2, 64, device="cuda", dtype=torch.bfloat16)
    o = sab.causal_attention(q, q, q)
    for ask in (lambda: sab.causal_attention(q, q, q), sab.check_device_status):
        assert lib.sa_selftest_wait_timeout(word, 2_000_000, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == _abi.SA_OK
        torch.cuda.synchronize()
        with pytest.raises(_abi.SimplicialAttnError, match=label):
            ask()
        ask()
    assert torch.equal(sab.causal_attention(q, q, q), o)


@gpu
def test_nothing_to_do():
    for q_rows, k_rows in ((0, 0), (0, 5), (5, 0)):
        q = torch.randn(2, q_rows, 4, 64, device="cuda", dtype=torch.bfloat16)
        k = torch.randn(2, k_rows, 2, 64, device="cuda", dtype=torch.bfloat16)
        got = step(q, k, k.clone(), q)
        assert all(not got[n].any() for n in ("o", "dq", "dk", "dv")) and torch.isinf(got["lse"]).all()


@gpu
def test_calls_through_ctypes_and_traces(monkeypatch):
    (q, k, v, d_o), (cu_q, cu_k), _ = make([(100, 100), (1, 30)], 4, 2, 64, "bf16", seed=16)
    plain = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
    with monkeypatch.context() as m:
        m.setattr(_abi, "_binding", False)
        got = step(q, k, v, d_o, cu_q=cu_q, cu_k=cu_k)
        sab.check_device_status()
    assert all(torch.equal(plain[n], got[n]) for n in plain)
    traced = torch.jit.trace(lambda a, b, c: sab.causal_attention(a, b, c, cu_q=cu_q, cu_k=cu_k), (q, k, v), check_trace=False)
    assert torch.equal(traced(q, k, v), plain["o"])
    o, lse, low = sab.causal_attention_fwd(q, k, v, 0.125, cu_q, cu_k, low=True)
    bw = sab.causal_attention_bwd(q, k, v, o, lse, d_o, 0.125, cu_q, cu_k, need=(True, False, True), o_low=low)
    fw = sab.causal_attention_fwd(q, k, v, 0.125, cu_q, cu_k)
    assert torch.equal(fw[0], o) and torch.equal(fw[1], lse) and len(fw) == 2
    with pytest.raises(ValueError, match="o_low"):
        sab.causal_attention_bwd(q, k, v, o, lse, d_o, 0.125, cu_q, cu_k, o_low=low[:50])
    assert torch.equal(fw[0], plain["o"]) and torch.equal(bw[0], plain["dq"]) and bw[1] is None and torch.equal(bw[2], plain["dv"])


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_no_second_derivative(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_abi, "_binding", False)
    q = torch.randn(1, 20, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    o = sab.causal_attention(q, q, q)
    g, = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative|once_differentiable"):
        g.float().sum().backward()


@gpu
def test_refusals_on_the_device():
    t = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dtype)
    q, k, cu = t(10, 4, 64), t(10, 2, 64), torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    call = sab.causal_attention
    for error, args, kw in [
        (ValueError, (q, k, k), {}),                                             # packed without cu_q
        (ValueError, (q[None], k[None], k[None]), dict(cu_q=cu)),                # batched with it
        (ValueError, (q[None], k[None], k[None]), dict(cu_k=cu)),
        (ValueError, (q, t(11, 2, 64), t(11, 2, 64)), dict(cu_q=cu)),            # other rows without cu_k
        (ValueError, (q, k, t(10, 4, 64)), dict(cu_q=cu)),
        (ValueError, (q, t(10, 3, 64), t(10, 3, 64)), dict(cu_q=cu)),            # 4 % 3
        (ValueError, (q, t(10, 2, 32), t(10, 2, 32)), dict(cu_q=cu)),
        (ValueError, (q, k, k), dict(cu_q=cu[:1])),
        (ValueError, (q, k, k), dict(cu_q=cu, cu_k=torch.tensor([0, 5, 10], dtype=torch.int32, device="cuda"))),
        (ValueError, (q, k, k), dict(cu_q=cu, max_q=-1)),
        (TypeError, (q, k, k), dict(cu_q=cu.long())),
        (TypeError, (q, k, k), dict(cu_q=cu.cpu())),
        (TypeError, (q, k.half(), k), dict(cu_q=cu)),
        (TypeError, (q.double(), k.double(), k.double()), dict(cu_q=cu)),
        (_abi.SimplicialAttnError, (t(10, 4, 300), t(10, 2, 300), t(10, 2, 300)), dict(cu_q=cu)),
    ]:
        for binding in (_abi.binding(), False):
            saved = _abi._binding
            _abi._binding = binding
            try:
                with pytest.raises(error):
                    call(*args, **kw)
            finally:
                _abi._binding = saved


# ------------------------------------------------------------------------------------------------ without a GPU
def params(**kw):
    p = _abi.CausalParams()
    p.B, p.Nq, p.Nk, p.H, p.Hkv, p.D = 1, 64, 64, 4, 2, 128
    p.dtype, p.algo, p.scale = _abi.SA_BF16, _abi.SA_ALGO_AUTO, 0.1
    for n in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv"):
        setattr(p, n, _abi.Strides(64 * 512, 512, 128))
    for n, x in kw.items():
        setattr(p, n, x)
    return ctypes.byref(p)


def test_entries_validate():
    lib = _abi.load()
    assert ctypes.sizeof(_abi.CausalParams) == 12 * 4 + 8 * 24
    nul, some = ctypes.c_void_p(0), ctypes.c_void_p(4096)
    fwd = lambda p, a=nul, ws=nul, n=0, status=some: lib.sa_causal_forward(p, *[a] * 4, nul, a, nul, nul, ws, n, status, nul)
    bwd = lambda p, a=nul, ws=nul, n=0, status=some: lib.sa_causal_backward(p, *[a] * 4, nul, *[a] * 5, nul, nul, ws, n, status, nul)
    for call in (fwd, bwd):
        assert call(None) == 1 and call(params()) == 1
        for bad in (dict(B=0), dict(Nq=0), dict(Nk=-1), dict(H=5), dict(Hkv=0), dict(D=0), dict(sequences=-1), dict(max_q=-1),
                    dict(sequences=2, B=2)):
            assert call(params(**bad), some) == 2, bad
        for bad in (dict(D=257), dict(dtype=3), dict(algo=3), dict(Nk=(1 << 30) + 1), dict(B=1 << 12, Nq=1 << 20)):
            assert call(params(**bad), some) == 4, bad
        assert call(params(sequences=2), some) == 1                       # no starts
        assert call(params(), some, status=nul) == 1
        assert call(params(), some, ctypes.c_void_p(256), 1 << 30, ctypes.c_void_p(4097)) == 5
    need = lib.sa_causal_backward_workspace_size(params())
    assert need >= 4 * 64 * 4 and bwd(params(), some, ctypes.c_void_p(256), need - 1) == 5
    assert bwd(params(), some, ctypes.c_void_p(128), need) == 5 and bwd(params(), some, nul, need) == 5
    assert lib.sa_causal_backward_workspace_size(params(D=0)) == 0
    r = lambda b=0, **kw: lib.sa_causal_resolve(params(**kw), b)
    assert r() == r(1) == r(1, Nq=1) == _abi.SA_ALGO_TCGEN05 and r(Nq=16) == _abi.SA_CAUSAL_FEW_ROWS and r(Nq=17) == _abi.SA_ALGO_TCGEN05
    assert r(Nq=4, algo=_abi.SA_ALGO_TCGEN05) == _abi.SA_ALGO_TCGEN05 and r(sequences=9, max_q=1, max_k=5) == _abi.SA_CAUSAL_FEW_ROWS
    assert r(D=96) == r(D=8) == r(1, D=40) == _abi.SA_ALGO_TCGEN05
    for general in (dict(D=100), dict(D=136), dict(dtype=_abi.SA_F32), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(algo=_abi.SA_ALGO_GENERAL),
                    dict(k=_abi.Strides(64 * 512, 512, 132))):
        assert r(**general) == r(1, **general) == _abi.SA_ALGO_GENERAL, general
    assert r(D=100, algo=_abi.SA_ALGO_TCGEN05) == -4
    assert lib.sa_causal_resolve(params(D=257), 0) == -4 and lib.sa_causal_resolve(params(H=3), 1) == -2


def test_python_layer_rejects_cpu_tensors(monkeypatch):
    x = torch.zeros(1, 8, 2, 64)
    for binding in (None, False):
        monkeypatch.setattr(_abi, "_binding", binding)
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            sab.causal_attention(x, x, x)
    with pytest.raises(ValueError):
        sab.CausalSelfAttention(64, 4, 16, kv_heads=3)


def test_module_parameters():
    m = sab.CausalSelfAttention(96, 4, 16, kv_heads=2, rotary=sab.RotaryPositions(16), dtype=torch.float32)
    assert {n: tuple(p.shape) for n, p in m.state_dict().items()} == {"in_proj.weight": (128, 96), "out_proj.weight": (96, 64)}
    assert m.scale == 0.25
