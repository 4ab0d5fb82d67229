"""Rotary positions against their definition in 64 bits, their refusals, and a layer stack that uses them.

The kernel computes x cos - y sin in 32 bits from sines and cosines in 32 bits and rounds once.  In units of 2^-24 a sine is
off by at most 3 (its argument's rounding 0.8, sincospif 2 with the final bit), the product with the magnitude and the
magnitude itself by one each, a product and the sum by one each: 7 units of magnitude (|x| + |y|), then half a step of the type.
"""
import ctypes
import math

import pytest
import torch

import simplical_attn_b200 as sab
from simplical_attn_b200 import _abi

gpu = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def pairs(rd, interleaved):
    return (torch.arange(0, rd, 2), torch.arange(1, rd, 2)) if interleaved else (torch.arange(rd // 2), torch.arange(rd // 2, rd))


def reference(x, f, pos, interleaved=False, magnitude=1.0, inverse=False):
    """x [..., heads, D] on the CPU, pos [...]: (value, bound of the error) in fp64."""
    v = x.detach().cpu().double()
    i, j = pairs(2 * f.numel(), interleaved)
    t = (pos.cpu().double()[..., None] * f.cpu().double())[..., None, :] * (-1 if inverse else 1)
    a, b = v[..., i], v[..., j]
    out, err = v.clone(), torch.zeros_like(v)
    out[..., i] = magnitude * (a * t.cos() - b * t.sin())
    out[..., j] = magnitude * (b * t.cos() + a * t.sin())
    # (far positions: the angle itself is rounded to 64 bits, here and in the kernel)
    e = abs(magnitude) * (a.abs() + b.abs()) * (7 * 2.0 ** -24 + t.abs() * 2.0 ** -50)
    err[..., i] = err[..., j] = e
    u = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    return out, err * (1 + u) + u * out.abs() * (err > 0) + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)


def check(got, x, f, pos, **kw):
    val, err = reference(x, f, pos, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype
    off = (got.detach().cpu().double() - val).abs()
    assert (off <= err).all(), f"{int((off > err).sum())} outside, worst {float((off / err.clamp(min=1e-300)).max()):.2f} times the bound"


# B, N, heads of the tensors, D, rd, interleaved, dtype, layout
CASES = [
    (1, 1, (1,), 64, 64, False, "bf16", "plain"),
    (2, 5, (4, 2), 64, 64, False, "bf16", "plain"),
    (2, 33, (16, 4, 4), 128, 128, True, "fp16", "fused"),
    (3, 7, (5, 1, 2, 9), 80, 40, False, "fp32", "plain"),
    (1, 129, (3, 3), 64, 24, True, "bf16", "bhnd"),
    (2, 17, (2,), 256, 64, False, "fp16", "bhnd"),
    (2, 9, (6, 3), 34, 34, False, "bf16", "plain"),          # pairs that no wide load reaches
    (2, 9, (6, 3), 33, 6, True, "fp32", "plain"),
    (1, 20, (4, 4), 64, 64, False, "bf16", "odd"),
    (2, 6, (4,), 64, 2, True, "bf16", "transposed"),
    (2, 6, (7,), 48, 46, False, "fp16", "plain"),
]


def tensors(case, seed=0):
    B, N, heads, D, rd, interleaved, dtype, layout = case
    g = torch.Generator().manual_seed(seed)
    xs = []
    buf = torch.randn(B, N, sum(heads) + 1, D + 1, generator=g).to(DT[dtype]).cuda()
    at = 0
    for h in heads:
        t = buf[:, :, at:at + h, :D]
        at += h
        if layout == "bhnd":
            t = t.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "transposed":
            t = t.transpose(1, 3).contiguous().transpose(1, 3)
        elif layout == "odd":
            t = buf[:, :, at - h:at, 1:]
        elif layout == "plain":
            t = t.contiguous()
        xs.append(t)
    if layout == "fused":
        whole = torch.cat(xs, 2).contiguous()
        xs = list(whole.split(heads, 2))
    return xs


@gpu
@pytest.mark.parametrize("case", CASES)
def test_against_definition(case):
    B, N, heads, D, rd, interleaved, dtype, layout = case
    f = sab.rotary_frequencies(rd, device="cuda")
    xs = [t.detach().requires_grad_() for t in tensors(case)]
    ds = [torch.randn(t.shape, device="cuda").to(t.dtype) for t in xs]
    for pos, kw in ((torch.randint(0, 5000, (B, N), device="cuda"), {}), (torch.randint(-9, 9, (N,), device="cuda", dtype=torch.int32), dict(magnitude=1.3)),
                    (None, dict(offset=100000)), (torch.randint(0, 2 ** 20, (B, 1), device="cuda").expand(B, N), dict(inverse=True, offset=-3))):
        ys = sab.rotary_positions(xs, f, pos, interleaved=interleaved, **kw)
        at = (torch.arange(N) if pos is None else pos.cpu()) + kw.pop("offset", 0)
        at = at.expand(B, N)
        for x, y in zip(xs, ys):
            check(y, x, f, at, interleaved=interleaved, **kw)
        kw["inverse"] = not kw.get("inverse", False)
        for d, g in zip(ds, torch.autograd.grad(ys, xs, ds)):
            check(g, d, f, at, interleaved=interleaved, **kw)


@gpu
@pytest.mark.parametrize("scaling", [None, "linear", "base", "parts"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_scaled_frequencies_and_far_positions(scaling, dtype):
    f = sab.rotary_frequencies(64, 500000.0, scaling, 8.0, 4096, device="cuda").to(dtype)
    x = torch.randn(6, 2, 64, device="cuda")
    pos = torch.tensor([0, 1, 4095, 1 << 20, (1 << 31) - 1, 1 << 40], device="cuda")
    check(sab.rotary_positions(x, f, pos), x, f, pos)


@gpu
def test_packed_positions_and_single_tensor():
    f = sab.rotary_frequencies(64, device="cuda")
    x = torch.randn(30, 3, 64, device="cuda", dtype=torch.bfloat16)
    pos = torch.cat([torch.arange(n) for n in (7, 1, 22)]).cuda()
    y = sab.rotary_positions(x, f, pos)
    assert isinstance(y, torch.Tensor)
    check(y, x, f, pos)
    back = sab.rotary_positions(y, f, pos, inverse=True)
    assert (back.float() - x.float()).abs().max() <= 2 ** -7 * 1.5 * x.float().abs().max() * 2      # two roundings, of a pair's length


@gpu
def test_in_place_and_into_buffers():
    f = sab.rotary_frequencies(32, device="cuda")
    whole = torch.randn(2, 9, 7, 64, device="cuda", dtype=torch.bfloat16)
    q, k, v = whole.split((4, 2, 1), 2)
    want = sab.rotary_positions((q, k), f)
    kept = v.clone()
    version = whole._version
    got = sab.rotary_positions((q, k), f, out=(q, k))
    assert got[0].data_ptr() == q.data_ptr() and whole._version > version
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)
    buf = torch.full((2, 9, 8, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    sab.rotary_positions(want[0], f, inverse=True, out=buf[:, :, 2:6])
    assert torch.equal(buf[:, :, 2:6], sab.rotary_positions(want[0], f, inverse=True)) and (buf[:, :, :2] == 7).all() and (buf[:, :, 6:] == 7).all()


@gpu
def test_refusals_on_the_device():
    f = sab.rotary_frequencies(64, device="cuda")
    x = torch.zeros(2, 5, 4, 64, device="cuda", dtype=torch.bfloat16)
    call = sab.rotary_positions
    for error, args in [
        (ValueError, ([x] * 5, f)), (TypeError, ([], f)), (TypeError, ([x, None], f)), (TypeError, ([x, x.half()], f)), (ValueError, ([x, x[:1]], f)),
        (ValueError, (x[0, 0], f)), (TypeError, (x.double(), f)), (TypeError, (x, f.half())), (TypeError, (x, f.cpu())), (ValueError, (x, f[None])),
        (ValueError, (x, f[:0])), (ValueError, (x[..., :62], f)), (TypeError, (x, f, torch.zeros(5, device="cuda"))),
        (ValueError, (x, f, torch.zeros(4, device="cuda", dtype=torch.long))), (ValueError, (x, f, torch.zeros(1, 5, device="cuda", dtype=torch.long))),
        (TypeError, (x, f, torch.zeros(5, dtype=torch.long))),
    ]:
        for binding in (_abi.binding(), False):
            saved, _abi._binding = _abi._binding, binding
            try:
                with pytest.raises(error):
                    call(*args)
            finally:
                _abi._binding = saved
    for binding in (_abi.binding(), False):
        saved, _abi._binding = _abi._binding, binding
        try:
            with pytest.raises(ValueError, match="no gradient"):
                call(x, f.clone().requires_grad_())
        finally:
            _abi._binding = saved
    whole = torch.zeros(2, 5, 9, 64, device="cuda", dtype=torch.bfloat16)
    for bad in (whole[:, :, 1:5], whole[:, :, 5:8], whole[:, :, :1].expand(2, 5, 4, 64), torch.empty(2, 5, 4, 64, device="cuda")):
        with pytest.raises((ValueError, TypeError)):
            call(whole[:, :, :4], f, out=bad)
    with pytest.raises(ValueError):
        call([whole[:, :, :4], whole[:, :, 4:8]], f, out=[whole[:, :, 4:8], whole[:, :, :4]])
    with pytest.raises(RuntimeError, match="records no gradient"):
        call(x.clone().requires_grad_(), f, out=torch.empty_like(x))


@gpu
def test_histories():
    """Some tensors need a gradient, some outputs are used, a second derivative, calls that are not plain, nothing to do."""
    f = sab.rotary_frequencies(64, device="cuda")
    q, k = (torch.randn(1, 6, 2, 64, device="cuda", requires_grad=r) for r in (True, False))
    yq, yk = sab.rotary_positions((q, k), f, offset=5)
    g, = torch.autograd.grad(yq.square().sum() / 2, q, create_graph=True)
    # |y|^2 / 2 is |x|^2 / 2: the gradient is x, and the gradient of sum(g c) is c, up to 4 turns of 7 units each and the pair's sum
    c = torch.randn_like(q)
    tol = 64 * 2.0 ** -24 * (q.abs().max() + c.abs().max())
    assert (g - q).abs().max() <= tol and (torch.autograd.grad((g * c).sum(), q)[0] - c).abs().max() <= tol
    with torch.no_grad():
        assert not sab.rotary_positions(q, f).requires_grad
    traced = torch.jit.trace(lambda a: sab.rotary_positions(a, f, offset=5), (q.detach(),), check_trace=False)
    assert torch.equal(traced(q.detach()), yq.detach())
    saved, _abi._binding = _abi._binding, False
    try:
        y2 = sab.rotary_positions((q, k), f, offset=5)
        assert torch.equal(y2[0], yq) and torch.equal(y2[1], yk)
        assert torch.equal(torch.autograd.grad(y2[0], q, c)[0], torch.autograd.grad(sab.rotary_positions(q, f, offset=5), q, c)[0])
    finally:
        _abi._binding = saved
    assert sab.rotary_positions(torch.zeros(0, 4, 64, device="cuda"), f).shape == (0, 4, 64)
    assert [t.shape[2] for t in sab.rotary_positions((torch.zeros(1, 3, 0, 64, device="cuda"), torch.zeros(1, 3, 2, 64, device="cuda")), f)] == [0, 2]


@gpu
def test_captured_rotation_follows_positions():
    f = sab.rotary_frequencies(64, device="cuda")
    x, pos = torch.randn(4, 1, 8, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(4, 1, device="cuda", dtype=torch.long)
    sab.rotary_positions(x, f, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = sab.rotary_positions(x, f, pos)
    for start in (3, 70000):
        pos.fill_(start)
        x.normal_()
        graph.replay()
        check(y, x, f, pos)


# ------------------------------------------------------------------------------------------------ the operators together
def _layer64(m, x, pos, seqs):
    """CausalSelfAttention in 64 bits over packed rows."""
    w = m.in_proj.weight.detach().double().cpu().requires_grad_()
    q, k, v = (t.unflatten(-1, (-1, m.head_dim)) for t in (x @ w.T).split(m.widths, -1))
    f = m.rotary.frequencies.cpu()
    i, j = pairs(2 * f.numel(), m.rotary.interleaved)
    t = (pos.double()[:, None] * f)[:, None]

    def turn(y):
        a, b = y[..., i], y[..., j]
        parts = torch.zeros_like(y).index_copy(-1, i, a * t.cos() - b * t.sin()).index_copy(-1, j, b * t.cos() + a * t.sin())
        return torch.cat((parts[..., :2 * f.numel()], y[..., 2 * f.numel():]), -1)

    q, k = turn(q), turn(k)
    G = m.num_heads // m.kv_heads
    rows = []
    for q0, n in seqs:
        s = slice(q0, q0 + n)
        p = torch.einsum("ihd,jhd->hij", q[s], k[s].repeat_interleave(G, 1)) * m.scale
        p = p.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -math.inf).softmax(-1)
        rows.append(torch.einsum("hij,jhd->ihd", p, v[s].repeat_interleave(G, 1)))
    return torch.cat(rows).flatten(-2) @ m.out_proj.weight.detach().double().cpu().T, w


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_layers_together(interleaved):
    """A packed batch through projection, rotation, attention and projection, then a 2-simplicial layer per sequence; fp32,
    forward and gradients.  Sums of at most 128 terms in 32 bits (2^-17 of sums of absolute values, which exceed the
    results by less than 16), in a chain of five: 1e-3 of the largest element leaves room for all of them."""
    torch.manual_seed(3)
    rot = sab.RotaryPositions(24, interleaved=interleaved, device="cuda")
    layer = sab.CausalSelfAttention(64, 4, 32, kv_heads=2, dtype=torch.float32, device="cuda", rotary=rot)
    second = sab.TwoSimplicialSelfAttention(64, 2, 32, 16, 8, dtype=torch.float32, device="cuda", rotary=rot)
    lens = (33, 1, 70)
    cu = torch.tensor([0, 33, 34, 104], dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    x = torch.randn(104, 64, device="cuda", requires_grad=True)
    y = layer(x, positions=pos, cu=cu, max_len=70)
    d = torch.randn_like(y)
    x64 = x.detach().double().cpu().requires_grad_()
    y64, w64 = _layer64(layer, x64, pos.cpu(), [(0, 33), (33, 1), (34, 70)])
    close = lambda a, b: float((a.detach().double().cpu() - b.detach()).abs().max()) <= 1e-3 * float(b.detach().abs().max())
    assert close(y, y64)
    gx, gw = torch.autograd.grad(y, [x, layer.in_proj.weight], d, retain_graph=True)
    rx, rw = torch.autograd.grad(y64, [x64, w64], d.double().cpu())
    assert close(gx, rx) and close(gw, rw)
    # the same rows, sequence by sequence, as a batch of one
    for a, n in ((0, 33), (33, 1), (34, 70)):
        assert close(layer(x[None, a:a + n])[0], y64[a:a + n])
    z = torch.cat([second(y[None, a:b])[0] for a, b in ((0, 33), (33, 34), (34, 104))])
    grads = torch.autograd.grad(z.square().sum(), [x, second.in_proj.weight, layer.out_proj.weight])
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)
    plain = sab.TwoSimplicialSelfAttention(64, 2, 32, 16, 8, dtype=torch.float32, device="cuda")
    plain.load_state_dict(second.state_dict())
    zero = torch.zeros(70, dtype=torch.long, device="cuda")
    assert close(second(y[None, 34:], positions=zero), plain(y[None, 34:]).detach().double().cpu())


# ------------------------------------------------------------------------------------------------ without a GPU
def test_frequencies():
    f = sab.rotary_frequencies(8, 100.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(sab.rotary_frequencies(8, 100.0, "linear", 4.0), f / 4, rtol=1e-15)
    b = sab.rotary_frequencies(8, 100.0, "base", 4.0)
    assert abs(float(b[0]) - 1) < 1e-15 and abs(float(b[-1] * 4 / f[-1]) - 1) < 1e-14
    p = sab.rotary_frequencies(64, 10000.0, "parts", 4.0, original_length=4096)
    turns = sab.rotary_frequencies(64) * 4096 / (2 * math.pi)
    ratio = p / sab.rotary_frequencies(64)
    assert (ratio[turns >= 32] == 1).all() and torch.allclose(ratio[turns <= 1], torch.tensor(0.25, dtype=torch.float64))
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and torch.allclose(ratio[mid], 0.25 + 0.75 * (turns[mid] - 1) / 31)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=-1.0), dict(rotary_dim=8, scaling="x"),
                dict(rotary_dim=8, scaling="parts"), dict(rotary_dim=2, scaling="base"), dict(rotary_dim=8, scaling="parts", original_length=64, low_turns=9, high_turns=9)):
        with pytest.raises(ValueError):
            sab.rotary_frequencies(**bad)


def test_module_keeps_its_frequencies():
    m = sab.RotaryPositions(64, scaling="linear", factor=2.0)
    want = m.frequencies.clone()
    for cast in (lambda: m.half(), lambda: m.to(torch.bfloat16), lambda: m.float()):
        cast()
        assert m.frequencies.dtype == torch.float64 and torch.equal(m.frequencies, want)
    assert not m.state_dict()


def test_entry_validates():
    lib = _abi.load()
    assert ctypes.sizeof(_abi.RotaryParams) == 280
    some = (ctypes.c_void_p * 4)(*[4096] * 4)

    def call(src=some, dst=some, freq=4096, pos=0, **kw):
        p = _abi.RotaryParams()
        p.tensors, p.B, p.N, p.D, p.rotary_dim, p.frequency_bits, p.position_bits = 2, 1, 4, 64, 64, 64, 64
        p.heads[:] = kw.pop("heads", [4, 2, 0, 0])
        for n, x in kw.items():
            setattr(p, n, x)
        return lib.sa_rotary(ctypes.byref(p), src, dst, pos, freq, 0)

    assert lib.sa_rotary(None, some, some, 0, 4096, 0) == 1 and call(src=None) == 1 and call(freq=0) == 1 and call(dst=(ctypes.c_void_p * 4)()) == 1
    for bad in (dict(tensors=0), dict(tensors=5), dict(B=0), dict(N=0), dict(D=0), dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=66),
                dict(heads=[4, 0, 0, 0])):
        assert call(**bad) == 2, bad
    for bad in (dict(dtype=3), dict(frequency_bits=16), dict(pos=4096, position_bits=16), dict(B=1 << 16, N=1 << 16), dict(D=4096, rotary_dim=2050)):
        assert call(**bad) == 4, bad


def test_python_layer_rejects_cpu_tensors(monkeypatch):
    x, f = torch.zeros(1, 8, 2, 64), sab.rotary_frequencies(64)
    for binding in (None, False):
        monkeypatch.setattr(_abi, "_binding", binding)
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            sab.rotary_positions(x, f)
