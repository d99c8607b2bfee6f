"""Rotation, and norm with rotation, against the formulas in float64 on the CPU.

Tolerances, from the arithmetic (u = 2^-24, a float32 rounding): a turned value is one FMA of values
whose cosine and sine are off by at most 3u (argument, sum, magnitude), so it is off by 4u (|x1| + |x2|);
the norm's factor by (E / 2 + 8) u of itself (a sum of E squares halved by the root, the mean, the root
and the quotient), the gradients by the same of each of their terms.  bf16 results are rounded once more,
2^-8 of the value.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def pairs(x, R, interleaved):
    return (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])


def unpairs(a, b, rest, interleaved):
    head = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([head, rest], -1)


def turn64(x, positions, freq, interleaved, mag, sign=1.0):
    """x (B, H, L, E) float64; positions (B, L) int64.  Also the magnitudes that go into each value."""
    R = 2 * freq.numel()
    ang = positions.double()[:, None, :, None] * freq
    c, s = ang.cos() * mag, ang.sin() * mag * sign
    a, b = pairs(x, R, interleaved)
    rest = x[..., R:]
    y = unpairs(a * c - b * s, b * c + a * s, rest, interleaved)
    size = (a.abs() + b.abs()) * mag
    return y, unpairs(size, size, rest.abs(), interleaved)


def close(got, ref, slack, dtype, name):
    got, ref, slack = (t.detach().double().cpu() for t in (got, ref, slack))
    bad = ~((got - ref).abs() <= slack + half_step(dtype) * (ref.abs() + slack))
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()}, worst {float((got - ref).abs().max()):.3e}"


def make(shape, dtype, gen, layout):
    B, H, L, E = shape
    if layout == "blhe":
        return torch.randn(B, L, H, E, generator=gen).to(dtype).to(DEV).transpose(1, 2)
    if layout == "slice":  # rows that start on no 16-byte boundary
        return torch.randn(B, H, L, E + 3, generator=gen).to(dtype).to(DEV)[..., 1:E + 1]
    if layout == "column":  # no unit stride along the head
        return torch.randn(B, H, E, L, generator=gen).to(dtype).to(DEV).transpose(2, 3)
    return torch.randn(B, H, L, E, generator=gen).to(dtype).to(DEV)


CASES = [  # B, H, Hkv, L, E, R, interleaved, layout, positions
    (1, 1, 1, 1, 1, 0, False, "bhle", "offset"),
    (1, 2, 1, 1, 2, 2, False, "bhle", "offset"),
    (2, 3, 3, 5, 7, 4, False, "bhle", "int64"),
    (2, 3, 1, 5, 7, 6, True, "bhle", "int32"),
    (1, 32, 8, 1, 128, 128, False, "blhe", "far"),
    (1, 32, 8, 1, 128, 128, True, "blhe", "far"),
    (3, 12, 12, 37, 64, 32, True, "blhe", "int64"),
    (3, 12, 12, 37, 64, 64, False, "slice", "offset"),
    (2, 8, 2, 129, 80, 80, False, "blhe", "int64"),
    (2, 8, 2, 129, 80, 40, False, "blhe", "row"),
    (2, 5, 5, 33, 100, 50, True, "bhle", "int64"),
    (2, 5, 5, 33, 96, 48, False, "column", "int64"),
    (1, 4, 4, 70, 256, 256, False, "bhle", "far"),
    (1, 2, 2, 19, 512, 512, True, "bhle", "int32"),
    (1, 2, 1, 19, 510, 256, False, "bhle", "int64"),
    (4, 16, 4, 600, 64, 64, False, "bhle", "int64"),
]


def positions_of(kind, B, L, gen):
    """(positions argument, offset argument, int64 (B, L))."""
    if kind == "offset":
        return None, 5, (5 + torch.arange(L)).expand(B, L)
    if kind == "row":
        p = torch.randperm(4 * L, generator=gen)[:L]
        return p.to(DEV), 0, p.expand(B, L)
    top = {"int32": 100, "int64": 100000, "far": (1 << 31) - 5000}[kind]
    p = torch.randint(-50, 50, (B, 1), generator=gen) + top + torch.arange(L)
    return (p.int() if kind == "int32" else p).to(DEV), 0, p


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_rotary(case, dtype):
    from densecore_amd import functional as F
    B, H, Hkv, L, E, R, inter, layout, kind = case
    gen = torch.Generator().manual_seed(1)
    freq, mag = F.rotary_frequencies(R, scaling="yarn", factor=4.0, original_length=64, device=DEV)
    pos, offset, p64 = positions_of(kind, B, L, gen)
    x = [make((B, n, L, E), dtype, gen, layout).requires_grad_(True) for n in (H, Hkv)]
    g = [make((B, n, L, E), dtype, gen, layout) for n in (H, Hkv)]
    y = F.rotary_embedding(*x, freq, positions=pos, offset=offset, interleaved=inter, magnitude=mag)
    dx = torch.autograd.grad(y, x, g)
    # The angle itself carries p f 2^-52, 2^-21 at the farthest position.
    ang = 2.0 ** -52 * float(p64.abs().max()) if R else 0.0
    for i, n in enumerate("qk"):
        assert y[i].is_contiguous() and dx[i].is_contiguous()
        for got, src, sign in ((y[i], x[i], 1.0), (dx[i], g[i], -1.0)):
            ref, size = turn64(src.detach().double().cpu(), p64, freq.cpu(), inter, mag, sign)
            close(got, ref, (4 * U + ang) * size, dtype, f"{n} {sign}")
    alone = F.rotary_embedding(x[0].detach(), None, freq, positions=pos, offset=offset, interleaved=inter, magnitude=mag)
    assert torch.equal(alone, y[0])


@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.bfloat16, torch.float32)], ids=["f32", "bf16", "mixed"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_qk_norm_rotary(case, dtype, wtype):
    from densecore_amd import functional as F
    B, H, Hkv, L, E, R, inter, layout, kind = case
    gen = torch.Generator().manual_seed(2)
    eps = 1e-3
    freq, mag = F.rotary_frequencies(R, scaling="yarn", factor=4.0, original_length=64, device=DEV)
    pos, offset, p64 = positions_of(kind, B, L, gen)
    x = [make((B, n, L, E), dtype, gen, layout).requires_grad_(True) for n in (H, Hkv)]
    g = [make((B, n, L, E), dtype, gen, layout) for n in (H, Hkv)]
    w = [(torch.randn(E, generator=gen) * 0.2 + 1).to(wtype).to(DEV).requires_grad_(True) for _ in range(2)]
    y = F.qk_norm_rotary(*x, *w, freq, positions=pos, offset=offset, interleaved=inter, magnitude=mag, eps=eps)
    d = torch.autograd.grad(y, (*x, *w), g)
    ang = 2.0 ** -52 * float(p64.abs().max()) if R else 0.0
    k = (E / 2 + 12) * U + ang
    for i, n in enumerate("qk"):
        x64, w64, g64 = (t.detach().double().cpu() for t in (x[i], w[i], g[i]))
        r = 1 / (x64.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        ref, size = turn64(x64 * r * w64, p64, freq.cpu(), inter, mag)
        close(y[i], ref, k * size, dtype, f"{n} out")
        t, tsize = turn64(g64, p64, freq.cpu(), inter, mag, -1.0)
        s = (t * w64 * x64).mean(-1, keepdim=True)
        ref = r * (t * w64 - x64 * r * r * s)
        size = r * (tsize * w64.abs() + x64.abs() * r * r * (tsize * w64.abs() * x64.abs()).mean(-1, keepdim=True))
        close(d[i], ref, 3 * k * size, dtype, f"d{n}")
        rows = x64.numel() // E
        size = (tsize * x64.abs() * r).sum((0, 1, 2))
        close(d[2 + i], (t * x64 * r).sum((0, 1, 2)), (k + rows * U) * size, wtype, f"dw{n}")


def test_gradients_against_differences():
    """d(sum y g) along a direction, from float64 differences of the plain form on the same values."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(3)
    B, H, L, E, eps = 2, 3, 9, 32, 1e-3
    freq, mag = F.rotary_frequencies(E, device=DEV)
    x, g, dirx = (torch.randn(B, H, L, E, generator=gen) for _ in range(3))
    w, dirw = torch.randn(E, generator=gen), torch.randn(E, generator=gen)
    xg, wg = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y, _ = F.qk_norm_rotary(xg, xg.detach(), wg, None, freq, eps=eps)
    dx, dw = torch.autograd.grad(y, (xg, wg), g.to(DEV))

    def f(h):
        a, b = x.double() + h * dirx.double(), w.double() + h * dirw.double()
        u = a / (a.pow(2).mean(-1, keepdim=True) + eps).sqrt() * b
        return float((turn64(u, torch.arange(L).expand(B, L), freq.cpu(), False, mag)[0] * g.double()).sum())
    h = 1e-5
    want = (f(h) - f(-h)) / (2 * h)
    got = float((dx.cpu().double() * dirx).sum() + (dw.cpu().double() * dirw).sum())
    # Float32 gradients of 1760 terms of size about 1: 1760 u (E / 2 + 16) at the very worst.
    assert abs(got - want) <= 1760 * (E / 2 + 16) * U


def test_no_weights_empty_frequencies_and_shared_tensor():
    from densecore_amd import functional as F
    x = torch.randn(2, 3, 11, 48, device=DEV)
    empty = F.rotary_frequencies(0, device=DEV)[0]
    q, k = F.qk_norm_rotary(x, x, None, None, empty, eps=1e-6)
    ref = x.double() / (x.double().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
    close(q, ref, 40 * U * ref.abs(), torch.float32, "norm alone")
    assert torch.equal(q, k)
    a, b = F.rotary_embedding(x, x, empty)
    assert torch.equal(a, x) and torch.equal(b, x)


def test_empty_tensors():
    from densecore_amd import functional as F
    freq = F.rotary_frequencies(8, device=DEV)[0]
    for shape in ((0, 2, 3, 8), (2, 2, 0, 8)):
        x, w = torch.zeros(shape, device=DEV, requires_grad=True), torch.ones(8, device=DEV, requires_grad=True)
        q, k = F.rotary_embedding(x, x, freq)
        assert q.shape == shape and k.shape == shape
        q, k = F.qk_norm_rotary(x, x, w, w, freq)
        dx, dw = torch.autograd.grad((q, k), (x, w), (torch.zeros(shape, device=DEV),) * 2)
        assert dx.shape == shape and torch.equal(dw, torch.zeros(8, device=DEV))


def test_values_that_are_not_finite_stay_in_their_pairs():
    from densecore_amd import functional as F
    x = torch.randn(1, 2, 6, 16, device=DEV)
    clean = F.rotary_embedding(x, None, F.rotary_frequencies(16, device=DEV)[0])
    x[0, 0, 2, 3] = float("nan")
    x[0, 1, 4, 9] = float("inf")
    y = F.rotary_embedding(x, None, F.rotary_frequencies(16, device=DEV)[0])
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[0, 0, 2, [3, 11]] = True
    hit[0, 1, 4, [1, 9]] = True
    assert torch.equal(y[~hit], clean[~hit]) and not torch.isfinite(y[hit]).any()


def test_broadcast_gradient_and_one_output_used():
    """A gradient of stride 0 (from a sum) and an output that takes no part in the loss."""
    from densecore_amd import functional as F
    freq = F.rotary_frequencies(64, device=DEV)[0]
    q = torch.randn(2, 4, 9, 64, device=DEV, requires_grad=True)
    k = torch.randn(2, 2, 9, 64, device=DEV, requires_grad=True)
    a, _ = F.rotary_embedding(q, k, freq, offset=3)
    dq, dk = torch.autograd.grad(a.sum(), (q, k))
    ones = torch.ones_like(q)
    ref, size = turn64(ones.double().cpu(), (3 + torch.arange(9)).expand(2, 9), freq.cpu(), False, 1.0, -1.0)
    close(dq, ref, 4 * U * size, torch.float32, "dq")
    assert torch.equal(dk, torch.zeros_like(k))


def test_weight_gradients_repeat_bit_for_bit():
    from densecore_amd import functional as F
    freq = F.rotary_frequencies(128, device=DEV)[0]
    q = torch.randn(4, 16, 1000, 128, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    w = torch.ones(128, device=DEV, requires_grad=True)
    g = torch.randn_like(q)
    runs = []
    for _ in range(3):
        a, b = F.qk_norm_rotary(q, q, w, w, freq)
        runs.append(torch.autograd.grad((a, b), (q, w), (g, g)))
    for r in runs[1:]:
        assert torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1])


def test_rows_beyond_31_bits():
    """A strided input whose last row starts past 2^31 elements."""
    from densecore_amd import functional as F
    base = torch.zeros((1 << 31) + 4096, device=DEV, dtype=torch.bfloat16)
    step = 1 << 30
    x = base.as_strided((3, 1, 2, 64), (step, 64, 64, 1))
    x.copy_(torch.randn(3, 1, 2, 64, device=DEV))
    freq = F.rotary_frequencies(64, device=DEV)[0]
    assert torch.equal(F.rotary_embedding(x, None, freq), F.rotary_embedding(x.contiguous(), None, freq))


def test_streams_and_graphs():
    """Two streams at once, then a captured forward and backward replayed on new inputs."""
    from densecore_amd import functional as F
    freq = F.rotary_frequencies(128, device=DEV)[0]
    weight = torch.rand(128, device=DEV) + 0.5

    def step(q, g):
        # Leaves of its own, and no autograd graph of them left behind: torch cannot capture a backward
        # pass while an eager graph of the same leaves lives.
        q, w = q.detach().requires_grad_(True), weight.detach().requires_grad_(True)
        a, b = F.qk_norm_rotary(q, q, w, None, freq, offset=7)
        return (a.detach(), b.detach(), *torch.autograd.grad((a, b), (q, w), (g, g)))
    xs = [torch.randn(2, 8, 333, 128, device=DEV) for _ in range(4)]
    gs = [torch.randn_like(x) for x in xs]
    ref = [step(x, g) for x, g in zip(xs, gs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None] * 4
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = step(xs[i], gs[i])
    torch.cuda.synchronize()
    for a, b in zip(ref, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    x, g = xs[0].clone(), gs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, g)
    for i in (1, 2, 3, 1):
        x.copy_(xs[i]), g.copy_(gs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(out, ref[i])), i
        assert np.isfinite(float(torch.randn(1000, device=DEV).sum()))  # eager work between replays


@pytest.mark.parametrize("bad", ["dtype", "freq", "freq_dim", "freq_dtype", "positions", "positions_dtype",
                                 "weight", "weight_types", "both"])
def test_refusals(bad):
    from densecore_amd import functional as F
    x, f = torch.zeros(2, 2, 3, 8, device=DEV), F.rotary_frequencies(8, device=DEV)[0]
    w, kw = None, {}
    k = x
    if bad == "dtype":
        k = x.bfloat16()
    if bad == "freq":
        f = f.cpu()
    if bad == "freq_dim":
        f = F.rotary_frequencies(10, device=DEV)[0]
    if bad == "freq_dtype":
        f = f.float()
    if bad == "positions":
        kw["positions"] = torch.zeros(4, device=DEV, dtype=torch.int64)
    if bad == "positions_dtype":
        kw["positions"] = torch.zeros(3, device=DEV)
    if bad == "both":
        kw.update(positions=torch.zeros(3, device=DEV, dtype=torch.int64), offset=1)
    if bad == "weight":
        w = torch.ones(7, device=DEV)
    wk = torch.ones(8, device=DEV, dtype=torch.bfloat16) if bad == "weight_types" else None
    if bad == "weight_types":
        w = torch.ones(8, device=DEV)
    with pytest.raises(ValueError):
        F.qk_norm_rotary(x, k, w, wk, f, **kw)


def test_head_dim_limit():
    from densecore_amd import functional as F
    x = torch.zeros(1, 1, 1, 514, device=DEV)
    with pytest.raises(NotImplementedError):
        F.rotary_embedding(x, x, F.rotary_frequencies(8, device=DEV)[0])
