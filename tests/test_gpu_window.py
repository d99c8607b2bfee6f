"""Window attention and its decode form against the formulas in float64.

Tolerances, from the arithmetic (u = 2^-24): a score is a sum of E products, off by (E + 8) u of the sum
of their magnitudes; its exponential by twice that (the score and the row's maximum or lse) and 2^-20 for
the base-2 functions and the lse's own rounding; P and dS in bf16 calls are carried to 2^-16.  Sums of n
terms are off by n u of their magnitudes, dsum takes the output as it was rounded, and results are rounded
once more, half a step of the type.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(p, S, window, sinks):
    s = torch.arange(S, device=p.device)
    return (s <= p[..., None]) & ((s > p[..., None] - window) | (s < sinks))


def close(got, ref, slack, dtype, name):
    got = got.detach().double().to(ref.device)
    bad = ~((got - ref).abs() <= slack + half_step(dtype) * (ref.abs() + slack) + 1e-30)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - ref).abs().max()):.3e}, "
                           f"first {bad.nonzero()[0].tolist()}")


def formulas(q, k, v, open_, scale, dtype, g=None):
    """{name: (value, slack)} in float64; open_ (L, S) or (B, 1, L, S)."""
    q, k, v = (t.detach().double() for t in (q, k, v))
    rep, E, n = q.shape[1] // k.shape[1], q.shape[-1], max(k.shape[2], q.shape[2] * (q.shape[1] // k.shape[1]))
    kk, vv = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = (q @ kk.transpose(2, 3)) * scale
    s = torch.where(open_, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    e = torch.where(open_, (s - torch.where(m == -math.inf, 0.0, m)).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    size = torch.where(open_, (q.abs() @ kk.abs().transpose(2, 3)) * abs(scale), 0.0)
    prel = 2 * (E + 8) * U * size.amax(-1, keepdim=True) + 2.0 ** -20 + (2.0 ** -16 if dtype == torch.bfloat16 else 0)
    o = p @ vv
    r = {"out": (o, (p * (prel + n * U)) @ vv.abs()),
         "lse": (torch.where(total == 0, 0.0, torch.where(m == -math.inf, 0.0, m) + total.log())[..., 0],
                 prel[..., 0] + 2.0 ** -20)}
    if g is None:
        return r
    g = g.detach().double()

    def group(t):
        return t.reshape(t.shape[0], k.shape[1], rep, *t.shape[2:]).sum(2)
    dp, dsum = g @ vv.transpose(2, 3), (g * o).sum(-1, keepdim=True)
    ds = p * (dp - dsum)
    osize = (g.abs() * o.abs()).sum(-1, keepdim=True)
    dslack = ((E + 8) * U * (g.abs() @ vv.abs().transpose(2, 3)) + (half_step(dtype) + (E + 8) * U + prel) * osize)
    dss = p * ((prel + 4 * U) * (dp - dsum).abs() + dslack) + (2.0 ** -16 if dtype == torch.bfloat16 else 4 * U) * ds.abs()
    ps, a = p * (prel + n * U), abs(scale)
    r["dq"] = ((ds @ kk) * scale, ((dss + n * U * ds.abs()) @ kk.abs()) * a)
    r["dk"] = (group(ds.transpose(2, 3) @ q) * scale, group((dss + n * U * ds.abs()).transpose(2, 3) @ q.abs()) * a)
    r["dv"] = (group(p.transpose(2, 3) @ g), group(ps.transpose(2, 3) @ g.abs()))
    return r


CASES = [  # B, H, Hkv, L, S, E, window, sinks, offset
    (1, 1, 1, 1, 1, 1, 1, 0, 0),
    (1, 2, 1, 1, 5, 7, 2, 1, 4),
    (2, 2, 2, 33, 33, 31, 1, 0, 0),
    (2, 2, 2, 33, 33, 32, 5, 0, 0),
    (1, 3, 1, 130, 130, 33, 32, 4, 0),
    (2, 4, 2, 200, 200, 64, 64, 4, 0),
    (1, 4, 4, 300, 300, 64, 100, 40, 0),
    (1, 2, 2, 257, 257, 80, 1000, 4, 0),
    (1, 2, 1, 500, 500, 96, 77, 130, 0),
    (1, 8, 2, 384, 384, 128, 128, 1, 0),
    (1, 2, 2, 700, 700, 128, 200, 0, 0),
    (2, 2, 2, 290, 290, 100, 65, 33, 0),
    (1, 8, 1, 5, 700, 64, 300, 4, 695),       # the last few queries: packed heads, split keys
    (2, 16, 2, 17, 2000, 128, 1024, 16, 1983),
    (1, 6, 2, 40, 900, 128, 90, 500, 300),    # queries in the middle of the keys
    (1, 2, 2, 3, 5000, 128, 3000, 4, 4997),
    (1, 2, 1, 150, 150, 64, 20, 0, 60),       # the last rows see no key
    (1, 2, 1, 150, 40, 64, 20, 3, 0),         # more queries than keys
    (1, 2, 2, 64, 64, 128, 8, 0, 500),        # no row sees a key
    (1, 2, 2, 160, 160, 64, 48, 200, 0),      # all sinks
    (1, 1, 1, 1000, 1000, 32, 129, 65, 0),
]


@TYPES
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradients(case, dtype):
    from densecore_amd import _native
    from densecore_amd import functional as F
    B, H, Hkv, L, S, E, window, sinks, offset = case
    gen = torch.Generator().manual_seed(1)
    q, k, v, g = (torch.randn(*s, E, generator=gen).to(dtype).to(DEV)
                  for s in ((B, H, L), (B, Hkv, S), (B, Hkv, S), (B, H, L)))
    ref = formulas(q, k, v, visible(offset + torch.arange(L, device=DEV), S, window, sinks), 1 / math.sqrt(E), dtype, g)
    out, lse = _native._window_attention(q, k, v, window, sinks, offset)
    close(out, *ref["out"], dtype, "out")
    close(lse, *ref["lse"], torch.float32, "lse")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    y = F.window_attention(*leaves, window, sinks, offset=offset)
    assert torch.equal(y, out)
    for name, d in zip(("dq", "dk", "dv"), torch.autograd.grad(y, leaves, g)):
        assert d.is_contiguous()
        close(d, *ref[name], dtype, name)


MANY = [  # enough rows and heads to fill the device (other kernels, grids and pieces than a few heads take)
    (16, 16, 4, 300, 300, 64, 100, 4, 0),
    (16, 16, 16, 257, 257, 24, 1, 0, 0),
    (9, 30, 10, 400, 400, 96, 130, 70, 0),
    (8, 16, 2, 513, 700, 128, 300, 4, 187),
    (8, 32, 32, 260, 130, 32, 64, 0, 3),
    (4, 64, 64, 300, 300, 128, 4000, 0, 0),
    (3, 8, 4, 1500, 1500, 80, 64, 4, 0),
    (17, 16, 8, 290, 290, 100, 30, 200, 0),
]


@TYPES
@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(map(str, c)))
def test_many_heads(case, dtype):
    test_forward_and_gradients(case, dtype)


@TYPES
def test_many_heads_with_values_that_are_not_finite(dtype):
    """As test_hidden_keys_have_no_influence, on a grid that fills the device."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(17)
    B, H, L, E, window = 8, 32, 300, 64, 50
    q, k, v, g = (torch.randn(B, H, L, E, generator=gen).to(dtype).to(DEV) for _ in range(4))
    ref = formulas(q, k, v, visible(torch.arange(L, device=DEV), L, window, 0), 1 / math.sqrt(E), dtype, g)
    k2, v2 = k.clone(), v.clone()
    k2[3, 7, 100], v2[3, 7, 100] = math.nan, math.inf
    leaves = [t.requires_grad_(True) for t in (q, k2, v2)]
    y = F.window_attention(*leaves, window)
    hit = torch.zeros(B, H, L, dtype=torch.bool, device=DEV)
    hit[3, 7, 100:100 + window] = True
    assert torch.isnan(y[hit]).all()
    near = torch.zeros_like(hit)
    near[3, 7, 100 - window + 1:100 + window] = True
    dq, dk, dv = torch.autograd.grad(y, leaves, g)
    for name, d, m in (("out", y, hit), ("dq", dq, hit), ("dk", dk, near), ("dv", dv, near)):
        close(d[~m], ref[name][0][~m], ref[name][1].expand_as(ref[name][0])[~m], dtype, name)


@TYPES
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_scales(scale, dtype):
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(2)
    q, k, v, g = (torch.randn(1, 2, 150, 32, generator=gen).to(dtype).to(DEV) for _ in range(4))
    ref = formulas(q, k, v, visible(torch.arange(150, device=DEV), 150, 40, 2), scale, dtype, g)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    y = F.window_attention(*leaves, 40, 2, scale=scale)
    close(y, *ref["out"], dtype, "out")
    for name, d in zip(("dq", "dk", "dv"), torch.autograd.grad(y, leaves, g)):
        close(d, *ref[name], dtype, name)


@TYPES
@pytest.mark.parametrize("layout", ["blhe", "slice", "column", "expand"])
def test_strides(layout, dtype):
    """Views are read as they lie: the results of their contiguous copies, bit for bit where rows keep
    their 16-byte alignment."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(3)
    B, H, L, E = 2, 4, 140, 64

    def make(heads):
        if layout == "blhe":
            return torch.randn(B, L, heads, E, generator=gen).to(dtype).to(DEV).transpose(1, 2)
        if layout == "slice":
            return torch.randn(B, heads, L + 3, E + 5, generator=gen).to(dtype).to(DEV)[:, :, 2:-1, 3:-2]
        if layout == "column":
            return torch.randn(B, heads, E, L, generator=gen).to(dtype).to(DEV).transpose(2, 3)
        return torch.randn(B, 1, L, E, generator=gen).to(dtype).to(DEV).expand(B, heads, L, E)
    x = [make(n) for n in (H, 2, 2)]
    g = make(H)

    def run(q, k, v, g):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        y = F.window_attention(*leaves, 50, 4)
        return (y, *torch.autograd.grad(y, leaves, g))
    a, b = run(*x, g), run(*(t.contiguous() for t in (*x, g)))
    ref = formulas(*x, visible(torch.arange(L, device=DEV), L, 50, 4), 1 / math.sqrt(E), dtype, g)
    for s, t, name in zip(a, b, ("out", "dq", "dk", "dv")):
        close(s, *ref[name], dtype, name)
        if layout != "slice":
            assert torch.equal(s, t), name


@TYPES
def test_hidden_keys_have_no_influence(dtype):
    """NaN and infinities in keys and values that a query does not see (before its window, behind it, past
    the end of what any query sees), and in queries that do not see a key: nothing changes."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(4)
    L, S, E, window, sinks, offset = 90, 300, 64, 32, 4, 100
    q, k, v, g = (torch.randn(1, 2, n, E, generator=gen).to(dtype).to(DEV) for n in (L, S, S, L))

    def run(q, k, v, g):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        y = F.window_attention(*leaves, window, sinks, offset=offset)
        return (y.detach(), *torch.autograd.grad(y, leaves, g))
    ref = formulas(q, k, v, visible(offset + torch.arange(L, device=DEV), S, window, sinks), 1 / math.sqrt(E), dtype, g)
    # Keys no query sees: 4 .. 68 and 190 ..; every kind of value there.
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max], device=DEV).to(dtype)
    k2, v2 = k.clone(), v.clone()
    hidden = torch.cat([torch.arange(sinks, offset - window + 1), torch.arange(offset + L, S)]).to(DEV)
    k2[:, :, hidden] = bad[torch.arange(len(hidden), device=DEV) % 4][:, None]
    v2[:, :, hidden] = bad[torch.arange(len(hidden), device=DEV) % 3][:, None]
    for name, d in zip(("out", "dq", "dk", "dv"), run(q, k2, v2, g)):
        close(d, *ref[name], dtype, name)
    # Key 120 is seen by the queries at 120 .. 151: with NaN there the others keep their results.
    k3, v3 = k.clone(), v.clone()
    k3[:, :, 120] = math.nan
    v3[:, :, 120] = math.nan
    out, dq, dk, dv = run(q, k3, v3, g)
    rows = torch.arange(L, device=DEV) + offset
    sees = (rows >= 120) & (rows < 120 + window)
    assert torch.isnan(out[:, :, sees]).all() and torch.isnan(dq[:, :, sees]).all()
    for name, d in (("out", out), ("dq", dq)):
        value, slack = (t[:, :, ~sees] for t in ref[name])
        close(d[:, :, ~sees], value, slack, dtype, name)
    # Their gradients reach the keys those queries see, and no others.
    s = torch.arange(S, device=DEV)
    touched = (s < sinks) | ((s > 120 - window) & (s < 120 + window))
    for name, d in (("dk", dk), ("dv", dv)):
        assert torch.isnan(d[:, :, touched]).all()
        value, slack = (t[:, :, ~touched] for t in ref[name])
        close(d[:, :, ~touched], value, slack, dtype, name)


@TYPES
def test_infinite_key_that_is_seen(dtype):
    """A key of -inf dims against queries of positive ones scores -inf: it takes no part."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(5)
    q, k, v = (torch.rand(1, 1, 70, 32, generator=gen).add_(0.1).to(dtype).to(DEV) for _ in range(3))
    k2 = k.clone()
    k2[:, :, 30] = -math.inf
    open_ = visible(torch.arange(70, device=DEV), 70, 16, 1)
    open_[:, 30] = False
    ref = formulas(q, k, v, open_, 1 / math.sqrt(32), dtype)
    close(F.window_attention(q, k2, v, 16, 1), *ref["out"], dtype, "out")


def test_large_values_float32():
    """Values near the type's largest: the split products overflow, the results do not."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(1, 1, 80, 32, generator=gen).to(DEV) for _ in range(3))
    v = v * 0 + 3.4e38 * (1 - 2.0 ** -10 * torch.rand(1, 1, 80, 32, generator=gen).to(DEV))
    out = F.window_attention(q, k, v, 20, 2)
    ref = formulas(q, k, v, visible(torch.arange(80, device=DEV), 80, 20, 2), 1 / math.sqrt(32), torch.float32)
    assert torch.isfinite(out).all()
    close(out, *ref["out"], torch.float32, "out")


@TYPES
def test_gradient_against_differences(dtype):
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(7)
    q, k, v, g, dq, dk, dv = (torch.randn(1, 2, 60, 32, generator=gen).to(dtype) for _ in range(7))
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    y = F.window_attention(*leaves, 20, 3)
    grads = torch.autograd.grad(y, leaves, g.to(DEV))
    open_ = visible(torch.arange(60), 60, 20, 3)

    def f(h):
        a = [t.double() + h * d.double() for t, d in zip((q, k, v), (dq, dk, dv))]
        s = torch.where(open_, a[0] @ a[1].transpose(2, 3) / math.sqrt(32), -math.inf)
        return float((torch.softmax(s, -1) @ a[2] * g.double()).sum())
    h = 1e-5
    want = (f(h) - f(-h)) / (2 * h)
    ref = formulas(*(t.to(DEV) for t in (q, k, v)), open_.to(DEV), 1 / math.sqrt(32), dtype, g.to(DEV))
    slack = sum(float(((half_step(dtype) * ref[n][0].abs() + ref[n][1]) * d.to(DEV).double().abs()).sum())
                for n, d in (("dq", dq), ("dk", dk), ("dv", dv)))
    got = sum(float((a.cpu().double() * d.double()).sum()) for a, d in zip(grads, (dq, dk, dv)))
    assert abs(got - want) <= slack + 1e-6


def test_rows_that_see_one_key_have_no_query_gradient():
    """Softmax over one key is 1 whatever the query: dq is 0 but for float32's rounding of terms of size
    |dO| |V|, also where the output was rounded to bf16 (2^-16 with its rest)."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(16)
    for dtype, u in ((torch.float32, U), (torch.bfloat16, 2.0 ** -16)):
        q, k, v, g = (torch.randn(1, 2, 100, 64, generator=gen).to(dtype).to(DEV) for _ in range(4))
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        dq = torch.autograd.grad(F.window_attention(*leaves, 1), leaves, g)[0]
        size = (g.double().abs() * v.detach().double().abs()).sum(-1, keepdim=True) * k.detach().double().abs() / 8
        assert (dq.double().abs() <= (64 + 8) * U * size + u * size).all()


@TYPES
def test_rows_behind_the_results_are_left_alone(dtype):
    """Outputs, gradients and workspaces in the middle of larger buffers."""
    from densecore_amd import _lib, _native
    B, H, Hkv, L, S, E = 1, 4, 2, 70, 131, 64
    gen = torch.Generator().manual_seed(8)
    q, k, v, g = (torch.randn(*s, E, generator=gen).to(dtype).to(DEV)
                  for s in ((B, H, L), (B, Hkv, S), (B, Hkv, S), (B, H, L)))
    d = _native._window_desc(q, k, v, 40, 4, 61, None, g)
    L_, mark, pad = _lib.lib(), 7.0, 4096

    def room(n, dt):
        return torch.full((n + 2 * pad,), mark, dtype=dt, device=DEV)
    out, lse = room(q.numel(), dtype), room(B * H * L, torch.float32)
    grads = [room(t.numel(), dtype) for t in (q, k, v)]
    fw, bw = L_.dc_window_fwd_workspace_size(d), L_.dc_window_bwd_workspace_size(d)
    ws = [room(max(n, 1) // 4 + 1, torch.float32) for n in (fw, bw)]

    def at(t):
        return t.data_ptr() + pad * t.element_size()
    st = _native._stream(q.device)
    _lib.check(L_.dc_window_fwd(d, q.data_ptr(), k.data_ptr(), v.data_ptr(), at(out), None, at(lse), at(ws[0]), fw, st))
    _lib.check(L_.dc_window_bwd(d, g.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), at(out), None, at(lse),
                                *(at(t) for t in grads), at(ws[1]), bw, st))
    torch.cuda.synchronize()
    for t in (out, lse, *grads, *ws):
        assert (t[:pad] == mark).all() and (t[-pad:] == mark).all()
    ref = formulas(q, k, v, visible(61 + torch.arange(L, device=DEV), S, 40, 4), 1 / math.sqrt(E), dtype, g)
    for t, name in zip((out, *grads), ("out", "dq", "dk", "dv")):
        close(t[pad:-pad].reshape(ref[name][0].shape), *ref[name], dtype, name)


DECODE = [  # B, H, Hkv, S, E, window, sinks, lengths
    (1, 1, 1, 1, 1, 1, 0, None),
    (1, 6, 6, 255, 64, 128, 4, None),
    (3, 4, 2, 100, 31, 7, 2, [100, 1, 0]),
    (4, 6, 2, 300, 80, 64, 4, [300, 64, 65, 70]),
    (2, 8, 1, 3000, 128, 1000, 16, [3000, 17]),
    (2, 14, 2, 2000, 128, 5000, 4, [1999, 2000]),
    (1, 16, 1, 4097, 256, 4096, 4, None),
    (5, 2, 2, 500, 96, 1, 0, [500, 499, 1, 2, 250]),
    (2, 3, 1, 333, 100, 50, 400, [333, 200]),
    (2, 5, 1, 700, 40, 300, 1, [-3, 900]),     # clamped to 0 and S
]


@TYPES
@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(map(str, c[:7])))
def test_decode(case, dtype):
    from densecore_amd import _native
    B, H, Hkv, S, E, window, sinks, lengths = case
    gen = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(*s, E, generator=gen).to(dtype).to(DEV) for s in ((B, H, 1), (B, Hkv, S), (B, Hkv, S)))
    n = torch.tensor(lengths or [S] * B)
    open_ = visible(n.clamp(0, S).to(DEV)[:, None] - 1, S, window, sinks)[:, None]
    ref = formulas(q, k, v, open_, 1 / math.sqrt(E), dtype)
    for kind in (torch.int64, torch.int32):
        out, lse = _native._window_decode(q, k, v, window, sinks, None if lengths is None else n.to(kind).to(DEV))
        close(out, *ref["out"], dtype, "out")
        close(lse, *ref["lse"], torch.float32, "lse")


@TYPES
def test_decode_does_not_read_hidden_rows(dtype):
    """Rows behind the length and outside the window hold NaN; the cache is a view of a longer one."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(10)
    B, H, Hkv, S, E, window, sinks = 3, 8, 2, 900, 64, 100, 4
    q = torch.randn(B, H, 1, E, generator=gen).to(dtype).to(DEV)
    k, v = (torch.randn(B, Hkv, S + 50, E, generator=gen).to(dtype).to(DEV) for _ in range(2))
    n = torch.tensor([900, 333, 102], device=DEV)
    open_ = visible(n[:, None] - 1, S, window, sinks)[:, None]
    ref = formulas(q, k[:, :, :S], v[:, :, :S], open_, 1 / math.sqrt(E), dtype)
    for t in (k, v):
        t[:, :, :S][~open_.expand(B, Hkv, 1, S)[:, :, 0]] = math.nan
        t[:, :, S:] = math.nan
    close(F.window_decode(q, k[:, :, :S], v[:, :, :S], window, sinks, lengths=n), *ref["out"], dtype, "out")


@TYPES
def test_decode_is_the_last_row_of_attention(dtype):
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(2, n, 777, 64, generator=gen).to(dtype).to(DEV) for n in (8, 2, 2))
    full = F.window_attention(q, k, v, 256, 4)
    open_ = visible(torch.tensor([776], device=DEV), 777, 256, 4)
    ref = formulas(q[:, :, -1:], k, v, open_, 0.125, dtype)
    close(F.window_decode(q[:, :, -1:], k, v, 256, 4), *ref["out"], dtype, "decode")
    close(full[:, :, -1:], *ref["out"], dtype, "attention")
    tail = F.window_attention(q[:, :, -9:], k, v, 256, 4, offset=768)
    close(tail[:, :, -1:], *ref["out"], dtype, "chunk")


def test_offsets_beyond_31_bits():
    """Caches of more than 2^31 elements: decode, forward and backward on their last head."""
    from densecore_amd import functional as F
    H, S, E = 17, 1 << 20, 128
    k = torch.zeros(1, H, S, E, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(1, H, S, E, dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator().manual_seed(12)
    tail = [torch.randn(1, H, 400, E, generator=gen).bfloat16().to(DEV) for _ in range(2)]
    k[:, :, -400:], v[:, :, -400:] = tail
    q = torch.randn(1, H, 40, E, generator=gen).bfloat16().to(DEV)
    # A window of 300 keys: the last 340 hold all that the last 40 queries see.
    ref = formulas(q, *tail, visible(360 + torch.arange(40, device=DEV), 400, 300, 0), 1 / math.sqrt(E), torch.bfloat16)
    close(F.window_attention(q, k, v, 300, offset=S - 40), *ref["out"], torch.bfloat16, "out")
    close(F.window_decode(q[:, :, -1:], k, v, 300), *(t[:, :, -1:] for t in ref["out"]), torch.bfloat16, "decode")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(F.window_attention(*leaves, 300, offset=S - 40), leaves, torch.ones_like(q))
    ref = formulas(q, *tail, visible(360 + torch.arange(40, device=DEV), 400, 300, 0), 1 / math.sqrt(E), torch.bfloat16,
                   torch.ones_like(q))
    close(dq, *ref["dq"], torch.bfloat16, "dq")
    close(dk[:, :, -400:], *ref["dk"], torch.bfloat16, "dk")
    close(dv[:, :, -400:], *ref["dv"], torch.bfloat16, "dv")
    assert not dk[:, :, :-400].any() and not dv[:, :, :-400].any()


@TYPES
def test_repeats_streams_and_graphs(dtype):
    """Bit-identical from run to run, on two streams at once, and captured with its backward."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(13)

    def inputs():
        return [torch.randn(1, n, 500, 64, generator=gen).to(dtype).to(DEV) for n in (4, 2, 2, 4)]

    def step(q, k, v, g):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        y = F.window_attention(*leaves, 100, 4)
        few = F.window_attention(q[:, :, -3:].detach(), k.detach(), v.detach(), 400, 4, offset=497)
        one = F.window_decode(q[:, :, -1:], k, v, 450, 4)
        return (y.detach(), few, one, *torch.autograd.grad(y, leaves, g))
    xs = [inputs() for _ in range(4)]
    ref = [step(*x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step(*xs[i]))
    torch.cuda.synchronize()
    for a, b in zip(ref, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    x = [t.clone() for t in xs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*x)
    for i in (1, 2, 3, 1):
        for s, t in zip(x, xs[i]):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(out, ref[i])), i
        assert float(torch.ones(1000, device=DEV).sum()) == 1000  # eager work between replays


@TYPES
def test_empty_tensors(dtype):
    from densecore_amd import functional as F
    for shape in ((0, 2, 3, 8), (1, 2, 0, 8)):
        x = torch.zeros(shape, dtype=dtype, device=DEV, requires_grad=True)
        y = F.window_attention(x, x, x, 4)
        assert y.shape == shape and torch.autograd.grad(y, x, torch.zeros_like(y))[0].shape == shape
    q = torch.randn(1, 2, 5, 8, dtype=torch.float32, device=DEV).to(dtype).requires_grad_(True)
    k = torch.zeros(1, 2, 0, 8, dtype=dtype, device=DEV, requires_grad=True)
    y = F.window_attention(q, k, k, 4, 2)
    dq, dk = torch.autograd.grad(y, (q, k), torch.ones_like(y))
    assert not y.any() and not dq.any() and dk.shape == k.shape
    assert not F.window_decode(q[:, :, :1], k, k, 4).any()
    none = torch.zeros(1, 2, 0, 8, dtype=dtype, device=DEV, requires_grad=True)
    z = F.window_attention(none, q.detach().requires_grad_(True), q, 4)
    assert z.shape == none.shape


def test_one_layer_from_projection_to_cache():
    """Norm and rotation, window attention and its gradients; then the same tokens one at a time through the
    cache: what the operators are for, together."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(14)
    B, L, H, Hkv, E, window, sinks = 2, 150, 8, 2, 64, 48, 4
    width = (H + 2 * Hkv) * E
    x = torch.randn(B, L, width, generator=gen).to(DEV)
    wq, wk = (torch.rand(E, generator=gen).add_(0.5).to(DEV) for _ in range(2))
    freq, mag = F.rotary_frequencies(E, scaling="yarn", factor=2.0, original_length=64, device=DEV)

    def layer(x, wq, wk):
        q, k, v = (t.unflatten(-1, (-1, E)).transpose(1, 2) for t in x.split((H * E, Hkv * E, Hkv * E), -1))
        q, k = F.qk_norm_rotary(q, k, wq, wk, freq, magnitude=mag)
        return F.window_attention(q, k, v, window, sinks), k, v
    leaves = [t.requires_grad_(True) for t in (x, wq, wk)]
    y, k, v = layer(*leaves)
    g = torch.randn(y.shape, generator=gen).to(DEV)
    grads = torch.autograd.grad(y, leaves, g)

    def plain(x, wq, wk):
        q, k, v = (t.unflatten(-1, (-1, E)).transpose(1, 2) for t in x.split((H * E, Hkv * E, Hkv * E), -1))

        def turn(t, w):
            t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
            ang = torch.arange(L, device=DEV).double()[:, None] * freq
            c, s, (a, b) = ang.cos() * mag, ang.sin() * mag, t.chunk(2, -1)
            return torch.cat([a * c - b * s, b * c + a * s], -1)
        q, k = turn(q, wq), turn(k, wk)
        k, v = (t.repeat_interleave(H // Hkv, 1) for t in (k, v))
        s = (q @ k.transpose(2, 3)) / math.sqrt(E)
        return torch.softmax(torch.where(visible(torch.arange(L, device=DEV), L, window, sinks), s, -math.inf), -1) @ v
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    y64 = plain(*wide)
    g64 = torch.autograd.grad(y64, wide, g.double())
    # Norm-wise: the chain's float32 roundings, some E + window of them, each u of a value's size.
    for a, b in zip((y, *grads), (y64, *g64)):
        a, b = a.detach(), b.detach()
        assert float((a.double() - b).norm()) <= 4 * (E + window) * U * float(b.norm()) * math.sqrt(B * L)
    y64 = y64.detach()
    kc, vc = (torch.full((B, Hkv, 200, E), math.nan, device=DEV) for _ in range(2))
    for t in range(L):
        q1, k1, v1 = (s.unflatten(-1, (-1, E)).transpose(1, 2)
                      for s in x[:, t:t + 1].detach().split((H * E, Hkv * E, Hkv * E), -1))
        q1, k1 = F.qk_norm_rotary(q1, k1, wq.detach(), wk.detach(), freq, offset=t, magnitude=mag)
        kc[:, :, t:t + 1], vc[:, :, t:t + 1] = k1, v1
        one = F.window_decode(q1, kc, vc, window, sinks, lengths=torch.full((B,), t + 1, device=DEV))
        assert float((one.double() - y64[:, :, t:t + 1]).norm()) <= \
            4 * (E + window) * U * float(y64[:, :, t:t + 1].norm()) * math.sqrt(B * L), t


@pytest.mark.parametrize("bad", ["device", "dtype", "types", "heads", "shape", "lengths", "lengths_type"])
def test_refusals(bad):
    from densecore_amd import functional as F
    q, k = torch.zeros(2, 4, 1, 8, device=DEV), torch.zeros(2, 2, 5, 8, device=DEV)
    v, n = k, None
    if bad == "device":
        v = k.cpu()
    if bad == "dtype":
        q, k, v = q.half(), k.half(), v.half()
    if bad == "types":
        v = k.bfloat16()
    if bad == "heads":
        k = v = torch.zeros(2, 3, 5, 8, device=DEV)
    if bad == "shape":
        v = k[:, :, :4]
    if bad == "lengths":
        n = torch.zeros(3, dtype=torch.int64, device=DEV)
    if bad == "lengths_type":
        n = torch.zeros(2, device=DEV)
    with pytest.raises(ValueError):
        F.window_decode(q, k, v, 4, lengths=n)
    if n is None:
        with pytest.raises(ValueError):
            F.window_attention(q, k, v, 4)


def test_head_dim_limits():
    from densecore_amd import functional as F
    x = torch.zeros(1, 1, 1, 129, device=DEV)
    with pytest.raises(NotImplementedError):
        F.window_attention(x, x, x, 4)
    x = torch.zeros(1, 1, 1, 257, device=DEV)
    with pytest.raises(NotImplementedError):
        F.window_decode(x, x, x, 4)


@TYPES
def test_decode_of_large_values(dtype):
    """Values near the type's largest, over one piece and over several."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(15)
    for S in (90, 4000):
        q, k, v = (torch.randn(1, 2, n, 64, generator=gen).to(dtype).to(DEV) for n in (1, S, S))
        v = (3.0e38 * (1 - 0.1 * torch.rand(1, 2, S, 64, generator=gen))).to(dtype).to(DEV)
        ref = formulas(q, k, v, visible(torch.tensor([S - 1], device=DEV), S, 3500, 4), 0.125, dtype)
        close(F.window_decode(q, k, v, 3500, 4), *ref["out"], dtype, "decode")
        close(F.window_attention(q, k, v, 3500, 4, offset=S - 1), *ref["out"], dtype, "attention")


@TYPES
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (16, 1), (17, 1), (40, 2), (24, 8)], ids=str)
def test_decode_heads_that_share_rows(heads, dtype):
    """Grouped heads of every size, over one piece and several, head dims between the instantiated ones."""
    from densecore_amd import functional as F
    H, Hkv = heads
    gen = torch.Generator().manual_seed(18)
    for S, E, window, sinks in ((70, 16, 33, 2), (1500, 48, 700, 5), (2600, 120, 2500, 0), (600, 72, 5000, 4)):
        q, k, v = (torch.randn(2, n, m, E, generator=gen).to(dtype).to(DEV) for n, m in ((H, 1), (Hkv, S), (Hkv, S)))
        n = torch.tensor([S, S // 2 + 1], device=DEV)
        open_ = visible(n[:, None] - 1, S, window, sinks)[:, None]
        ref = formulas(q, k, v, open_, 1 / math.sqrt(E), dtype)
        close(F.window_decode(q, k, v, window, sinks, lengths=n), *ref["out"], dtype, f"S{S} E{E}")


@TYPES
def test_decode_of_infinite_values(dtype):
    """An infinite value that is seen makes its dim infinite, and no other; a NaN key makes its sequence NaN."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(19)
    q, k, v = (torch.randn(3, n, m, 64, generator=gen).to(dtype).to(DEV) for n, m in ((8, 1), (2, 900), (2, 900)))
    ref = formulas(q, k, v, visible(torch.tensor([899], device=DEV), 900, 600, 4), 0.125, dtype)
    v2, k2 = v.clone(), k.clone()
    v2[0, 1, 500, 7] = math.inf
    v2[1, 0, 899, 63] = -math.inf
    k2[2, 0, 2] = math.nan
    out = F.window_decode(q, k2, v2, 600, 4)
    assert (out[0, 4:, 0, 7] == math.inf).all() and (out[1, :4, 0, 63] == -math.inf).all()
    assert torch.isnan(out[2, :4]).all()
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, 4:, 0, 7] = hit[1, :4, 0, 63] = hit[2, :4] = True
    value, slack = (t.expand_as(out)[~hit] for t in ref["out"])
    close(out[~hit], value, slack, dtype, "others")


@pytest.mark.parametrize("offset", [2 ** 30, 2 ** 31 + 1, 2 ** 64, 2 ** 64 + 5])
def test_offsets_out_of_range(offset):
    from densecore_amd import functional as F
    x = torch.zeros(1, 2, 3, 8, device=DEV)
    with pytest.raises(NotImplementedError, match="offset"):
        F.window_attention(x, x, x, 4, 0, offset)
    f = torch.zeros(4, dtype=torch.float64, device=DEV)
    if offset >= 2 ** 53:
        for o in (offset, -offset):
            with pytest.raises(NotImplementedError, match="offset"):
                F.rotary_embedding(x, x, f, offset=o)


def test_host_threads_on_one_stream():
    """Calls of several kernels from host threads whose launches interleave on one stream."""
    import threading
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(31)
    xs = [[torch.randn(1, n, 2000, 64, generator=gen).to(DEV) for n in (4, 2, 2, 4)] for _ in range(4)]

    def work(q, k, v, g):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        few = F.window_attention(q[:, :, -3:], k, v, 1900, 4, offset=1997)
        one = F.window_decode(q[:, :, -1:], k, v, 1900, 4)
        return (few, one, *torch.autograd.grad(F.window_attention(*leaves, 100, 4), leaves, g))
    ref = [work(*x) for x in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]

    def run(i):
        for _ in range(10):
            got[i].append(work(*xs[i]))
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, runs in zip(ref, got):
        assert len(runs) == 10
        assert all(torch.equal(s, t) for b in runs for s, t in zip(a, b))


@pytest.mark.parametrize("sizes", [(1, 700, 700, 0, 0), (300, 2000, 200, 1700, 4), (2000, 300, 64, 0, 0),
                                   (500, 1500, 128, 250, 200), (64, 1111, 3000, 900, 0)], ids=str)
def test_gradient_pieces(sizes):
    """The longest key tile without sinks, which sets the pieces, wherever it lies."""
    from densecore_amd import functional as F
    L, S, window, offset, sinks = sizes
    gen = torch.Generator().manual_seed(L + S)
    q, k, v, g = (torch.randn(1, h, n, 32, generator=gen).to(DEV) for h, n in ((2, L), (1, S), (1, S), (2, L)))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    y = F.window_attention(*leaves, window, sinks, offset)
    dq, dk, dv = torch.autograd.grad(y, leaves, g)
    open_ = visible(torch.arange(offset, offset + L, device=DEV), S, window, sinks)
    ref = formulas(q, k, v, open_, 32 ** -0.5, torch.float32, g)
    for name, x in (("out", y), ("dq", dq), ("dk", dk), ("dv", dv)):
        close(x, *ref[name], torch.float32, name)


def _random_case(seed):
    import random
    r = random.Random(seed)
    Hkv, rep = r.choice([1, 2, 3, 5]), r.choice([1, 1, 2, 3, 4, 8])
    E = r.choice([8, 16, 24, 32, 40, 48, 64, 64, 72, 96, 128, 128, r.randint(1, 128)])
    S = r.choice([r.randint(1, 70), r.randint(60, 400), r.randint(400, 1500)])
    L = r.choice([1, 2, r.randint(1, 70), min(S, 300), r.randint(60, 300)])
    offset = r.choice([0, max(S - L, 0), max(S - L, 0), r.randint(0, 2 * S)])
    window = r.choice([1, r.randint(1, 40), r.randint(30, 300), S, 5 * S])
    sinks = r.choice([0, 0, 1, 4, r.randint(0, 200)])
    return r.randint(1, 3), Hkv * rep, Hkv, L, S, E, window, sinks, offset


@TYPES
@pytest.mark.parametrize("seed", range(40))
def test_random_sizes(seed, dtype):
    test_forward_and_gradients(_random_case(seed), dtype)


@TYPES
@pytest.mark.parametrize("seed", range(30))
def test_decode_of_random_sizes(seed, dtype):
    import random
    r = random.Random(seed)
    B, H, Hkv, _, S, E, window, sinks, _ = _random_case(1000 + seed)
    test_decode((B, H, Hkv, S, r.choice([E, 2 * E]), window, sinks, r.choice([None, [r.randint(0, S) for _ in range(B)]])), dtype)


@TYPES
@pytest.mark.parametrize("what", ["all", "queries", "keys", "values", "gradients", "some"])
def test_results_that_are_not_finite(what, dtype):
    """NaN where the formulas have it and nowhere else: rows that see no key stay 0, the others' hidden
    neighbours finite; sinks, pieces of keys and a few rows over many keys among them."""
    from densecore_amd import functional as F
    gen = torch.Generator().manual_seed(41)
    for B, H, Hkv, L, S, E, window, sinks, offset in ((1, 4, 2, 400, 400, 64, 70, 4, 0), (2, 2, 1, 260, 200, 40, 30, 0, 0),
                                                      (1, 4, 1, 9, 1500, 128, 900, 3, 1491)):
        q, k, v, g = (torch.randn(B, h, n, E, generator=gen).to(dtype).to(DEV) for h, n in ((H, L), (Hkv, S), (Hkv, S), (H, L)))
        for name, t in (("queries", q), ("keys", k), ("values", v), ("gradients", g)):
            if what in ("all", name):
                t.fill_(math.nan)
            elif what == "some":
                t[:, :, t.shape[2] // 2] = math.nan
        open_ = visible(offset + torch.arange(L, device=DEV), S, window, sinks)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        y = F.window_attention(*leaves, window, sinks, offset)
        dq, dk, dv = torch.autograd.grad(y, leaves, g)

        def dirty(t):  # rows, (B, H, rows)
            return torch.isnan(t.detach().float()).any(-1)

        def shared(t):
            return t.repeat_interleave(H // Hkv, 1)
        pair = open_[None, None]
        q_, k_, v_, g_ = dirty(q), shared(dirty(k)), shared(dirty(v)), dirty(g)
        score = pair & (q_[..., None] | k_[:, :, None])          # pairs whose score is NaN
        row = score.any(-1)                                      # rows whose P is NaN
        out = row | (pair & v_[:, :, None]).any(-1)
        sees = open_.any(-1)[None, None].expand(B, H, L)
        ds = sees & (out | g_)                                   # dsum takes both
        p_pair, ds_pair = pair & row[..., None], pair & (ds[..., None] | v_[:, :, None])

        def group(t):
            return t.reshape(B, Hkv, H // Hkv, S).any(2)
        want = {"out": out, "dq": (ds_pair | (pair & k_[:, :, None])).any(-1),
                "dk": group((ds_pair | (pair & q_[..., None])).any(2)), "dv": group((p_pair | (pair & g_[..., None])).any(2))}
        for name, t in (("out", y), ("dq", dq), ("dk", dk), ("dv", dv)):
            assert torch.equal(torch.isnan(t).all(-1), want[name]), (name, L)
            assert torch.equal(torch.isnan(t).any(-1), want[name]), (name, L)
        assert not y[~sees].any() and not dq[~sees].any()
