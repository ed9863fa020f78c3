"""Layer norm, gated linear recurrence and AdamW over many tensors on the GPU against their definitions in 64 bits.

Tolerances: U = 2^-24 is half a step of float32, half(t) that of the results' type.  A chain of k float32 operations is off by at most
k U of the sum of its terms' magnitudes (1 + k U covers the higher orders by far at these lengths); each test says what k is."""
import itertools

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def half(torch, t):
    return torch.finfo(t).eps / 2


def tiny(torch, t):
    """half the spacing of the numbers nearest to zero: what rounds to them is off by that much at most"""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def gen(torch, seed):
    return torch.Generator("cuda").manual_seed(seed)


def near(torch, got, want, slack, what):
    """|got - want| <= slack + half a step of got's type"""
    got64 = got.double()
    bound = slack + half(torch, got.dtype) * (want.abs() + slack) + tiny(torch, got.dtype)
    off = (got64 - want).abs() - bound
    assert torch.isfinite(got64).all(), f"{what}: not finite"
    assert (off <= 0).all(), f"{what}: {off.max().item():.3g} beyond the bound, at {off.argmax().item()} of {tuple(off.shape)}"


# ---- layer norm ----
def norm_reference(torch, x, w, b, eps, dy=None):
    """64-bit results and, for each, the sum of magnitudes its error goes by"""
    n = x.shape[-1]
    x = x.double().reshape(-1, n)
    w_ = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b_ = torch.zeros_like(w_) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh * w_ + b_
    # a sum of n terms in the kernels: at most 64 in a lane (8 vectors of 8), 10 steps over lanes and waves: k = 80 with the rounding of
    # the parts.  x - mean is off by (80 + 1) U mean|x| + U |x - mean|; squares double that relative to sd
    k = 80 * U
    e_mean = k * x.abs().mean(1, keepdim=True)
    e_rstd = k + 2 * e_mean * rstd                           # relative
    e_xh = e_mean * rstd + xh.abs() * (e_rstd + 4 * U)
    e_y = e_xh * w_.abs() + 4 * U * (y.abs() + b_.abs())
    if dy is None:
        return y, e_y
    dy = dy.double().reshape(-1, n)
    q = dy * w_
    s1, s2 = q.mean(1, keepdim=True), (q * xh).mean(1, keepdim=True)
    dx = rstd * (q - s1 - xh * s2)
    qa = q.abs()
    e_s1 = k * qa.mean(1, keepdim=True)
    e_s2 = k * (qa * xh.abs()).mean(1, keepdim=True) + (qa * e_xh).mean(1, keepdim=True)
    e_dx = rstd * (4 * U * (qa + s1.abs() + (xh * s2).abs()) + e_s1 + xh.abs() * e_s2 + e_xh * s2.abs()) + (e_rstd + 4 * U) * dx.abs()
    # columns: rows / workgroups in a thread, then up to 1024 partial sums in 32 lanes of 32, summed: at most 1024 + 64 with the rows' own
    kc = (1100 + x.shape[0] / 64) * U
    dw, e_dw = (dy * xh).sum(0), kc * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)
    db, e_db = dy.sum(0), kc * dy.abs().sum(0)
    return y, e_y, dx, e_dx, dw, e_dw, db, e_db


NORM_SHAPES = [(1, 1), (5, 1), (3, 7), (145, 32), (1000, 33), (64, 64), (17, 255), (4, 256), (9, 257), (9, 600), (33, 1000), (7, 1024), (5, 1025), (6, 2049),
               (700, 4096), (3, 10007), (5, 13001), (9, 16384), (2, 16385), (4, 20005), (3, 24570), (2, 30001), (3, 32768), (2, 40001), (3, 70001)]


@pytest.mark.parametrize("rows,n", NORM_SHAPES)
@pytest.mark.parametrize("xt,wt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32")])
def test_layer_norm(torch_mod, rows, n, xt, wt):
    torch = torch_mod
    from sound_bubble_amd import functional as F
    xt, wt = getattr(torch, xt), getattr(torch, wt)
    g = gen(torch, rows * 100003 + n)
    x = (torch.randn(rows, n, generator=g, device="cuda") * 2 + 1).to(xt).requires_grad_(True)
    w = (1 + 0.3 * torch.randn(n, generator=g, device="cuda")).to(wt).requires_grad_(True)
    b = (0.3 * torch.randn(n, generator=g, device="cuda")).to(wt).requires_grad_(True)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(xt)
    y = F.layer_norm(x, w, b, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ref = norm_reference(torch, x.detach(), w.detach(), b.detach(), 1e-5, dy)
    for got, want, slack, what in zip((y.detach(), dx, dw, db), ref[::2], ref[1::2], ("y", "dx", "dw", "db")):
        assert got.dtype == (xt if what in ("y", "dx") else wt)
        near(torch, got, want, slack, what)
    again = torch.autograd.grad(F.layer_norm(x, w, b, 1e-5), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again)), "the same call gives the same bits"
    with torch.no_grad():
        assert torch.equal(F.layer_norm(x, w, b, 1e-5), y)


@pytest.mark.parametrize("affine", ["none", "weight", "bias"])
@pytest.mark.parametrize("xt", ["float32", "bfloat16"])
def test_layer_norm_without_weight_or_bias(torch_mod, affine, xt):
    torch = torch_mod
    from sound_bubble_amd import functional as F
    xt = getattr(torch, xt)
    g = gen(torch, 5)
    x = torch.randn(3, 11, 77, generator=g, device="cuda").to(xt).requires_grad_(True)
    p = torch.randn(77, generator=g, device="cuda").to(xt).requires_grad_(True)
    w, b = (p if affine == "weight" else None), (p if affine == "bias" else None)
    dy = torch.randn(3, 11, 77, generator=g, device="cuda").to(xt)
    y = F.layer_norm(x, w, b)
    assert y.shape == x.shape
    leaves = (x,) if affine == "none" else (x, p)
    got = torch.autograd.grad(y, leaves, dy)
    ref = norm_reference(torch, x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), 1e-5, dy)
    near(torch, y.detach().reshape(-1, 77), ref[0], ref[1], "y")
    near(torch, got[0].reshape(-1, 77), ref[2], ref[3], "dx")
    if affine != "none":
        i = 4 if affine == "weight" else 6
        near(torch, got[1], ref[i], ref[i + 1], "dp")


def test_layer_norm_layouts(torch_mod):
    """sliced rows at odd addresses, transposed and broadcast inputs, expanded gradients, frozen parameters, empty batches"""
    torch = torch_mod
    from sound_bubble_amd import functional as F
    g = gen(torch, 6)
    base = torch.randn(40, 101, generator=g, device="cuda")
    w = torch.randn(64, generator=g, device="cuda")
    for dt in (torch.float32, torch.float16):
        wide = base.to(dt)
        cuts = [wide[:, 3:67], wide[1::3, 37:], wide[:, :64].reshape(8, 5, 64).transpose(0, 1), wide[:1, :64].expand(7, 64),
                base[:40, :].to(dt).t()[:64, :].t()]
        for x in cuts:
            y = F.layer_norm(x, w)
            ref = norm_reference(torch, x.contiguous(), w, None, 1e-5)
            near(torch, y.reshape(-1, 64), ref[0], ref[1], "y")
    x = wide[:, 3:67].detach().float().requires_grad_(True)
    (dx,) = torch.autograd.grad(F.layer_norm(x, w).sum(), x)                    # an expanded gradient of strides 0
    ref = norm_reference(torch, x.detach(), w, None, 1e-5, torch.ones_like(x))
    near(torch, dx, ref[2], ref[3], "dx")
    e = torch.zeros(0, 64, device="cuda", requires_grad=True)
    wl = w.clone().requires_grad_(True)
    y = F.layer_norm(e, wl)
    (dw,) = torch.autograd.grad(y, wl, torch.zeros_like(y))
    assert y.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


def test_layer_norm_values(torch_mod):
    """a far mean, equal rows, rows with NaN and infinity beside clean ones, subnormals"""
    torch = torch_mod
    from sound_bubble_amd import functional as F
    g = gen(torch, 7)
    for n in (48, 3001):
        x = torch.randn(6, n, generator=g, device="cuda")
        x[0] += 1e4
        x[1] = 3.25
        x[4] *= 1e-30
        ref = norm_reference(torch, x, None, None, 1e-5)
        near(torch, F.layer_norm(x), ref[0], ref[1], "y")
        clean = F.layer_norm(x)
        x[2, 5], x[3, 7] = float("nan"), float("inf")
        y = F.layer_norm(x)
        assert torch.isnan(y[2]).all() and torch.isnan(y[3]).any()
        assert torch.equal(y[[0, 1, 4, 5]], clean[[0, 1, 4, 5]])


# ---- gated scan ----
def scan_reference(torch, x, gate, h0, dim, form, reverse, lengths, dh=None, dlast=None):
    """64-bit results with error sums.  h_t is a sum of terms b_j a_{j+1} .. a_t: each carries at most 6 U a step behind j (the
    gate's own 4 U -- exponential, sum, reciprocal, product --, the product, the addition), however the products are grouped:
    E_t = |a_t| E_{t-1} + 8 U H_t with H_t = |a_t| H_{t-1} + |b_t| adds up to that, and the same holds for the gradient's walk.
    Gradual underflow: a float32 operation is off by U |value| + 2^-150 at most (half the spacing of subnormals).  The second part is 8
    operations a step here too; where it falls on a product of gates it is carried on times a state, of at most `top`.  A gate's logistic
    function counts e^-|z| as 0 behind |z| = 87: that is 1.7e-38 at most, times a state again."""
    xs, zs = x.double().movedim(dim, 0), gate.double().movedim(dim, 0)
    a = torch.sigmoid(zs) if form == "sigmoid" else zs
    ol = torch.sigmoid(-zs) if form == "sigmoid" else torch.ones_like(zs)
    T, rest = xs.shape[0], xs.shape[1:]
    live = torch.ones((T,) + (1,) * len(rest), dtype=torch.bool, device=x.device)
    if lengths is not None:
        ln = lengths.reshape(lengths.shape + (1,) * (len(rest) - lengths.dim()))
        live = torch.arange(T, device=x.device).reshape((T,) + (1,) * len(rest)) < ln
    live = live.expand((T,) + tuple(rest))
    a, ol = torch.where(live, a, 1.0), torch.where(live, ol, 0.0)
    xs = torch.where(live, xs, 0.0)
    b = ol * xs
    order = range(T - 1, -1, -1) if reverse else range(T)
    h = torch.zeros(rest, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    tops = [t.double().abs().nan_to_num(0, 0, 0).max().item() for t in (xs, h, dh, dlast) if t is not None and t.numel()]
    top = 1 + sum(tops) * T                              # (|a| <= 1: a state is at most the sum of all that enters)
    low = (8 * 2.0 ** -150 + (1.7e-38 if form == "sigmoid" else 0.0)) * top
    H, E = h.abs(), torch.zeros_like(h)
    before, hs, es, eb = (torch.zeros_like(xs) for _ in range(4))
    for t in order:
        before[t], eb[t] = h, E
        h, H = a[t] * h + b[t], a[t].abs() * H + b[t].abs()
        E = a[t].abs() * E + 8 * U * H + low
        hs[t], es[t] = h, E
    out = {"h": (torch.where(live, hs, 0.0).movedim(0, dim), es.movedim(0, dim)), "last": (h, E)}
    if dh is None and dlast is None:
        return out
    d = torch.zeros_like(xs) if dh is None else torch.where(live, dh.double().movedim(dim, 0), 0.0)
    c = torch.zeros(rest, dtype=torch.float64, device=x.device) if dlast is None else dlast.double()
    C_, Ec = c.abs(), torch.zeros_like(c)
    dx, dg, ex, eg = (torch.zeros_like(xs) for _ in range(4))
    for t in reversed(list(order)):
        G, GA = d[t] + c, d[t].abs() + C_
        EG = Ec + U * GA + low
        c, C_ = a[t] * G, a[t].abs() * GA
        Ec = a[t].abs() * EG + 8 * U * C_ + low
        if form == "sigmoid":
            dx[t], ex[t] = ol[t] * G, ol[t] * (EG + 6 * U * GA) + low
            s = a[t] * ol[t]
            dg[t] = G * (before[t] - xs[t]) * s
            eg[t] = s * (EG * (before[t] - xs[t]).abs() + G.abs() * (eb[t] + U * (before[t].abs() + xs[t].abs())) + 12 * U * (G * (before[t] - xs[t])).abs()) + low * top
        else:
            dx[t], ex[t] = G, EG
            dg[t], eg[t] = G * before[t], EG * before[t].abs() + G.abs() * eb[t] + 4 * U * (G * before[t]).abs() + low * top
    z = torch.zeros((), dtype=torch.float64, device=x.device)
    out["dx"] = (torch.where(live, dx, z).movedim(0, dim), ex.movedim(0, dim))
    out["dgate"] = (torch.where(live, dg, z).movedim(0, dim), eg.movedim(0, dim))
    out["dh0"] = (c, Ec)
    return out


def scan_inputs(torch, shape, dim, xt, gt, form, seed, ragged=False, h0=True):
    g = gen(torch, seed)
    x = torch.randn(shape, generator=g, device="cuda").to(xt)
    z = torch.randn(shape, generator=g, device="cuda") * 2 + 1
    gate = (z if form == "sigmoid" else torch.tanh(z)).to(gt)
    rest = shape[:dim] + shape[dim + 1:]
    h = torch.randn(rest, generator=g, device="cuda") if h0 else None
    lengths = torch.randint(0, shape[dim] + 1, shape[:dim], generator=g, device="cuda") if ragged else None
    dh = torch.randn(shape, generator=g, device="cuda").to(xt)
    dlast = torch.randn(rest, generator=g, device="cuda")
    return x, gate, h, lengths, dh, dlast


def check_scan(torch, x, gate, h0, lengths, dh, dlast, **kw):
    from sound_bubble_amd import functional as F
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, h0) if t is not None]
    h, last = F.gated_scan(leaves[0], leaves[1], leaves[2] if h0 is not None else None, lengths=lengths, **kw)
    assert h.dtype == x.dtype and last.dtype == torch.float32 and h.shape == x.shape
    outs, grads = [(h, dh), (last, dlast)], None
    outs = [(o, g) for o, g in outs if g is not None]
    grads = torch.autograd.grad([o for o, _ in outs], leaves, [g for _, g in outs])
    ref = scan_reference(torch, x, gate, h0, kw.get("dim", 1), kw.get("form", "sigmoid"), kw.get("reverse", False), lengths, dh, dlast)
    got = {"h": h.detach(), "last": last.detach(), "dx": grads[0], "dgate": grads[1]}
    if h0 is not None:
        got["dh0"] = grads[2]
    for name, t in got.items():
        near(torch, t, *ref[name], name)
    with torch.no_grad():
        h2, last2 = F.gated_scan(x, gate, h0, lengths=lengths, **kw)
    assert torch.equal(h2, h) and torch.equal(last2, last), "inference and training give the same bits"
    return got


SCAN_SHAPES = [((1, 1, 1), 1), ((2, 1, 64), 1), ((3, 7, 5), 1), ((2, 8, 8), 1), ((5, 65, 33), 1), ((2, 257, 130), 1), ((1, 1031, 3), 1), ((3, 300, 1), 1),
               ((4, 9, 6, 20), 1), ((4, 9, 37, 20), 2), ((70, 40, 9, 2), 2), ((33, 12, 145, 32), 2), ((5, 6), 1), ((9,), 0), ((600, 4, 7, 64), 2),
               ((1, 5000, 16), 1), ((2, 3000, 200), 1), ((4, 700, 1501), 1), ((3, 130, 3001), 1), ((5, 20, 1000), 1), ((1500, 90, 3), 1)]


@pytest.mark.parametrize("shape,dim", SCAN_SHAPES)
@pytest.mark.parametrize("xt,gt,form,reverse,ragged", [("float32", "float32", "sigmoid", False, False), ("bfloat16", "float32", "decay", True, False),
                                                      ("float16", "float16", "sigmoid", True, True), ("float32", "float32", "decay", False, True)])
def test_gated_scan(torch_mod, shape, dim, xt, gt, form, reverse, ragged):
    torch = torch_mod
    xt, gt = getattr(torch, xt), getattr(torch, gt)
    ins = scan_inputs(torch, shape, dim, xt, gt, form, sum(shape) + dim, ragged, h0=not ragged or len(shape) % 2 == 1)
    check_scan(torch, *ins, dim=dim, form=form, reverse=reverse)


@pytest.mark.parametrize("what", ["dh only", "dlast only"])
def test_gated_scan_one_gradient(torch_mod, what):
    torch = torch_mod
    x, gate, h0, _, dh, dlast = scan_inputs(torch, (3, 200, 24), 1, torch.float32, torch.float32, "sigmoid", 3)
    check_scan(torch, x, gate, h0, None, dh if what == "dh only" else None, dlast if what == "dlast only" else None)


def test_gated_scan_layouts(torch_mod):
    """halves of one projection, transposed, broadcast and unaligned inputs, expanded gradients"""
    torch = torch_mod
    g = gen(torch, 11)
    dlast = torch.randn(3, 21, generator=g, device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        proj = torch.randn(3, 90, 43, generator=g, device="cuda").to(dt)
        x, gate = proj[..., 1:22], proj[..., 22:]
        ones = torch.ones(1, 1, 1, device="cuda", dtype=dt).expand(3, 90, 21)
        check_scan(torch, x, gate, None, None, ones, dlast)
        check_scan(torch, x.transpose(0, 1), gate.transpose(0, 1), None, None, ones.transpose(0, 1), dlast, dim=0)
        check_scan(torch, x.transpose(1, 2), gate.transpose(1, 2), None, None, ones.transpose(1, 2), dlast, dim=2)
        check_scan(torch, x[:1].expand(3, 90, 21), gate[:, :1].expand(3, 90, 21), None, None, ones, dlast, reverse=True)
        check_scan(torch, x, gate, torch.randn(21, generator=g, device="cuda").expand(3, 21), None, ones, dlast, dim=-2)


def test_gated_scan_values(torch_mod):
    """saturated and infinite gates, NaN behind a sequence's length and in one channel, lengths of 0 and beyond the steps"""
    torch = torch_mod
    from sound_bubble_amd import functional as F
    x, gate, h0, _, dh, dlast = scan_inputs(torch, (4, 77, 12), 1, torch.float32, torch.float32, "sigmoid", 12)
    gate[0, 20:30] = 90.0
    gate[1, 20:30] = -90.0
    gate[2, 40] = float("-inf")
    gate[3, 50:] = float("inf")
    check_scan(torch, x, gate, h0, None, dh, dlast)
    lengths = torch.tensor([0, 1, 500, -3], device="cuda")
    lim = lengths.clamp(0, 77)
    ref = check_scan(torch, x, gate, h0, lim, dh, dlast)
    got = F.gated_scan(x, gate, h0, lengths=lengths)
    assert torch.equal(got[0], ref["h"]) and torch.equal(got[1], ref["last"])
    assert torch.equal(F.gated_scan(x, gate, h0, lengths=lengths.int())[0], ref["h"])
    assert torch.equal(ref["last"][0], h0[0]) and torch.equal(ref["dh0"][0], dlast[0]) and not ref["h"][0].any()
    bx, bg, bd = (t.clone() for t in (x, gate, dh))
    for t in (bx, bg, bd):
        t[0], t[1, 1:] = float("nan"), float("inf")
        t[3] = float("nan")
    again = check_scan(torch, bx, bg, h0, lim, bd, dlast)
    assert all(torch.equal(ref[k], again[k]) for k in ref), "what lies behind a length does not matter"
    bx = x.clone()
    bx[2, 30, 5] = float("nan")
    h, last = F.gated_scan(bx, gate, h0)
    clean, _ = F.gated_scan(x, gate, h0)
    assert torch.isnan(h[2, 30:, 5]).all() and torch.isnan(last[2, 5])
    h[2, 30:, 5] = clean[2, 30:, 5]
    assert torch.equal(h, clean), "a NaN stays in its channel and behind its step"


def test_gated_scan_against_differences(torch_mod):
    """the gradient of a scalar against central differences in 64 bits of the definition, through random directions"""
    torch = torch_mod
    from sound_bubble_amd import functional as F
    for form, reverse in itertools.product(("sigmoid", "decay"), (False, True)):
        x, gate, h0, lengths, dh, dlast = scan_inputs(torch, (2, 40, 6), 1, torch.float32, torch.float32, form, 21, ragged=True)
        leaves = [t.requires_grad_(True) for t in (x, gate, h0)]
        h, last = F.gated_scan(*leaves, lengths=lengths, form=form, reverse=reverse)
        grads = torch.autograd.grad(((h * dh).sum() + (last * dlast).sum()), leaves)

        def value(*t):
            r = scan_reference(torch, *t, 1, form, reverse, lengths)
            return (r["h"][0] * dh).sum() + (r["last"][0] * dlast).sum()
        for seed in range(3):
            g = gen(torch, 100 + seed)
            step = [torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) for t in leaves]
            eps = 1e-5
            hi, lo = (value(*(t.detach().double() + s * eps * v for t, v in zip(leaves, step))) for s in (1, -1))
            want = sum((a.double() * v).sum() for a, v in zip(grads, step))
            scale = sum((a.double() * v).abs().sum() for a, v in zip(grads, step))
            # differences: eps^2 of third derivatives and 2^-52 / eps; the gradients' own float32 errors, 100 U of their terms
            assert abs((hi - lo) / (2 * eps) - want) <= scale * (100 * U + 1e-8)


def test_gated_scan_step(torch_mod):
    """steps one by one are the scan; the state is the caller's, rows may be strided"""
    torch = torch_mod
    from sound_bubble_amd import functional as F
    for xt, gt, form in ((torch.float32, torch.float32, "sigmoid"), (torch.bfloat16, torch.float32, "decay"), (torch.float16, torch.float16, "sigmoid")):
        for rows, n in ((1, 1), (3, 5), (7, 130)):
            x, gate, h0, _, _, _ = scan_inputs(torch, (rows, 9, n), 1, xt, gt, form, rows + n)
            state = h0.clone()
            ys = [F.gated_scan_step(x[:, t], gate[:, t], state, form=form) for t in range(9)]
            ref = scan_reference(torch, x, gate, h0, 1, form, False, None)
            near(torch, torch.stack(ys, 1), *ref["h"], "h")
            near(torch, state, *ref["last"], "last")
    x = torch.zeros(0, 4, device="cuda")
    assert F.gated_scan_step(x, x, x.clone()).shape == (0, 4)


def test_gated_scan_empty(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import functional as F
    h0 = torch.randn(2, 3, device="cuda").requires_grad_(True)
    x = torch.zeros(2, 0, 3, device="cuda", requires_grad=True)
    h, last = F.gated_scan(x, x, h0)
    assert h.shape == (2, 0, 3) and torch.equal(last, h0)
    (d,) = torch.autograd.grad(last, h0, torch.ones_like(last))
    assert torch.equal(d, torch.ones_like(d))
    assert torch.equal(F.gated_scan(x.detach(), x.detach())[1], torch.zeros(2, 3, device="cuda"))


# ---- AdamW ----
def dither(n, step, seed):
    x = (np.arange(n, dtype=np.uint64) + np.uint64((seed * 0x9E3779B9 + step * 0x6A09E667) & 0xFFFFFFFF)) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x5BE0CD19) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x1F83D9AB) & 0xFFFFFFFF
    return x ^ (x >> 16)


def inverses(torch):
    """2^(127 - byte) as tensor operations give it on the device: for some exponents one ulp below the power of two"""
    return torch.ldexp(torch.ones(256, device="cuda"), 127 - torch.arange(256, device="cuda", dtype=torch.int32)).cpu().numpy()


def encode(x, inverse, mant, bias, top, u16, floor):
    """the 8-bit format's definition in integers of 64 bits and float64 (numpy): -> codes, scale bytes.  inverse[byte]: what a
    block is multiplied by before it is cut, in float32"""
    blocks = x.reshape(-1, 256).astype(np.float64)
    big = np.abs(blocks).max(1)
    largest = (2 - 0.25) * 2.0 ** top
    with np.errstate(divide="ignore"):
        k = np.where(big > 0, np.ceil(np.log2(np.maximum(big, 1e-300) / largest)), -127)
    k = np.where(big > 0, k + (big > largest * 2.0 ** k) - (big <= largest * 2.0 ** (k - 1)), k)      # (log2's own rounding)
    k = np.clip(k, -127, 127)
    y = (np.abs(blocks).astype(np.float32) * inverse[(k + 127).astype(int)][:, None]).astype(np.float64)
    e = np.maximum(np.floor(np.log2(np.maximum(y, 1e-300))), 1 - bias)
    unit = 2.0 ** (e - mant)                                          # spacing of the codes around y
    part = y / unit
    u = (u16.reshape(-1, 256) + 0.5) / 65536
    # the fraction counts to 23 - mant bits, as the float's own below the spacing
    frac = np.floor((part - np.floor(part)) * 2.0 ** (23 - mant)) / 2.0 ** (23 - mant)
    n = np.floor(part) + (frac + u >= 1)
    value = n * unit
    e2 = np.maximum(np.floor(np.log2(np.maximum(value, 1e-300))), 1 - bias)
    m = np.round(value / 2.0 ** (e2 - mant)).astype(np.int64)
    code = np.where(m >= 1 << mant, ((e2 + bias).astype(np.int64) << mant) + m - (1 << mant), m)
    if floor:
        code = np.where((code == 0) & (blocks > 0), 1, code)
    else:
        code = code | (np.signbit(blocks).astype(np.int64) << 7)
    return code.reshape(-1).astype(np.uint8), (k + 127).astype(np.uint8)


def adamw_reference(p, g, m, v, step, lr, b1, b2, eps, wd, scale=1.0):
    g = g * scale
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr / (1 - b1 ** step) * m / (np.sqrt(v) / np.sqrt(1 - b2 ** step) + eps), m, v


def laid(ts):
    out = []
    for t in ts:
        t = t.detach().double().cpu().numpy().ravel()
        out.append(np.pad(t, (0, -t.size % 256)))
    return np.concatenate(out)


HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.05)


@pytest.mark.parametrize("sizes", [[1], [255, 256, 257, 3], [5000, 1, 4096, 4097, 70000], [3] * 150, [1 << 20]])
@pytest.mark.parametrize("pt,gt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32")])
@pytest.mark.parametrize("clip", [0.0, 0.7])
def test_adamw_32(torch_mod, sizes, pt, gt, clip):
    torch = torch_mod
    from sound_bubble_amd import ops
    pt, gt = getattr(torch, pt), getattr(torch, gt)
    g = gen(torch, len(sizes))
    ps = [torch.randn(n, generator=g, device="cuda").to(pt) for n in sizes]
    st = ops.adamw_state(ps)
    w = laid([p.float() for p in ps])
    m, v = np.zeros_like(w), np.zeros_like(w)
    mask = laid([torch.ones(n) for n in sizes]) > 0
    for step in (1, 2, 3):
        gs = [torch.randn(n, generator=g, device="cuda").to(gt) for n in sizes]
        ops.adamw_step(ps, gs, st, step, clip=clip, gscale=0.5, **HYPER)
        gl = laid(gs)
        scale = 0.5 * (min(1.0, clip / (np.sqrt((gl ** 2).sum()) * 0.5 + 1e-6)) if clip else 1.0)
        # the rates are rounded to float32, a value takes at most 12 roundings beside; the state that goes into the next step is the
        # kernel's own
        w0, m0, v0 = w, m, v
        w, m, v = adamw_reference(w, gl, m, v, step, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], scale)
        got_m, got_v = st["exp_avg"].double().cpu().numpy(), st["exp_avg_sq"].double().cpu().numpy()
        am = np.abs(m0) + 0.1 * np.abs(gl * scale)
        assert (np.abs(got_m - m) <= 12 * U * am)[mask].all() and (np.abs(got_v - v) <= 12 * U * v + 1e-44)[mask].all()
        dw = np.abs(w - w0 * (1 - HYPER["lr"] * HYPER["weight_decay"]))
        upd = 24 * U * (dw + HYPER["lr"] / (1 - 0.9 ** step) * am / (np.sqrt(v) / np.sqrt(1 - 0.99 ** step) + HYPER["eps"]))
        got_w = st["master"].double().cpu().numpy() if pt != torch.float32 else laid(ps)
        assert (np.abs(got_w - w) <= 4 * U * np.abs(w0) + upd)[mask].all()
        assert not got_m[~mask].any() and not got_v[~mask].any()
        if pt != torch.float32:
            assert np.array_equal(laid(ps)[mask], laid([torch.from_numpy(got_w).float().to(pt)])[:mask.size][mask])
        w, m, v = got_w, got_m, got_v


@pytest.mark.parametrize("sizes", [[1], [255, 256, 257, 3], [5000, 70000]])
@pytest.mark.parametrize("pt", ["float32", "bfloat16"])
def test_adamw_8(torch_mod, sizes, pt):
    """every code and scale is the definition's, made from the formula's float32 values"""
    torch = torch_mod
    from sound_bubble_amd import ops
    pt = getattr(torch, pt)
    g = gen(torch, 40 + len(sizes))
    ps = [torch.randn(n, generator=g, device="cuda").to(pt) for n in sizes]
    st = ops.adamw_state(ps, bits=8)
    f = np.float32
    b1, b2 = HYPER["betas"]
    for step in (1, 2, 3, 4):
        spread = [torch.exp(2 * torch.randn(n, generator=g, device="cuda")) for n in sizes]      # (v spans far more than a code's range)
        gs = [(torch.randn(n, generator=g, device="cuda") * s * 1e-3).to(pt) for n, s in zip(sizes, spread)]
        if step == 2:
            gs[0][:] = 0
        m0 = (st["exp_avg"].float().view(-1, 256) * st["exp_avg_scale"].float()[:, None]).view(-1).cpu().numpy()
        v0 = (st["exp_avg_sq"].float().view(-1, 256) * st["exp_avg_sq_scale"].float()[:, None]).view(-1).cpu().numpy()
        ops.adamw_step(ps, gs, st, step, seed=7, **HYPER)
        gl = laid(gs).astype(f)
        m = m0 * f(b1) + gl * f(1 - b1)
        v = v0 * f(b2) + (gl * gl) * f(1 - b2)
        u = dither(m.size, step, 7).astype(np.int64)
        mc, ms = encode(m, inverses(torch), 3, 7, 8, u & 0xFFFF, False)
        vc, vs = encode(v, inverses(torch), 2, 15, 15, u >> 16, True)
        assert np.array_equal(st["exp_avg_scale"].view(torch.uint8).cpu().numpy(), ms)
        assert np.array_equal(st["exp_avg_sq_scale"].view(torch.uint8).cpu().numpy(), vs)
        assert np.array_equal(st["exp_avg"].view(torch.uint8).cpu().numpy(), mc)
        assert np.array_equal(st["exp_avg_sq"].view(torch.uint8).cpu().numpy(), vc)


def test_adamw_8_scales(torch_mod):
    """blocks of every magnitude, each of 16 mantissas of its largest element, and values that are a code's own: the definition's codes"""
    torch = torch_mod
    from sound_bubble_amd import ops
    g = gen(torch, 44)
    f, (b1, b2) = np.float32, HYPER["betas"]
    unit = torch.arange(-60, 60, device="cuda").repeat_interleave(16)
    blocks = unit.numel()
    x = torch.randn(blocks, 256, generator=g, device="cuda") * torch.exp2(unit.float())[:, None]
    x[:, 0] = torch.exp2(unit.float()) * (1 + torch.arange(blocks, device="cuda") % 16 / 16) * 4
    x[:, 128:192] = torch.exp2(unit.float())[:, None] * torch.exp2(-torch.arange(64, device="cuda").float() / 8).round(decimals=2)
    p = torch.zeros(blocks * 256, device="cuda")
    st = ops.adamw_state([p], bits=8)
    ops.adamw_step([p], [x.view(-1)], st, 1, seed=3, **HYPER)
    gl = x.view(-1).cpu().numpy()
    u = dither(gl.size, 1, 3).astype(np.int64)
    for k, a, fmt, part in (("exp_avg", gl * f(1 - b1), (3, 7, 8), u & 0xFFFF), ("exp_avg_sq", (gl * gl) * f(1 - b2), (2, 15, 15), u >> 16)):
        code, scale = encode(a, inverses(torch), *fmt, part, k == "exp_avg_sq")
        assert np.array_equal(st[k + "_scale"].view(torch.uint8).cpu().numpy(), scale), k
        assert np.array_equal(st[k].view(torch.uint8).cpu().numpy(), code), k


def test_adamw_8_follows_a_falling_gradient(torch_mod):
    """v falls by 0.1 % a step, far less than the codes' spacing of 12 .. 25 %: on average over 4096 elements it does.  A step's rounding
    is unbiased, so the mean of v is off by at most 5 standard deviations: each of 400 steps adds a variance of at most
    (spacing 1/4) x (drift 1/1000) of v^2, the mean over 4096 has a 4096th of it"""
    torch = torch_mod
    from sound_bubble_amd import ops
    p = [torch.zeros(4096, device="cuda")]
    st = ops.adamw_state(p, bits=8)
    ops.adamw_step(p, [torch.ones(4096, device="cuda")], st, 1, lr=0.0)
    v1 = (st["exp_avg_sq"].float().view(-1, 256) * st["exp_avg_sq_scale"].float()[:, None]).mean().item()
    zero = [torch.zeros(4096, device="cuda")]
    for step in range(2, 402):
        ops.adamw_step(p, zero, st, step, lr=0.0)
    v = (st["exp_avg_sq"].float().view(-1, 256) * st["exp_avg_sq_scale"].float()[:, None]).mean().item()
    want = v1 * 0.999 ** 400
    assert abs(v - want) <= 5 * want * (400 * 0.25 / 1000 / 4096) ** 0.5 + 1e-5 * want


def test_adamw_8_values(torch_mod):
    """a NaN marks its block and no other; v > 0 never becomes 0; blocks of zeros; the largest and smallest magnitudes"""
    torch = torch_mod
    from sound_bubble_amd import ops
    g = gen(torch, 50)
    p = [torch.zeros(1024, device="cuda")]
    gr = torch.randn(1024, generator=g, device="cuda")
    gr[300] = float("nan")
    gr[512:768] = 0
    gr[768:] = 1e-4
    gr[800] = 1e15
    st = ops.adamw_state(p, bits=8)
    ops.adamw_step(p, [gr], st, 1, lr=0.1, weight_decay=0.0)
    for k in ("exp_avg", "exp_avg_sq"):
        s = st[k + "_scale"].float()
        assert torch.isnan(s[1]) and torch.isfinite(s[[0, 2, 3]]).all()
        v = st[k].float().view(-1, 256) * s[:, None]
        assert torch.isfinite(v[[0, 2, 3]]).all() and not v[2].any()
    assert (v[3] > 0).all() and v[3, 32] == v[3].max()
    assert torch.isnan(p[0][300]) and torch.isfinite(p[0][:256]).all() and torch.isfinite(p[0][512:]).all()


def test_adamw_skips_and_order(torch_mod):
    """parameters without a gradient are left alone with their states; mixed types; views at odd addresses; the neighbours stay"""
    torch = torch_mod
    from sound_bubble_amd import ops
    g = gen(torch, 60)
    flat = torch.randn(2000, generator=g, device="cuda")
    keep = flat.clone()
    ps = [flat[1:300], torch.randn(500, generator=g, device="cuda").bfloat16(), flat[301:800], torch.randn(40, generator=g, device="cuda").half(),
          torch.zeros(0, device="cuda")]
    gs = [torch.randn(p.shape, generator=g, device="cuda").to(p.dtype) for p in ps]
    gs[2] = None
    gs[1] = gs[1].float()
    st = ops.adamw_state(ps)
    ops.adamw_step(ps, gs, st, 1, clip=1.0, **HYPER)
    assert torch.equal(flat[300:], keep[300:]) and flat[0] == keep[0] and not torch.equal(flat[1:300], keep[1:300])
    b = ops.adamw_blocks([p.numel() for p in ps])
    assert not st["exp_avg"][b[2] * 256:b[3] * 256].any() and st["exp_avg"][b[3] * 256:].any()
    alone = [keep[1:300].clone(), *(p.clone() for p in ps[1:])]
    norm = torch.cat([t.double() for t in gs if t is not None]).norm()
    one = ops.adamw_state(alone[:1])
    ops.adamw_step(alone[:1], gs[:1], one, 1, gscale=min(1.0, float(1.0 / (norm + 1e-6))), **HYPER)
    assert torch.allclose(alone[0], flat[1:300], rtol=8 * U, atol=8 * U * 4)


def test_adamw_step_and_lr_on_the_device(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import ops
    g = gen(torch, 61)
    a = [torch.randn(700, generator=g, device="cuda")]
    b = [a[0].clone()]
    sa, sb = ops.adamw_state(a, 8), ops.adamw_state(b, 8)
    t, lr = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), 0.25, device="cuda")
    kw = {k: v for k, v in HYPER.items() if k != "lr"}
    for step in range(1, 5):
        gr = [torch.randn(700, generator=g, device="cuda")]
        t.add_(1)
        ops.adamw_step(a, gr, sa, step, lr=0.25, **kw)
        ops.adamw_step(b, gr, sb, t, lr=lr, **kw)
    assert torch.equal(a[0], b[0]) and all(torch.equal(sa[k].view(torch.uint8), sb[k].view(torch.uint8)) for k in sa)


# ---- refusals, streams, graphs ----
def test_refusals(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    x, h = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(2, 8, device="cuda")
    bad = [lambda: F.layer_norm(x.double()), lambda: F.layer_norm(x, torch.ones(7, device="cuda")), lambda: F.layer_norm(x, torch.ones(8)),
           lambda: F.layer_norm(x, torch.ones(8, device="cuda").half()), lambda: F.layer_norm(x[..., :0]),
           lambda: F.layer_norm(x.half(), torch.ones(8, device="cuda"), torch.ones(8, device="cuda").half()),
           lambda: F.gated_scan(x, x.half()), lambda: F.gated_scan(x, x[:1]), lambda: F.gated_scan(x, x, form="tanh"), lambda: F.gated_scan(x, x, dim=3),
           lambda: F.gated_scan(x, x, h[:1]), lambda: F.gated_scan(x, x, h.half()), lambda: F.gated_scan(x, x, lengths=torch.tensor([1, 2])),
           lambda: F.gated_scan(x, x, lengths=torch.ones(3, dtype=torch.int64, device="cuda")), lambda: F.gated_scan(x, x.cpu()),
           lambda: F.gated_scan(x.long(), x), lambda: F.gated_scan_step(h, h, h.t().contiguous().t()), lambda: F.gated_scan_step(h, h, h.half()),
           lambda: ops.gated_scan_bwd(x, None, x, x, torch.zeros(3, device="cuda"))]
    p = [torch.zeros(300, device="cuda")]
    st = ops.adamw_state(p)
    step = lambda ps=p, gs=p, s=st, t=1, **kw: ops.adamw_step(ps, gs, s, t, **{"lr": 0.1, **kw})  # noqa: E731
    bad += [lambda: step(gs=[p[0][:5]]), lambda: step(gs=[p[0].half()]), lambda: step(gs=[p[0].cpu()]), lambda: step(t=0), lambda: step(clip=-1.0),
            lambda: step(s=ops.adamw_state([p[0][:3]])), lambda: step(s={}), lambda: step(ps=[p[0].double()]), lambda: step(gs=[]),
            lambda: step(ps=[torch.zeros(600, device="cuda")[::2]]), lambda: step(t=torch.ones(1, device="cuda")),
            lambda: step(lr=torch.ones(2, device="cuda")), lambda: step(ps=[p[0].half()], gs=[p[0]])]
    for i, call in enumerate(bad):
        with pytest.raises(E):
            call()
            pytest.fail(f"call {i} was not refused")


def test_other_stream(torch_mod):
    """launches go to the current stream, behind what it waits for"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops
    x, gate, h0, _, dh, dlast = scan_inputs(torch, (4, 3000, 256), 1, torch.float32, torch.float32, "sigmoid", 70)
    want = F.gated_scan(F.layer_norm(x), gate, h0)
    s = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 0
        for _ in range(20):
            big = big @ big * 1e-4
        y += x + 0 * big[0, 0]
        got = F.gated_scan(F.layer_norm(y), gate, h0)
        p = [y.clone()]
        st = ops.adamw_state(p)
        ops.adamw_step(p, [y], st, 1, clip=1.0, lr=0.1)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = [x.clone()]
    st2 = ops.adamw_state(q)
    ops.adamw_step(q, [x], st2, 1, clip=1.0, lr=0.1)
    assert torch.equal(p[0], q[0])


def test_block_trains_and_a_graph_replays_it(torch_mod):
    """The three together, as a block of a model uses them: layer norm, projection, scan, projection, residual; AdamW on every
    parameter.  The captured step, replayed with eager work between the replays, takes the eager step's values."""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops
    B, T, C, H = 2, 150, 24, 40

    def fresh():
        g = gen(torch, 80)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        ps = [1 + 0.1 * r(C), 0.1 * r(C), 0.2 * r(C, 2 * H), 0.2 * r(H, C)]
        return [p.requires_grad_(True) for p in ps]

    def loss_of(ps, x, target):
        u = F.layer_norm(x, ps[0], ps[1])
        v, z = (u.reshape(B * T, C) @ ps[2]).reshape(B, T, 2 * H).chunk(2, -1)
        h, last = F.gated_scan(v, z)
        y = x + (h.reshape(B * T, H) @ ps[3]).reshape(B, T, C)
        return ((y - target) ** 2).mean() + (last ** 2).mean()

    def step(ps, st, t, x, target):
        loss = loss_of(ps, x, target)
        gs = torch.autograd.grad(loss, ps)
        t.add_(1)
        with torch.no_grad():
            ops.adamw_step(ps, gs, st, t, lr=1e-2, clip=1.0)
        return loss.detach()

    g = gen(torch, 81)
    data = [(torch.randn(B, T, C, generator=g, device="cuda"), torch.randn(B, T, C, generator=g, device="cuda")) for _ in range(6)]
    # the gradients of the whole against the same block in 64 bits
    ps = fresh()
    gs = torch.autograd.grad(loss_of(ps, *data[0]), ps)
    p64 = [p.detach().double().requires_grad_(True) for p in ps]
    x64, t64 = (d.double() for d in data[0])
    mean = x64.mean(-1, keepdim=True)
    u = (x64 - mean) / ((x64 - mean).square().mean(-1, keepdim=True) + 1e-5).sqrt() * p64[0] + p64[1]
    v, z = (u.reshape(B * T, C) @ p64[2]).reshape(B, T, 2 * H).chunk(2, -1)
    h, hs = torch.zeros(B, H, dtype=torch.float64, device="cuda"), []
    for t in range(T):
        a = torch.sigmoid(z[:, t])
        h = a * h + (1 - a) * v[:, t]
        hs.append(h)
    y = x64 + (torch.stack(hs, 1).reshape(B * T, H) @ p64[3]).reshape(B, T, C)
    want = torch.autograd.grad(((y - t64) ** 2).mean() + (h ** 2).mean(), p64)
    for a, b in zip(gs, want):
        assert (a.double() - b).norm() <= 1000 * U * b.norm() * 4      # sums over 300 positions of terms some 10 times the result
    del gs, p64, want, y, hs, h, v, z, u

    eager, st_e, t_e = fresh(), None, torch.zeros(1, dtype=torch.int32, device="cuda")
    st_e = ops.adamw_state(eager)
    losses = [step(eager, st_e, t_e, *d) for d in data]
    ps, t = fresh(), torch.zeros(1, dtype=torch.int32, device="cuda")
    st = ops.adamw_state(ps)
    x, target = (d.clone() for d in data[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):                       # warm up on copies: libraries and the allocator
        warm = fresh()
        step(warm, ops.adamw_state(warm), torch.zeros(1, dtype=torch.int32, device="cuda"), x, target)
        del warm
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(ps, st, t, x, target)
    for d, want in zip(data, losses):
        x.copy_(d[0])
        target.copy_(d[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        F.layer_norm(torch.randn(50, 333, device="cuda"))
    assert int(t) == 6 and all(torch.equal(a, b) for a, b in zip(ps, eager))
    with pytest.raises(Exception, match="int32 tensor"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.adamw_step(ps, [p.detach() for p in ps], st, 7, lr=0.1)


def test_two_graphs_do_not_share_memory(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import functional as F
    ins = [scan_inputs(torch, (1, 6000, 24), 1, torch.float32, torch.float32, "sigmoid", 90 + k) for k in range(2)]
    F.gated_scan(*ins[0][:3])
    want = [F.gated_scan(*i[:3]) for i in ins]
    graphs, outs = [], []
    for i in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(F.gated_scan(*i[:3]))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o[0].fill_(7)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_calls_with_and_without_python_in_between(torch_mod, monkeypatch):
    """the library's own calls (csrc/seq/sb_seq_torch.cpp) and the Python wrappers: the same bits, refusals and version counts"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops, ops_seq
    assert ops_seq.native() is not None
    ins = scan_inputs(torch, (3, 200, 24), 1, torch.bfloat16, torch.float32, "sigmoid", 97, ragged=True)

    def everything():
        x, gate, h0, lengths, dh, dlast = ins
        out = []
        for t in (x, x.transpose(0, 1), x[:, ::2]):
            w = torch.ones(24, device="cuda", requires_grad=True)
            leaf = t.detach().requires_grad_(True)
            y = F.layer_norm(leaf, w, w.detach())
            out += [y.detach(), *torch.autograd.grad(y, (leaf, w), t)]
        for rev in (False, True):
            leaves = [t.detach().requires_grad_(True) for t in (x, gate, h0)]
            h, last = F.gated_scan(*leaves, lengths=lengths.int(), reverse=rev)
            out += [h.detach(), last.detach(), *torch.autograd.grad((h, last), leaves, (dh, dlast))]
        out += F.gated_scan(x, gate, dim=-1, form="decay")
        state = h0.clone()
        v = state._version
        out += [F.gated_scan_step(x[:, 0], gate[:, 0], state), state]
        assert state._version == v + 1
        for bits, dt in ((32, torch.float32), (8, torch.bfloat16)):
            g = gen(torch, 3)
            ps = [torch.randn(n, generator=g, device="cuda").to(dt) for n in [5] * 130 + [70000]]
            st = ops.adamw_state(ps, bits)
            v = ps[0]._version
            for step in (1, 2):
                ops.adamw_step(ps, [p.clone() for p in ps], st, step, lr=1e-2, clip=0.5, seed=9)
            assert ps[0]._version == v + 2
            out += ps + [t.view(torch.uint8) for t in st.values()]
        return out
    a = everything()
    monkeypatch.setattr(ops_seq, "_NATIVE", False)
    b = everything()
    assert len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


def test_refusals_without_the_native_calls(torch_mod, monkeypatch):
    from sound_bubble_amd import ops_seq
    monkeypatch.setattr(ops_seq, "_NATIVE", False)
    test_refusals(torch_mod)
    test_gated_scan_layouts(torch_mod)
    test_layer_norm_layouts(torch_mod)
    test_adamw_skips_and_order(torch_mod)


def test_more_refusals(torch_mod):
    """lazily negated and sparse tensors, a state that is no buffer of its own, gradients through the step"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    neg = torch.randn(4, 8, dtype=torch.complex64, device="cuda").conj().imag
    assert neg.is_neg()
    h = torch.zeros(4, 8, device="cuda")
    leaf = h.clone().requires_grad_(True)
    for call in (lambda: F.layer_norm(neg), lambda: F.gated_scan(h, neg), lambda: F.layer_norm(h.to_sparse()), lambda: F.gated_scan_step(h, h, neg),
                 lambda: F.gated_scan_step(leaf, h, h), lambda: F.gated_scan_step(h, h, h.t().contiguous().t()), lambda: F.layer_norm([1.0])):
        with pytest.raises(E):
            call()
    p = torch.ones(4, 8, device="cuda")
    for g in (neg, h.to_sparse()):
        with pytest.raises(E, match="gradient 0"):
            ops.adamw_step([p], [g], ops.adamw_state([p]), 1, lr=0.1)
    assert p.eq(1).all()


@pytest.mark.parametrize("how", ["native", "python"])
def test_lazily_negated_gradients(torch_mod, monkeypatch, how):
    """a gradient that reaches the backward pass as a negated view"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops_seq
    monkeypatch.setattr(ops_seq, "_PYTHON", how == "python")
    x = torch.randn(3, 40, 8, generator=gen(torch, 5), device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    dy = torch.randn(3, 40, 8, dtype=torch.complex64, device="cuda").conj().imag
    assert dy.is_neg()
    y, (h, last) = F.layer_norm(x, w), F.gated_scan(x, x * 2)
    dl = dy[:, 0]
    for lazy, plain in zip(torch.autograd.grad((y, h, last), (x, w), (dy, dy, dl), retain_graph=True),
                           torch.autograd.grad((y, h, last), (x, w), (dy.resolve_neg(), dy.resolve_neg(), dl.resolve_neg()))):
        assert torch.equal(lazy, plain)


@pytest.mark.parametrize("how", ["native", "python"])
def test_tangents_are_refused(torch_mod, monkeypatch, how):
    """forward-mode differentiation has no rule here: said, not dropped"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops_seq
    import torch.autograd.forward_ad as fwAD
    monkeypatch.setattr(ops_seq, "_PYTHON", how == "python")
    x, t = torch.randn(2, 5, 8, device="cuda"), torch.ones(2, 5, 8, device="cuda")
    with torch.enable_grad(), fwAD.dual_level():
        d = fwAD.make_dual(x, t)
        for call in (lambda: F.layer_norm(d), lambda: F.layer_norm(x, d[0, 0]), lambda: F.gated_scan(d, x), lambda: F.gated_scan(x, d),
                     lambda: F.gated_scan_step(d, x, torch.zeros_like(x))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
        assert torch.equal(F.layer_norm(x), F.layer_norm(x.clone()))


def test_adamw_refuses_what_it_cannot_mean(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import ops
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    p = torch.ones(300, device="cuda")
    two = [p, torch.ones(20, device="cuda"), p]
    st = ops.adamw_state(two)
    with pytest.raises(E, match="twice"):
        ops.adamw_step(two, two, st, 1, lr=0.1)
    one = ops.adamw_state([p])
    for kw in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(eps=float("nan")), dict(clip=float("nan"))):
        with pytest.raises(E):
            ops.adamw_step([p], [p], one, 1, lr=0.1, **kw)
    assert p.eq(1).all()


@pytest.mark.parametrize("how", ["native", "python", "dispatcher"])
def test_capture_refuses_leaves_of_a_live_eager_graph(torch_mod, monkeypatch, how):
    """the forward call under capture says so (its backward pass would end the process); without the eager graph it goes on"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops_seq
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    monkeypatch.setattr(ops_seq, "_PYTHON", how == "python")
    norm, scan = F.layer_norm, F.gated_scan
    if how == "dispatcher":
        from sound_bubble_amd import torch_ops  # noqa: F401
        norm = lambda x, w: torch.ops.sound_bubble.layer_norm(x, w, None, 1e-5)[0]  # noqa: E731
        scan = lambda x, z: torch.ops.sound_bubble.gated_scan(x, z, None, None, 1, "sigmoid", False)  # noqa: E731
    x = torch.randn(4, 50, 16, device="cuda")
    w = torch.ones(16, device="cuda", requires_grad=True)
    z = torch.zeros(4, 50, 16, device="cuda", requires_grad=True)
    eager = norm(x, w), scan(x, z)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            for call in (lambda: norm(x, w), lambda: scan(x, z)):
                with pytest.raises(E, match="eager graph"):
                    call()
            keep = x + 1
        finally:
            graph.capture_end()
    torch.cuda.current_stream().wait_stream(s)
    del eager, keep
    want = torch.autograd.grad(norm(x, w).sum() + scan(x, z)[0].sum(), (w, z))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(norm(x, w).sum() + scan(x, z)[0].sum(), (w, z))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        F.layer_norm(x)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_more_than_2_31_elements(torch_mod):
    """offsets that pass 32 bits: the far end of a large tensor is what the same rows, steps and blocks give by themselves"""
    torch = torch_mod
    from sound_bubble_amd import ops
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GiB of free GPU memory")
    n, rows, tail = 1024, (1 << 21) + 3, 100
    x, dy = (torch.randn(rows, n, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    w = torch.randn(n, device="cuda").bfloat16()
    y, mean, rstd = ops.layer_norm_fwd(x, w, None)
    assert torch.equal(y[-tail:], ops.layer_norm_fwd(x[-tail:], w, None)[0])
    dx = ops.layer_norm_bwd(dy, x, w, mean, rstd, want_dw=False, want_db=False)[0]
    assert torch.equal(dx[-tail:], ops.layer_norm_bwd(dy[-tail:], x[-tail:], w, mean[-tail:], rstd[-tail:], want_dw=False, want_db=False)[0])
    del y, dx, mean, rstd
    # gates of 0: h is x, and dgate_t is dh_t x_{t-1}
    gate = torch.zeros_like(x)
    h, last, states = ops.gated_scan_fwd(x, gate, dim=0, form="decay")
    assert torch.equal(h, x) and torch.equal(last, x[-1].float())
    del h
    dx, dgate, _ = ops.gated_scan_bwd(dy, None, x, gate, states, dim=0, form="decay")
    assert torch.equal(dx, dy)
    assert torch.equal(dgate[-tail:], (dy[-tail:].float() * x[-tail - 1:-1].float()).bfloat16())
    del dx, dgate, gate, states, x, dy
    # a strided view over as much memory: 3 sequences, more than 2^32 bytes apart
    far = (1 << 30) + 5
    big = torch.empty(2 * far + 64 * 48, device="cuda")
    x = big.as_strided((3, 64, 48), (far, 48, 1))
    x.copy_(torch.randn(3, 64, 48, device="cuda"))
    dense = x.contiguous()
    assert torch.equal(ops.layer_norm_fwd(x, None, None)[0], ops.layer_norm_fwd(dense, None, None)[0])
    for a, b in zip(ops.gated_scan_fwd(x, x), ops.gated_scan_fwd(dense, dense)):
        assert torch.equal(a, b)
    states = ops.gated_scan_fwd(x, x)[2]
    for a, b in zip(ops.gated_scan_bwd(x, None, x, x, states), ops.gated_scan_bwd(dense, None, dense, dense, states)):
        assert torch.equal(a, b)
    del big, x
    size, tail = (1 << 31) + 300, 44 + 5 * 256      # (the tail begins with a block)
    p, g = torch.zeros(size, device="cuda"), torch.zeros(size, device="cuda")
    p[-tail:], g[-tail:] = torch.randn(tail, device="cuda"), torch.randn(tail, device="cuda")
    q, gq = p[-tail:].clone(), g[-tail:].clone()
    sp, sq = ops.adamw_state([p]), ops.adamw_state([q])
    for step in (1, 2):
        ops.adamw_step([p], [g], sp, step, lr=0.1, clip=0.5)
        ops.adamw_step([q], [gq], sq, step, lr=0.1, clip=0.5)
    assert torch.equal(p[-tail:], q) and not p[:-tail].any()
    assert all(torch.equal(sp[k][-sq[k].numel():], sq[k]) for k in sq)
