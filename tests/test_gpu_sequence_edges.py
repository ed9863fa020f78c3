"""Sequence-block operators at the edges of their arguments, on the GPU, against their definitions in 64 bits."""
import numpy as np
import pytest

import test_gpu_sequence_ops as plain
from test_gpu_sequence_ops import U, dither, encode, gen, near

pytestmark = pytest.mark.gpu


# ---- layer norm: groups that take one row after the other ----
# more than two rows for every group of the forward grid (as many lanes as 4096 waves have, a row's lanes and vectors by its width), and of the
# backward one; the column sums of wide rows (128 parts) with several rows a part, and with parts that have none
MANY = [(600001, 1), (150001, 2), (70001, 7), (150001, 8), (40003, 33), (20011, 100), (9001, 255), (9001, 500), (9001, 600), (9001, 1000), (9001, 1500), (4501, 2040),
        (2501, 1025), (2501, 4096), (2503, 5000), (2503, 8192), (1301, 6100), (1301, 12000), (1301, 16384), (601, 10007), (601, 13001), (601, 20005), (130, 16385),
        (300, 24576), (129, 24577), (601, 30001), (601, 32768), (1301, 33001), (1100, 40001)]


@pytest.mark.parametrize("rows,n", MANY)
@pytest.mark.parametrize("xt,wt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32")])
def test_layer_norm_of_many_rows(torch_mod, rows, n, xt, wt):
    plain.test_layer_norm(torch_mod, rows, n, xt, wt)


# ---- gated scan: gates beyond 1 ----
def walk(torch, x, gate, h0, dh, dlast, reverse):
    """the "decay" recurrence along axis 1 in 64 bits: h, last, dx, dgate, dh0"""
    x, gate, dh = (t.double().flip(1) if reverse else t.double() for t in (x, gate, dh))
    T = x.shape[1]
    h = torch.zeros_like(x[:, 0]) if h0 is None else h0.double()
    before, hs, G = [], [], [None] * T
    for t in range(T):
        before.append(h)
        h = gate[:, t] * h + x[:, t]
        hs.append(h)
    c = dlast.double()
    for t in reversed(range(T)):
        G[t] = dh[:, t] + c
        c = gate[:, t] * G[t]
    hs, before, G = (torch.stack(v, 1) for v in (hs, before, G))
    out = {"h": hs, "dx": G, "dgate": G * before, "before": before}
    out = {k: v.flip(1) if reverse else v for k, v in out.items()}
    return {**out, "last": h, "dh0": c}


def check_walk(torch, x, gate, h0, dh, dlast, reverse):
    """Every term is positive, so every result is off by the roundings of its terms' factors: a term is a product of at most T gates, T - 1
    roundings however they are grouped, and as many additions at most; 64 for the joins.  dgate has two such factors.
    What is below float32's smallest number is lost: h and G are off by 2^-140 by that (2^10 half steps of 2^-150), and dgate, their product,
    by 2^-140 of each: a G of 1e-60 beside an h of 1e36 is 0, not 1e-24."""
    from sound_bubble_amd import functional as F, ops_seq
    B, T, C = x.shape
    assert ops_seq._scan_plan(B, T, C, ops_seq._TYPES[x.dtype])[1] > 0, "time is cut at this size"
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, h0) if t is not None]
    h, last = F.gated_scan(leaves[0], leaves[1], leaves[2] if h0 is not None else None, form="decay", reverse=reverse)
    grads = torch.autograd.grad((h, last), leaves, (dh, dlast))
    got = {"h": h.detach(), "last": last.detach(), **dict(zip(("dx", "dgate", "dh0"), grads))}
    want = walk(torch, x, gate, h0, dh, dlast, reverse)
    for k, v in got.items():
        assert want[k].abs().max() < 1e37
        lost = 1 + (want["dx"] + want["before"] if k == "dgate" else 0)
        near(torch, v, want[k], (2 * T + 64) * U * (2 if k == "dgate" else 1) * want[k] + 2.0 ** -140 * lost, k)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("top", [1.5, 200.0])
@pytest.mark.parametrize("xt", ["float32", "bfloat16"])
def test_gates_beyond_one_and_a_silent_start(torch_mod, xt, top, reverse):
    """nothing but zeros until the last steps, a loss on the first ones only: everything between is 0, whatever the gates' products are"""
    torch = torch_mod
    xt, live = getattr(torch, xt), 10
    g = gen(torch, 1)
    r = lambda *s: torch.rand(*s, generator=g, device="cuda") + 0.25  # noqa: E731
    x, dh = torch.zeros(2, 2048, 24, device="cuda", dtype=xt), torch.zeros(2, 2048, 24, device="cuda", dtype=xt)
    gate = top * (1 - 0.1 * torch.rand(2, 2048, 24, generator=g, device="cuda"))
    x[:, -live:], dh[:, :live] = r(2, live, 24).to(xt), r(2, live, 24).to(xt)
    if reverse:
        x, dh = x.flip(1).contiguous(), dh.flip(1).contiguous()
    check_walk(torch, x, gate, None, dh, torch.zeros(2, 24, device="cuda"), reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("shape", [(2, 2048, 24), (1, 3000, 7), (3, 1100, 130)])
def test_gates_whose_products_leave_float32(torch_mod, shape, reverse):
    """256 steps that grow by 2^150 and 256 that shrink by as much: states stay within float32, products over either do not"""
    torch = torch_mod
    B, T, C = shape
    g = gen(torch, 2)
    r = lambda *s: torch.rand(*s, generator=g, device="cuda") + 0.5  # noqa: E731
    place = torch.arange(T, device="cuda")
    gate = torch.where(place // 256 % 2 == 0, 1.5, 1 / 1.5)[None, :, None].expand(shape).contiguous()
    x, dh = 1e-16 * r(*shape), 1e-26 * r(*shape)
    # what comes back from behind has the steps behind the last whole pair of 256 to go first
    left = T % 512
    c = 1e20 * 1.5 ** (-left if left <= 256 else left - 512)      # (its smallest, 1e-25, where the shrinking begins)
    if reverse:
        gate, x, dh = (t.flip(1).contiguous() for t in (gate, x, dh))
    check_walk(torch, x, gate, 1e-15 * r(B, C), dh, c * r(B, C), reverse)


@pytest.mark.parametrize("gate", [2.0 ** -0.5, 0.65, 0.4])
def test_a_large_state_that_decays_over_segments(torch_mod, gate):
    """segments whose products are between 2^-278 and 2^-126, or below: what they leave of a state of 1e36 is within float32"""
    torch = torch_mod
    g = gen(torch, 9)
    r = lambda *s: torch.rand(*s, generator=g, device="cuda") + 0.5  # noqa: E731
    shape = (2, 1100, 24)
    x, dh = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    x[:, ::100], dh[:, ::100] = 1e-20 * r(2, 11, 24), 1e-20 * r(2, 11, 24)
    z = torch.full(shape, gate, device="cuda")
    # (walk's own small values below float32's are within the 2^-140)
    check_walk(torch, x, z, 1e36 * r(2, 24), dh, 1e16 * r(2, 24), False)


def test_as_many_segments_as_there_are(torch_mod):
    """gates of 1 over 1.2 M steps: sums, forwards and backwards.  A term goes through at most 16 additions in a lane, 8 joins for each of a
    segment's 24 chunks, or 24 x 16 of a wave's part and 8 joins, and 409 segments: below 1100 roundings"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops_seq
    T, C = 1250000, 3
    assert ops_seq._scan_plan(1, T, C, 0)[1] // (2 * C) == 409 + 103
    x = (torch.rand(1, T, C, generator=gen(torch, 10), device="cuda") + 0.5).requires_grad_(True)
    gate = torch.ones(1, T, C, device="cuda", requires_grad=True)
    h, last = F.gated_scan(x, gate, form="decay")
    want = x.detach().double().cumsum(1)
    near(torch, h.detach(), want, 1100 * U * want, "h")
    dh = torch.rand(1, T, C, generator=gen(torch, 11), device="cuda") + 0.5
    dx, dgate = torch.autograd.grad(h, (x, gate), dh)
    G = dh.double().flip(1).cumsum(1).flip(1)
    near(torch, dx, G, 1100 * U * G, "dx")
    before = torch.cat([torch.zeros_like(want[:, :1]), want[:, :-1]], 1)
    near(torch, dgate, G * before, 2201 * U * G * before, "dgate")


# ---- calls out of the ordinary ----
def test_a_state_made_under_inference_mode(torch_mod):
    """streaming under no_grad goes on with a state that inference mode made (it has no version count)"""
    torch = torch_mod
    from sound_bubble_amd import functional as F
    x, gate = torch.randn(2, 3, 40, generator=gen(torch, 3), device="cuda")
    with torch.inference_mode():
        state = torch.zeros(3, 40, device="cuda")
        F.gated_scan_step(x, gate, state)
    with torch.no_grad():
        y = F.gated_scan_step(x, gate, state)
    want, _ = F.gated_scan(torch.stack([x, x], 1), torch.stack([gate, gate], 1))
    assert torch.equal(y, want[:, 1]) and torch.equal(state, want[:, 1])
    assert torch.equal(F.gated_scan(x[None], gate[None], reverse=1)[0], F.gated_scan(x[None], gate[None], reverse=True)[0])


@pytest.mark.parametrize("how", ["native", "python"])
def test_a_step_whose_inputs_are_views_of_its_state(torch_mod, monkeypatch, how):
    """the inputs are those from before the call, in whatever order they lie on the state's memory"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops_seq
    monkeypatch.setattr(ops_seq, "_PYTHON", how == "python")
    n = 4096
    views = {"itself": lambda b: b[n:2 * n].view(64, 64), "transposed": lambda b: b[n:2 * n].view(64, 64).t(), "one row": lambda b: b[n:n + 64].expand(64, 64),
             "behind": lambda b: b[n + 1:2 * n + 1].view(64, 64), "in front": lambda b: b[n - 4:2 * n - 4].view(64, 64),
             "apart": lambda b: b[2 * n:].view(64, 64), "16 bits": lambda b: b.view(torch.bfloat16)[2 * n:3 * n].view(64, 64)}
    for name, view in views.items():
        for gate_too in (False, True):
            buf = torch.randn(3 * n, generator=gen(torch, 6), device="cuda")
            state, x = buf[n:2 * n].view(64, 64), view(buf)
            if name == "16 bits":
                x.copy_(torch.randn(64, 64, generator=gen(torch, 8), device="cuda"))
            gate = x if gate_too else torch.randn(64, 64, generator=gen(torch, 7), device="cuda")
            want = state.clone()
            y = F.gated_scan_step(x.clone(), gate.clone(), want)
            assert torch.equal(F.gated_scan_step(x, gate, state), y) and torch.equal(state, want), name


# ---- AdamW ----
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-19])
@pytest.mark.parametrize("pt,bits", [("float32", 32), ("bfloat16", 32), ("float32", 8)])
def test_adamw_of_tiny_gradients(torch_mod, pt, bits, eps):
    """v below 2^-126 beside an eps that does not cover it: the update is the formula's, from the kernel's own m and v"""
    torch = torch_mod
    from sound_bubble_amd import ops
    pt = getattr(torch, pt)
    g = gen(torch, 4)
    p = torch.randn(3000, generator=g, device="cuda").to(pt)
    # v = g^2 / 1000 in the first step: 1e-43 .. 1e-35, subnormal up to 1.2e-38
    grad = 10 ** (-20 + 4 * torch.rand(3000, generator=g, device="cuda")) * torch.randn(3000, generator=g, device="cuda").sign()
    state = ops.adamw_state([p], bits)
    lr, wd = 1e-3, 0.01
    for step in (1, 2, 3):
        w0 = (state["master"][:3000] if pt != torch.float32 else p).double().cpu().numpy()
        old = {k: v[:3000].double().cpu().numpy() for k, v in ops.adamw_state_values(state).items()}
        ops.adamw_step([p], [grad], state, step, lr=lr, eps=eps, weight_decay=wd)
        m, v = (x[:3000].double().cpu().numpy() for x in ops.adamw_state_values(state).values())
        if bits == 8:      # (the update goes by the values before their rounding to 8 bits, float32 operations on the decoded ones)
            f, gr = np.float32, grad.cpu().numpy()
            m = (old["exp_avg"].astype(f) * f(0.9) + gr * f(1 - 0.9)).astype(np.float64)
            v = (old["exp_avg_sq"].astype(f) * f(0.999) + (gr * gr) * f(1 - 0.999)).astype(np.float64)
        assert (v < 2.0 ** -126).sum() > 1000 and (v > 0).all()
        update = lr / (1 - 0.9 ** step) * m / (np.sqrt(v) / np.sqrt(1 - 0.999 ** step) + eps)
        got = (state["master"][:3000] if pt != torch.float32 else p).double().cpu().numpy()
        # root and reciprocal are off by 2 U each, the products, the sum and the rates (rounded to float32) by U: 12 in all; p's own 4
        bound = 12 * U * np.abs(update) + 4 * U * np.abs(w0)
        assert (np.abs(got - (w0 * (1 - lr * wd) - update)) <= bound).all()


@pytest.mark.parametrize("size", [1e20, 1e30])
@pytest.mark.parametrize("count", [1, 150])
def test_clipping_far_beyond_the_norm(torch_mod, count, size):
    """gradients whose squares' sum leaves float32: they are scaled to the norm that clip asks for"""
    torch = torch_mod
    from sound_bubble_amd import ops
    g = gen(torch, 5)
    ps = [torch.zeros(700, device="cuda") for _ in range(count)]
    gs = [size * torch.randn(700, generator=g, device="cuda") for _ in ps]
    st = ops.adamw_state(ps)
    ops.adamw_step(ps, gs, st, 1, lr=0.1, clip=2.0, gscale=0.5)
    flat = torch.cat([t.double() for t in gs]) * 0.5
    flat *= 2.0 / (flat.norm() + 1e-6)
    m = torch.cat([st["exp_avg"][768 * k:768 * k + 700] for k in range(count)]).double()
    v = torch.cat([st["exp_avg_sq"][768 * k:768 * k + 700] for k in range(count)]).double()
    # the coefficient and its product with gscale: 2 U; two products: 2 U, twice that squared; 1 - beta rounded: U
    assert ((m - 0.1 * flat).abs() <= 8 * U * 0.1 * flat.abs()).all()
    assert ((v - 0.001 * flat ** 2).abs() <= 16 * U * 0.001 * flat ** 2 + 2.0 ** -149).all()
    assert abs(float(m.norm()) / 0.1 - 2.0) < 1e-5
    gs[0][3] = float("inf")      # (a coefficient of 0, and of it nothing: as torch.nn.utils.clip_grad_norm_)
    ops.adamw_step(ps, gs, st, 2, lr=0.1, clip=2.0)
    assert torch.isnan(ps[0][3]) and torch.isfinite(ps[0][4:]).all()


@pytest.mark.parametrize("which", ["exp_avg", "exp_avg_sq"])
def test_8_bit_codes_at_their_borders(torch_mod, which):
    """Values whose part cut off and dither add up to exactly 1, in a block of every scale: rounded up, as the format's exact powers of two
    have it; a scale that is off by one ulp rounds them down.  betas of 0: the moments are g and g^2"""
    torch = torch_mod
    from sound_bubble_amd import ops
    mant, bias, top, lo, hi = (3, 7, 8, 7, 246) if which == "exp_avg" else (2, 15, 15, 15, 239)
    bytes_, cut, rng = np.arange(lo, hi + 1).repeat(256), 23 - (3 if which == "exp_avg" else 2), np.random.default_rng(1)
    n = bytes_.size
    u = dither(n, 1, 0).astype(np.int64)
    u16 = u & 0xFFFF if which == "exp_avg" else u >> 16
    add = (u16 << (cut - 16)) + (1 << (cut - 17))
    g, found = np.zeros(n, np.float32), np.zeros(n, bool)
    for _ in range(200):      # (not every float32 is a square: other leading bits are tried until one is)
        e, lead = rng.integers(1 - bias, top, n), rng.integers(0, 1 << mant, n)
        x = np.ldexp(1 + (lead * 2.0 ** cut + (1 << cut) - add) / 2.0 ** 23, e + bytes_ - 127).astype(np.float32)
        with np.errstate(over="ignore"):
            c = x if which == "exp_avg" else np.sqrt(x)
            ok = ~found & (c.astype(np.float32) == c) & ((c if which == "exp_avg" else c * c) == x)
        g[ok], found = c[ok], found | ok
    largest = np.ldexp(1.0, top + bytes_[::256] - 127)      # (1 .. 1.75 of it give this scale)
    g[::256] = largest if which == "exp_avg" else np.sqrt(largest * np.where((top + bytes_[::256] - 127) % 2, 1.125, 1.0))
    assert found.mean() > 0.99
    p = torch.zeros(n, device="cuda")
    state = ops.adamw_state([p], bits=8)
    ops.adamw_step([p], [torch.from_numpy(g).cuda()], state, 1, lr=0.1, betas=(0.0, 0.0))
    exact = np.ldexp(np.float32(1), 127 - np.arange(256))
    with np.errstate(over="ignore"):
        want, scale = encode(g if which == "exp_avg" else g * g, exact, mant, bias, top, u16, which != "exp_avg")
    assert np.array_equal(scale, bytes_[::256].astype(np.uint8))
    assert np.array_equal(state[which + "_scale"].view(torch.uint8).cpu().numpy(), scale)
    got = state[which].view(torch.uint8).cpu().numpy()
    assert np.array_equal(got, want), np.unique(bytes_[got != want])


def test_adamw_skipped(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import ops
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    p = torch.ones(300, device="cuda")
    state = ops.adamw_state([p])
    for skipped in (torch.zeros(1, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32),
                    torch.zeros(1, dtype=torch.int64, device="cuda")):
        with pytest.raises(E, match="skipped"):
            ops.adamw_step([p], [p.clone()], state, 1, lr=0.1, skipped=skipped)
    assert p.eq(1).all()
    ops.adamw_step([p], [p.clone()], state, 1, lr=0.1, skipped=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert not p.eq(1).any()


@pytest.mark.parametrize("how", ["native", "python"])
def test_adamw_refuses_parameters_that_share_memory(torch_mod, monkeypatch, how):
    """two workgroups would update the same elements; neighbours in one buffer are fine"""
    torch = torch_mod
    from sound_bubble_amd import ops, ops_seq
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    monkeypatch.setattr(ops_seq, "_PYTHON", how == "python")
    flat = torch.ones(1000, device="cuda")
    for ps in ([flat[:301], flat[300:]], [flat[5:6], flat], [flat, flat[999:]], [flat[:500], flat[500:], flat[200:300]]):
        with pytest.raises(E, match="share memory"):
            ops.adamw_step(ps, [p.clone() for p in ps], ops.adamw_state(ps), 1, lr=0.1)
    assert flat.eq(1).all()
    ps = [flat[500:], flat[:0], flat[:300], flat[300:500], flat[100:200]]      # (the last one is not updated)
    ops.adamw_step(ps, [p.clone() for p in ps[:-1]] + [None], ops.adamw_state(ps), 1, lr=0.1)
    assert not flat.eq(1).any()


@pytest.mark.parametrize("key,value", [("lr", 1e-4), ("weight_decay", 0.0), ("betas", (0.8, 0.999)), ("eps", 1e-6), ("maximize", True)])
def test_fused_adamw_refuses_states_of_several_groups(torch_mod, key, value):
    """one group's values would go to all parameters; groups that differ in nothing are fine"""
    torch = torch_mod
    from sound_bubble_amd.train import FusedAdamW
    ps = [torch.nn.Parameter(torch.ones(n, device="cuda")) for n in (30, 5)]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = FusedAdamW(ps, lr=1e-2)
    opt.step()
    keep = [t.clone() for t in opt.state.values()]
    for same in (False, True):
        other = torch.optim.AdamW([{"params": ps[:1]}, {"params": ps[1:], **({} if same else {key: value})}], lr=1e-3)
        other.step()
        if same:
            opt.load_state_dict(other.state_dict())
            assert opt.param_groups[0]["lr"] == 1e-3 and opt.step_count == 1
            continue
        with pytest.raises(ValueError, match=key):
            opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == 1e-2 and all(torch.equal(a, b) for a, b in zip(keep, opt.state.values()))


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_does_not_count(torch_mod, capturable):
    torch = torch_mod
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    from sound_bubble_amd.train import FusedAdamW
    p = torch.nn.Parameter(torch.ones(30, device="cuda").bfloat16())
    opt = FusedAdamW([p], capturable=capturable)
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(E, match="clip"):
        opt.step(grad_clip=-1.0)
    assert opt.step_count == 1
    opt.step()
    assert opt.step_count == 2
