"""FusedAdamW beside torch.optim.AdamW, its checkpoints, a training run through the harness, and the dispatcher forms of the
sequence-block operators."""
import json
import os

import numpy as np
import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def params_of(torch, seed=0, dtype=None):
    g = torch.Generator("cuda").manual_seed(seed)
    shapes = [(7,), (64, 33), (1,), (300, 5), (4096,)]
    return [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda").to(dtype or torch.float32)) for s in shapes], g


@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("capturable", [False, True])
def test_fused_adamw_is_torch_adamw(torch_mod, clip, capturable):
    torch = torch_mod
    from sound_bubble_amd.train import FusedAdamW
    ps, g = params_of(torch)
    qs = [torch.nn.Parameter(p.detach().double()) for p in ps]
    kw = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.1)
    opt, ref = FusedAdamW(ps, capturable=capturable, **kw), torch.optim.AdamW(qs, **kw)
    for step in range(5):
        if step == 3:
            opt.param_groups[0]["lr"] = ref.param_groups[0]["lr"] = 5e-4
        for p, q in zip(ps, qs):
            p.grad = torch.randn(p.shape, generator=g, device="cuda")
            q.grad = p.grad.double() / 2
        if clip:
            torch.nn.utils.clip_grad_norm_(qs, clip)
        opt.step(grad_clip=clip, world_size=2)
        ref.step()
    assert opt.step_count == 5
    for p, q in zip(ps, qs):
        # 5 steps of lr times an update of at most 10 (1 / sqrt(1 - b2)); the moments' roundings are 12 U of those a step, the
        # parameter's 4 U; where clipping scales all gradients alike the update hardly changes
        assert ((p.double() - q).abs() <= 5 * (4 * U * (q.abs() + 1) + 2e-3 * 10 * 40 * U)).all()


def test_fused_adamw_checkpoint(torch_mod):
    """torch's layout both ways; a resumed run goes on to the same bits, in 32 and in 8 bits, with master copies"""
    torch = torch_mod
    from sound_bubble_amd.train import FusedAdamW
    for bits, dtype in ((32, torch.float32), (8, torch.float32), (8, torch.bfloat16), (32, torch.float16)):
        ps, g = params_of(torch, 3, dtype)
        opt = FusedAdamW(ps, lr=1e-2, state_bits=bits, seed=5)
        grads = [[torch.randn(p.shape, generator=g, device="cuda").to(dtype) * 1e-2 for p in ps] for _ in range(4)]

        def run(o, p, which):
            for k in which:
                for q, t in zip(p, grads[k]):
                    q.grad = t.clone()
                o.step(grad_clip=1.0)
        run(opt, ps, (0, 1))
        sd = opt.state_dict()
        qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        two = FusedAdamW(qs, lr=1.0, state_bits=bits, seed=5)
        two.load_state_dict(sd)
        assert two.step_count == 2
        for k in opt.state:
            if bits == 32 or k == "master":
                assert torch.equal(opt.state[k], two.state[k])
        run(opt, ps, (2, 3))
        run(two, qs, (2, 3))
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
        a, b = opt.state_dict()["state"], two.state_dict()["state"]
        assert all(torch.equal(a[i][k], b[i][k]) for i in a for k in ("exp_avg", "exp_avg_sq"))
    # torch's own optimiser takes the layout, and its state comes in
    ps, g = params_of(torch, 4)
    opt = FusedAdamW(ps, lr=1e-2)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g, device="cuda")
    opt.step()
    ref = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=1.0)
    ref.load_state_dict(opt.state_dict())
    assert torch.equal(ref.state[ref.param_groups[0]["params"][1]]["exp_avg"], opt.state_dict()["state"][1]["exp_avg"])
    opt8 = FusedAdamW(ps, state_bits=8)
    opt8.load_state_dict(ref.state_dict())
    v, w = opt8.state_dict()["state"], opt.state_dict()["state"]
    for i in v:
        x, y = v[i]["exp_avg_sq"], w[i]["exp_avg_sq"]
        top = max(float(t["exp_avg_sq"].max()) for t in w.values())
        # half a code's spacing (2^-3), below the normal codes half of the smallest, and no positive value becomes 0
        assert ((x - y).abs() <= y * 2.0 ** -3 + top * 2.0 ** -30).all() and (x[y > 0] > 0).all()
        x, y = v[i]["exp_avg"], w[i]["exp_avg"]
        top = max(float(t["exp_avg"].abs().max()) for t in w.values())
        assert ((x - y).abs() <= y.abs() * 2.0 ** -4 + top * 2.0 ** -16).all()


def test_fused_adamw_over_a_model_and_parameters_without_gradients(torch_mod):
    torch = torch_mod
    from sound_bubble_amd.train import FlatBucket, FusedAdamW
    m = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 4)).cuda()
    bucket = FlatBucket(m)
    opt = FusedAdamW(bucket, lr=1e-2)
    x = torch.randn(16, 20, device="cuda")
    first = None
    for _ in range(3):
        bucket.zero_grad()
        loss = (m(x) ** 2).mean()
        loss.backward()
        opt.step(grad_clip=1.0)
        first = first if first is not None else loss.detach().clone()
    ps, _ = params_of(torch, 6)
    v0 = [p._version for p in ps]
    opt = FusedAdamW(ps, lr=1e-2)
    keep = [p.detach().clone() for p in ps]
    ps[1].grad = torch.ones_like(ps[1])
    opt.step()
    assert not torch.equal(ps[1], keep[1]) and all(torch.equal(a, b) for i, (a, b) in enumerate(zip(ps, keep)) if i != 1)
    assert [p._version - v for p, v in zip(ps, v0)] == [0, 1, 0, 0, 0]
    opt.zero_grad()
    assert ps[1].grad is None
    with pytest.raises(ValueError):
        FusedAdamW([])
    with pytest.raises(NotImplementedError):
        FusedAdamW(ps, amsgrad=True)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_optimiser_step(torch_mod, bits):
    """a captured step counts on at every replay and takes the learning rate that sync_lr() put there"""
    torch = torch_mod
    from sound_bubble_amd.train import FusedAdamW
    ps, g = params_of(torch, 7)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = (FusedAdamW(p, lr=1e-2, state_bits=bits, capturable=True) for p in (ps, qs))
    for p, q in zip(ps, qs):
        p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step(grad_clip=1.0)
    for k in range(4):
        if k == 2:
            a.param_groups[0]["lr"] = b.param_groups[0]["lr"] = 1e-3
            b.sync_lr()
        for p, q in zip(ps, qs):
            p.grad.normal_(generator=g)
            q.grad.copy_(p.grad)
        a.step(grad_clip=1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert a.step_count == b.step_count == 4


@pytest.mark.parametrize("params", [{"lr": 1e-3}, {"lr": 1e-3, "weight_decay": 0.05, "state_bits": 8}])
def test_harness_takes_adamw(torch_mod, tmp_path, params):
    """the experiment JSON's optimizer by its dotted path: two steps, a checkpoint, a resumed step"""
    torch = torch_mod
    from sound_bubble_amd.harness import PLModule
    from sound_bubble_amd.train import FusedAdamW, train_step
    cfg = json.load(open(os.path.join(ROOT, "experiments", "bubble_small_synthetic.json")))["pl_module_args"]
    cfg = dict(cfg, optimizer="torch.optim.AdamW", optimizer_params=params, grad_clip=1.0, model_params=dict(cfg["model_params"], B=1))
    torch.manual_seed(0)
    pl = PLModule(**cfg)
    assert isinstance(pl.optimizer, FusedAdamW) and abs(pl.get_current_lr() - 1e-4) < 1e-12      # (its LinearLR starts at 0.1)
    n_ch = cfg["model_params"]["num_ch"]
    g = torch.Generator("cuda").manual_seed(1)
    inp = {"mixture": torch.randn(2, n_ch, 192 * 6, generator=g, device="cuda")}
    if "dis_type" in cfg["model_params"]:
        inp["dis_embed"] = torch.eye(3, device="cuda")[:2]
    tgt = torch.randn(2, 1, 192 * 6, generator=g, device="cuda")
    pl.model.train()
    for _ in range(2):
        loss = train_step(pl.model, pl.bucket, pl.optimizer, inp, tgt, 100.0, grad_clip=pl.grad_clip)
        assert torch.isfinite(loss)
    path = str(tmp_path / "last.pt")
    pl.dump_state(path)
    two = PLModule(**cfg)
    two.load_state(path)
    two.model.train()
    assert two.optimizer.step_count == 2
    for (k, p), q in zip(pl.model.named_parameters(), two.model.parameters()):
        assert torch.equal(p, q), k
    a = pl.optimizer.state_dict()["state"]
    b = two.optimizer.state_dict()["state"]
    assert all(torch.equal(a[i][k], b[i][k]) for i in a for k in ("exp_avg", "exp_avg_sq"))
    with pytest.raises(NotImplementedError):
        PLModule(**dict(cfg, optimizer="torch.optim.SGD"))


def test_dispatcher_operators(torch_mod):
    """the same bits as the functional forms, opcheck, and a whole compiled block"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, torch_ops  # noqa: F401
    sb = torch.ops.sound_bubble
    g = torch.Generator("cuda").manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w, b, dy = r(3, 9, 40), r(40), r(40), r(3, 9, 40)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = sb.layer_norm(*leaves, 1e-5)[0]
    got = torch.autograd.grad(y, leaves, dy)
    ref = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = F.layer_norm(*ref, 1e-5)
    assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad(want, ref, dy)))
    gate, h0, ln = r(3, 9, 40), r(3, 40), torch.tensor([9, 0, 4], device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (x, gate, h0)]
    h, last, _ = sb.gated_scan(*leaves, ln, 1, "sigmoid", True)
    got = torch.autograd.grad((h, last), leaves, (dy, h0))
    ref = [t.clone().requires_grad_(True) for t in (x, gate, h0)]
    wh, wl = F.gated_scan(*ref, dim=1, reverse=True, lengths=ln)
    assert torch.equal(h, wh) and torch.equal(last, wl)
    assert all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad((wh, wl), ref, (dy, h0))))
    s1, s2 = h0.clone(), h0.clone()
    assert torch.equal(sb.gated_scan_step(x[:, 0], gate[:, 0], s1, "decay"), F.gated_scan_step(x[:, 0], gate[:, 0], s2, form="decay"))
    assert torch.equal(s1, s2)
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(sb.layer_norm.default, (x, w, None, 1e-5), test_utils=checks)
    torch.library.opcheck(sb.layer_norm_backward.default, (dy, x, w, r(3, 9), r(3, 9), True, False, False), test_utils=checks)
    torch.library.opcheck(sb.gated_scan.default, (x, gate, None, ln, 1, "decay", False), test_utils=checks)
    torch.library.opcheck(sb.gated_scan_step.default, (x[:, 0].contiguous(), gate[:, 0].contiguous(), s1, "sigmoid"), test_utils=checks)

    def block(x, w, b, p):
        u = sb.layer_norm(x, w, b, 1e-5)[0]
        v, z = (u @ p).chunk(2, -1)
        return sb.gated_scan(v, z, None, None, 1, "sigmoid", False)[0].sum()
    p = r(40, 80) * 0.2
    fast = torch.compile(block, fullgraph=True, backend="aot_eager")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, p)]
    ref = [t.clone().requires_grad_(True) for t in (x, w, b, p)]
    a, c = fast(*leaves), block(*ref)
    assert torch.equal(a, c)
    assert all(torch.equal(m, n) for m, n in zip(torch.autograd.grad(a, leaves), torch.autograd.grad(c, ref)))


def test_no_second_derivative(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import functional as F
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(F.layer_norm(x).pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    x = torch.randn(2, 5, 8, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(F.gated_scan(x, x.detach())[0].pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
