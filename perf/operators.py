"""What the framework's sequence-block operators are measured on: layer norm, gated linear recurrence and multi-tensor AdamW.

`own` false: the plain form in elementary torch operations; `own` true: the framework's entry points.  Sizes are those of the
separator's own grid (16 clips x 625 frames x 145 bins x 32 channels, 8 ms streaming chunks) or generic ones.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256                      # elements that share a scale where the optimiser's states are held in 8 bits
BETAS, LR, EPS, WD = (0.9, 0.999), 1e-3, 1e-8, 0.01


def listed():
    return [
        # one streaming chunk's rows of the separator: latency counts
        {"name": "norm_chunk", "op": "norm", "rows": 145, "n": 32, "dtype": "f32", "wdtype": "f32", "affine": "both", "train": False},
        # a training batch of the separator: very many, very short rows
        {"name": "norm_grid", "op": "norm", "rows": 16 * 625 * 145, "n": 32, "dtype": "f32", "wdtype": "f32", "affine": "both", "train": True},
        # a wide training step in bf16
        {"name": "norm_wide", "op": "norm", "rows": 16384, "n": 4096, "dtype": "bf16", "wdtype": "bf16", "affine": "both", "train": True},
        # odd rows that start at no vector's border, no bias, fp32 weight beside fp16 activations
        {"name": "norm_odd", "op": "norm", "rows": 2309, "n": 10007, "dtype": "f16", "wdtype": "f32", "affine": "weight", "train": True},
        # one token of a streaming batch: the state is carried in place
        {"name": "scan_step", "op": "step", "rows": 64, "n": 2048, "dtype": "bf16", "gdtype": "bf16", "form": "sigmoid"},
        # the separator's grid along time: many sequences of a clip's length, training
        {"name": "scan_frames", "op": "scan", "b": 16, "t": 625, "f": 145, "c": 32, "dim": 1, "dtype": "f32", "gdtype": "f32",
         "form": "sigmoid", "reverse": False, "ragged": False, "h0": True, "split": False, "train": True},
        # a training batch in bf16, x and gate being the halves of one projection
        {"name": "scan_train", "op": "scan", "b": 8, "t": 4096, "f": 1, "c": 2048, "dim": 1, "dtype": "bf16", "gdtype": "bf16",
         "form": "sigmoid", "reverse": False, "ragged": False, "h0": False, "split": True, "train": True},
        # one long recording, few channels: the time axis itself has to be split
        {"name": "scan_long", "op": "scan", "b": 1, "t": 131072, "f": 1, "c": 512, "dim": 1, "dtype": "bf16", "gdtype": "f32",
         "form": "decay", "reverse": False, "ragged": False, "h0": True, "split": False, "train": True},
        # a padded batch of clips walked backwards, inference
        {"name": "scan_ragged", "op": "scan", "b": 6, "t": 3001, "f": 1, "c": 1000, "dim": 1, "dtype": "f16", "gdtype": "f16",
         "form": "sigmoid", "reverse": True, "ragged": True, "h0": True, "split": False, "train": False},
        # a model of the separator's size: half a million parameters in many small tensors, clipped
        {"name": "adamw_small", "op": "adamw", "total": 500_000, "tensors": 160, "layout": 1, "dtype": "f32", "bits": 32, "clip": 1.0},
        # 16-bit parameters with an fp32 master copy
        {"name": "adamw_master", "op": "adamw", "total": 96_000_000, "tensors": 60, "layout": 2, "dtype": "bf16", "bits": 32, "clip": 1.0},
        # states in 8 bits
        {"name": "adamw_8bit", "op": "adamw", "total": 64_000_000, "tensors": 40, "layout": 3, "dtype": "f32", "bits": 8, "clip": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "scan", "scan", "scan", "step", "adamw", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        n = _log(rng, 8, 16384)
        rows = _log(rng, 1, max(2, 64_000_000 // n))
        return {"op": op, "rows": rows, "n": n, "dtype": dtype, "wdtype": rng.choice([dtype, "f32"]),
                "affine": rng.choice(["both", "both", "weight", "none"]), "train": rng.random() < 0.7}
    if op == "step":
        return {"op": op, "rows": _log(rng, 1, 512), "n": _log(rng, 16, 8192), "dtype": dtype, "gdtype": rng.choice([dtype, "f32"]),
                "form": rng.choice(["sigmoid", "decay"])}
    if op == "scan":
        t = _log(rng, 1, 65536)
        grid = rng.random() < 0.4
        f = _log(rng, 2, 257) if grid else 1
        c = _log(rng, 1, 128) if grid else _log(rng, 16, 4096)
        b = _log(rng, 1, 64)
        while b * t * f * c > 48_000_000:
            b, t = max(1, b // 2), (t + 1) // 2 if b == 1 else t
        return {"op": op, "b": b, "t": t, "f": f, "c": c, "dim": 2 if grid and rng.random() < 0.5 else 1, "dtype": dtype,
                "gdtype": rng.choice([dtype, "f32"]), "form": rng.choice(["sigmoid", "decay"]), "reverse": rng.random() < 0.4,
                "ragged": rng.random() < 0.3, "h0": rng.random() < 0.5, "split": False, "train": rng.random() < 0.7}
    return {"op": op, "total": _log(rng, 10_000, 60_000_000), "tensors": _log(rng, 1, 150), "layout": rng.randrange(1 << 20),
            "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "bits": rng.choice([32, 8]), "clip": rng.choice([0.0, 1.0])}


# ---- inputs ----
def _sizes(case):
    """the tensors' sizes: log-spread, most of them odd, summing to about `total`"""
    r = random.Random(case["layout"])
    w = [math.exp(r.uniform(0.0, 6.0)) for _ in range(case["tensors"])]
    return [max(1, int(case["total"] * x / sum(w))) for x in w]


def _padded(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed * 7919 + 1)
    dt = DT[case["dtype"]]

    def normal(*shape, dtype=torch.float32, mean=0.0, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).add_(mean).to(dtype)

    s = {"case": case}
    if case["op"] == "norm":
        r, n, wt = case["rows"], case["n"], DT[case["wdtype"]]
        s["x"] = normal(r, n, dtype=dt, mean=0.5, std=2.0)
        s["w"] = normal(n, dtype=wt, mean=1.0, std=0.2) if case["affine"] != "none" else None
        s["b"] = normal(n, dtype=wt, std=0.2) if case["affine"] == "both" else None
        s["dy"] = normal(r, n, dtype=dt) if case["train"] else None
        return s
    if case["op"] == "adamw":
        sizes = _sizes(case)
        starts = [0]
        for n in sizes:
            starts.append(starts[-1] + (n + 3) // 4 * 4)
        flat = normal(starts[-1], std=0.05)                       # the parameters: views of one buffer, as a module's bucket
        s["flat"] = flat.to(dt)
        s["params"] = [s["flat"][o:o + n] for o, n in zip(starts, sizes)]
        s["grads"] = [t.clone() for t in normal(starts[-1], std=0.02, dtype=dt).split([b - a for a, b in zip(starts, starts[1:])])]
        s["grads"] = [t[:n] for t, n in zip(s["grads"], sizes)]
        # the states: one buffer each, every tensor from a multiple of BLOCK on
        m = _lay([normal(n, std=0.003) for n in sizes])
        v = _lay([normal(n, std=0.02).square_() for n in sizes])
        s["state"] = {"exp_avg": m, "exp_avg_sq": v}
        if case["bits"] == 8:
            zero = torch.full_like(m, 1 << 15, dtype=torch.int64)
            mc, ms = _to8(m, 4, zero)
            vc, vs = _to8(v, 5, zero)
            s["state"] = {"exp_avg": mc, "exp_avg_scale": ms, "exp_avg_sq": vc, "exp_avg_sq_scale": vs}
        if case["dtype"] != "f32":
            s["state"]["master"] = _lay([flat[o:o + n] for o, n in zip(starts, sizes)])
        s["step"] = 100 + seed % 50
        return s
    gt = DT[case["gdtype"]]

    def gate(*shape):
        z = normal(*shape, mean=2.0, std=1.5)                      # decays between about 0.3 and 0.99
        return z.to(gt) if case["form"] == "sigmoid" else torch.sigmoid(z).to(gt)

    if case["op"] == "step":
        r, n = case["rows"], case["n"]
        s["x"], s["gate"], s["h"] = normal(r, n, dtype=dt), gate(r, n), normal(r, n)
        return s
    b, t, f, c, dim = case["b"], case["t"], case["f"], case["c"], case["dim"]
    shape = [b, t, f, c] if f > 1 else [b, t, c]
    if case["split"]:
        both = normal(*shape[:-1], 2 * c, dtype=dt)
        both[..., c:] += 2.0
        s["x"], s["gate"] = both[..., :c], both[..., c:]
    else:
        s["x"], s["gate"] = normal(*shape, dtype=dt), gate(*shape)
    rest = shape[:dim] + shape[dim + 1:]
    s["h0"] = normal(*rest) if case["h0"] else None
    s["lengths"] = torch.randint(0, shape[dim] + 1, shape[:dim], generator=g, device="cuda") if case["ragged"] else None
    if case["train"]:
        s["dh"], s["dlast"] = normal(*shape, dtype=dt), normal(*rest)
    return s


# ---- one pass ----
def run(s):
    case = s["case"]
    return {"norm": _norm, "step": _step, "scan": _scan, "adamw": _adamw}[case["op"]](s, case)


def _norm(s, case):
    if own:
        from sound_bubble_amd import functional as F
        if not case["train"]:
            with torch.no_grad():
                return {"y": F.layer_norm(s["x"], s["w"], s["b"], EPS_NORM)}
        leaves = {k: s[k].detach().requires_grad_(True) for k in ("x", "w", "b") if s[k] is not None}
        y = F.layer_norm(leaves["x"], leaves.get("w"), leaves.get("b"), EPS_NORM)
        grads = torch.autograd.grad(y, list(leaves.values()), s["dy"])
        return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + EPS_NORM).rsqrt()
    xh = (x - mean) * rstd
    y = xh * s["w"].float() if s["w"] is not None else xh
    y = y + s["b"].float() if s["b"] is not None else y
    out = {"y": y.to(s["x"].dtype)}
    if case["train"]:
        dy = s["dy"].float()
        dxh = dy * s["w"].float() if s["w"] is not None else dy
        dx = rstd * (dxh - dxh.mean(1, keepdim=True) - xh * (dxh * xh).mean(1, keepdim=True))
        out["dx"] = dx.to(s["x"].dtype)
        if s["w"] is not None:
            out["dw"] = (dy * xh).sum(0).to(s["w"].dtype)
        if s["b"] is not None:
            out["db"] = dy.sum(0).to(s["b"].dtype)
    return out


EPS_NORM = 1e-5


def _step(s, case):
    if own:
        from sound_bubble_amd import functional as F
        y = F.gated_scan_step(s["x"], s["gate"], s["h"], form=case["form"])
        return {"y": y, "state": s["h"]}
    a, b = _coefficients(s["x"].float(), s["gate"].float(), case["form"])
    s["h"].copy_(a * s["h"] + b)
    return {"y": s["h"].to(s["x"].dtype), "state": s["h"]}


def _coefficients(x, gate, form):
    """h_t = a_t h_{t-1} + b_t"""
    if form == "decay":
        return gate, x
    return 1 / (1 + (-gate).exp()), x / (1 + gate.exp())


def _prefix(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, from zero: pairs (a, b) joined over distances 1, 2, 4, ..."""
    k = 1
    while k < a.shape[1]:
        b = torch.cat([b[:, :k], a[:, k:] * b[:, :-k] + b[:, k:]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return a, b


def _scan(s, case):
    kw = {"dim": case["dim"], "form": case["form"], "reverse": case["reverse"]}
    if own:
        from sound_bubble_amd import functional as F
        if not case["train"]:
            with torch.no_grad():
                h, last = F.gated_scan(s["x"], s["gate"], s["h0"], lengths=s["lengths"], **kw)
            return {"h": h, "last": last}
        leaves = {k: s[k].detach().requires_grad_(True) for k in ("x", "gate", "h0") if s[k] is not None}
        h, last = F.gated_scan(leaves["x"], leaves["gate"], leaves.get("h0"), lengths=s["lengths"], **kw)
        grads = torch.autograd.grad((h, last), list(leaves.values()), (s["dh"], s["dlast"]))
        return {"h": h.detach(), "last": last.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}
    dim, form, shape = case["dim"], case["form"], s["x"].shape
    outer, t, inner = math.prod(shape[:dim]), shape[dim], math.prod(shape[dim + 1:])

    def grid(v):                                                  # [outer, T, inner], walked from the first step on
        v = v.float().reshape(outer, t, inner)
        return v.flip(1) if case["reverse"] else v

    def back(v, dtype):
        return (v.flip(1) if case["reverse"] else v).reshape(shape).to(dtype)

    x, gate = grid(s["x"]), grid(s["gate"])
    a, b = _coefficients(x, gate, form)
    live = None
    if s["lengths"] is not None:
        live = torch.arange(t, device="cuda")[None, :, None] < s["lengths"].reshape(outer, 1, 1)
        live = live.flip(1) if case["reverse"] else live
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
    h0 = s["h0"].reshape(outer, 1, inner) if s["h0"] is not None else torch.zeros(outer, 1, inner, device="cuda")
    pa, pb = _prefix(a, b)
    h = pa * h0 + pb
    before = torch.cat([h0, h[:, :-1]], 1)
    shown = torch.where(live, h, 0.0) if live is not None else h
    rest = shape[:dim] + shape[dim + 1:]
    out = {"h": back(shown, s["x"].dtype), "last": h[:, -1].reshape(rest)}
    if case["train"]:
        dh, last = grid(s["dh"]), s["dlast"].reshape(outer, 1, inner)
        if live is not None:
            dh = torch.where(live, dh, 0.0)
        # G_t = dh_t + a_{t+1} G_{t+1}, with a = 1 behind the last step
        ra = torch.cat([torch.ones_like(last), a.flip(1)[:, :-1]], 1)
        pa, pb = _prefix(ra, dh.flip(1))
        G = (pa * last + pb).flip(1)
        if form == "decay":
            dx, dg = G, G * before
        else:
            dx, dg = G / (1 + gate.exp()), G * (before - x) * a / (1 + gate.exp())
        if live is not None:
            dx, dg = torch.where(live, dx, 0.0), torch.where(live, dg, 0.0)
        out["dx"], out["dgate"] = back(dx, s["x"].dtype), back(dg, s["gate"].dtype)
        if s["h0"] is not None:
            out["dh0"] = (a[:, 0] * G[:, 0]).reshape(rest)
    return out


# ---- AdamW: states of 32 or 8 bits ----
def _lay(tensors):
    """one buffer, every tensor from a multiple of BLOCK on, zeros behind it"""
    return torch.cat([torch.nn.functional.pad(t.reshape(-1).float(), (0, _padded(t.numel()) - t.numel())) for t in tensors])


def _dither(n, step, seed=0):
    """32 bits for each element index, from a counter: Weyl sequence and two multiply-xorshift rounds"""
    key = (seed * 0x9E3779B9 + step * 0x6A09E667) & 0xFFFFFFFF
    i = torch.arange(n, device="cuda", dtype=torch.int64)
    x = ((i & 0xFFFFFFFF) + (i >> 32) * 0x3C6EF372 + key) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x5BE0CD19) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x1F83D9AB) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _to8(x, exponent_bits, u16):
    """(codes, scales): E4M3 (signed) or E5M2 (x >= 0) codes with a power-of-two scale for each BLOCK; a code is rounded up where the
    part cut off and (u16 + 1/2) / 2^16 reach 1 together, and never down to zero in E5M2"""
    mant, bias, top = (3, 7, 8) if exponent_bits == 4 else (2, 15, 15)
    y = x.abs().reshape(-1, BLOCK)
    big = y.amax(1)                                               # NaN where one is in the block
    bits = big.view(torch.int32).to(torch.int64)
    e = (bits >> 23) - 127 + ((bits & 0x7FFFFF) > 0x600000).long() - top
    e = e.clamp(-127, 127)
    scale = torch.where(torch.isfinite(big), e + 127, 255)
    y = (y * torch.ldexp(torch.ones_like(big), (-e).int())[:, None]).reshape(-1)
    cut = 23 - mant
    yb = y.view(torch.int32).to(torch.int64)
    add = (u16 << (cut - 16)) + (1 << (cut - 17))
    normal = ((yb + add) >> cut) - ((127 - bias) << mant)
    lowest = 2.0 ** (1 - bias)
    small = ((y * (2.0 ** (bias - 1 + mant + cut))).clamp(max=2.0 ** 25).to(torch.int64) + add) >> cut
    code = torch.where(y >= lowest, normal, small)
    if exponent_bits == 5:
        code = torch.where((code == 0) & (x > 0), 1, code)
    else:
        code = code | (torch.signbit(x).long() << 7)
    code = torch.where(torch.isfinite(y), code, 0)
    kind = torch.float8_e4m3fn if exponent_bits == 4 else torch.float8_e5m2
    return code.to(torch.uint8).view(kind), scale.to(torch.uint8).view(torch.float8_e8m0fnu)


def _from8(codes, scales):
    return (codes.float().reshape(-1, BLOCK) * scales.float()[:, None]).reshape(-1)


def _adamw(s, case):
    s["step"] += 1
    step, st = s["step"], s["state"]
    if own:
        from sound_bubble_amd import ops
        ops.adamw_step(s["params"], s["grads"], st, step, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, clip=case["clip"])
        return {"params": s["flat"], **st}
    b1, b2 = BETAS
    g = _lay(s["grads"])
    if case["clip"]:
        norm = g.double().square().sum().float().sqrt()           # a long sum: in 64 bits
        g = g * (case["clip"] / (norm + 1e-6)).clamp(max=1.0)
    eight = case["bits"] == 8
    m = _from8(st["exp_avg"], st["exp_avg_scale"]) if eight else st["exp_avg"]
    v = _from8(st["exp_avg_sq"], st["exp_avg_sq_scale"]) if eight else st["exp_avg_sq"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = st["master"] if "master" in st else _lay(s["params"])
    p = p * (1 - LR * WD) - (LR / (1 - b1 ** step)) * (m / (v.sqrt() / math.sqrt(1 - b2 ** step) + EPS))
    if "master" in st:
        st["master"].copy_(p)
    parts = p.split([_padded(t.numel()) for t in s["params"]])
    torch._foreach_copy_(s["params"], [q[:t.numel()] for q, t in zip(parts, s["params"])])
    if eight:
        u = _dither(m.numel(), step)
        new = _to8(m, 4, u & 0xFFFF) + _to8(v, 5, u >> 16)
        for k, t in zip(("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"), new):
            st[k].view(torch.uint8).copy_(t.view(torch.uint8))
    else:
        st["exp_avg"].copy_(m)
        st["exp_avg_sq"].copy_(v)
    return {"params": s["flat"], **st}


# ---- what a pass cannot do without ----
def work(case):
    d = SIZE[case["dtype"]]
    if case["op"] == "norm":
        e, w = case["rows"] * case["n"], case["n"] * SIZE[case["wdtype"]] * {"both": 2, "weight": 1, "none": 0}[case["affine"]]
        return {"bytes": e * d * (4 if case["train"] else 2) + w * (2 if case["train"] else 1), "flops": e * (22 if case["train"] else 8)}
    if case["op"] == "step":
        e = case["rows"] * case["n"]
        return {"bytes": e * (2 * d + SIZE[case["gdtype"]] + 8), "flops": 8 * e}
    if case["op"] == "scan":
        b, t, f, c, gd = case["b"], case["t"], case["f"], case["c"], SIZE[case["gdtype"]]
        e = b * t * f * c
        state = 4 * e // (t if case["dim"] == 1 else f) * (1 + case["h0"])
        if not case["train"]:
            return {"bytes": e * (2 * d + gd) + state, "flops": 8 * e}
        return {"bytes": e * (4 * d + 2 * gd) + 2 * state, "flops": 28 * e}
    n = sum(_sizes(case))
    state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
    weights = 2 * d if case["dtype"] == "f32" else d + 8
    return {"bytes": n * (d + weights + state), "flops": n * (16 if case["bits"] == 32 else 50)}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    d = lambda t: None if t is None else t.double()  # noqa: E731
    if case["op"] == "norm":
        x, w, b = d(s["x"]), d(s["w"]), d(s["b"])
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        sd = (var + EPS_NORM).sqrt()
        xh = (x - mean) / sd
        y = xh * (1 if w is None else w) + (0 if b is None else b)
        if not case["train"]:
            return {"y": y}
        dy = d(s["dy"])
        q = dy * (1 if w is None else w)
        out = {"y": y, "dx": (q - (q.sum(1, keepdim=True) + xh * (q * xh).sum(1, keepdim=True)) / case["n"]) / sd}
        if w is not None:
            out["dw"] = torch.einsum("rn,rn->n", dy, xh)
        if b is not None:
            out["db"] = dy.sum(0)
        return out
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    sig = case["form"] == "sigmoid"
    if case["op"] == "step":
        a = d(s["gate"]).sigmoid() if sig else d(s["gate"])
        h = a * d(s["h"]) + d(s["x"]) * ((-d(s["gate"])).sigmoid() if sig else 1)
        return {"y": h, "state": h}
    dim, shape = case["dim"], s["x"].shape
    steps = shape[dim]
    if steps > 40000 and s["x"].numel() > 1 << 27:
        return None
    rest = shape[:dim] + shape[dim + 1:]
    x, z = d(s["x"]).movedim(dim, 0), d(s["gate"]).movedim(dim, 0)
    a, one_less = (z.sigmoid(), (-z).sigmoid()) if sig else (z, None)
    n = s["lengths"]
    order = list(range(steps))[::-1] if case["reverse"] else list(range(steps))
    h = d(s["h0"]) if s["h0"] is not None else x.new_zeros(rest)
    hs, before = torch.zeros_like(x), torch.zeros_like(x)
    on = [None] * steps
    if n is not None:
        mask = n.reshape(n.shape + (1,) * (len(rest) - n.dim())).expand(rest)
        on = (torch.arange(steps, device="cuda").reshape((-1,) + (1,) * len(rest)) < mask).unbind(0)
    for t in order:
        before[t] = h
        new = torch.addcmul(x[t] * one_less[t] if sig else x[t], a[t], h)
        h = new if n is None else torch.where(on[t], new, h)
        hs[t] = new if n is None else torch.where(on[t], new, 0.0)
    out = {"h": hs.movedim(0, dim), "last": h}
    if not case["train"]:
        return out
    dh, G = d(s["dh"]).movedim(dim, 0), d(s["dlast"])
    Gs = torch.zeros_like(x)
    for t in order[::-1]:
        g = G + dh[t]
        Gs[t] = g if n is None else torch.where(on[t], g, 0.0)
        G = a[t] * g if n is None else torch.where(on[t], a[t] * g, G)
    out["dx"] = (Gs * one_less if sig else Gs).movedim(0, dim)
    out["dgate"] = (Gs * (before - x) * a * one_less if sig else Gs * before).movedim(0, dim)
    if s["h0"] is not None:
        out["dh0"] = G
    return out


def _exact_adamw(case, s):
    """each tensor for itself; states in 8 bits have no value of their own in 64"""
    step, st, (b1, b2) = s["step"] + 1, s["state"], BETAS
    scale = 1.0
    if case["clip"]:
        norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in s["grads"]))
        scale = min(1.0, case["clip"] / (norm + 1e-6))
    values = {k: st[k].double() for k in ("exp_avg", "exp_avg_sq")}
    if case["bits"] == 8:
        values = {k: v * st[k + "_scale"].double().repeat_interleave(BLOCK) for k, v in values.items()}
    out = {"params": s["flat"].double().clone(), **{k: v.double().clone() for k, v in values.items()}}
    if "master" in st:
        out["master"] = st["master"].double().clone()
    at = 0
    for p, g in zip(s["params"], s["grads"]):
        n, o = p.numel(), p.storage_offset()
        g = g.double() * scale
        m = out["exp_avg"][at:at + n].mul_(b1).add_(g, alpha=1 - b1)
        v = out["exp_avg_sq"][at:at + n].mul_(b2).add_(g ** 2, alpha=1 - b2)
        w = out["master"][at:at + n] if "master" in st else out["params"][o:o + n]
        new = w - LR * WD * w - LR * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + EPS)
        w.copy_(new)
        out["params"][o:o + n] = new
        at += _padded(n)
    if case["bits"] == 8:
        out.update({k: None for k in st if k != "master"})
    return out
