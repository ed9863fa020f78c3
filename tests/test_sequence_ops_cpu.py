"""Sequence-block operators without a GPU: the C ABI (include/sound_bubble_seq.h) and its ctypes mirror, the refusals of the C entry
points and of the Python wrappers, the layout of AdamW's state buffers."""
import ctypes as C
import os
import re
import subprocess

import pytest

from conftest import ROOT


def test_library_exports_every_declared_symbol():
    from sound_bubble_amd import _lib
    hdr = open(os.path.join(ROOT, "include", "sound_bubble_seq.h")).read()
    declared = set(re.findall(r"^\s*(?:int|int64_t)\s+(sb_\w+)\s*\(", hdr, flags=re.M))
    assert declared and declared == set(_lib.SEQ_SYMBOLS), declared ^ set(_lib.SEQ_SYMBOLS)
    lib = _lib.load()
    for name in declared:
        assert getattr(lib, name) is not None


def test_struct_layouts_match_header(tmp_path):
    from sound_bubble_amd import _lib
    pairs = {"sb_layer_norm_args": _lib.LayerNormArgs, "sb_layer_norm_bwd_args": _lib.LayerNormBwdArgs,
             "sb_gated_scan_args": _lib.GatedScanArgs, "sb_gated_scan_bwd_args": _lib.GatedScanBwdArgs,
             "sb_adamw_tensor": _lib.AdamwTensor, "sb_adamw_args": _lib.AdamwArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "sound_bubble_seq.h"', "int main(void) {"]
    want = []
    for cname, cls in pairs.items():
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        want.append(C.sizeof(cls))
        for fname, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({cname}, {fname}));')
            want.append(getattr(cls, fname).offset)
    for name, value in (("SB_ADAMW_BLOCK", _lib.ADAMW_BLOCK), ("SB_ADAMW_MAX", _lib.ADAMW_MAX), ("SB_ADAMW_NORM_SLOTS", _lib.ADAMW_NORM_SLOTS)):
        lines.append(f'  printf("%d\\n", {name});')
        want.append(value)
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    exe = tmp_path / "probe"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    assert [int(x) for x in subprocess.check_output([str(exe)]).split()] == want
    assert C.sizeof(_lib.AdamwArgs) <= 4000          # it is passed by value, beside the kernel's other arguments


def test_c_entries_refuse_bad_arguments():
    """every refusal is made before anything is launched"""
    from sound_bubble_amd import _lib as L
    lib = L.load()
    p = 64                                            # (never looked at: the refusals are the host's)
    assert lib.sb_layer_norm_fwd(None, None) < 0 and lib.sb_layer_norm_bwd(None, None) < 0
    ok = dict(rows=4, n=8, ldx=8, xtype=1, wtype=0, eps=1e-5, x=p, y=p)
    for bad in (dict(n=0), dict(rows=-1), dict(ldx=-8), dict(wtype=2), dict(xtype=7, wtype=7), dict(x=None), dict(y=None), dict(mean=p)):
        assert lib.sb_layer_norm_fwd(L.LayerNormArgs(**{**ok, **bad}), None) <= -1000, bad
    ok = dict(rows=4, n=8, ldx=8, lddy=8, xtype=0, wtype=0, x=p, dy=p, dx=p, mean=p, rstd=p)
    for bad in (dict(n=-1), dict(lddy=-1), dict(dy=None), dict(mean=None), dict(dw=p), dict(wtype=1)):
        assert lib.sb_layer_norm_bwd(L.LayerNormBwdArgs(**{**ok, **bad}), None) <= -1000, bad
    ok = dict(outer=2, steps=5, inner=8, xtype=1, gtype=1, form=1, x=p, gate=p, so_x=40, st_x=8, so_g=40, st_g=8, h=p, h_last=p)
    for bad in (dict(outer=-1), dict(gtype=2), dict(form=2), dict(xtype=3, gtype=3), dict(st_x=-8), dict(so_g=-1), dict(x=None), dict(h_last=None)):
        assert lib.sb_gated_scan_fwd(L.GatedScanArgs(**{**ok, **bad}), None) <= -1000, bad
    ok = dict(outer=2, steps=5, inner=8, xtype=0, gtype=0, form=0, x=p, gate=p, states=p, dx=p, dgate=p, so_x=40, st_x=8, so_g=40, st_g=8)
    for bad in (dict(steps=-1), dict(states=None), dict(dx=None), dict(so_d=-1), dict(gtype=1), dict(form=-1)):
        assert lib.sb_gated_scan_bwd(L.GatedScanBwdArgs(**{**ok, **bad}), None) <= -1000, bad
    # one long sequence is cut in time: that needs the scratch
    assert lib.sb_gated_scan_fwd(L.GatedScanArgs(outer=1, steps=1 << 20, inner=8, xtype=0, gtype=0, form=0, x=p, gate=p, so_x=8 << 20, st_x=8,
                                                 so_g=8 << 20, st_g=8, h=p, h_last=p), None) <= -1000
    assert lib.sb_gated_scan_step(None, p, p, p, 4, 8, 8, 8, 0, 0, 0, None) <= -1000
    assert lib.sb_gated_scan_step(p, p, p, p, -4, 8, 8, 8, 0, 0, 0, None) <= -1000
    assert lib.sb_gated_scan_step(p, p, p, p, 4, 8, 8, 8, 1, 2, 0, None) <= -1000

    def args(**kw):
        a = L.AdamwArgs(count=1, bits=32, m=p, v=p, step=1)
        a.t[0] = L.AdamwTensor(p, p, 10, 0, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    for bad in (dict(count=0), dict(count=L.ADAMW_MAX + 1), dict(bits=16), dict(bits=8), dict(m=None), dict(step=0), dict(ptype=1),
                dict(ptype=5), dict(gtype=1), dict(clip=1.0), dict(clip=-1.0), dict(count=2)):
        assert lib.sb_adamw_step(args(**bad), None) <= -1000, bad
    assert lib.sb_adamw_norm(args(), p, 500, 100, None) <= -1000
    assert lib.sb_adamw_norm(args(), None, 0, 1, None) <= -1000
    a = args()
    a.t[0].n = 0
    assert lib.sb_adamw_step(a, None) <= -1000


@pytest.mark.parametrize("outer,steps,inner", [(1, 1, 1), (3, 17, 5), (1, 1 << 17, 512), (16, 625, 4640), (10000, 145, 32), (0, 5, 3), (2, 0, 3)])
@pytest.mark.parametrize("xtype", [0, 1, 2])
def test_scan_plan(outer, steps, inner, xtype):
    """the buffers a plan asks for cover the sequence: kept states at least every 1024 steps, two pairs a segment"""
    from sound_bubble_amd import ops_seq
    chunks, fwd, bwd = ops_seq._scan_plan(outer, steps, inner, xtype)
    if outer * steps * inner == 0:
        assert (chunks, fwd, bwd) == (0, 0, 0)
        return
    assert steps / 1024 <= chunks <= (steps + 7) // 8
    for n in (fwd, bwd):
        assert n % (2 * outer * inner) == 0 and n // (2 * outer * inner) in (0, *range(2, 513))


def test_wrappers_refuse_what_is_not_on_the_gpu(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    x = torch.zeros(2, 3, 4)
    for call in (lambda: F.layer_norm(x), lambda: F.layer_norm(x.requires_grad_(True)), lambda: F.gated_scan(x, x), lambda: ops.adamw_state([x]),
                 lambda: F.gated_scan_step(x.detach(), x.detach(), x.detach()),
                 lambda: ops.adamw_step([x], [x], {}, 1, lr=0.1), lambda: ops.adamw_step([x], [], {}, 1, lr=0.1)):
        with pytest.raises(E):
            call()
    with pytest.raises(E):
        ops.adamw_state([], bits=4)
    with pytest.raises(E, match="no gradient"):
        F.gated_scan_step(x, x.detach(), x.detach())


def test_adamw_layout():
    from sound_bubble_amd import ops
    assert ops.adamw_blocks([]) == [0]
    assert ops.adamw_blocks([1, 256, 257, 0, 5]) == [0, 1, 2, 4, 4, 5]


def test_fake_implementations_propagate_shapes(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import torch_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    sb = torch.ops.sound_bubble
    with FakeTensorMode():
        x = torch.empty(3, 300, 40, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(40, device="cuda")
        y, mean, rstd = sb.layer_norm(x, w, None, 1e-5)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == rstd.shape == (3, 300) and mean.dtype == torch.float32
        dx, dw, db = sb.layer_norm_backward(y, x, w, mean, rstd, True, False, False)
        assert dx.shape == x.shape and dw.shape == (40,) and dw.dtype == torch.float32 and db.shape == (0,)
        h, last, states = sb.gated_scan(x, x, None, None, 1, "sigmoid", False)
        assert h.shape == x.shape and last.shape == (3, 40) and last.dtype == states.dtype == torch.float32 and states.numel() % 120 == 0
        dx, dg, d0 = sb.gated_scan_backward(h, None, x, x, states, None, 1, "sigmoid", False)
        assert dx.shape == dg.shape == x.shape and d0.shape == (3, 40)
        assert sb.gated_scan_step(x[:, 0], x[:, 0], last, "decay").shape == (3, 40)
    with pytest.raises((NotImplementedError, RuntimeError)):
        sb.layer_norm(torch.zeros(2, 3), None, None, 1e-5)


def test_adamw_states_pack_exactly(torch_mod):
    """8-bit states -> float32 -> 8-bit states keeps every value; a value is rounded to the nearest code"""
    torch = torch_mod
    from sound_bubble_amd import ops_seq as Q
    g = torch.Generator().manual_seed(1)
    st = {}
    for k, (kind, _) in Q._EIGHT.items():
        top = 0x7F if kind is torch.float8_e4m3fn else 0x7C
        code = torch.randint(0, top, (2048,), generator=g, dtype=torch.uint8)
        if k == "exp_avg":
            code |= torch.randint(0, 2, (2048,), generator=g, dtype=torch.uint8) << 7
        code[256:512] = 0
        st[k] = code.view(kind)
        st[k + "_scale"] = torch.randint(60, 180, (8,), generator=g, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    st["exp_avg"].view(torch.uint8)[512:768] = 0x01                     # a block of the smallest code only: another scale, the same values
    want = Q.adamw_state_values(st)
    two = {k: torch.zeros_like(v.view(torch.uint8)).view(v.dtype) for k, v in st.items()}
    Q.adamw_state_pack(two, want)
    got = Q.adamw_state_values(two)
    assert all(torch.equal(got[k], want[k]) for k in want)
    x = {"exp_avg": torch.randn(2048, generator=g), "exp_avg_sq": torch.randn(2048, generator=g).square()}
    x["exp_avg_sq"][5] = 1e-30
    x["exp_avg"][300] = float("inf")
    Q.adamw_state_pack(two, x)
    got = Q.adamw_state_values(two)
    assert got["exp_avg_sq"][5] > 0 and torch.isnan(got["exp_avg"][256:512]).all()
    fine = torch.ones(2048, dtype=torch.bool)
    fine[256:512] = False
    for k, half in (("exp_avg", 2.0 ** -4), ("exp_avg_sq", 2.0 ** -3)):
        low = x[k][fine].abs().max() * (2.0 ** -17 if k == "exp_avg" else 2.0 ** -30)      # half the smallest code, at most
        assert ((got[k] - x[k]).abs()[fine] <= x[k].abs()[fine] * half + low).all()


def test_replicas_share_the_optimiser_state(torch_mod, tmp_path):
    """broadcast_replica moves whatever state_tensors() names (two ranks over gloo; FusedAdam's moments here)"""
    torch = torch_mod
    import subprocess
    import sys
    src = tmp_path / "rank.py"
    src.write_text("""
import sys, torch, torch.distributed as dist
sys.path.insert(0, %r)
from sound_bubble_amd.train import broadcast_replica
rank = int(sys.argv[1])
dist.init_process_group("gloo", init_method="tcp://127.0.0.1:%%s" %% sys.argv[2], rank=rank, world_size=2)
class Bucket: flat = torch.full((4,), float(rank))
class Optim:
    step_count, param_groups = 3 + rank, [{"lr": 0.5 + rank}]
    codes = torch.full((5,), 7 + rank, dtype=torch.uint8).view(torch.float8_e4m3fn)
    def state_tensors(self): return [self.codes.view(torch.uint8)]
o = Optim()
broadcast_replica(Bucket, o)
assert Bucket.flat.eq(0).all() and o.codes.view(torch.uint8).eq(7).all() and o.step_count == 3 and o.param_groups[0]["lr"] == 0.5
""" % ROOT)
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = str(s.getsockname()[1])
    procs = [subprocess.Popen([sys.executable, str(src), str(r), port]) for r in range(2)]
    assert [p.wait(timeout=120) for p in procs] == [0, 0]
