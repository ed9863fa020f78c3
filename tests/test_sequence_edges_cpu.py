"""Sequence-block operators without a GPU: what is refused, and what a failed call leaves behind."""
import os
import runpy
import subprocess
import sys

import pytest

from conftest import ROOT


def test_refused_inside_on_stream(torch_mod):
    """a call's scratch would be reused by the current stream while the other one works on it"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    x = torch.zeros(2, 3, 4)
    leaf = x.clone().requires_grad_(True)
    calls = [lambda: F.layer_norm(x), lambda: F.layer_norm(leaf), lambda: ops.layer_norm_bwd(x, x, None, x[..., 0], x[..., 0]),
             lambda: F.gated_scan(x, x), lambda: F.gated_scan(leaf, x), lambda: ops.gated_scan_bwd(x, None, x, x, x.view(-1)),
             lambda: F.gated_scan_step(x, x, x.clone()), lambda: ops.adamw_step([x], [x], {}, 1, lr=0.1)]
    for call in calls:
        with ops.on_stream(1), pytest.raises(E, match="on_stream"):
            call()


class Stub:
    """native calls that have done their work, or the first launch of it, and then raise"""

    def __init__(self, error):
        self.error, self.calls = error, []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            raise self.error
        return call


@pytest.mark.parametrize("text", ["sound_bubble: sb_adamw_step failed with status -719", "HIP error: unspecified launch failure"])
def test_a_failed_native_call_is_not_run_again(torch_mod, monkeypatch, text):
    """an update that has been launched must not be launched a second time by the wrapper"""
    torch = torch_mod
    from sound_bubble_amd import _lib as L, functional as F, ops_seq
    stub, launched = Stub(RuntimeError(text)), []
    monkeypatch.setattr(ops_seq, "native", lambda: stub)
    monkeypatch.setattr(ops_seq, "_launch", lambda fn, *a: launched.append(fn))
    for name in ("layer_norm_fwd", "gated_scan_fwd", "gated_scan_step"):
        monkeypatch.setattr(ops_seq, name, lambda *a, **k: launched.append(a))
    x = torch.zeros(2, 3, 4)
    calls = [lambda: F.layer_norm(x, x[0, 0], None, 1e-5), lambda: F.gated_scan(x, x, reverse=True), lambda: F.gated_scan(x, x, x[:, 0], lengths=x[:, 0, 0]),
             lambda: F.gated_scan_step(x, x, x.clone(), form="decay"),
             lambda: ops_seq.adamw_step([x], [x], {"exp_avg": x, "exp_avg_sq": x}, 1, lr=0.1)]
    for call in calls:
        with pytest.raises(RuntimeError) as e:
            call()
        assert str(e.value) == text and not launched
        assert isinstance(e.value, L.SoundBubbleHipError) == text.startswith("sound_bubble:")
    assert stub.calls == ["layer_norm", "gated_scan", "gated_scan", "gated_scan_step", "adamw_step"]


def test_arguments_of_another_kind_are_said_to_be(torch_mod, monkeypatch):
    """what a native call cannot even take (nothing has been done) is for the wrappers to name"""
    torch = torch_mod
    from sound_bubble_amd import functional as F, ops_seq
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    stub = Stub(TypeError("no such kind"))
    monkeypatch.setattr(ops_seq, "native", lambda: stub)
    x = torch.zeros(2, 3, 4)
    calls = [lambda: F.layer_norm([1.0]), lambda: F.gated_scan(x, None), lambda: F.gated_scan_step(x, x, 3.0),
             lambda: ops_seq.adamw_step([x], [x], {"exp_avg": x}, 1, lr=0.1), lambda: ops_seq.adamw_step([x], [x], {"exp_avg": x, "exp_avg_sq": x}, 1, lr="0.1")]
    for call in calls:
        with pytest.raises(E):
            call()


def test_adamw_refuses_a_counter_that_the_kernel_cannot_count(torch_mod):
    torch = torch_mod
    from sound_bubble_amd import ops
    from sound_bubble_amd._lib import SoundBubbleHipError as E
    x = torch.zeros(4)
    for skipped in (torch.zeros(1, dtype=torch.int32), torch.zeros(1), 3):
        with pytest.raises(E, match="skipped"):
            ops.adamw_step([x], [x], {}, 1, lr=0.1, skipped=skipped)


def test_the_c_entry_refuses_a_clip_that_is_no_number(torch_mod):
    """(it counted as none)"""
    from sound_bubble_amd import _lib as L
    a = L.AdamwArgs(count=1, bits=32, m=64, v=64, step=1, clip=float("nan"))      # (64: never looked at, the refusal is the host's)
    a.t[0] = L.AdamwTensor(64, 64, 10, 0, 0)
    assert L.load().sb_adamw_step(a, None) <= -1000


# ---- the build ----
class Started:
    def __init__(self, cmd):
        self.cmd = cmd

    def wait(self):
        return 0


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """the compiler lines of a build into an empty folder, none of them run"""
    from sound_bubble_amd import build as B
    got = []
    for name in ("LIBDIR", "LIB", "TORCH_LIB"):
        monkeypatch.setattr(B, name, str(tmp_path if name == "LIBDIR" else tmp_path / os.path.basename(getattr(B, name))))
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **k: got.append(list(cmd)) or 0)
    monkeypatch.setattr(subprocess, "Popen", lambda cmd, **k: got.append(list(cmd)) or Started(cmd))
    return got


@pytest.mark.parametrize("script,args,own", [("build_variant.py", ["x", "-DSB_X"], "_x.o"), ("exp_gate_recompute.py", ["build"], "_rc1.o")])
def test_experiment_libraries_have_every_unit(commands, monkeypatch, script, args, own):
    """_lib.load() asks a variant of the library for the sequence-block operators' entries too"""
    from sound_bubble_amd import build as B
    monkeypatch.setattr(B, "build", lambda *a, **k: None)
    monkeypatch.setattr(sys, "argv", [script] + args)
    runpy.run_path(os.path.join(ROOT, "scripts", script), run_name="__main__")
    links = [c for c in commands if "-shared" in c]
    assert links
    units = [os.path.basename(u).replace(".hip", "") for u in B.SOURCES + B.SEQ_SOURCES] + [stem for _, stem, _ in B.EXTRA_UNITS]
    for link in links:
        objs = [os.path.basename(o) for o in link if o.endswith(".o")]
        assert len(objs) == len(units) and all(any(o == u + ".o" or o.startswith(u + "_") for o in objs) for u in units)
    assert any(o.endswith(own) for link in links for o in link)


@pytest.mark.parametrize("missing", ["torch", "g++", "Python.h"])
def test_the_library_is_built_without_the_torch_side(commands, monkeypatch, tmp_path, missing):
    """the C ABI library needs none of them; a stale torch side does not stay beside it"""
    import importlib.util
    import shutil
    import sysconfig
    from sound_bubble_amd import build as B
    if missing == "torch":
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    elif missing == "g++":
        monkeypatch.setattr(shutil, "which", lambda *a, **k: None)
    else:
        monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(tmp_path / "nowhere")})
    open(B.TORCH_LIB, "w").close()
    assert B.build(force=True, verbose=False) == B.LIB
    assert len(commands) == len(B.SOURCES + B.SEQ_SOURCES + B.EXTRA_UNITS) + 1 and "-shared" in commands[-1]
    assert not any(B.TORCH_SOURCE in c for c in commands) and not os.path.exists(B.TORCH_LIB)


def test_the_torch_side_is_built_again_for_another_torch(commands, monkeypatch, tmp_path):
    import importlib.util
    from sound_bubble_amd import build as B
    home = tmp_path / "torch"
    (home / "lib").mkdir(parents=True)
    (home / "lib" / "libc10_hip.so").touch()
    (home / "version.py").write_text("__version__ = '1'")
    spec = importlib.util.spec_from_loader("torch", None, is_package=True)
    spec.submodule_search_locations = [str(home)]
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec)

    def torch_side():
        del commands[:]
        B.build(verbose=False)
        open(B.TORCH_LIB, "w").close()
        return sum(B.TORCH_SOURCE in c for c in commands)
    assert [torch_side(), torch_side()] == [1, 0]
    (home / "version.py").write_text("__version__ = '2'")
    assert [torch_side(), torch_side()] == [1, 0]
