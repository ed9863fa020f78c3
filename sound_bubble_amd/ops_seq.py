"""Tensor-level wrappers of the sequence-block operators (include/sound_bubble_seq.h): layer norm, gated linear recurrence, AdamW
over many tensors.

float32, bfloat16 and float16 on a HIP device; anything else raises, there is no eager fallback.  The launches go to the current
stream of the tensors' own device; what a call needs besides its results is allocated for the call.
"""
import ctypes as C
import functools
import importlib.machinery
import importlib.util
import itertools
import os

import numpy as np
import torch

from . import _lib as L

_OPS = None         # the module ops, which imports this one (it sets the name)

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
FORMS = {"decay": 0, "sigmoid": 1}


def _fail(msg):
    raise L.SoundBubbleHipError(msg)


_NATIVE = None      # the operators of libsoundbubble_torch.so, False: there is no such library


class _Native:
    def __init__(self, path):
        lib, name = L.load(), "libsoundbubble_torch"
        spec = importlib.util.spec_from_file_location(name, path, loader=importlib.machinery.ExtensionFileLoader(name, path))
        self.module = importlib.util.module_from_spec(spec)      # (registers the operators too)
        spec.loader.exec_module(self.module)
        ops = torch.ops.sound_bubble_seq
        ops.bind([C.cast(getattr(lib, name), C.c_void_p).value for name in _ENTRIES])
        self.layer_norm, self.gated_scan = ops.layer_norm.default, ops.gated_scan.default
        self.gated_scan_step, self.adamw_step = ops.gated_scan_step.default, self.module.adamw_step
        self.refuse_held_leaves = ops.refuse_held_leaves.default


_ENTRIES = ("sb_layer_norm_fwd", "sb_layer_norm_bwd_scratch", "sb_layer_norm_bwd", "sb_gated_scan_plan", "sb_gated_scan_fwd", "sb_gated_scan_bwd",
            "sb_gated_scan_step", "sb_adamw_chunk", "sb_adamw_norm", "sb_adamw_step")      # csrc/seq/sb_seq_torch.cpp: Entries
_PYTHON = os.environ.get("SB_SEQ_HOST", "") == "python"


def _library():
    global _NATIVE
    if _NATIVE is None:
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libsoundbubble_torch.so")
        _NATIVE = False
        if os.path.exists(path):
            _NATIVE = _Native(path)
    return _NATIVE


def native():
    """The plain calls without Python in between (csrc/seq/sb_seq_torch.cpp): same kernels, same results, a fraction of the host time.
    They answer with an empty list (0) what they do not take; None where the library has not been built, with SB_SEQ_HOST=python, or
    inside ops.on_stream, which the wrappers refuse."""
    lib = _library()
    return lib if lib and not _PYTHON and _OPS._STREAM_OVERRIDE is None else None


def said(e):
    """the error to raise for one of the native calls' own: theirs begin with the library's name, others (out of memory, say) stay"""
    return L.SoundBubbleHipError(str(e)) if str(e).startswith("sound_bubble:") else e


def refuse_held_leaves(*leaves):
    """Under capture: raises where an eager graph made on another stream holds one of the leaves (the captured backward pass would
    wait for that stream, which ends the process)."""
    leaves = [t for t in leaves if isinstance(t, torch.Tensor) and t.is_cuda and t.requires_grad]
    if leaves and torch.cuda.is_current_stream_capturing() and _library():
        try:
            _library().refuse_held_leaves(leaves)
        except RuntimeError as e:
            raise L.SoundBubbleHipError(str(e)) from None


def _need(t, name, dtypes, device=None, shape=None):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.layout is torch.strided):
        _fail(f"{name}: expected a tensor of {' / '.join(str(d)[6:] for d in dtypes)} on the GPU, got "
              f"{type(t).__name__} {getattr(t, 'dtype', '')} {getattr(t, 'device', '')}")
    if t.is_neg():
        _fail(f"{name}: a lazily negated tensor (call .resolve_neg())")
    if device is not None and t.device != device:
        _fail(f"{name}: is on {t.device}, the call's tensors are on {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        _fail(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _not_on_stream(name):
    """Inside ops.on_stream a call's scratch and copies would be made on the current stream and given back to its allocator while the other
    stream still uses them: refused."""
    if _OPS._STREAM_OVERRIDE is not None:
        _fail(f"{name}: not inside ops.on_stream (use torch.cuda.stream)")


def _launch(fn, device, *args):
    """fn(*args, stream) on the tensors' own device and its current stream"""
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _launch(fn, device, *args)
    rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        L.check(rc, fn.__name__)


def _like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


# ---- layer norm ----
def _rows(t, n):
    """-> (tensor, row stride): the last axis dense, all others one axis of rows; a copy where the strides do not allow that"""
    if t.is_contiguous():
        return t, n
    t2 = t.reshape(-1, n)
    if n > 1 and t2.stride(1) != 1:
        t2 = t2.contiguous()
    return t2, t2.stride(0) if t2.shape[0] > 1 else n


def _norm_params(x, weight, bias):
    if x.dim() < 1 or x.shape[-1] == 0:
        _fail(f"layer_norm: x needs a last axis of at least one element, got shape {tuple(x.shape)}")
    n = x.shape[-1]
    for t, name in ((weight, "layer_norm: weight"), (bias, "layer_norm: bias")):
        if t is not None:
            _need(t, name, (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32), x.device, (n,))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        _fail(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    return n


def layer_norm_fwd(x, weight, bias, eps=1e-5, stats=True):
    """-> (y, mean, rstd): y = (x - mean) rstd weight + bias over the last axis, x's type; mean and rstd float32 of the leading
    shape (None without `stats`).  weight / bias (None: 1 / 0) in x's type or float32."""
    _not_on_stream("layer_norm")
    _need(x, "layer_norm: x", _TYPES)
    n = _norm_params(x, weight, bias)
    y = _like(x)
    mean = rstd = None
    if stats:
        mean, rstd = (x.new_empty(x.shape[:-1], dtype=torch.float32) for _ in range(2))
    rows = x.numel() // n
    if rows == 0:
        return y, mean, rstd
    xr, ldx = _rows(x, n)
    w, b = (t.contiguous() if t is not None else None for t in (weight, bias))
    wt = w if w is not None else b
    a = L.LayerNormArgs(rows, n, ldx, _TYPES[x.dtype], _TYPES[wt.dtype] if wt is not None else 0, eps, xr.data_ptr(), _ptr(w), _ptr(b),
                        y.data_ptr(), _ptr(mean), _ptr(rstd))
    _launch(L.load().sb_layer_norm_fwd, x.device, a)
    return y, mean, rstd


def layer_norm_bwd(dy, x, weight, mean, rstd, want_dw=True, want_db=True, wdtype=None, check=True):
    """-> (dx, dw, db) of layer_norm_fwd; dw / db (None where not wanted) in `wdtype` (the weight's, or given for a bias alone),
    summed over the rows in float32 in an order that the shape alone fixes"""
    _not_on_stream("layer_norm_bwd")
    if check:      # (False: they are layer_norm_fwd's own, and autograd has seen to dy)
        _need(x, "layer_norm_bwd: x", _TYPES)
        _norm_params(x, weight, None)
        _need(dy, "layer_norm_bwd: dy", (x.dtype,), x.device, x.shape)
        for t, name in ((mean, "mean"), (rstd, "rstd")):
            if not _need(t, f"layer_norm_bwd: {name}", (torch.float32,), x.device, x.shape[:-1]).is_contiguous():
                _fail(f"layer_norm_bwd: {name} must be contiguous")
        if wdtype is not None and wdtype not in (x.dtype, torch.float32):
            _fail(f"layer_norm_bwd: wdtype is {x.dtype} or float32, got {wdtype}")
    n = x.shape[-1]
    wdtype = weight.dtype if weight is not None else (wdtype or x.dtype)
    dx = _like(x)
    dw = x.new_empty(n, dtype=wdtype) if want_dw else None
    db = x.new_empty(n, dtype=wdtype) if want_db else None
    rows = x.numel() // n
    xt = _TYPES[x.dtype]
    lib = L.load()
    scratch = None
    if (want_dw or want_db) and rows:
        scratch = x.new_empty(lib.sb_layer_norm_bwd_scratch(rows, n, xt), dtype=torch.float32)
    (xr, ldx), (dyr, lddy) = _rows(x, n), _rows(dy, n)
    w = weight.contiguous() if weight is not None else None
    a = L.LayerNormBwdArgs(rows, n, ldx, lddy, xt, _TYPES[wdtype], xr.data_ptr(), dyr.data_ptr(), _ptr(w), mean.data_ptr(), rstd.data_ptr(),
                           dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(scratch))
    if rows or want_dw or want_db:
        _launch(lib.sb_layer_norm_bwd, x.device, a)
    return dx, dw, db


# ---- gated linear recurrence ----
def _steps(t, outer, steps, inner):
    """-> (tensor, outer stride, step stride) of the [outer, steps, inner] view with a dense inner axis; a copy where there is none"""
    if t.is_contiguous():
        return t, steps * inner, inner
    t3 = t.reshape(outer, steps, inner)
    if inner > 1 and t3.stride(2) != 1:
        t3 = t3.contiguous()
    return t3, t3.stride(0), t3.stride(1)


def _scan_sizes(x, gate, dim, form, h0, lengths):
    _not_on_stream("gated_scan")
    _need(x, "gated_scan: x", _TYPES)
    _need(gate, "gated_scan: gate", (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32), x.device, x.shape)
    if form not in FORMS:
        _fail(f"gated_scan: form is one of {sorted(FORMS)}, got {form!r}")
    if not (isinstance(dim, int) and 0 <= (dim if dim >= 0 else dim + x.dim()) < x.dim()):
        _fail(f"gated_scan: dim {dim} is no axis of a tensor of shape {tuple(x.shape)}")
    dim = dim % x.dim()
    rest = x.shape[:dim] + x.shape[dim + 1:]
    if h0 is not None:
        _need(h0, "gated_scan: h0", (torch.float32,), x.device, rest)
    if lengths is not None:
        _need(lengths, "gated_scan: lengths", (torch.int64, torch.int32), x.device, x.shape[:dim])
    outer = x.shape[:dim].numel()
    return dim, rest, outer, x.shape[dim], x.shape[dim + 1:].numel()


@functools.lru_cache(maxsize=256)
def _scan_plan(outer, steps, inner, xt):
    """(a function of the sizes alone)"""
    got = [C.c_int64() for _ in range(3)]
    L.check(L.load().sb_gated_scan_plan(outer, steps, inner, xt, *(C.byref(v) for v in got)), "sb_gated_scan_plan")
    return tuple(v.value for v in got)


def gated_scan_fwd(x, gate, h0=None, *, dim=1, form="sigmoid", reverse=False, lengths=None, save=True):
    """-> (h, h_last, states): h_t = a_t h_{t-1} + b_t along axis `dim`, from h0 (float32, x's shape without `dim`; None: zeros).
    form "decay": a = gate, b = x; "sigmoid": a = sigmoid(gate), b = (1 - a) x.  h in x's type, h_last float32.
    lengths (int64 / int32, x.shape[:dim]): steps behind a sequence's length leave its state alone and give 0.
    states (None without `save`): what gated_scan_bwd needs, fp32."""
    dim, rest, outer, steps, inner = _scan_sizes(x, gate, dim, form, h0, lengths)
    h = _like(x)
    if x.numel() == 0:
        last = torch.zeros(rest, dtype=torch.float32, device=x.device) if h0 is None else h0.clone()
        return h, last, torch.empty(0, dtype=torch.float32, device=x.device) if save else None
    last = x.new_empty(rest, dtype=torch.float32)
    xt = _TYPES[x.dtype]
    chunks, scratch_n, _ = _scan_plan(outer, steps, inner, xt)
    states = x.new_empty(chunks * outer * inner, dtype=torch.float32) if save else None
    scratch = x.new_empty(scratch_n, dtype=torch.float32) if scratch_n else None
    x3, so_x, st_x = _steps(x, outer, steps, inner)
    g3, so_g, st_g = _steps(gate, outer, steps, inner)
    h0 = h0.contiguous() if h0 is not None else None
    lengths = lengths.to(torch.int64).contiguous() if lengths is not None else None
    a = L.GatedScanArgs(outer, steps, inner, xt, _TYPES[gate.dtype], FORMS[form], int(bool(reverse)), x3.data_ptr(), so_x, st_x,
                        g3.data_ptr(), so_g, st_g, _ptr(h0), _ptr(lengths), h.data_ptr(), last.data_ptr(), _ptr(states), _ptr(scratch))
    _launch(L.load().sb_gated_scan_fwd, x.device, a)
    return h, last, states


def gated_scan_bwd(dh, dlast, x, gate, states, *, dim=1, form="sigmoid", reverse=False, lengths=None, want_dh0=True):
    """-> (dx, dgate, dh0): gradients of gated_scan_fwd's (h, h_last); dh / dlast None: zero.  `states` from gated_scan_fwd with the
    same sizes.  dh0 float32 (None where not wanted)."""
    dim, rest, outer, steps, inner = _scan_sizes(x, gate, dim, form, None, lengths)
    if dh is not None:
        _need(dh, "gated_scan_bwd: dh", (x.dtype,), x.device, x.shape)
    if dlast is not None:
        _need(dlast, "gated_scan_bwd: dlast", (torch.float32,), x.device, rest)
    dx = _like(x)
    dgate = _like(gate)
    if x.numel() == 0:
        dh0 = None
        if want_dh0:
            dh0 = torch.zeros(rest, dtype=torch.float32, device=x.device) if dlast is None else dlast.clone()
        return dx, dgate, dh0
    xt = _TYPES[x.dtype]
    chunks, _, scratch_n = _scan_plan(outer, steps, inner, xt)
    _need(states, "gated_scan_bwd: states", (torch.float32,), x.device, (chunks * outer * inner,))
    dh0 = x.new_empty(rest, dtype=torch.float32) if want_dh0 else None
    scratch = x.new_empty(scratch_n, dtype=torch.float32) if scratch_n else None
    x3, so_x, st_x = _steps(x, outer, steps, inner)
    g3, so_g, st_g = _steps(gate, outer, steps, inner)
    d3, so_d, st_d = _steps(dh, outer, steps, inner) if dh is not None else (None, 0, 0)
    dlast = dlast.contiguous() if dlast is not None else None
    lengths = lengths.to(torch.int64).contiguous() if lengths is not None else None
    a = L.GatedScanBwdArgs(outer, steps, inner, xt, _TYPES[gate.dtype], FORMS[form], int(bool(reverse)), x3.data_ptr(), so_x, st_x,
                           g3.data_ptr(), so_g, st_g, _ptr(d3), so_d, st_d, _ptr(dlast), _ptr(lengths), states.contiguous().data_ptr(),
                           dx.data_ptr(), dgate.data_ptr(), _ptr(dh0), _ptr(scratch))
    _launch(L.load().sb_gated_scan_bwd, x.device, a)
    return dx, dgate, dh0


def _rows_beside(t, state, n):
    """_rows; a copy where they lie on the state's memory in another order, in which other threads write it"""
    r, ld = _rows(t, n)
    at, to = r.data_ptr(), state.data_ptr()
    size = ((t.numel() // n - 1) * ld + n) * r.element_size()
    if at < to + state.nbytes and to < at + size and not (at == to and ld == n and r.dtype == torch.float32):
        return t.clone(memory_format=torch.contiguous_format), n
    return r, ld


def gated_scan_step(x, gate, state, *, form="sigmoid"):
    """one step: `state` (float32, dense, x's shape) becomes a state + b in place -> its value in x's type"""
    _not_on_stream("gated_scan_step")
    _need(x, "gated_scan_step: x", _TYPES)
    _need(gate, "gated_scan_step: gate", (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32), x.device, x.shape)
    _need(state, "gated_scan_step: state", (torch.float32,), x.device, x.shape)
    if form not in FORMS:
        _fail(f"gated_scan_step: form is one of {sorted(FORMS)}, got {form!r}")
    if not state.is_contiguous():
        _fail("gated_scan_step: state is updated in place and must be contiguous")
    y = _like(x)
    if x.numel() == 0:
        return y
    n = x.shape[-1] if x.dim() else 1
    (xr, ldx), (gr, ldg) = _rows_beside(x, state, n), _rows_beside(gate, state, n)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    _launch(L.load().sb_gated_scan_step, x.device, xr.data_ptr(), gr.data_ptr(), state.data_ptr(), y.data_ptr(), x.numel() // n, n, ldx, ldg,
            _TYPES[x.dtype], _TYPES[gate.dtype], FORMS[form])
    return y


# ---- AdamW over many tensors ----
def adamw_blocks(sizes):
    """first block of each of the tensors in the state buffers, and behind the last one: a tensor starts at a multiple of
    ADAMW_BLOCK elements"""
    return list(itertools.accumulate(((n + L.ADAMW_BLOCK - 1) // L.ADAMW_BLOCK for n in sizes), initial=0))


def adamw_state(params, bits=32):
    """zero states for adamw_step: exp_avg, exp_avg_sq in one buffer each (float32, or float8_e4m3fn / float8_e5m2 codes with a
    float8_e8m0fnu scale for every ADAMW_BLOCK elements), and `master`, float32, where a parameter has 16 bits"""
    params = list(params)
    if bits not in (32, 8):
        _fail(f"adamw_state: bits is 32 or 8, got {bits}")
    for p in params:
        _need(p, "adamw_state: parameter", _TYPES, params[0].device)
    starts = adamw_blocks([p.numel() for p in params])
    blocks, dev = starts[-1], params[0].device if params else "cuda"
    n = blocks * L.ADAMW_BLOCK
    if bits == 32:
        st = {k: torch.zeros(n, dtype=torch.float32, device=dev) for k in ("exp_avg", "exp_avg_sq")}
    else:
        st = {}
        for k, t in (("exp_avg", torch.float8_e4m3fn), ("exp_avg_sq", torch.float8_e5m2)):
            st[k] = torch.zeros(n, dtype=torch.uint8, device=dev).view(t)
            st[k + "_scale"] = torch.zeros(blocks, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
    if any(p.dtype != torch.float32 for p in params):
        st["master"] = torch.zeros(n, dtype=torch.float32, device=dev)
        for p, b in zip(params, starts):
            st["master"][b * L.ADAMW_BLOCK:b * L.ADAMW_BLOCK + p.numel()].copy_(p.detach().reshape(-1))
    return st


_EIGHT = {"exp_avg": (torch.float8_e4m3fn, 448.0), "exp_avg_sq": (torch.float8_e5m2, 57344.0)}


def adamw_state_values(state):
    """the float32 values that adamw_step's states stand for (exact): {"exp_avg", "exp_avg_sq"}"""
    out = {}
    for k in _EIGHT:
        v = state[k]
        out[k] = v if v.dtype == torch.float32 else (v.float().view(-1, L.ADAMW_BLOCK) * state[k + "_scale"].float()[:, None]).view(-1)
    return out


def adamw_state_pack(state, values):
    """`values` (float32 of the buffers' length) into `state`; where that has 8 bits each is rounded to the nearest code, values of
    adamw_state_values come back exactly, and no positive exp_avg_sq becomes 0"""
    for k, (kind, largest) in _EIGHT.items():
        x = values[k]
        if state[k].dtype == torch.float32:
            state[k].copy_(x)
            continue
        x = x.float().view(-1, L.ADAMW_BLOCK)
        big = x.abs().amax(1)
        man, exp = torch.frexp(big / largest)                    # big <= largest * 2^e, e the smallest
        e = torch.where(man == 0.5, exp - 1, exp).clamp(-127, 127)
        e = torch.where(big == 0, -127, e)
        byte = torch.where(torch.isfinite(big), e + 127, 255).to(torch.uint8)
        scale = byte.view(torch.float8_e8m0fnu).float()[:, None]
        y = torch.where(torch.isfinite(big)[:, None], x / scale, 0.0)
        code = y.clamp(-largest, largest).to(kind).view(torch.uint8)
        if k == "exp_avg_sq":
            code = torch.where((code == 0) & (x > 0), 1, code)
        state[k].view(torch.uint8).copy_(code.reshape(-1))
        state[k + "_scale"].view(torch.uint8).copy_(byte)


_ROW = np.dtype([("p", "u8"), ("g", "u8"), ("n", "i8"), ("first_block", "i4"), ("first_chunk", "i4")])      # sb_adamw_tensor


@functools.lru_cache(maxsize=32)
def _adamw_layout(sizes, take, ptypes, gtypes):
    """-> (blocks of the state buffers, [(ptype, gtype, places among the taken tensors (None: all of them), table rows)]): one entry a
    launch, tensors of one pair of types, pointers left open.  A function of the sizes and types alone."""
    chunk = L.load().sb_adamw_chunk()
    starts = adamw_blocks(sizes)
    take = range(len(sizes)) if take is None else take
    groups = {}
    for j, key in enumerate(zip(ptypes, gtypes)):
        groups.setdefault(key, []).append(j)
    out = []
    for (pt, gt), js in groups.items():
        for k in range(0, len(js), L.ADAMW_MAX):
            ids, at = js[k:k + L.ADAMW_MAX], 0
            rows = np.zeros(len(ids), dtype=_ROW)
            for r, j in zip(rows, ids):
                r["n"], r["first_block"], r["first_chunk"] = sizes[take[j]], min(starts[take[j]], (1 << 31) - 1), at
                at += (sizes[take[j]] + chunk - 1) // chunk
            out.append((pt, gt, None if len(ids) == len(take) else np.array(ids), rows))
    return starts[-1], out


def _adamw_check_state(state, blocks, device, need_master):
    n = blocks * L.ADAMW_BLOCK
    eight = isinstance(state.get("exp_avg"), torch.Tensor) and state["exp_avg"].dtype == torch.float8_e4m3fn
    want = {"exp_avg": (torch.float8_e4m3fn, n), "exp_avg_sq": (torch.float8_e5m2, n), "exp_avg_scale": (torch.float8_e8m0fnu, blocks),
            "exp_avg_sq_scale": (torch.float8_e8m0fnu, blocks)} if eight else {k: (torch.float32, n) for k in ("exp_avg", "exp_avg_sq")}
    if need_master:
        want["master"] = (torch.float32, n)
    for k, (t, size) in want.items():
        b = _need(state.get(k), f"adamw_step: state[{k!r}]", (t,), device, (size,))
        if not b.is_contiguous() or b.data_ptr() % 16:
            _fail(f"adamw_step: state[{k!r}] must be contiguous and start at a multiple of 16 bytes")
    return 8 if eight else 32


def adamw_step(params, grads, state, step, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, gscale=1.0, clip=0.0, seed=0,
               skipped=None):
    """One AdamW step (torch.optim.AdamW without amsgrad) over all tensors: `params` (no two updated ones share memory) and `state`
    (adamw_state of the same parameters) are updated in place.

    grads: one a parameter, of its type or float32, None: that parameter and its states are left alone.
    step: the step's number, from 1 on -- an int, or an int32 tensor of one element, which a captured graph reads at every replay.
    lr: a number or a float32 tensor of one element.  clip > 0: the gradients, scaled by gscale, are clipped to that norm over all
    tensors.  seed: of the 8-bit states' rounding.  skipped (int32, one element): counts a step that the device's watchdog word turned into a no-op
    (ops.adam_step)."""
    _not_on_stream("adamw_step")
    params, grads = list(params), list(grads)
    step_dev = lr_dev = None
    if isinstance(step, torch.Tensor):
        step_dev, step = step, 0
    elif params and getattr(params[0], "is_cuda", False) and torch.cuda.is_current_stream_capturing():
        _fail("adamw_step: a captured graph would repeat this step's number at every replay: pass step as an int32 tensor")
    if isinstance(lr, torch.Tensor):
        lr_dev, lr = lr, 0.0
    if skipped is not None and not (isinstance(skipped, torch.Tensor) and skipped.dtype is torch.int32 and skipped.is_cuda and skipped.numel() == 1 and
                                    (not params or skipped.get_device() == params[0].get_device())):      # (the kernel counts it up)
        _fail("adamw_step: skipped is an int32 tensor of one element on the parameters' GPU")
    fast = native()
    if fast is not None and params and isinstance(state.get("exp_avg"), torch.Tensor):
        bits = 8 if state["exp_avg"].dtype == torch.float8_e4m3fn else 32
        keys = ["exp_avg", "exp_avg_sq"] + ["exp_avg_scale", "exp_avg_sq_scale"] * (bits == 8) + ["master"] * (params[0].dtype != torch.float32)
        done = False
        try:
            buffers = [state[k] for k in keys]
            guard = _OPS._SCHED_STATUS.get(params[0].get_device())
            done = fast.adamw_step(params, grads, buffers, bits, step, step_dev, lr, lr_dev, *betas, eps, weight_decay, gscale, clip,
                                   seed & 0xFFFFFFFF, guard.data_ptr() if guard is not None else 0,
                                   skipped.data_ptr() if guard is not None and skipped is not None else 0)
        except (TypeError, KeyError, OverflowError):      # an argument of another kind, nothing has been done: what it is, is said below
            pass
        except RuntimeError as e:      # a launch that failed, perhaps behind others that did not: the step is not begun again
            raise said(e)
        if done:
            return
    if len(params) != len(grads):
        _fail(f"adamw_step: {len(params)} parameters, {len(grads)} gradients")
    if not params:
        return
    dev = params[0].device
    index, T = params[0].get_device(), torch.Tensor
    ptypes = [p.dtype for p in params]
    if index < 0 or {*map(T.get_device, params)} != {index} or not _TYPES.keys() >= {*ptypes} or not all(map(T.is_contiguous, params)):
        i = next(i for i, p in enumerate(params) if not (p.is_cuda and p.device == dev and p.dtype in _TYPES and p.is_contiguous()))
        _fail(f"adamw_step: parameter {i}: expected a contiguous float32 / bfloat16 / float16 tensor on one GPU, got {params[i].dtype} on "
              f"{params[i].device}{'' if params[i].is_contiguous() else ', not contiguous'}")
    sizes = tuple(map(T.numel, params))
    if any(g is None for g in grads) or 0 in sizes:
        take = tuple(i for i, g in enumerate(grads) if g is not None and sizes[i])
        ps, gs, pts = [params[i] for i in take], [grads[i] for i in take], [ptypes[i] for i in take]
    else:
        take, ps, gs, pts = None, params, grads, ptypes
    for i, g in enumerate(gs):
        if g.layout is not torch.strided or g.is_neg():
            what = "a lazily negated one (call .resolve_neg())" if g.layout is torch.strided else g.layout
            _fail(f"adamw_step: gradient {take[i] if take else i}: expected a dense tensor, got {what}")
    gtypes = [g.dtype for g in gs]
    if {*map(T.get_device, gs)} - {index} or not all(map(T.is_same_size, ps, gs)) or \
            (gtypes != pts and any(a is not b and a is not torch.float32 for a, b in zip(gtypes, pts))):
        i, p, g = next((i, p, g) for i, (p, g) in enumerate(zip(ps, gs)) if not (g.is_cuda and g.device == dev and g.shape == p.shape and
                                                                               g.dtype in (p.dtype, torch.float32)))
        _fail(f"adamw_step: gradient {take[i] if take else i}: expected {p.dtype} or float32 of shape {tuple(p.shape)} on {dev}, got {g.dtype} "
              f"{tuple(g.shape)} on {g.device}")
    if not all(map(T.is_contiguous, gs)):
        gs = [g.contiguous() for g in gs]
    blocks, batches = _adamw_layout(sizes, take, tuple(map(_TYPES.get, pts)), tuple(map(_TYPES.get, gtypes)))
    need_master = {*ptypes} != {torch.float32}
    bits = _adamw_check_state(state, blocks, dev, need_master)
    if blocks >= 1 << 31:
        _fail("adamw_step: more than 2^31 blocks of states")
    if step_dev is not None:
        if _need(step_dev, "adamw_step: step", (torch.int32,), dev).numel() != 1:
            _fail("adamw_step: step is one number")
    elif step < 1 or step >= 1 << 31:
        _fail(f"adamw_step: step counts from 1, got {step}")
    if lr_dev is not None and _need(lr_dev, "adamw_step: lr", (torch.float32,), dev).numel() != 1:
        _fail("adamw_step: lr is one number")
    if not all(0 <= b < 1 for b in betas) or not eps >= 0:
        _fail(f"adamw_step: betas are in [0, 1) and eps is not negative, got {betas}, {eps}")
    if len({p.data_ptr() for p, n in zip(params, sizes) if n}) < sum(n > 0 for n in sizes):
        _fail("adamw_step: a parameter is given twice, or two of them share memory")
    places = sorted((p.data_ptr(), p.data_ptr() + p.nbytes) for p in ps)
    if any(a[1] > b[0] for a, b in zip(places, places[1:])):
        _fail("adamw_step: two parameters share memory")
    if not clip >= 0:
        _fail(f"adamw_step: clip is a norm (0: none), got {clip}")
    if not batches:
        return
    lib = L.load()
    pp, gp = (np.array([*map(T.data_ptr, ts)], dtype=np.uint64) for ts in (ps, gs))
    calls = []
    for pt, gt, ids, rows in batches:
        a = L.AdamwArgs()
        table = rows.copy()
        table["p"], table["g"] = (pp, gp) if ids is None else (pp[ids], gp[ids])
        C.memmove(C.addressof(a), table.__array_interface__["data"][0], table.nbytes)
        a.count, a.ptype, a.gtype, a.bits = len(table), pt, gt, bits
        a.m, a.v = state["exp_avg"].data_ptr(), state["exp_avg_sq"].data_ptr()
        if bits == 8:
            a.m_scale, a.v_scale = state["exp_avg_scale"].data_ptr(), state["exp_avg_sq_scale"].data_ptr()
        if need_master:
            a.master = state["master"].data_ptr()
        a.lr, (a.beta1, a.beta2), a.eps, a.weight_decay = lr, betas, eps, weight_decay
        a.lr_dev, a.step_dev, a.step, a.seed = _ptr(lr_dev), _ptr(step_dev), step, seed & 0xFFFFFFFF
        a.gscale, a.clip = gscale, clip
        calls.append(a)
    calls[-1].last = 1
    guard = _OPS._SCHED_STATUS.get(index)
    torch.autograd.graph.increment_version(ps)
    if clip > 0:
        slots = L.ADAMW_NORM_SLOTS // len(calls)
        if slots == 0:
            _fail(f"adamw_step: clipping over more than {L.ADAMW_NORM_SLOTS * L.ADAMW_MAX} tensors")
        part = params[0].new_empty(L.ADAMW_NORM_SLOTS, dtype=torch.float64)
        for k, a in enumerate(calls):
            _launch(lib.sb_adamw_norm, dev, a, part.data_ptr(), k * slots, slots)
    for a in calls:
        if clip > 0:
            a.norm_part, a.norm_slots = part.data_ptr(), slots * len(calls)
        if guard is not None:
            a.guard, a.skipped = guard.data_ptr(), _ptr(skipped)
        _launch(lib.sb_adamw_step, dev, a)
