"""Sequence-block operators with gradients: layer norm and the gated linear recurrence, beside the fused stages of functional.py.

    u = layer_norm(x, w, b);  h, last = gated_scan(*proj(u).chunk(2, -1), h0)

Any leading shape, float32 / bfloat16 / float16; the sums, statistics and states inside are float32.
"""
import torch

from . import _lib as L
from . import ops_seq


_T, _M, _N = torch.Tensor, (torch.Tensor, type(None)), (int, float)
_KINDS = {"layer_norm": (_T, _M, _M, _N), "gated_scan": (_T, _T, _M, _M, int, int, bool), "gated_scan_step": (_T, _T, _T, int)}


def _native(name, *args):
    """the call without Python in between, where it is one of the plain ones; empty: not taken, the wrappers see to it or say what is
    wrong"""
    native = ops_seq.native()
    if native is None:
        return ()
    try:
        return getattr(native, name)(*args)
    except (RuntimeError, TypeError) as e:
        if not all(isinstance(a, k) and (k is bool or not isinstance(a, bool)) for a, k in zip(args, _KINDS[name])):      # (nothing has been done)
            return ()
        raise ops_seq.said(e)


def _recorded(*tensors):
    """whether autograd is concerned: with gradients, or with tangents (which the autograd functions refuse)"""
    forward = torch.autograd.forward_ad
    if forward._current_level >= 0 and any(forward.unpack_dual(t).tangent is not None for t in tensors if isinstance(t, torch.Tensor)):
        return True
    return torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in tensors)


def _once_differentiable(backward):
    """torch's once_differentiable where somebody asks for a graph of the gradients, nothing around the call where nobody does (a
    backward pass of a small operator is its Python calls)"""
    checked = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, *grads: (checked if torch.is_grad_enabled() else backward)(ctx, *grads)


class LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = ops_seq.layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.wdtype = bias.dtype if bias is not None else None
        return y

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx, dw, db = ops_seq.layer_norm_bwd(dy.resolve_neg(), *ctx.saved_tensors, need[1], need[2], ctx.wdtype, check=False)
        return dx if need[0] else None, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, in x's type; weight / bias of shape (n,) in x's type or
    float32"""
    out = _native("layer_norm", x, weight, bias, eps)
    if out:
        return out[0]
    if _recorded(x, weight, bias):
        ops_seq.refuse_held_leaves(x, weight, bias)
        return LayerNormFn.apply(x, weight, bias, eps)
    return ops_seq.layer_norm_fwd(x, weight, bias, eps, stats=False)[0]


class GatedScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lengths, dim, form, reverse):
        h, last, states = ops_seq.gated_scan_fwd(x, gate, h0, dim=dim, form=form, reverse=reverse, lengths=lengths)
        ctx.save_for_backward(x, gate, states, lengths)
        ctx.how = dict(dim=dim, form=form, reverse=reverse)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @_once_differentiable
    def backward(ctx, dh, dlast):
        x, gate, states, lengths = ctx.saved_tensors
        if dh is None and dlast is None:
            return (None,) * 7
        need = ctx.needs_input_grad
        dh, dlast = (t if t is None else t.resolve_neg() for t in (dh, dlast))
        dx, dgate, dh0 = ops_seq.gated_scan_bwd(dh, dlast, x, gate, states, lengths=lengths, want_dh0=need[2], **ctx.how)
        return dx if need[0] else None, dgate if need[1] else None, dh0, None, None, None, None


def gated_scan(x, gate, h0=None, *, dim=1, form="sigmoid", reverse=False, lengths=None):
    """-> (h, last): h_t = a_t h_{t-1} + b_t along axis `dim`; last (float32) is the state behind the last step.

    form "sigmoid": a = sigmoid(gate), b = (1 - a) x; "decay": a = gate, b = x.  Steps are joined by products of gates: with "decay"
    gates beyond 1 in magnitude, products of 16 of them in a row have to stay within float32 (longer ones need not).
    h0: float32, x's shape without `dim` (None: zeros).  reverse: from the last step to the first.
    lengths (int64 / int32, x.shape[:dim]): a padded batch; steps at and behind a sequence's length leave its state alone, their
    outputs and gradients are 0 and their inputs are not looked at (reverse: the walk begins at a sequence's last own step).
    x and gate may be halves of one projection: a dense last axis is enough, other layouts are copied."""
    out = _native("gated_scan", x, gate, h0, lengths, dim, ops_seq.FORMS.get(form, -1), reverse)
    if out:
        return tuple(out)
    if _recorded(x, gate, h0):
        ops_seq.refuse_held_leaves(x, gate, h0)
        return GatedScanFn.apply(x, gate, h0, lengths, dim, form, reverse)
    return ops_seq.gated_scan_fwd(x, gate, h0, dim=dim, form=form, reverse=reverse, lengths=lengths, save=False)[:2]


def gated_scan_step(x, gate, state, *, form="sigmoid"):
    """One step of gated_scan for streaming: state (float32, x's shape, dense) is updated in place; -> its value in x's type.  No
    gradients: gated_scan with one step has them."""
    out = _native("gated_scan_step", x, gate, state, ops_seq.FORMS.get(form, -1))
    if out:
        return out[0]
    if _recorded(x, gate, state):
        raise L.SoundBubbleHipError("gated_scan_step updates the state in place and has no gradient: call gated_scan, or this under "
                                    "torch.no_grad()")
    return ops_seq.gated_scan_step(x, gate, state, form=form)
