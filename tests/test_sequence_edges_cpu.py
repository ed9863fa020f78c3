"""Sequence-block operators without a GPU: what is refused, and what a failed call leaves behind."""
import pytest


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
