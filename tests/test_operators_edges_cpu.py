"""What the channels-last GroupNorm, the gradient norms and the fused SGD step refuse beside their arguments' shapes and types: no GPU needed."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from lgd_amd import hip, ops, optim


@pytest.mark.parametrize("which", ["map", "second map", "weight", "bias", "gradient", "clipped gradient"])
def test_forward_mode_is_refused(which):
    """an input with a tangent: an error, not an output without one"""
    x, y, w, b, g = torch.ones(1, 4, 2, 2), torch.ones(1, 4, 3, 3), torch.ones(4), torch.zeros(4), torch.ones(5)
    with fw.dual_level():
        dual = lambda t, name: fw.make_dual(t, torch.ones_like(t)) if name == which else t  # noqa: E731
        with pytest.raises(hip.LgdHipError, match="forward-mode"):
            if which == "gradient":
                optim.grad_norm([torch.ones(3), dual(g, which)])
            elif which == "clipped gradient":
                p = torch.nn.Parameter(torch.ones(5))
                p.grad = dual(g, which)
                optim.clip_grad_norm_([p], 1.0)
            else:
                ops.group_norm_act([dual(x, "map"), dual(y, "second map")], 2, dual(w, "weight"), dual(b, "bias"))
