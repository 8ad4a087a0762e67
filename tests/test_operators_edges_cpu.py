"""What the channels-last GroupNorm, the gradient norms and the fused SGD step refuse beside their arguments' shapes and types: no GPU needed."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from lgd_amd import hip, ops, optim


@pytest.fixture(scope="module", autouse=True)
def built():
    import os
    if not os.path.exists(hip.lib_path()):
        import __graft_entry__ as g
        g.build()


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


# batch, channels, groups, map, type, bytes of an element: rows of more than 320 vectors, that a vector of 16 bytes divides or not
WIDE = [(8, 2049, 3, (16, 16), 1, 2), (8, 1025, 5, (32, 32), 1, 2), (2, 2047, 23, (30, 30), 0, 4), (8, 1331, 11, (16, 16), 2, 2), (3, 517, 11, (60, 60), 1, 2),
        (4, 2048, 32, (40, 40), 0, 4), (2, 4096, 32, (40, 40), 1, 2), (1, 5001, 3, (64, 64), 0, 4)]


@pytest.mark.parametrize("B,C,G,hw,dtype,size", WIDE, ids=str)
def test_workspace_of_wide_rows_stays_below_the_maps(B, C, G, hw, dtype, size):
    """a row over several column blocks: what the workgroups leave for one another is less than the maps themselves"""
    shape = hip.int_array(list(hw))
    maps = B * C * hw[0] * hw[1] * size
    for backward in (0, 1):
        assert hip.load().lgd_gn_act_ws_bytes(shape, 1, B, C, G, dtype, backward) < maps


def test_the_fused_step_by_norm_is_not_offered_for_what_it_refuses():
    """a parameter in two optimizers, or more optimizers than it takes: the trainer stays on torch's step instead of failing"""
    from types import SimpleNamespace
    clip = lambda kind: SimpleNamespace(ENABLED=True, CLIP_TYPE=kind, CLIP_VALUE=1.0, NORM_TYPE=2.0)  # noqa: E731
    param = lambda: SimpleNamespace(is_cuda=True, dtype=torch.float32, is_contiguous=lambda: True)  # noqa: E731
    shared = param()

    def sgd(*params):
        o = torch.optim.SGD([torch.nn.Parameter(torch.zeros(1))], 0.1)
        o.param_groups[0]["params"] = list(params)
        return o
    two, many = [sgd(shared, param()), sgd(param(), shared)], [sgd(param()) for _ in range(17)]
    assert optim.supported(two, clip("value")) and optim.supported(many, clip("value"))
    assert not optim.supported(two, clip("full_model")) and not optim.supported(many, clip("full_model"))
    assert optim.supported(many[:16], clip("full_model"))
