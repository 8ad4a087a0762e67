"""Calls of the channels-last GroupNorm, the gradient norms and the fused SGD step at their edges: differentiating again."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _rand(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(DEV)


def _map(form):
    """a leaf of each memory order, (2, 8, 5, 6)"""
    x = _rand((2, 8, 5, 6), 1)
    if form == "channels-last":
        return x.to(memory_format=torch.channels_last).requires_grad_(True)
    if form == "nchw":
        return x.requires_grad_(True)
    wide = _rand((2, 8, 7, 8), 2).to(memory_format=torch.channels_last).requires_grad_(True)
    return wide[:, :, 1:6, 1:7]


def _parameters(kind):
    w, b = _rand((8,), 3, 0.3) + 1, _rand((8,), 4)
    if kind == "none":
        return None, None
    if kind == "frozen":
        return w, b
    if kind == "trainable":
        return w.requires_grad_(True), b.requires_grad_(True)
    both = torch.stack([w, b], 1).requires_grad_(True)   # columns: strided
    return both[:, 0], both[:, 1]


@pytest.mark.parametrize("kind", ["none", "frozen", "trainable", "strided"])
@pytest.mark.parametrize("form", ["channels-last", "nchw", "slice"])
def test_a_second_derivative_raises_for_every_memory_order(form, kind):
    """a gradient penalty through group_norm_act: an error in every form of the call, never a penalty that is left out"""
    from lgd_amd import ops
    x, (w, b) = _map(form), _parameters(kind)
    dy = _rand((2, 8, 5, 6), 5)
    ask = lambda leaf: torch.autograd.grad(ops.group_norm_act([x], 2, w, b, act="silu")[0], [leaf], dy, create_graph=True)[0]  # noqa: E731
    first, = torch.autograd.grad(ops.group_norm_act([x], 2, w, b, act="silu")[0], [x], dy)
    for leaf in [x] + ([w, b] if w is not None and w.requires_grad else []):
        g = ask(leaf)
        assert g.requires_grad
        if leaf is x:
            assert torch.equal(g, first)
        for other in [x] + ([w] if w is not None and w.requires_grad else []):
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(g.square().sum(), [other], retain_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            (ops.group_norm_act([x], 2, w, b, act="silu")[0].sum() + g.square().sum()).backward()


@pytest.mark.parametrize("form", ["channels-last", "nchw"])
def test_a_derivative_by_the_output_gradient_raises(form):
    """the backward is linear in dy, which may carry a graph of its own; a frozen map and parameters otherwise"""
    from lgd_amd import ops
    x, dy = _map(form), _rand((2, 8, 5, 6), 5).requires_grad_(True)
    g, = torch.autograd.grad(ops.group_norm_act([x], 2)[0], [x], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(g.square().sum(), [dy])
