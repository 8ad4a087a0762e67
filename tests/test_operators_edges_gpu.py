"""Calls of the channels-last GroupNorm, the gradient norms and the fused SGD step at their edges: differentiating again, optimizer states that come and go,
long sums."""
import copy

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


def test_threads_that_differentiate_one_graph():
    """two threads run backward over one graph, a third one releases it in between: the right gradients or the error of a freed graph, nothing else"""
    import threading
    from lgd_amd import ops
    x, (w, b), dy = _map("nchw"), _parameters("trainable"), _rand((2, 8, 5, 6), 5)
    want = torch.autograd.grad(ops.group_norm_act([x], 2, w, b, act="silu")[0], [x, w, b], dy)
    torch.cuda.synchronize()
    for keep in (True, False):
        y, = ops.group_norm_act([x], 2, w, b, act="silu")
        got, errors, start = [], [], threading.Barrier(3)

        def work(times, retain):
            start.wait()
            for _ in range(times):
                try:
                    got.append(torch.autograd.grad(y, [x, w, b], dy, retain_graph=retain))
                except RuntimeError as e:
                    errors.append(str(e))
        threads = [threading.Thread(target=work, args=a) for a in ((20, True), (20, True), (1, keep))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert len(got) + len(errors) == 41 and all("freed" in e for e in errors) and (not keep or not errors) and got
        assert all(torch.equal(g, v) for grads in got for g, v in zip(grads, want))


def test_a_derivative_of_the_norm_raises():
    """a gradient penalty by grad_norm: an error, not a penalty that is left out; without a graph the norm has none either"""
    from lgd_amd import optim
    w = _rand((8, 8), 6).requires_grad_(True)
    g, = torch.autograd.grad((w * w * w).sum(), [w], create_graph=True)
    n = optim.grad_norm([g, torch.ones(3, device=DEV)])
    assert n.requires_grad
    with pytest.raises(RuntimeError, match="no derivative"):
        ((w * w).sum() + n).backward()
    with torch.no_grad():
        assert torch.equal(optim.grad_norm([g, torch.ones(3, device=DEV)]), n) and not optim.grad_norm([g]).requires_grad
    assert not optim.grad_norm([g.detach()]).requires_grad
    w.grad = g
    assert not optim.clip_grad_norm_([w], 1.0).requires_grad


def test_a_tangent_of_the_output_gradient_raises():
    """forward over reverse: an error, not an input gradient without a tangent"""
    import torch.autograd.forward_ad as fw
    from lgd_amd import ops
    x, dy = _map("nchw"), _rand((2, 8, 5, 6), 5)
    y, = ops.group_norm_act([x], 2)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, [x], fw.make_dual(dy, torch.ones_like(dy)))


def _sgd(count, seed=7):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(5 + 3 * i, generator=g).to(DEV)) for i in range(count)]
    return ps, [torch.optim.SGD(ps[:2], 0.1, momentum=0.9), torch.optim.SGD(ps[2:], 0.2, momentum=0.8, weight_decay=1e-3)]


def _load(optimizers, factor, times):
    for o in optimizers:
        for k in range(times):
            sd = copy.deepcopy(o.state_dict())
            for st in sd["state"].values():
                st["momentum_buffer"] = st["momentum_buffer"] * factor + 1.0
            o.load_state_dict(sd)


def _replace(optimizers):
    for o in optimizers:
        for st in o.state.values():
            st["momentum_buffer"] = st["momentum_buffer"] * -2.0


def _drop(optimizers):
    for o in optimizers:
        o.state.clear()


def _forget(optimizers):   # the key leaves the inner dict: both sides begin again at zero
    for o in optimizers:
        for st in o.state.values():
            st.pop("momentum_buffer")


CHANGES = {"load": lambda o: _load(o, -1.5, 1), "load twice": lambda o: _load(o, -1.5, 2), "load four times": lambda o: _load(o, 0.5, 4),
           "replaced buffers": _replace, "cleared": _drop, "one optimizer": lambda o: _load(o[1:], 2.0, 2), "forgotten": _forget}


@pytest.mark.parametrize("limit", [None, 0.5])
@pytest.mark.parametrize("count", [6, 90])
@pytest.mark.parametrize("change", list(CHANGES))
def test_the_step_follows_the_optimizers_state(change, count, limit):
    """momentum that is loaded, replaced or dropped between two steps counts in the next one, and the optimizers hold what the step wrote.  Tolerance: torch's own
    step rounds each operation and its norm is fp32; 2e-5 of the value covers a few steps of that (2^-24 each), 2e-6 the cancelled ones"""
    from lgd_amd import optim
    (pa, oa), (pb, ob) = _sgd(count), _sgd(count)
    fused = optim.FusedClipSGD(ob, clip_norm=limit)
    for step in range(4):
        for i, (a, b) in enumerate(zip(pa, pb)):
            a.grad = _rand(tuple(a.shape), 100 * step + i)
            b.grad = a.grad.clone()
        for o in oa:
            if limit is not None:
                torch.nn.utils.clip_grad_norm_([p for g in o.param_groups for p in g["params"]], limit)
            o.step()
        fused.step()
        for a, b, k in zip(pa, pb, [0, 0] + [1] * count):
            assert torch.allclose(a, b, rtol=2e-5, atol=2e-6), (step, k)
            assert torch.allclose(oa[k].state[a]["momentum_buffer"], ob[k].state[b]["momentum_buffer"], rtol=2e-5, atol=2e-6), (step, k)
        if step in (0, 2):
            CHANGES[change](oa)
            CHANGES[change](ob)


@pytest.mark.parametrize("limit", [None, 0.5])
def test_the_step_refuses_tensors_that_no_longer_fit(limit):
    """`.data` of a momentum buffer, a parameter or a gradient replaced by another type, device, order or size between two steps: refused, nothing is changed"""
    from lgd_amd import hip, optim
    for what, other in [("m", lambda t: t.half()), ("m", lambda t: t.cpu()), ("m", lambda t: torch.zeros(2 * t.numel(), device=DEV)[::2]),
                        ("g", lambda t: torch.ones(3, device=DEV)), ("g", lambda t: torch.ones(2 * t.numel(), device=DEV)),
                        ("g", lambda t: t.half()), ("p", lambda t: t.half()), ("p", lambda t: t.cpu())]:
        ps, opts = _sgd(4)
        fused = optim.FusedClipSGD(opts, clip_norm=limit)
        for p in ps:
            p.grad = torch.ones_like(p)
        fused.step()
        t = {"m": opts[1].state[ps[2]]["momentum_buffer"], "g": ps[2].grad, "p": ps[2]}[what]
        t.data = other(t.data)
        before = [p.detach().clone() for p in ps]
        with pytest.raises(hip.LgdHipError, match="fused SGD needs"):
            fused.step()
        assert all(torch.equal(p, b) for p, b in zip(ps, before)), what


@pytest.mark.parametrize("clip", [dict(), dict(clip_value=0.5), dict(clip_norm=0.5)])
@pytest.mark.parametrize("count", [6, 90])
def test_a_step_is_not_captured(count, clip):
    """with any kind of clipping: the table is the host's of the call; a first step neither, which would leave its buffers in the graph's memory; afterwards
    the step goes on eagerly"""
    from lgd_amd import hip, optim
    ps, opts = _sgd(count)
    fused = optim.FusedClipSGD(opts, **clip)
    for p in ps:
        p.grad = torch.ones_like(p)
    for first in (True, False):
        before = [p.detach().clone() for p in ps]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(hip.LgdHipError, match="captured"):
            with torch.cuda.graph(graph):
                fused.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, b) for p, b in zip(ps, before))
        assert not first or not any(o.state for o in opts)
        fused.step()
        assert not any(torch.equal(p, b) for p, b in zip(ps, before))


def test_parameter_gradients_over_millions_of_pixels():
    """dgamma and dbeta of like-signed terms, 2^22 pixels: x = 1 and -1 in turn (mean 0, variance 1), dy = c in the even channels and c x in the odd ones, so that
    dbeta = n c or 0, dgamma = 0 or n c r with r = 1 / sqrt(1 + eps).  At most 256 terms are added in fp32: 256 U, and a few U for the terms and the
    sums' roundings"""
    from lgd_amd import ops
    n, C, c = 2048 * 2048, 256, torch.tensor(0.6, dtype=torch.float32)
    x = torch.ones(1, 2048, 2048, C, device=DEV)
    x[:, :, 1::2] = -1.0
    dy = torch.full((1, 2048, 2048, C), float(c), device=DEV)
    dy[..., 1::2] *= x[..., 1::2]
    x, dy = x.permute(0, 3, 1, 2), dy.permute(0, 3, 1, 2)
    w, b = torch.ones(C, device=DEV, requires_grad=True), torch.zeros(C, device=DEV, requires_grad=True)
    y, = ops.group_norm_act([x], 32, w, b, act="none", eps=1e-5)
    dw, db = torch.autograd.grad(y, [w, b], dy)
    total, r = n * float(c), (1 + 1e-5) ** -0.5
    assert float((db[0::2].double() - total).abs().max()) <= 264 * U * total
    assert float((dw[1::2].double() - total * r).abs().max()) <= 264 * U * total
    assert float(db[1::2].abs().max()) <= 264 * U * total and float(dw[0::2].abs().max()) <= 264 * U * total


@pytest.mark.parametrize("C,G,dtype,act", [(33, 3, torch.bfloat16, "silu"), (24, 2, torch.float16, "relu"), (20, 5, torch.float32, "none")])
def test_group_norm_act_over_long_chunks(C, G, dtype, act):
    """maps of 0.7 GB, where a thread's sums are cut into blocks of 256 terms: odd rows over several vectors, one and several groups a vector; all results against
    64 bits, at the tolerances of the small maps (256 U of the terms' magnitudes)"""
    from test_operators_gpu import _check, _params, _run
    side = int((0.7e9 / C / dtype.itemsize) ** 0.5)
    g = torch.Generator(device=DEV).manual_seed(C)
    x, dy = ((torch.randn(1, side, side + 3, C, device=DEV, generator=g) * k + m).to(dtype).permute(0, 3, 1, 2) for k, m in ((1.3, 0.4), (1.0, 0.2)))
    w, b = _params(C, torch.float32, 9)
    ys, dxs, dw, db = _run([x], G, w, b, act, 1e-5, [dy])
    _check([x], G, w, b, act, 1e-5, [dy], ys, dxs, dw, db)


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("B,C,G,hws,dtype", [
    (2, 2047, 23, [(30, 30)], torch.float32), (8, 1331, 11, [(16, 16)], torch.float16), (8, 2049, 3, [(16, 16), (1, 1)], torch.bfloat16),
    (3, 517, 11, [(60, 60), (7, 9)], torch.bfloat16), (4, 2048, 32, [(40, 40)], torch.float32), (2, 4096, 32, [(40, 40), (3, 5)], torch.bfloat16),
    (1, 4096, 1, [(25, 21)], torch.float32), (1, 1285, 257, [(200, 33)], torch.float32), (2, 5001, 3, [(2, 3)], torch.float32)], ids=str)
def test_group_norm_act_wide_rows(B, C, G, hws, dtype, act):
    """rows over two to sixteen column blocks, whole groups or cut ones: fewer chunks than workgroups, several maps; all results against 64 bits"""
    from test_operators_gpu import _check, _maps, _params, _run
    xs, dys = _maps(B, C, hws, dtype, 60, 1.3, 0.4), _maps(B, C, hws, dtype, 70)
    w, b = _params(C, torch.float32, 80)
    ys, dxs, dw, db = _run(xs, G, w, b, act, 1e-5, dys)
    _check(xs, G, w, b, act, 1e-5, dys, ys, dxs, dw, db)
