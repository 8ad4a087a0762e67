"""What the channels-last GroupNorm, the gradient norms and the clipping refuse, and their host logic: no GPU needed (every refusal is decided
before anything is launched)."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from lgd_amd import hip, ops, optim


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(hip.lib_path()):
        import __graft_entry__ as g
        g.build()
    return hip.load()


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,what", [
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 4), "split"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 0), "split"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 2, act="gelu"), "activation"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 2, eps=-1.0), "eps"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 2, eps=float("nan")), "eps"),
    (lambda: ops.group_norm_act([_x(1, 6, 2)], 2), "maps of one call"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2), _x(1, 4, 2, 2)], 2), "maps of one call"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2), _x(2, 6, 2, 2)], 2), "maps of one call"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2), _x(1, 6, 2, 2, dtype=torch.bfloat16)], 2), "one type"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2, dtype=torch.float64)], 2), "fp32, bf16 or fp16"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)] * 17, 2), "at most 16"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 2, _x(5)), "weight"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 2, _x(6), _x(6, dtype=torch.int32)), "bias"),
    (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 2, _x(6), _x(6, dtype=torch.bfloat16)), "one type"),
    (lambda: optim.grad_norm([_x(3)], 3.0), "norm_type"),
    (lambda: optim.grad_norm([_x(3, dtype=torch.float64)]), "strided fp32"),
    (lambda: optim.grad_norm([_x(3), torch.zeros(3, dtype=torch.int32)]), "strided fp32"),
    (lambda: optim.grad_norm([torch.zeros(3, 3).to_sparse()]), "strided fp32"),
    (lambda: optim.clip_grad_norm_([], -1.0), "max_norm"),
    (lambda: optim.clip_grad_norm_([], float("nan")), "max_norm"),
    (lambda: optim.grad_norm([1.0]), "expected tensors"),
    (lambda: ops.group_norm_act([None], 2), "expected tensors"),
    (lambda: optim.FusedClipSGD([], 1.0, clip_norm=1.0), "not both"),
])
def test_refusals(call, what):
    with pytest.raises(hip.LgdHipError, match=what):
        call()


def _param(grad):
    p = torch.nn.Parameter(torch.empty(grad.shape))
    p.grad = grad
    return p


def test_gradients_that_share_memory_are_refused():
    buf = torch.zeros(100)
    for grads in ([buf[:60], buf[59:]], [buf, buf], [buf[10:20], buf[:50], buf[60:]], [buf[:1].expand(4), buf[50:60]],
                  [buf.view(10, 10)[:, 3], buf.view(10, 10)[:, 3]]):
        with pytest.raises(hip.LgdHipError, match="share memory|expanded"):
            optim.clip_grad_norm_([_param(g) for g in grads], 1.0)


def test_views_side_by_side_do_not_share():
    buf, mat = torch.zeros(100), torch.zeros(10, 10)
    for grads in ([buf[:50], buf[50:]], [buf[60:], buf[:60], buf[5:5], buf[60:60]], [buf[:0], buf], [mat[:, 2], mat[:, 3]],
                  [torch.zeros(4, 3, 2, 2).to(memory_format=torch.channels_last), mat.t()]):
        with pytest.raises(hip.LgdHipError, match="GPU|device tensor"):   # nothing to say against them but where they are
            optim.clip_grad_norm_([_param(g) for g in grads], 1.0)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU failure mode")
def test_no_gpu_no_answer():
    for call in (lambda: ops.group_norm_act([_x(1, 6, 2, 2)], 2), lambda: optim.grad_norm([_x(3)]),
                 lambda: optim.clip_grad_norm_([_param(_x(3))], 1.0)):
        with pytest.raises(hip.LgdHipError, match="GPU|device tensor"):
            call()


def test_nothing_to_do():
    assert ops.group_norm_act([], 4) == []
    assert float(optim.grad_norm([])) == 0.0
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0   # no gradients


def test_c_entries_refuse_bad_arguments(lib):
    hw, big = hip.int_array([8, 8]), hip.int_array([1 << 16, 1 << 15])
    ptrs = (ctypes.c_void_p * 1)(4096)
    none = (ctypes.c_void_p * 1)(None)
    one = ctypes.c_void_p(4096)   # never dereferenced: every call below is refused on the host
    fwd = lambda x=ptrs, hw=hw, L=1, B=1, C=6, G=2, dt=0, pt=0, eps=1e-5, act=0, ws=one, st=one, y=ptrs: lib.lgd_gn_act_fwd(  # noqa: E731
        x, hw, L, B, C, G, dt, None, None, pt, eps, act, ws, st, y, None)
    for bad in (dict(x=None), dict(x=none), dict(y=None), dict(y=none), dict(L=0), dict(L=17), dict(B=0), dict(C=0), dict(G=0), dict(G=4), dict(dt=3),
                dict(dt=-1), dict(pt=3), dict(eps=-1.0), dict(eps=float("nan")), dict(act=3), dict(act=-1), dict(hw=hip.int_array([80, 800]), ws=None), dict(st=None),
                dict(hw=hip.int_array([0, 8])), dict(hw=None), dict(hw=big)):
        assert fwd(**bad) == -1, bad
    assert lib.lgd_gn_act_bwd(ptrs, None, hw, 1, 1, 6, 2, 0, None, None, 0, 0, one, one, ptrs, None, None, None) == -1
    assert lib.lgd_gn_act_bwd(ptrs, ptrs, hw, 1, 2, 6, 2, 0, None, None, 0, 0, None, one, ptrs, None, None, None) == -1   # the workspace
    assert lib.lgd_gn_act_bwd(ptrs, ptrs, hw, 1, 1, 6, 2, 0, None, None, 0, 0, one, one, none, None, None, None) == -1
    bytes_of = lambda hw, B, back: lib.lgd_gn_act_ws_bytes(hw, 1, B, 6, 2, 0, back)  # noqa: E731
    assert bytes_of(big, 1, 0) == bytes_of(big, 1, 1) == ctypes.c_size_t(-1).value and bytes_of(hip.int_array([80, 800]), 1, 0) > 0
    assert bytes_of(hw, 2, 0) == 0 and bytes_of(hw, 1, 1) == 0 and bytes_of(hw, 2, 1) > 0   # small: no workspace but for the parameters' gradients

    one_px = hip.int_array([1, 1])   # more workgroups or statistics than a launch numbers
    assert lib.lgd_gn_act_ws_bytes(one_px, 1, 1 << 25, 64, 64, 0, 0) == lib.lgd_gn_act_ws_bytes(one_px, 1, 1 << 21, 520, 520, 0, 1) == ctypes.c_size_t(-1).value

    def norm(rec, n=1, kind=0, ws=one, out=one, clip=None):
        r = (hip.GradTensor * 1)(rec)
        if clip is not None:
            return lib.lgd_grad_clip(r, n, kind, clip, ws, out, None)
        return lib.lgd_grad_norm(r, n, kind, ws, out, None)
    ok = hip.GradTensor(4096, 8, 0, 0)
    for bad in (hip.GradTensor(None, 8, 0, 0), hip.GradTensor(4096, -1, 0, 0), hip.GradTensor(4096, 8, 3, 0), hip.GradTensor(4098, 8, 0, 0),
                hip.GradTensor(4097, 8, 1, 0)):
        assert norm(bad) == -1
    assert norm(ok, n=-1) == -1 and norm(ok, kind=3) == -1 and norm(ok, ws=None) == -1 and norm(ok, out=None) == -1
    assert norm(ok, clip=-1.0) == -1 and norm(ok, clip=float("nan")) == -1
    assert lib.lgd_grad_norm(None, 1, 0, one, one, None) == -1

    off, blk = hip.int_array([0, 1, 2]), hip.int_array([0, 1, 3])
    step = lambda tab=one, nt=2, nb=3, o=off, b=blk, ng=2, kind=0, m=1.0, ws=one, out=one: lib.lgd_sgd_norm_step(  # noqa: E731
        tab, one, nt, nb, o, b, ng, kind, m, ws, out, None)
    for bad in (dict(tab=None), dict(nt=0), dict(nt=3), dict(nb=4), dict(nb=-1), dict(o=None), dict(b=None), dict(ng=0), dict(ng=17), dict(kind=3), dict(m=-1.0),
                dict(m=float("nan")), dict(ws=None), dict(out=None), dict(o=hip.int_array([0, 3, 2])), dict(b=hip.int_array([0, 4, 3])),
                dict(o=hip.int_array([1, 1, 2])), dict(o=hip.int_array([0, 0, 2]), b=hip.int_array([0, 1, 3]))):
        assert step(**bad) == -1, bad
    recs = (ctypes.c_uint8 * (48 * 73))()   # the form with the table in host memory: refused before anything of it is used
    host = lambda tab=recs, nt=2, nb=3, o=off, b=blk, ng=2, kind=0, m=1.0, ws=one, out=one: lib.lgd_sgd_norm_step_host(  # noqa: E731
        tab, b, nt, nb, o, b, ng, kind, m, ws, out, None)
    for bad in (dict(tab=None), dict(nt=0), dict(nt=73), dict(nb=4), dict(b=None), dict(o=None), dict(ng=17), dict(kind=3), dict(m=-1.0), dict(ws=None), dict(out=None)):
        assert host(**bad) == -1, bad
    assert lib.lgd_sgd_norm_ws_bytes(0) == 0 and lib.lgd_sgd_norm_ws_bytes(2) > 0


def test_clip_by_the_whole_gradient_on_the_cpu():
    """CLIP_TYPE 'full_model': each optimizer's gradient as one vector (torch's clip_grad_norm_ off the GPU)"""
    from lgd_amd.engine import Trainer
    t = Trainer.__new__(Trainer)
    a, b, c = (torch.nn.Parameter(torch.zeros(n)) for n in (4, 2, 3))
    a.grad, b.grad = torch.full((4,), 3.0), torch.full((2,), 4.0)
    t.stu_optimizer, t.tea_optimizer = torch.optim.SGD([a, b], 0.1), torch.optim.SGD([c], 0.1)
    c.grad = torch.tensor([0.1, 0.2, 0.2])
    t.clip = SimpleNamespace(CLIP_TYPE="full_model", CLIP_VALUE=0.5, NORM_TYPE=2.0)
    t._clip()
    assert abs(float(torch.cat([a.grad, b.grad]).norm()) - 0.5) < 1e-6
    assert torch.equal(a.grad / a.grad[0], torch.ones(4)) and abs(float(b.grad[0] / a.grad[0]) - 4 / 3) < 1e-6
    assert torch.equal(c.grad, torch.tensor([0.1, 0.2, 0.2]))   # 0.3 < 0.5


def test_fused_step_is_offered_for_the_clip_types_it_has():
    clip = lambda kind, norm=2.0: SimpleNamespace(ENABLED=True, CLIP_TYPE=kind, CLIP_VALUE=1.0, NORM_TYPE=norm)  # noqa: E731
    assert optim.supported([], clip("value")) and optim.supported([], clip("full_model")) and optim.supported([], clip("full_model", float("inf")))
    assert not optim.supported([], clip("norm")) and not optim.supported([], clip("full_model", 3.0))
    p = torch.nn.Parameter(torch.zeros(2))
    with pytest.raises(hip.LgdHipError, match="share no parameter"):
        optim.FusedClipSGD([torch.optim.SGD([p], 0.1), torch.optim.SGD([p], 0.1)], clip_norm=1.0)
    with pytest.raises(hip.LgdHipError, match="norm_type"):
        optim.FusedClipSGD([torch.optim.SGD([p], 0.1)], clip_norm=1.0, norm_type=3)
