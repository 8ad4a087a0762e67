"""Channels-last GroupNorm + activation, gradient norms, clipping and the SGD step that clips by norm, against their definitions in 64 bits.
Tolerances: H = half a step of the output's type (torch.finfo(t).eps / 2, relative), U = 2^-24 (fp32's); what a kernel does in fp32 between its
64-bit statistics and its one rounding is counted in U at each test."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _half(t):
    return torch.finfo(t).eps / 2


def _tiny(t):   # below the smallest normal number the step no longer shrinks: fp16 2^-25, the other types nothing that counts
    return 2.0 ** -25 if t == torch.float16 else 1e-37


def _rand(shape, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.float64) * scale + shift


def _maps(B, C, hws, dtype, seed, scale=1.0, shift=0.0):
    return [_rand((B, h, w, C), seed + i, scale, shift).to(dtype).to(DEV).permute(0, 3, 1, 2) for i, (h, w) in enumerate(hws)]


def _ref(xs, G, w, b, act, eps, dys):
    """definition in fp64 on the CPU's own arithmetic (on the GPU): per map z, y, dx and the magnitudes its error bound hangs on; dw, db"""
    out, dw, db, mw, mb = [], 0.0, 0.0, 0.0, 0.0
    for x, dy in zip(xs, dys):
        B, C, H, W = x.shape
        v = x.detach().double().reshape(B, G, -1)
        mu = v.mean(2, keepdim=True)
        r = 1 / ((v - mu).square().mean(2, keepdim=True) + eps).sqrt()
        xh = ((v - mu) * r).reshape(B, C, H, W)
        ga = (w.detach().double() if w is not None else torch.ones(C, device=DEV, dtype=torch.float64)).view(1, C, 1, 1)
        be = (b.detach().double() if b is not None else torch.zeros(C, device=DEV, dtype=torch.float64)).view(1, C, 1, 1)
        z = xh * ga + be
        s = torch.sigmoid(z)
        y, d1 = {"none": (z, torch.ones_like(z)), "relu": (z.clamp(min=0), (z > 0).double()), "silu": (z * s, s * (1 + z * (1 - s)))}[act]
        g = dy.double() * d1
        grp = lambda t: t.reshape(B, G, -1).mean(2, keepdim=True).expand(B, G, C // G).reshape(B, C, 1, 1)  # noqa: E731
        rc = r.expand(B, G, C // G).reshape(B, C, 1, 1)
        dx = rc * (ga * g - grp(ga * g) - xh * grp(ga * g * xh))
        K = 16 + 4 * z.abs() if act == "silu" else torch.full_like(z, 8.0)
        # per element K U |gamma dy|; the means carry fp32 sums of up to a few hundred terms per thread and workgroup: 256 U of the terms' magnitudes
        mag = rc * (K * (ga * dy.double()).abs() * 1.1 + 256 * (grp((ga * g).abs()) + xh.abs() * grp((ga * g * xh).abs())))
        # the variance is sum x^2 / n - mean^2 in fp64: partial sums rounded to 2^-53 of mean^2 + var leave it off by some 2^-52 (mean^2 + var), so that
        # 1 / deviation, and with it xh gamma, is off by up to 2^-52 (mean^2 / var + 1) of itself; where beta cancels xh gamma that is not relative to z
        far = grp(v.reshape(B, C, H, W) ** 2) * rc ** 2
        out.append((z, y, dx, mag, K, 2.0 ** -52 * far * (xh * ga).abs() * (2 if act == "silu" else 1)))
        dw, db = dw + (g * xh).sum((0, 2, 3)), db + g.sum((0, 2, 3))
        mw = mw + ((256 + K) * (dy.double() * 1.1 * xh).abs()).sum((0, 2, 3))
        mb = mb + ((256 + K) * (dy.double() * 1.1).abs()).sum((0, 2, 3))
    return out, dw, db, mw, mb


def _check(xs, G, w, b, act, eps, dys, ys, dxs, dw, db):
    out, rw, rb, mw, mb = _ref(xs, G, w, b, act, eps, dys)
    T = xs[0].dtype
    for i, (x, y, (z, yr, dxr, mag, K, stat)) in enumerate(zip(xs, ys, out)):
        if not x.numel():
            continue
        assert y.dtype == T and y.shape == x.shape and y.is_contiguous(memory_format=torch.channels_last)
        err = (y.double() - yr).abs() - (_half(T) * yr.abs() + U * K * z.abs() + stat + _tiny(T))
        assert float(err.max()) <= 0, ("y", i, float(err.max()))
        if dxs is not None:
            assert dxs[i].dtype == T and dxs[i].is_contiguous(memory_format=torch.channels_last)
            err = (dxs[i].double() - dxr).abs() - (_half(T) * dxr.abs() * (1 + 2.0 ** -8) + U * mag + _tiny(T))
            assert float(err.max()) <= 0, ("dx", i, float(err.max()))
    for got, ref, m, p in ((dw, rw, mw, w), (db, rb, mb, b)):
        if got is not None:
            assert got.dtype == p.dtype and got.shape == p.shape
            err = (got.double() - ref).abs() - (_half(p.dtype) * ref.abs() * (1 + 2.0 ** -8) + U * m + _tiny(p.dtype))
            assert float(err.max()) <= 0, ("param", float(err.max()))


def _run(xs, G, w, b, act, eps, dys):
    from lgd_amd import ops
    xs = [x.detach().requires_grad_(True) for x in xs]
    ys = ops.group_norm_act(xs, G, w, b, act=act, eps=eps)
    leaves = xs + [p for p in (w, b) if p is not None]
    got = torch.autograd.grad(ys, leaves, dys)
    rest = list(got[len(xs):])
    return [y.detach() for y in ys], list(got[:len(xs)]), rest.pop(0) if w is not None else None, rest.pop(0) if b is not None else None


def _params(C, dtype, seed):
    return tuple((_rand((C,), seed + k, 0.3, 1.0 - k)).to(dtype).to(DEV).requires_grad_(True) for k in (0, 1))


GN_SHAPES = [
    (2, 64, 8, [(13, 21), (7, 11), (1, 1)]),         # several maps, one of them a single pixel
    (1, 7, 7, [(1, 1), (1, 2), (5, 3)]),             # groups of one channel: with one pixel the variance is 0
    (3, 33, 3, [(9, 7)]),                            # odd channels: vectors wrap round the row's end, samples start unaligned
    (2, 330, 11, [(11, 5), (6, 3)]),                 # groups of 30: no multiple of a vector
    (1, 1, 1, [(37, 29)]),                           # one channel
    (2, 6, 2, [(64, 65)]),                           # few channels, many pixels
    (2, 2056, 8, [(3, 5)]),                          # 257 (514) vectors a row: column blocks
    (1, 1025, 5, [(4, 3)]),                          # odd and wide: column blocks over wrapped rows
    (2, 1026, 1026, [(2, 3)]),                       # as many groups as channels, over column blocks
    (2, 2600, 8, [(9, 11)]),                         # column blocks that cut groups (fp32) or hold them whole
    (1, 2048, 32, [(23, 19)]), (2, 4096, 64, [(21, 22)]),   # column blocks of whole groups (fp32; all types)
    (3, 517, 11, [(20, 21)]),                        # an odd row over two column blocks: every block has all channels
    (2, 1280, 32, [(30, 31)]), (2, 660, 4, [(37, 31)]),   # 160 and 165 vectors a row: 320 and 192 threads
    (1, 256, 32, [(40, 67)]),                        # more than one chunk a sample
    (5, 96, 1, [(17, 19), (2, 2)]),                  # one group
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape", GN_SHAPES, ids=lambda s: "%dx%dg%d" % s[:3])
def test_group_norm_act(shape, act, dtype):
    B, C, G, hws = shape
    T = TYPES[dtype]
    xs, dys = _maps(B, C, hws, T, 100, 1.3, 0.4), _maps(B, C, hws, T, 200)
    w, b = _params(C, T, 300)
    ys, dxs, dw, db = _run(xs, G, w, b, act, 1e-5, dys)
    _check(xs, G, w, b, act, 1e-5, dys, ys, dxs, dw, db)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1040, 520, [(80, 81)]), (1, 96, 48, [(150, 203)]), (2, 1040, 520, [(9, 11), (120, 61)]), (1, 1025, 205, [(67, 66)])], ids=str)
def test_group_norm_act_many_groups(shape, dtype):
    """more groups and chunks than the apply kernels reduce themselves: the records go through kernels of their own; parameters frozen, too"""
    B, C, G, hws = shape
    T = TYPES[dtype]
    xs, dys = _maps(B, C, hws, T, 400, 0.7, -0.3), _maps(B, C, hws, T, 500)
    w, b = _params(C, torch.float32, 600)
    ys, dxs, dw, db = _run(xs, G, w, b, "silu", 1e-5, dys)
    _check(xs, G, w, b, "silu", 1e-5, dys, ys, dxs, dw, db)
    yf, df, _, _ = _run(xs, G, None, None, "relu", 1e-5, dys)
    _check(xs, G, None, None, "relu", 1e-5, dys, yf, df, None, None)
    from lgd_amd import ops
    gw, gb = torch.autograd.grad(ops.group_norm_act(xs, G, w, b, act="silu"), [w, b], dys)   # maps without gradients
    assert torch.equal(gw, dw) and torch.equal(gb, db)


@pytest.mark.parametrize("seed", range(60))
def test_group_norm_act_over_the_range(seed):
    """drawn shapes: batches, groups of 1 to 325 channels, one to sixteen maps of any sides, every type, parameters of another type"""
    import random
    r = random.Random(seed)
    G, B, L = r.choice([1, 2, 3, 5, 7, 8, 11, 16, 32, 33, 64]), r.choice([1, 1, 2, 3, 9]), r.choice([1, 1, 2, 3, 5, 16])
    C = G * r.choice([1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 17, 20, 24, 31, 40, 64, 80, 325])
    side = max(1, int((2e6 / (B * C * L)) ** 0.5))
    hws = [(max(1, int(side * r.uniform(0.2, 2))), max(1, int(side * r.random()))) for _ in range(L)]
    dtype, act, ptype = r.choice(list(TYPES)), r.choice(["none", "relu", "silu"]), r.choice(list(TYPES))
    T = TYPES[dtype]
    xs, dys = _maps(B, C, hws, T, 1000 * seed, r.choice([0.1, 1.0, 3.0]), r.choice([0.0, 0.5, -20.0])), _maps(B, C, hws, T, 1000 * seed + 500)
    w, b = _params(C, TYPES[ptype], 7 * seed)
    ys, dxs, dw, db = _run(xs, G, w, b, act, 1e-5, dys)
    _check(xs, G, w, b, act, 1e-5, dys, ys, dxs, dw, db)


@pytest.mark.parametrize("weight,bias,ptype", [(True, False, "fp32"), (False, True, "bf16"), (False, False, "fp32"), (True, True, "fp16"), (True, True, "fp32")])
def test_group_norm_act_parameters(weight, bias, ptype):
    """either parameter may be missing, and theirs may be another type than the maps'"""
    hws = [(12, 9), (5, 5)]
    xs, dys = _maps(2, 40, hws, torch.bfloat16, 1, 2.0, -1.0), _maps(2, 40, hws, torch.bfloat16, 2)
    w, b = _params(40, TYPES[ptype], 3)
    w, b = w if weight else None, b if bias else None
    ys, dxs, dw, db = _run(xs, 5, w, b, "silu", 1e-3, dys)
    _check(xs, 5, w, b, "silu", 1e-3, dys, ys, dxs, dw, db)


def test_group_norm_act_far_mean_and_constant_groups():
    """mean / spread = 4000 in fp32 (sums of squares lose 24 of their bits there), and groups that are one value: z = beta exactly"""
    x = _maps(2, 16, [(31, 17)], torch.float32, 5, 1.0, 4000.0)
    dy = _maps(2, 16, [(31, 17)], torch.float32, 6)
    w, b = _params(16, torch.float32, 7)
    ys, dxs, dw, db = _run(x, 4, w, b, "relu", 1e-5, dy)
    _check(x, 4, w, b, "relu", 1e-5, dy, ys, dxs, dw, db)
    from lgd_amd import ops
    c = torch.full((1, 8, 9, 7), 1234.5, device=DEV).to(memory_format=torch.channels_last)
    y, = ops.group_norm_act([c], 2, w.detach()[:8], b.detach()[:8], act="none")
    assert torch.equal(y, b.detach()[:8].view(1, 8, 1, 1).expand_as(y))


def test_group_norm_act_memory_orders():
    """maps in NCHW order, slices of larger maps, an expanded output gradient, non-contiguous parameters: same values as the dense ones"""
    from lgd_amd import ops
    big = _maps(4, 24, [(20, 15)], torch.float32, 11)[0]
    w, b = (torch.cat([p.detach(), p.detach()]).view(2, 24).t().contiguous()[:, 0] for p in _params(24, torch.float32, 12))
    views = [big, big.contiguous(), big[:, :, 2:9, 1:8], big[1::2], big[:, :, ::2].transpose(2, 3)]
    for v in views:
        x = v.detach().requires_grad_(True)
        y, = ops.group_norm_act([x], 6, w, b, act="silu")
        dx, = torch.autograd.grad(y, x, torch.ones(1, device=DEV).expand(y.shape))
        dense = torch.empty(v.shape, device=DEV).to(memory_format=torch.channels_last).copy_(v).requires_grad_(True)
        yd, = ops.group_norm_act([dense], 6, w.contiguous(), b.contiguous(), act="silu")
        dd, = torch.autograd.grad(yd, dense, torch.ones_like(yd))
        assert torch.equal(y, yd) and torch.equal(dx, dd)


def test_group_norm_act_empty_and_partial_gradients():
    from lgd_amd import ops
    w, b = _params(8, torch.float32, 1)
    full, none = _maps(2, 8, [(4, 4)], torch.float32, 2)[0].requires_grad_(True), torch.zeros(2, 8, 0, 5, device=DEV).requires_grad_(True)
    ys = ops.group_norm_act([none, full], 2, w, b)
    assert ys[0].shape == none.shape
    dn, df, dw, db = torch.autograd.grad(ys[0].sum() + ys[1].sum(), [none, full, w, b])
    ys1 = ops.group_norm_act([full], 2, w, b)
    f1, w1, b1 = torch.autograd.grad(ys1[0].sum(), [full, w, b])
    assert dn.shape == none.shape and torch.equal(df, f1) and torch.equal(dw, w1) and torch.equal(db, b1)
    e = torch.zeros(0, 8, 3, 3, device=DEV).requires_grad_(True)
    y, = ops.group_norm_act([e], 2, w, b)
    de, dw, db = torch.autograd.grad(y.sum(), [e, w, b])
    assert de.shape == e.shape and not dw.any() and not db.any()
    # only some inputs want gradients; one output is not used
    a = _maps(2, 8, [(4, 4), (3, 5)], torch.float32, 3)
    y = ops.group_norm_act(a, 2, w, None)
    gw, = torch.autograd.grad(y[0].sum(), [w])
    yr = F.relu(F.group_norm(a[0].double(), 2)) * 0
    ref, = torch.autograd.grad(F.relu(F.group_norm(a[0].double(), 2, wd := w.detach().double().requires_grad_(True))).sum(), [wd])
    assert yr.shape == y[0].shape and float((gw.double() - ref).abs().max()) < 1e-4
    with torch.no_grad():
        assert torch.equal(ops.group_norm_act(a, 2, w, None)[1], y[1])
    x = a[0].detach().requires_grad_(True)
    first, = torch.autograd.grad(ops.group_norm_act([x], 2, w, None, act="silu")[0].sum(), [x])
    g, = torch.autograd.grad(ops.group_norm_act([x], 2, w, None, act="silu")[0].sum(), [x], create_graph=True)
    assert torch.equal(g, first)
    with pytest.raises(RuntimeError, match="second derivative"):   # an error, not a wrong value
        (g * x).sum().backward()


def test_group_norm_act_saved_tensors_kept_elsewhere():
    """what the backward needs, kept on the host in another memory order; the same map twice in one call; a second backward of a kept graph"""
    from lgd_amd import ops
    x, = _maps(2, 24, [(9, 11)], torch.float32, 31)
    dys = _maps(2, 24, [(9, 11), (9, 11)], torch.float32, 32)
    w, b = _params(24, torch.float32, 33)
    x.requires_grad_(True)
    ys = ops.group_norm_act([x, x], 6, w, b, act="silu")
    want = torch.autograd.grad(ys, [x, w, b], dys, retain_graph=True)
    assert all(torch.equal(g, a) for g, a in zip(torch.autograd.grad(ys, [x, w, b], dys), want))
    with pytest.raises(RuntimeError, match="freed"):
        torch.autograd.grad(ys, [x], dys)
    one, two = (torch.autograd.grad(ops.group_norm_act([x], 6, w, b, act="silu"), [x], [dy])[0] for dy in dys)
    assert torch.equal(one + two, want[0])
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        ys = ops.group_norm_act([x, x], 6, w, b, act="silu")
    assert all(torch.equal(g, a) for g, a in zip(torch.autograd.grad(ys, [x, w, b], dys), want))


def test_group_norm_act_captured_beside_an_eager_graph_of_the_same_leaves():
    """refused before the engine makes the eager graph's stream wait inside the capture"""
    from lgd_amd import ops
    x, dy = _maps(1, 16, [(5, 5)], torch.float32, 41)[0].requires_grad_(True), _maps(1, 16, [(5, 5)], torch.float32, 42)[0]
    w, b = _params(16, torch.float32, 43)
    kept = ops.group_norm_act([x], 4, w, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="held by a graph"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(ops.group_norm_act([x], 4, w, b), [x, w, b], [dy])
    torch.cuda.synchronize()
    want = torch.autograd.grad(kept, [x, w, b], [dy])
    assert all(torch.isfinite(g).all() for g in want)


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_group_norm_act_not_finite_stays_in_its_group(act):
    """inf and NaN spoil their own (sample, group) as in torch, and nothing else"""
    from lgd_amd import ops
    x = _maps(3, 12, [(6, 7)], torch.float32, 4)[0].clone(memory_format=torch.channels_last)
    x[0, 1, 2, 3], x[2, 8, 0, 0] = float("inf"), float("nan")
    y, = ops.group_norm_act([x], 4, act=act)
    ref = F.group_norm(x, 4)
    ref = {"none": lambda t: t, "relu": torch.relu, "silu": F.silu}[act](ref)
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and int(torch.isnan(y).sum()) == 2 * 3 * 42
    ok = ~torch.isnan(ref)
    assert torch.allclose(y[ok], ref[ok], rtol=1e-5, atol=1e-5)


def test_group_norm_act_gradient_against_differences():
    """directional derivatives of a 64-bit sum over the fp32 outputs: step 2^-6, third-derivative error below 1e-3 of the value at these sizes"""
    from lgd_amd import ops
    x, d = _maps(2, 12, [(9, 8)], torch.float32, 21)[0], _maps(2, 12, [(9, 8)], torch.float32, 22)[0]
    w, b = _params(12, torch.float32, 23)
    dw, db = (_rand((12,), 24 + k).float().to(DEV) for k in (0, 1))
    q = _maps(2, 12, [(9, 8)], torch.float32, 26)[0]
    f = lambda x, w, b: (ops.group_norm_act([x], 3, w, b, act="silu")[0].double() * q).sum()  # noqa: E731
    xl = x.detach().requires_grad_(True)
    gx, gw, gb = torch.autograd.grad(f(xl, w, b), [xl, w, b])
    h = 2.0 ** -6
    w, b = w.detach(), b.detach()
    for got, lo, hi in ((float((gx.double() * d).sum()), f(x - h * d, w, b), f(x + h * d, w, b)), (float((gw.double() * dw).sum()), f(x, w - h * dw, b), f(x, w + h * dw, b)),
                        (float((gb.double() * db).sum()), f(x, w, b - h * db), f(x, w, b + h * db))):
        num = float(hi - lo) / (2 * h)
        assert abs(num - got) <= 2e-3 * max(abs(got), 1.0), (num, got)


def test_group_norm_act_beyond_32_bits():
    """2.5 * 2^30 elements in all: the last sample equals what it is alone"""
    from lgd_amd import ops
    H = W = 1024
    C, B = 512, 5
    x = torch.empty(B, H, W, C, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(5)
    for i in range(B):
        x[i].copy_(torch.randn(H, W, C, device=DEV, generator=g, dtype=torch.float32) + 0.5 * i)
    x = x.permute(0, 3, 1, 2)
    w, b = (p.detach() for p in _params(C, torch.float32, 6))
    y, = ops.group_norm_act([x], 32, w, b, act="relu")
    one, = ops.group_norm_act([x[B - 1:]], 32, w, b, act="relu")
    # statistics differ in the order of 64-bit sums only: at most a rounding tie of bf16 falls the other way
    diff = (y[B - 1:].float() - one.float()).abs()
    assert float(diff.max()) <= 2.0 ** -7 * float(one.float().abs().max()) and int((diff > 0).sum()) < 64
    xl = x.detach().requires_grad_(True)
    dx, = torch.autograd.grad(ops.group_norm_act([xl], 32, w, b, act="relu"), [xl], [y])
    ol = x[B - 1:].detach().requires_grad_(True)
    do, = torch.autograd.grad(ops.group_norm_act([ol], 32, w, b, act="relu"), [ol], [y[B - 1:]])
    diff = (dx[B - 1:].float() - do.float()).abs()
    # the means differ by fp32 sums over other chunks (256 U of about 1): bf16 values next to a tie may fall the other way, by one step
    assert float(diff.max()) <= 2.0 ** -7 * float(do.float().abs().max())


def test_group_norm_act_same_bits_streams_and_graph():
    """the same call twice, two calls at once on two streams, and a captured forward + backward replayed over changing inputs: the eager bits"""
    from lgd_amd import ops
    hws = [(33, 40), (17, 20)]
    w, b = _params(48, torch.float32, 1)
    ins = [(_maps(2, 48, hws, torch.bfloat16, 10 * k), _maps(2, 48, hws, torch.bfloat16, 10 * k + 5)) for k in range(1, 5)]

    def eager(k):
        return _run(ins[k][0], 6, w, b, "silu", 1e-5, ins[k][1])

    def same(p, q):
        flat = lambda r: [*r[0], *r[1], r[2], r[3]]  # noqa: E731
        assert all(torch.equal(u, v) for u, v in zip(flat(p), flat(q)))
    want = [eager(k) for k in range(4)]
    for k in range(4):
        same(eager(k), want[k])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        r1 = [eager(0) for _ in range(4)]
    with torch.cuda.stream(s2):
        r2 = [eager(1) for _ in range(4)]
    torch.cuda.synchronize()
    for r in r1:
        same(r, want[0])
    for r in r2:
        same(r, want[1])
    xs = [torch.empty_like(x) for x in ins[0][0]]
    dys = [torch.empty_like(x) for x in ins[0][1]]
    w2, b2 = (p.detach().clone().requires_grad_(True) for p in (w, b))   # leaves no eager graph holds
    load = lambda k: [t.copy_(v) for t, v in zip(xs + dys, ins[k][0] + ins[k][1])]  # noqa: E731
    load(0)
    s1.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        _run(xs, 6, w2, b2, "silu", 1e-5, dys)
    torch.cuda.current_stream().wait_stream(s1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(xs, 6, w2, b2, "silu", 1e-5, dys)
    for k in (1, 2, 3, 0, 2):
        load(k)
        graph.replay()
        torch.cuda.synchronize()
        same(out, want[k])
        same(eager(3), want[3])


# ------------------------------------------------------------------------------------------- norms and clipping
LISTS = {
    "one": [1],
    "few": [5, 64, 1, 4097, 16384, 33000],
    "empty": [0, 3, 0, 0, 8195, 0],
    "many": [(i * 37) % 911 for i in range(160)],          # exactly what fits the kernel arguments (empty ones do not count)
    "more": [1 + (i * 53) % 1201 for i in range(401)],     # a table in the workspace, written by three launches
    "long": [3_000_017, 8, 5_000_000],                     # every workgroup walks several chunks
}


def _tensors(sizes, kind, seed, bucket):
    """gradients of one type or all three in turn; bucket: views at running offsets of one buffer per type, at whatever alignment"""
    types = list(TYPES.values()) if kind == "mixed" else [TYPES[kind]]
    out, bufs, offs = [], {t: torch.zeros(sum(sizes) + 8, dtype=t, device=DEV) for t in types}, {t: 1 for t in types}
    for i, n in enumerate(sizes):
        t = types[i % len(types)]
        v = _rand((n,), seed + i).to(t).to(DEV)
        if bucket:
            o, offs[t] = offs[t], offs[t] + n
            bufs[t][o:o + n] = v
            v = bufs[t][o:o + n]
        out.append(v)
    return out, bufs


def _norm64(ts, p):
    return torch.linalg.vector_norm(torch.cat([t.double() for t in ts] + [torch.zeros(1, dtype=torch.float64, device=DEV)]), p)


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("kind,bucket", [("fp32", False), ("bf16", True), ("fp16", True), ("mixed", False), ("mixed", True)])
@pytest.mark.parametrize("sizes", list(LISTS))
def test_grad_norm_and_clip(sizes, kind, bucket, p):
    from lgd_amd import optim
    ts, bufs = _tensors(LISTS[sizes], kind, 7, bucket)
    ref = _norm64(ts, p)
    got = optim.grad_norm(ts, p)
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - float(ref)) <= 2 * U * float(ref)        # 64-bit sums, one rounding
    assert torch.equal(got, optim.grad_norm(ts, p))
    before, edges = [t.clone() for t in ts], {t: b.clone() for t, b in bufs.items()}
    params = [torch.nn.Parameter(torch.empty_like(t)) for t in ts]
    for q, t in zip(params, ts):
        q.grad = t
    limit = 0.37 * float(ref)
    total = optim.clip_grad_norm_(params, limit, p)
    assert torch.equal(total, got)
    c = limit / (float(ref) + 1e-6)
    for t, o in zip(ts, before):
        want = o.double() * min(1.0, c)
        # the factor carries the norm's rounding and its own (3 U), the product one rounding to fp32 and one to the type
        assert float(((t.double() - want).abs() - (_half(t.dtype) * (1 + 2.0 ** -8) + 6 * U) * want.abs() - _tiny(t.dtype)).max() if t.numel() else 0) <= 0
    if bucket:   # nothing outside the views was touched
        for t, b in bufs.items():
            n = sum(x.numel() for x in ts if x.dtype == t)
            assert b[0] == edges[t][0] and torch.equal(b[1 + n:], edges[t][1 + n:])
    # a threshold above the norm: not a bit changes
    after, version = [t.clone() for t in ts], [t._version for t in ts]
    optim.clip_grad_norm_(params, 2 * float(ref) + 1, p)
    assert all(torch.equal(t, a) for t, a in zip(ts, after)) and all(t._version > v for t, v in zip(ts, version))


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_norm_of_values_at_the_ends_of_the_range(p):
    from lgd_amd import optim
    for v in (3e38, 1e-38, 1e-44, 0.0):
        t = torch.full((1000,), v, device=DEV)
        ref = float(_norm64([t], p))
        got = float(optim.grad_norm([t], p))
        assert got == math.inf if ref > 3.4028235e38 else abs(got - ref) <= 2 * U * ref + 2.0 ** -150, (v, got, ref)
    t = torch.ones(70001, device=DEV)
    t[65537] = math.inf
    assert float(optim.grad_norm([t], p)) == math.inf
    t[3] = math.nan
    assert math.isnan(float(optim.grad_norm([t], p)))
    for bad, limit in ((math.nan, 1.0), (math.inf, 1.0), (1.0, 0.0), (1.0, math.inf)):   # torch's arithmetic on what is not finite, and at the limits
        a, b = (torch.nn.Parameter(torch.zeros(5000, device=DEV)) for _ in range(2))
        g = torch.linspace(-1, 1, 5000, device=DEV)
        g[17] = bad
        a.grad, b.grad = g.clone(), g.clone()
        optim.clip_grad_norm_([a], limit, p)
        torch.nn.utils.clip_grad_norm_([b], limit, p, foreach=False)
        assert torch.allclose(a.grad, b.grad, rtol=1e-5, atol=0, equal_nan=True)


def test_clip_memory_orders():
    """channels-last filters are scaled where they lie; strided views through a copy; what lies between stays"""
    from lgd_amd import optim
    base = torch.randn(64, 40, device=DEV)
    keep = base.clone()
    gs = [torch.randn(16, 8, 3, 3, device=DEV).to(memory_format=torch.channels_last), base[:, 3], base[::2, 10:20], torch.randn(7, 5, device=DEV).t(),
          torch.randn((), device=DEV)]
    ps = [torch.nn.Parameter(torch.empty_like(g)) for g in gs]
    for q, g in zip(ps, gs):
        q.grad = g
    gs = [q.grad for q in ps]
    ref = [g.double().clone() for g in gs]
    total = optim.clip_grad_norm_(ps, 0.5)
    norm = math.sqrt(sum(float(r.square().sum()) for r in ref))
    assert abs(float(total) - norm) <= 2 * U * norm
    for g, r in zip(gs, ref):
        assert float(((g.double() - r * (0.5 / (norm + 1e-6))).abs() - 8 * U * r.abs()).max()) <= 0
    mask = torch.ones_like(base, dtype=torch.bool)
    mask[:, 3] = False
    mask[::2, 10:20] = False
    assert torch.equal(base[mask], keep[mask])


def test_norm_beyond_32_bits():
    from lgd_amd import optim
    n = (1 << 31) + 4099
    t = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    t[-1], t[1 << 31] = 3.0, -2.0
    assert float(optim.grad_norm([t])) == pytest.approx(math.sqrt(n - 2 + 9 + 4), rel=2 * U)
    assert float(optim.grad_norm([t], 1.0)) == pytest.approx(n - 2 + 5, rel=2 * U)
    assert float(optim.grad_norm([t], math.inf)) == 3.0
    p = torch.nn.Parameter(torch.empty(0, device=DEV))
    q = torch.nn.Parameter(t)
    q.grad = t
    optim.clip_grad_norm_([p, q], 1.5, math.inf)
    assert float(t[0]) == 0.5 and float(t[-1]) == 1.5 and float(t[1 << 31]) == -1.0 and float(t[(1 << 31) - 1]) == 0.5


def test_norm_streams_and_graph():
    """two calls at once on two streams; captured clipping (short and long lists) replayed over changing gradients, eager work in between"""
    from lgd_amd import optim
    sets = [_tensors(LISTS["more"], "mixed", 1000 * k, True)[0] for k in range(3)]
    want = [optim.grad_norm(s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s, k in zip(streams, (0, 1)):
            with torch.cuda.stream(s):
                got.append((k, optim.grad_norm(sets[k])))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[k]) for k, v in got)
    for name in ("few", "more"):
        sets = [_tensors(LISTS[name], "mixed", 1000 * k, False)[0] for k in range(3)]
        ps = [torch.nn.Parameter(torch.empty_like(t)) for t in sets[0]]
        for p, t in zip(ps, sets[0]):
            p.grad = t.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            total = optim.clip_grad_norm_(ps, 1.0)
        for k in (0, 1, 2, 1):
            for p, t in zip(ps, sets[k]):
                p.grad.copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            qs = [torch.nn.Parameter(torch.empty_like(t)) for t in sets[k]]
            for q, t in zip(qs, sets[k]):
                q.grad = t.clone()
            assert torch.equal(optim.clip_grad_norm_(qs, 1.0), total)
            assert all(torch.equal(p.grad, q.grad) for p, q in zip(ps, qs))


# ------------------------------------------------------------------------------------------- the step
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_fused_step_clips_by_norm(p):
    """FusedClipSGD(clip_norm=) against torch: clip_grad_norm_ of each optimizer's parameters, then its step(); three steps, the second without one
    parameter's gradient, the third without any in the second optimizer; unaligned gradient views"""
    from lgd_amd import optim
    sizes = [(1,), (3,), (255,), (64, 3, 7, 7), (4097,), (256, 256, 3, 3), (720,), (5,), (0,)]

    def make():
        g = torch.Generator().manual_seed(4)
        ps = [torch.nn.Parameter(torch.randn(*s, generator=g).to(DEV)) for s in sizes]
        return ps, [torch.optim.SGD(ps[:5], 0.02, momentum=0.9, weight_decay=1e-4), torch.optim.SGD(ps[5:], 0.05, momentum=0.8, weight_decay=1e-3)]
    (pa, oa), (pb, ob) = make(), make()
    fused = optim.FusedClipSGD(ob, clip_norm=2.5, norm_type=p)
    bucket = torch.zeros(300, device=DEV)
    for step in range(3):
        for i, (a, b) in enumerate(zip(pa, pb)):
            if (step == 1 and i == 1) or (step == 2 and i >= 5):
                a.grad = b.grad = None
                continue
            g = _rand(tuple(a.shape), 50 * step + i, 3.0 if i % 2 else 0.3).float().to(DEV)
            a.grad, b.grad = g, g.clone()
            if i == 2:
                bucket[1:256] = g
                b.grad = bucket[1:256]
        norms = [torch.nn.utils.clip_grad_norm_([q for g in o.param_groups for q in g["params"]], 2.5, p) for o in oa]
        for o in oa:
            o.step()
        fused.step()
        assert fused.total_norms.shape == (2,)
        for k, n in enumerate(norms):
            assert abs(float(fused.total_norms[k]) - float(n)) <= 1e-5 * float(n)    # torch's norm is a sum of fp32 norms
        for i, (a, b) in enumerate(zip(pa, pb)):
            assert torch.allclose(a, b, rtol=2e-5, atol=2e-6), (step, i)
            assert (a.grad is None) == (b.grad is None)
            if a.grad is not None:
                assert torch.allclose(a.grad, b.grad, rtol=2e-5, atol=1e-9), (step, i)
                o = 0 if i < 5 else 1
                assert torch.allclose(oa[o].state[a]["momentum_buffer"], ob[o].state[b]["momentum_buffer"], rtol=2e-5, atol=2e-6)
    # far above the norm: exactly the step without clipping, gradients untouched; and no gradients at all
    (pc, oc), (pd, od) = make(), make()
    free, high = optim.FusedClipSGD(oc), optim.FusedClipSGD(od, clip_norm=1e9, norm_type=p)
    for i, (c, d) in enumerate(zip(pc, pd)):
        c.grad = _rand(tuple(c.shape), 900 + i).float().to(DEV)
        d.grad = c.grad.clone()
    free.step()
    high.step()
    assert all(torch.equal(c, d) and torch.equal(c.grad, d.grad) for c, d in zip(pc, pd)) and free.total_norms is None
    high.zero_grad()
    high.step()
    assert torch.equal(high.total_norms, torch.zeros(2, device=DEV)) and all(torch.equal(c, d) for c, d in zip(pc, pd))


@pytest.mark.parametrize("count", [72, 73, 300])
def test_fused_step_by_norm_many_tensors(count):
    """tables that travel in the kernels' arguments and tables in device memory; three optimizers, the last without a gradient; the set of parameters that
    have a gradient changes between the steps, and a state dict is loaded"""
    from lgd_amd import optim
    sizes = [1 + (i * 397) % 5003 for i in range(count)]

    def make():
        g = torch.Generator().manual_seed(14)
        ps = [torch.nn.Parameter(torch.randn(n, generator=g).to(DEV)) for n in sizes]
        extra = torch.nn.Parameter(torch.ones(3, device=DEV))
        return ps, [torch.optim.SGD(ps[:count // 3], 0.02, momentum=0.9, weight_decay=1e-4), torch.optim.SGD(ps[count // 3:], 0.05, momentum=0.8),
                    torch.optim.SGD([extra], 0.1)]
    (pa, oa), (pb, ob) = make(), make()
    fused = optim.FusedClipSGD(ob, clip_norm=5.0)
    for step in range(4):
        for i, (a, b) in enumerate(zip(pa, pb)):
            a.grad = b.grad = None
            if step != 1 or i % 2:
                a.grad = _rand((sizes[i],), 70 * step + i).float().to(DEV)
                b.grad = a.grad.clone()
        if step == 3:
            for o in ob:
                o.load_state_dict(o.state_dict())
        want = [float(torch.nn.utils.clip_grad_norm_([q for g in o.param_groups for q in g["params"]], 5.0)) for o in oa]
        for o in oa:
            o.step()
        version = pb[1]._version
        fused.step()
        assert pb[1]._version > version
        assert all(abs(float(x) - w) <= 1e-5 * w for x, w in zip(fused.total_norms, want))
        for i, (a, b) in enumerate(zip(pa, pb)):
            assert torch.allclose(a, b, rtol=2e-5, atol=2e-6), (step, i)
            assert a.grad is None or torch.allclose(a.grad, b.grad, rtol=2e-5, atol=1e-9)


def test_fused_step_refusals():
    """gradients that share memory (by norm), strided gradients and strided parameters; nothing has been changed when the step refuses"""
    from lgd_amd import hip, optim
    p, q = (torch.nn.Parameter(torch.ones(8, 4, device=DEV)) for _ in range(2))
    buf = torch.ones(48, device=DEV)
    f = optim.FusedClipSGD([torch.optim.SGD([p, q], 0.1)], clip_norm=1.0)
    p.grad, q.grad = buf[:32].view(8, 4), buf[16:].view(8, 4)
    with pytest.raises(hip.LgdHipError, match="share memory"):
        f.step()
    p.grad, q.grad = torch.ones(8, 4, device=DEV), torch.ones(4, 8, device=DEV).t()
    with pytest.raises(hip.LgdHipError, match="contiguous fp32 gradients"):
        f.step()
    assert torch.equal(p, torch.ones_like(p)) and torch.equal(q, torch.ones_like(q)) and torch.equal(buf, torch.ones_like(buf))
    s = torch.nn.Parameter(torch.ones(4, 8, device=DEV).t())
    f = optim.FusedClipSGD([torch.optim.SGD([s], 0.1)], clip_norm=1.0)
    s.grad = torch.ones(8, 4, device=DEV)
    with pytest.raises(hip.LgdHipError, match="contiguous"):
        f.step()


def test_fused_step_by_norm_is_not_captured():
    from lgd_amd import hip, optim
    p = torch.nn.Parameter(torch.ones(8, device=DEV))
    f = optim.FusedClipSGD([torch.optim.SGD([p], 0.1)], clip_norm=1.0)
    p.grad = torch.ones(8, device=DEV)
    f.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(hip.LgdHipError, match="captured"):
        with torch.cuda.graph(graph):
            f.step()
    torch.cuda.synchronize()
    f.clip_norm = -1.0
    with pytest.raises(hip.LgdHipError, match="negative"):
        f.step()


@pytest.mark.parametrize("limit,clips", [(0.7, False), (0.1, True)])   # the gradients' norm is about 0.6
def test_tower_norms_clip_and_step_together(limit, clips):
    """a two-layer channels-last tower over two maps, three training steps: group_norm_act with its gradients, clipping by the norm of them all
    inside the fused step, against torch's own modules in fp64"""
    from lgd_amd import ops, optim
    C, G, hws = 32, 4, [(14, 18), (7, 9)]
    g = torch.Generator().manual_seed(9)
    init = [torch.randn(C, C, generator=g, dtype=torch.float64) / C ** 0.5, torch.ones(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64)] * 2
    ours = [torch.nn.Parameter(t.float().to(DEV)) for t in init]
    refs = [torch.nn.Parameter(t.float().double().to(DEV)) for t in init]
    oo, ro = torch.optim.SGD(ours, 0.05, momentum=0.9, weight_decay=1e-4), torch.optim.SGD(refs, 0.05, momentum=0.9, weight_decay=1e-4)
    fused = optim.FusedClipSGD([oo], clip_norm=limit)
    for step in range(3):
        xs, ts = _maps(2, C, hws, torch.float32, 30 + step), _maps(2, C, hws, torch.float32, 60 + step)
        h = xs
        for k in (0, 3):
            h = [(m.permute(0, 2, 3, 1) @ ours[k]).permute(0, 3, 1, 2) for m in h]
            h = ops.group_norm_act(h, G, ours[k + 1], ours[k + 2], act="silu")
        loss = sum(((m - t) ** 2).mean() for m, t in zip(h, ts))
        fused.zero_grad()
        loss.backward()
        r = [x.double() for x in xs]
        for k in (0, 3):
            r = [F.silu(F.group_norm((m.permute(0, 2, 3, 1) @ refs[k]).permute(0, 3, 1, 2), G, refs[k + 1], refs[k + 2])) for m in r]
        rloss = sum(((m - t.double()) ** 2).mean() for m, t in zip(r, ts))
        ro.zero_grad()
        rloss.backward()
        for a, b in zip(ours, refs):
            assert float((a.grad.double() - b.grad).norm()) <= 1e-4 * float(b.grad.norm())   # two fp32 products with 32 terms and their weights' drift
        want = optim.grad_norm([a.grad for a in ours])
        total = torch.nn.utils.clip_grad_norm_(refs, limit)
        fused.step()
        ro.step()
        assert abs(float(fused.total_norms[0]) - float(total)) <= 1e-4 * float(total) and (float(total) > limit) == clips
        assert abs(float(fused.total_norms[0]) - float(want)) <= 4 * U * float(want)
        for a, b in zip(ours, refs):
            assert float((a.double() - b).norm()) <= 1e-4 * float(b.norm())


@pytest.mark.parametrize("fused", [True, False])
def test_trainer_clips_the_whole_gradient(fused):
    """SOLVER.CLIP_GRADIENTS.CLIP_TYPE full_model through the trainer, in the fused step and in front of torch's optimizers"""
    import os
    from lgd_amd import config
    from lgd_amd.data import synthetic_batch
    from lgd_amd.distillator import build_model
    from lgd_amd.engine import Trainer
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cfg = config.setup_cfg(os.path.join(root, "configs", "lgd_retinanet_r50.yaml"),
                           ["MODEL.DEVICE", "cuda:0", "SOLVER.CLIP_GRADIENTS.ENABLED", "True", "SOLVER.CLIP_GRADIENTS.CLIP_TYPE", "full_model",
                            "SOLVER.CLIP_GRADIENTS.CLIP_VALUE", "0.05"])
    torch.manual_seed(0)
    tr = Trainer(cfg, build_model(cfg), fused_sgd=fused)
    assert (tr._fused_sgd is not None) == fused
    tr.step(synthetic_batch(2, 256, 320, 5, seed=2), 40000)
    for k, o in enumerate((tr.stu_optimizer, tr.tea_optimizer)):
        grads = [p.grad for g in o.param_groups for p in g["params"] if p.grad is not None]
        assert grads
        after = float(_norm64([g.reshape(-1) for g in grads], 2.0))
        if fused:
            before = float(tr._fused_sgd.total_norms[k])
            assert abs(after - min(before, 0.05)) <= 1e-4 * after
        assert after <= 0.05 * (1 + 1e-5)
