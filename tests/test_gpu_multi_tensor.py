"""GPU: the global norm, clipping by it and the Adam step over lists of tensors, against 64-bit formulas.

Tolerances, u = 2^-24: the norm is summed in double and rounded once, u |s| (2 u allowed for the root).  A clipped entry is
one product with a factor that is off by 2 u, and one rounding to the type (eps / 2).  An Adam moment is three roundings of
terms of the moment's size; the updated parameter is x minus a step of at most `step`, whose factors (m, sqrt(v), quotient,
lr) carry some 12 u between them."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope='module')
def la(gpu_device):
    from bayes_vi_amd import linalg
    return linalg


def tensors(shapes, dtypes, size, seed, dev):
    gen = torch.Generator(device=dev); gen.manual_seed(seed)
    return [(size * torch.randn(*s, generator=gen, device=dev)).to(d) for s, d in zip(shapes, dtypes)]


def norm64(ts):
    return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in ts))


LISTS = [[(1,)], [(7,), (3, 5), (1, 1)], [(4096,), (4097,), (4095,)], [(100, 33)] * 79, [(3,)] * 80, [(5,)] * 81, [(2, 9)] * 200,
         [(1_000_003,), (2,), (513, 1025)], [(0,), (4,), (0, 3)], [(3_000_000, 4)]]


@pytest.mark.parametrize('mix', ['float32', 'bfloat16', 'float16', 'mixed'])
@pytest.mark.parametrize('shapes', LISTS, ids=lambda s: '%d x %s' % (len(s), s[0]))
def test_norm_and_clipping(la, gpu_device, shapes, mix):
    kinds = [torch.float32, torch.bfloat16, torch.float16]
    dtypes = [kinds[k % 3] if mix == 'mixed' else getattr(torch, mix) for k in range(len(shapes))]
    ts = tensors(shapes, dtypes, 0.25, len(shapes), gpu_device)
    keep = [t.clone() for t in ts]
    s = norm64(ts)
    assert abs(float(la.global_norm(ts)) - s) <= 2 * U * s
    for clip in (s * 0.3, s * 3.0, 1e-3):
        out, norm = la.clip_by_global_norm(ts, clip)
        assert abs(float(norm) - s) <= 2 * U * s
        factor = min(1.0, clip / s)
        for o, t in zip(out, keep):
            f = torch.finfo(t.dtype)
            ref = t.double() * factor
            assert o.dtype == t.dtype and o.shape == t.shape
            assert bool(((o.double() - ref).abs() <= (f.eps / 2 + 4 * U) * ref.abs() + f.smallest_normal * f.eps).all())
            if factor == 1.0:
                assert torch.equal(o, t)
        assert all(torch.equal(t, k) for t, k in zip(ts, keep))
        twice, _ = la.clip_by_global_norm(ts, clip)
        assert all(torch.equal(a, b) for a, b in zip(out, twice))
        own = [t.clone() for t in ts]
        res, norm2 = la.clip_by_global_norm(own, clip, inplace=True)
        assert all(r is o for r, o in zip(res, own)) and torch.equal(norm, norm2)
        assert all(torch.equal(a, b) for a, b in zip(out, own))


def test_alignment_and_layout(la, gpu_device):
    base = torch.randn(10_001, device=gpu_device)
    half = torch.randn(10_001, device=gpu_device).half()
    ts = [base[1:5000], base[5003:], half[3:4000], half[4001:4003], base[:9000].view(90, 100).T]
    s = norm64(ts)
    assert abs(float(la.global_norm(ts)) - s) <= 2 * U * s
    out, _ = la.clip_by_global_norm(ts, 0.5 * s)
    for o, t in zip(out, ts):
        f = torch.finfo(t.dtype)
        ref = t.double() * 0.5
        assert bool(((o.double() - ref).abs() <= (f.eps / 2 + 4 * U) * ref.abs() + f.smallest_normal * f.eps).all())
    own = base.clone()
    la.clip_by_global_norm([own[1:77]], 1e-3, inplace=True)           # the neighbours stay as they were
    assert torch.equal(own[:1], base[:1]) and torch.equal(own[77:], base[77:])


def test_special_norms(la, gpu_device):
    one = lambda *v: torch.tensor(v, device=gpu_device)
    out, norm = la.clip_by_global_norm([one(0., 0.), None, one(0.)], 1.0)
    assert float(norm) == 0.0 and out[1] is None and all(bool((o == 0).all()) for o in (out[0], out[2]))
    for bad in (float('inf'), float('nan')):
        out, norm = la.clip_by_global_norm([one(1., bad), one(2.)], 1.0)
        assert not math.isfinite(float(norm)) and all(bool(torch.isnan(o).all()) for o in out)
    # squares that leave float's range at either end
    out, norm = la.clip_by_global_norm([one(3e30, 4e30)], 1.0)
    assert abs(float(norm) / 5e30 - 1) < 4 * U and torch.allclose(out[0], one(.6, .8), rtol=8 * U, atol=0)
    assert abs(float(la.global_norm([one(3e-30, 4e-30)])) / 5e-30 - 1) < 4 * U
    out, norm = la.clip_by_global_norm([one(3., 4.)], 1.0, use_norm=one(10.))
    assert float(norm) == 10.0 and torch.allclose(out[0], one(.3, .4), rtol=4 * U, atol=0)
    out, _ = la.clip_by_global_norm([one(3., 4.)], float('inf'))
    assert torch.equal(out[0], one(3., 4.))


def test_refusals(la, gpu_device):
    t = torch.ones(6, device=gpu_device)
    with pytest.raises(ValueError, match='positive'):
        la.clip_by_global_norm([t], 0.0)
    with pytest.raises(ValueError, match='overlap'):
        la.clip_by_global_norm([t, t], 1.0, inplace=True)
    with pytest.raises(ValueError, match='overlap'):
        la.clip_by_global_norm([t[:4], t[3:]], 1.0, inplace=True)
    with pytest.raises(ValueError, match='contiguous'):
        la.clip_by_global_norm([t[::2]], 1.0, inplace=True)
    with pytest.raises(ValueError, match='use_norm'):
        la.clip_by_global_norm([t], 1.0, use_norm=torch.ones(2, device=gpu_device))
    with pytest.raises(TypeError):
        la.global_norm([t.double()])
    out, norm = la.clip_by_global_norm([t, t], 1.0)              # read twice, written apart
    assert abs(float(norm) - math.sqrt(12)) < 1e-6 and torch.equal(out[0], out[1])


def test_clipping_in_a_graph(la, gpu_device):
    ts = tensors([(300, 50), (7,), (20_000,)], [torch.float32, torch.bfloat16, torch.float32], 1.0, 4, gpu_device)
    la.clip_by_global_norm(ts, 2.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, norm = la.clip_by_global_norm(ts, 2.0)
    for k in range(4):
        for t in ts:
            t.copy_(torch.randn(t.shape, device=gpu_device) * (10.0 ** -k))
        graph.replay()
        want, n = la.clip_by_global_norm(ts, 2.0)
        assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(out, want))
        torch.cuda.synchronize()


def adam64(x, g, m, v, t, lr, clip, joint):
    norm = lambda a: math.sqrt(float((a * a).sum()))
    g = [k * min(1.0, clip / norm(k)) if clip > 0 and norm(k) > 0 else k for k in g]
    s = math.sqrt(math.fsum(float((k * k).sum()) for k in g))
    if joint:
        g = [k * min(1.0, joint / s) if s > 0 else k for k in g]
    m = [0.9 * a + 0.1 * k for a, k in zip(m, g)]
    v = [0.999 * a + 0.001 * k * k for a, k in zip(v, g)]
    step = lr * math.sqrt(1 - 0.999 ** t) / (1 - 0.9 ** t)
    return [a - step * b / (c.sqrt() + 1e-7) for a, b, c in zip(x, m, v)], g, m, v


@pytest.mark.parametrize('shapes', [[(5,)], [(20, 32), (32,), (32, 32), (32,), (32, 1), (1,)], [(70_000, 3), (7,)],
                                    [(3,)] * 90, [(300_001,), (4096, 16), (1,), (0,)]], ids=lambda s: str(s[:2]))
@pytest.mark.parametrize('clip,joint,size', [(1.0, 0.5, 0.3), (1.0, 50.0, 0.3), (0.0, 0.7, 1.0), (1.0, 2.0, 1e-6)])
def test_adam_steps(gpu_device, shapes, clip, joint, size):
    from bayes_vi_amd.inference.vi.vi import Adam
    gen = torch.Generator(device=gpu_device); gen.manual_seed(len(shapes))
    params = [torch.nn.Parameter(torch.randn(*s, generator=gen, device=gpu_device)) for s in shapes]
    opt = Adam(learning_rate=0.01, global_clipnorm=joint).bind(params)
    x = [p.detach().double() for p in params]
    m, v = [torch.zeros_like(a) for a in x], [torch.zeros_like(a) for a in x]
    for t in range(1, 4):
        for p in params:
            p.grad = size * torch.randn(p.shape, generator=gen, device=gpu_device)
        g = [p.grad.double() for p in params]
        opt.clip_and_step(clip)
        x, g, m, v = adam64(x, g, m, v, t, 0.01, clip, joint)
        assert float(opt.t) == t
        for p, a, b, c, d, pm, pv in zip(params, x, g, m, v, opt.m, opt.v):
            assert bool(((p.grad.double() - b).abs() <= 6 * U * b.abs() + 1e-44).all())
            # moments: t steps, each a few roundings of terms no larger than the largest so far
            big = max(float(b.abs().max()) if b.numel() else 0.0, float(c.abs().max()) if c.numel() else 0.0)
            assert bool(((pm.double() - c).abs() <= 12 * t * U * big + 1e-44).all())
            assert bool(((pv.double() - d).abs() <= 16 * t * U * d.abs() + 1e-44).all())
            step = 0.01 * 1.1 * t
            assert bool(((p.detach().double() - a).abs() <= t * U * a.abs() + 64 * t * U * step + 3 * step * 12 * t * U * big
                         / (d.sqrt() + 1e-7)).all())


def test_adam_without_a_joint_clip_keeps_its_results(gpu_device):
    """Small variables go through the one-workgroup step as before; a large one takes the step over the list, with the
    same numbers."""
    from bayes_vi_amd import _native
    from bayes_vi_amd.inference.vi import vi
    gen = torch.Generator(device=gpu_device); gen.manual_seed(9)
    shape = (300, 301)
    a = [torch.randn(*shape, generator=gen, device=gpu_device) for _ in range(2)]
    g = 0.1 * torch.randn(*shape, generator=gen, device=gpu_device)
    p = torch.nn.Parameter(a[0].clone()); p.grad = g.clone()
    opt = vi.Adam(learning_rate=0.05).bind([p])
    assert p.numel() > vi.ONE_WORKGROUP_MAX
    opt.clip_and_step(1.0)
    x, gg, m, v = a[0].clone(), g.clone(), torch.zeros_like(g), torch.zeros_like(g)
    t = torch.zeros((), dtype=torch.float64, device=gpu_device)
    _native.check(_native.lib().bvi_clip_adam_step(x.numel(), _native._ptr(x), _native._ptr(gg), _native._ptr(m),
                                                   _native._ptr(v), _native._ptr(t), 1, 0.05, 0.9, 0.999, 1e-7, 1.0,
                                                   _native._stream()), 'bvi_clip_adam_step')
    # two factors that may differ by a rounding or two: g and m by 4 u, v by 8 u, the quotient m / sqrt(v) by 8 u
    assert bool(((p.grad - gg).abs() <= 4 * U * gg.abs()).all()) and bool(((opt.m[0] - m).abs() <= 8 * U * m.abs()).all())
    assert bool(((p.detach() - x).abs() <= 2 * U * x.abs() + 0.05 * 1.1 * 32 * U).all())


def test_a_variable_twice_is_refused(gpu_device):
    from bayes_vi_amd.inference.vi.vi import Adam
    p = torch.nn.Parameter(torch.ones(5, device=gpu_device))
    p.grad = torch.ones(5, device=gpu_device)
    with pytest.raises(ValueError, match='twice'):
        Adam(global_clipnorm=1.0).bind([p, p]).clip_and_step(1.0)


def test_clipping_in_place_is_seen_by_autograd(la, gpu_device):
    x = torch.ones(4, device=gpu_device, requires_grad=True)
    y = x * 2.0
    z = (y * y).sum()
    la.clip_by_global_norm([y.detach()], 0.5, inplace=True)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        z.backward()


def test_adam_non_finite_gradient(gpu_device):
    from bayes_vi_amd.inference.vi.vi import Adam
    ps = [torch.nn.Parameter(torch.ones(5, device=gpu_device)) for _ in range(2)]
    opt = Adam(global_clipnorm=1.0).bind(ps)
    ps[0].grad, ps[1].grad = torch.full((5,), float('nan'), device=gpu_device), torch.ones(5, device=gpu_device)
    opt.clip_and_step(1.0)
    assert all(bool(torch.isnan(p).all()) for p in ps)       # one norm for all, as tf.clip_by_global_norm signals it


def test_a_large_variable_twice_is_stepped_twice(gpu_device):
    """Without the joint clip a variable that is listed twice, and two variables with one gradient, are stepped one after
    the other whatever their size: the same bits as bvi_clip_adam_step in that order."""
    from bayes_vi_amd import _native
    from bayes_vi_amd.inference.vi import vi
    gen = torch.Generator(device=gpu_device); gen.manual_seed(21)
    n = 3 * vi.ONE_WORKGROUP_MAX + 1
    a, b = (torch.randn(n, generator=gen, device=gpu_device) for _ in range(2))
    g = 0.1 * torch.randn(n, generator=gen, device=gpu_device)
    for tied in ('variable', 'gradient'):
        p = torch.nn.Parameter(a.clone())
        q = p if tied == 'variable' else torch.nn.Parameter(b.clone())
        p.grad = g.clone()
        q.grad = p.grad
        opt = vi.Adam(learning_rate=0.05).bind([p, q])
        xs, gg = [a.clone(), b.clone()], g.clone()
        if tied == 'variable':
            xs[1] = xs[0]
        m, v = [torch.zeros_like(g) for _ in range(2)], [torch.zeros_like(g) for _ in range(2)]
        t = torch.zeros((), dtype=torch.float64, device=gpu_device)
        for _ in range(2):
            opt.clip_and_step(1.0)
            for k in range(2):
                _native.check(_native.lib().bvi_clip_adam_step(
                    n, _native._ptr(xs[k]), _native._ptr(gg), _native._ptr(m[k]), _native._ptr(v[k]), _native._ptr(t),
                    1 if k == 0 else 0, 0.05, 0.9, 0.999, 1e-7, 1.0, _native._stream()), 'bvi_clip_adam_step')
        assert float(opt.t) == 2.0 and torch.equal(p.detach(), xs[0]) and torch.equal(q.detach(), xs[1])
        assert torch.equal(p.grad, gg) and all(torch.equal(x, y) for x, y in zip(opt.m + opt.v, m + v))


def test_variables_that_share_memory_are_refused_by_the_joint_step(gpu_device):
    from bayes_vi_amd.inference.vi.vi import Adam
    base = torch.ones(20, device=gpu_device)
    for ps in ([base[:12], base[8:]], [base[:5], base[:5]]):
        ps = [torch.nn.Parameter(p) for p in ps]
        for p in ps:
            p.grad = torch.ones_like(p)
        with pytest.raises(ValueError, match='share memory'):
            Adam(global_clipnorm=1.0).bind(ps).clip_and_step(1.0)
    ps = [torch.nn.Parameter(torch.ones(5, device=gpu_device)) for _ in range(2)]
    ps[0].grad = ps[1].grad = torch.ones(5, device=gpu_device)
    with pytest.raises(ValueError, match='share memory'):
        Adam(global_clipnorm=1.0).bind(ps).clip_and_step(1.0)
    assert bool((ps[0] == 1).all()) and bool((base == 1).all())


def test_the_norm_to_use_may_not_be_written(la, gpu_device):
    """In place, use_norm inside a tensor of the list would be read by some workgroups after others had scaled it."""
    t = torch.full((70_000,), 3.0, device=gpu_device)
    for norm in (t[5], t[:1], t[-1:]):
        with pytest.raises(ValueError, match='use_norm lies'):
            la.clip_by_global_norm([torch.ones(4, device=gpu_device), t], 1.0, use_norm=norm, inplace=True)
    assert bool((t == 3).all())
    out, norm = la.clip_by_global_norm([t], 1.0, use_norm=t[5])          # written apart: fine
    assert float(norm) == 3.0 and bool((out[0] == 1).all())
    la.clip_by_global_norm([t[:7]], 1.0, use_norm=t[7], inplace=True)    # beside the tensor: fine
    assert bool((t[:7] == 1).all()) and bool((t[7:] == 3).all())


def test_lists_of_many_launches(la, gpu_device):
    """Tensors beyond what one launch's arguments hold, large enough for several workgroups each: the norm and the clipped
    values, in place and apart, and again the same bits from a graph."""
    for count, n in ((81, 60_000), (400, 5_000)):
        ts = tensors([(n + k % 3,) for k in range(count)], [torch.float32, torch.bfloat16] * count, 0.5, count, gpu_device)
        s = norm64(ts)
        out, norm = la.clip_by_global_norm(ts, 0.25 * s)
        assert abs(float(norm) - s) <= 2 * U * s and abs(float(la.global_norm(ts)) - s) <= 2 * U * s
        for o, t in zip(out, ts):
            f = torch.finfo(t.dtype)
            ref = t.double() * 0.25
            assert bool(((o.double() - ref).abs() <= (f.eps / 2 + 4 * U) * ref.abs() + f.smallest_normal * f.eps).all())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            again, norm2 = la.clip_by_global_norm(ts, 0.25 * s)
        for _ in range(3):
            graph.replay()
            eager, _ = la.clip_by_global_norm(ts, 0.25 * s)
            assert torch.equal(norm2, norm) and all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(again, out, eager))
        own = [t.clone() for t in ts]
        la.clip_by_global_norm(own, 0.25 * s, inplace=True)
        assert all(torch.equal(a, b) for a, b in zip(own, out))
