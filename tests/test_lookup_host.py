"""Host side of the lookup / clipping / grouped-regression operators: what is refused before anything is launched, the
C entry points' status codes, and how a likelihood with gathered group effects is recognised."""
import collections
import ctypes

import numpy as np
import pytest
import torch

import bayes_vi_amd.distributions as tfd
from bayes_vi_amd import _native, embedding, linalg, symbolic as sym
from bayes_vi_amd.inference.vi.vi import Adam
from bayes_vi_amd.model import Model


def test_python_refusals_without_a_gpu():
    t, i = torch.zeros(4, 3), torch.zeros(5, dtype=torch.int64)
    with pytest.raises(_native.BviError, match='no CPU fallback'):
        embedding.lookup(t, i)
    with pytest.raises(_native.BviError, match='no CPU fallback'):
        embedding.LookupPlan(i, 4)
    with pytest.raises(TypeError, match='int32 or int64'):
        embedding.lookup(t, i.float())
    with pytest.raises(TypeError, match='int32 or int64'):
        embedding.lookup(t, [0, 1])
    with pytest.raises(ValueError, match='rows, width'):
        embedding.lookup(torch.zeros(2, 2, 2), i)
    with pytest.raises(ValueError, match='no entries'):
        embedding.lookup(torch.zeros(0, 3), i)
    with pytest.raises(ValueError, match='shape'):
        embedding.lookup_grad(torch.zeros(4, 3), i, 4)
    with pytest.raises(ValueError, match='num_rows'):
        embedding.lookup_grad(torch.zeros(5, 3), i, 0)
    with pytest.raises(TypeError, match='list'):
        linalg.global_norm(t)
    with pytest.raises(ValueError, match='no tensor'):
        linalg.clip_by_global_norm([None], 1.0)
    with pytest.raises(_native.BviError, match='no CPU fallback'):
        linalg.clip_by_global_norm([t], 1.0)
    with pytest.raises(TypeError, match='float32'):
        linalg.global_norm([t.double()])
    for bad in (0.0, -1.0, float('nan')):
        with pytest.raises(ValueError, match='positive'):
            Adam(global_clipnorm=bad)


def test_c_entry_points_refuse_before_launching():
    """Every call here must return its status from the argument checks: the pointers are not device memory."""
    lib = _native.lib()
    p = ctypes.c_void_p(4096)
    z = ctypes.c_size_t(0)
    one = _native._int64s([3])
    assert lib.bvi_lookup(None, 0, 4, 3, 3, p, 0, 5, 1.0, p, None) == -1
    assert lib.bvi_lookup(p, 7, 4, 3, 3, p, 0, 5, 1.0, p, None) == -1
    assert lib.bvi_lookup(p, 0, 4, 3, 2, p, 0, 5, 1.0, p, None) == -1          # row stride below the width
    assert lib.bvi_lookup(p, 0, 4, 3, 3, p, 2, 5, 1.0, p, None) == -1
    assert lib.bvi_lookup(p, 0, 4, 3, 3, p, 0, -1, 1.0, p, None) == -1
    assert lib.bvi_lookup(p, 0, 4, 3, 3, None, 0, 0, 1.0, None, None) == 0     # no ids: nothing to do
    assert lib.bvi_lookup_plan_bytes(0, 5, ctypes.byref(z), ctypes.byref(z)) == -1
    assert lib.bvi_lookup_plan_bytes(1 << 31, 5, ctypes.byref(z), ctypes.byref(z)) == -2
    assert lib.bvi_lookup_plan(p, 1, 5, 4, p, 16, p, 16, None) == -3
    assert lib.bvi_lookup_plan(None, 1, 5, 4, p, 1 << 30, p, 1 << 30, None) == -1
    assert lib.bvi_lookup_grad_ws_bytes(4, 0, 5, 0, ctypes.byref(z)) == -1
    assert lib.bvi_lookup_grad(p, 0, 5, 3, 3, None, 0, None, 4, 1.0, p, p, 16, None) == -1      # neither ids nor a plan
    assert lib.bvi_lookup_grad(p, 0, 5, 3, 3, p, 5, None, 4, 1.0, p, p, 16, None) == -1
    assert lib.bvi_lookup_grad(p, 0, 5000, 3, 3, p, 0, p, 4, 1.0, p, None, 0, None) == -3
    assert lib.bvi_lookup_grad(p, 0, 5000, 3, 3, p, 0, None, 4, 1.0, p, p, 16, None) == -3
    # addresses between elements, scratch off its alignment
    odd = ctypes.c_void_p(4098)
    assert lib.bvi_lookup(odd, 0, 4, 3, 3, p, 0, 5, 1.0, p, None) == -1
    assert lib.bvi_lookup(p, 0, 4, 3, 3, odd, 0, 5, 1.0, p, None) == -1
    assert lib.bvi_lookup_plan(p, 1, 5000, 4, odd, 1 << 30, p, 1 << 30, None) == -1
    assert lib.bvi_lookup_grad(p, 0, 5000, 3, 3, p, 0, None, 4, 1.0, p, odd, 1 << 30, None) == -1
    assert lib.bvi_lookup_grad(odd, 0, 5000, 3, 3, p, 0, None, 4, 1.0, p, p, 1 << 30, None) == -1
    ptrs, types = (ctypes.c_void_p * 1)(4096), (ctypes.c_int * 1)(0)
    assert lib.bvi_global_norm(0, ptrs, one, types, p, p, 1 << 20, None) == -1
    assert lib.bvi_global_norm(1, ptrs, one, (ctypes.c_int * 1)(9), p, p, 1 << 20, None) == -1
    assert lib.bvi_global_norm(1, ptrs, one, types, p, p, 8, None) == -3
    assert lib.bvi_global_norm(1, (ctypes.c_void_p * 1)(4097), one, types, p, p, 1 << 20, None) == -1    # misaligned
    assert lib.bvi_clip_by_global_norm(1, ptrs, ptrs, one, types, 0.0, None, p, p, 1 << 20, None) == -1
    assert lib.bvi_clip_by_global_norm(1, ptrs, ptrs, _native._int64s([-1]), types, 1.0, None, p, p, 1 << 20, None) == -1
    assert lib.bvi_adam_step(1, ptrs, ptrs, ptrs, ptrs, one, p, .1, .9, .999, 1e-7, 1., 1., p, 8, None) == -3
    assert lib.bvi_adam_step(1, ptrs, ptrs, ptrs, ptrs, one, None, .1, .9, .999, 1e-7, 1., 1., p, 1 << 20, None) == -1
    assert lib.bvi_grouped_packed_bytes(5, 65, 1, one, 0, ctypes.byref(z), ctypes.byref(z)) == -2
    assert lib.bvi_grouped_packed_bytes(5, 1, 9, _native._int64s([1] * 9), 0, ctypes.byref(z), ctypes.byref(z)) == -2
    assert lib.bvi_grouped_packed_bytes(5, 1, 1, _native._int64s([0]), 0, ctypes.byref(z), ctypes.byref(z)) == -1
    assert lib.bvi_grouped_packed_bytes(5, 1, 2, _native._int64s([1 << 24, (1 << 24) + 1]), 0, ctypes.byref(z),
                                        ctypes.byref(z)) == -2
    assert lib.bvi_grouped_ws_bytes(5, 1, 1, one, 0, ctypes.byref(z)) == -1
    assert lib.bvi_grouped_logp_grad(odd, 5, 1, 1, one, 0, p, 4, p, p, None, p, 1 << 30, None) == -1
    assert lib.bvi_adam_step(1, (ctypes.c_void_p * 1)(4098), ptrs, ptrs, ptrs, one, p, .1, .9, .999, 1e-7, 1., 1., p, 1 << 20,
                             None) == -1
    assert lib.bvi_grouped_ws_bytes(5, 1, 1, one, (1 << 20) + 1, ctypes.byref(z)) == -2
    assert lib.bvi_grouped_logp_grad(p, 5, 1, 1, one, 0, p, 4, p, p, None, p, 16, None) == -3


def _priors(**sizes):
    return collections.OrderedDict((k, tfd.HalfNormal(1.) if k == 'scale' else tfd.Normal(0., 1.) if n == 0 else
                                    tfd.Normal(torch.zeros(n), torch.ones(n))) for k, n in sizes.items())


def test_recognise_varying_intercepts_and_slopes():
    feats = dict(school=torch.zeros(6), x=torch.zeros(6), year=torch.zeros(6))
    m = Model(_priors(mu=0, u=5, scale=0), lambda mu, u, scale, features: tfd.Normal(
        loc=mu + sym.gather(u, features['school']), scale=scale))
    d = m.describe_likelihood(feats)
    assert d['family'] == 'grouped' and d['columns'] == []
    assert d['index'] == [0, 6, 1, 2, 3, 4, 5]
    assert d['lookups'] == [('school', 5, [(None, 1.0)])]
    m = Model(_priors(mu=0, w=0, scale=0, u=3, v=4), lambda mu, w, scale, u, v, features: tfd.Normal(
        loc=mu + w * features['x'] + 0.5 * sym.gather(u, features['school']) * features['x']
        - sym.gather(v, features['year']) + 2.0 * features['x'], scale=scale))
    d = m.describe_likelihood(feats)
    assert d['index'] == list(range(10)) and d['columns'] == [[('x', 1.0)]] and d['offset'] == [('x', 2.0)]
    assert d['lookups'] == [('school', 3, [('x', 0.5)]), ('year', 4, [(None, -1.0)])]
    feats['x'] = torch.arange(6.)
    feats['year'] = torch.tensor([0., 1., 2., 3., 0., 1.])
    (i0, z0), (i1, z1) = m.lookup_columns(d, feats)
    assert i1.dtype == torch.int64 and i1.tolist() == [0, 1, 2, 3, 0, 1]
    assert torch.equal(z0, 0.5 * feats['x']) and torch.equal(z1, -torch.ones(6))
    X, y = m.design_matrix(d, feats, torch.zeros(6))
    assert torch.equal(X[:, 0], feats['x']) and torch.equal(y, -2.0 * feats['x'])
    # two uses of one table with the same groups are one lookup
    m = Model(_priors(mu=0, u=3, scale=0), lambda mu, u, scale, features: tfd.Normal(
        loc=mu + sym.gather(u, features['school']) * features['x'] + sym.gather(u, features['school']), scale=scale))
    assert m.describe_likelihood(feats)['lookups'] == [('school', 3, [('x', 1.0), (None, 1.0)])]


def test_unsupported_uses_of_gather():
    feats = dict(g=torch.zeros(6), x=torch.zeros(6))
    bad = [lambda u, scale, features: tfd.Normal(loc=sym.gather(u[0], features['g']), scale=scale),
           lambda u, scale, features: tfd.Normal(loc=sym.gather(u, u), scale=scale),
           lambda u, scale, features: tfd.Normal(loc=sym.gather(u, features['g']) * u[0], scale=scale),
           lambda u, scale, features: tfd.Normal(loc=0., scale=sym.gather(u, features['g']))]
    for f in bad:
        with pytest.raises(sym.UnsupportedLikelihood):
            Model(_priors(u=3, scale=0), f).describe_likelihood(feats)
    many = Model(_priors(u=3, scale=0), lambda u, scale, features: tfd.Normal(
        loc=sum(sym.gather(u, features['g%d' % k]) for k in range(9)), scale=scale))
    with pytest.raises(sym.UnsupportedLikelihood, match='at most 8'):
        many.describe_likelihood({'g%d' % k: torch.zeros(6) for k in range(9)})


def test_group_numbers():
    assert sym.whole_numbers(torch.tensor([0., 3., 1.])).tolist() == [0, 3, 1]
    with pytest.raises(ValueError, match='not whole'):
        sym.whole_numbers(torch.tensor([0.5]))
    with pytest.raises(ValueError, match='not whole'):
        sym.whole_numbers(torch.tensor([float('nan')]))
    with pytest.raises(ValueError, match='2\\^24'):
        sym.whole_numbers(torch.tensor([2.0 ** 25]))
    with pytest.raises(TypeError):
        sym.whole_numbers(torch.tensor([True]))


def test_gather_on_host_draws():
    u = torch.arange(6.).reshape(2, 3)
    assert torch.equal(sym.gather(u, torch.tensor([2., 0.])), u[:, [2, 0]])
    with pytest.raises(IndexError):
        sym.gather(u, torch.tensor([3.]))


def test_global_clipnorm_on_the_host_path():
    """`step` on CPU parameters: Keras' order, the joint clip before the moments."""
    rng = np.random.default_rng(0)
    p = [torch.nn.Parameter(torch.tensor(rng.normal(size=s), dtype=torch.float32)) for s in (3, (2, 2))]
    g = [rng.normal(size=q.shape) for q in p]
    opt = Adam(learning_rate=0.1, global_clipnorm=0.5).bind(p)
    x0 = [q.detach().double().numpy().copy() for q in p]
    for q, k in zip(p, g):
        q.grad = torch.tensor(k, dtype=torch.float32)
    opt.step()
    f = min(1.0, 0.5 / np.sqrt(sum((k.astype(np.float32).astype(np.float64) ** 2).sum() for k in g)))
    for q, k, x in zip(p, g, x0):
        m, v = 0.1 * f * k, 0.001 * (f * k) ** 2
        lr = 0.1 * np.sqrt(1 - 0.999) / (1 - 0.9)
        # m, v, sqrt, quotient, product: 6 roundings of the step of size <= 0.1, one of the result
        np.testing.assert_allclose(q.detach().double().numpy(), x - lr * m / (np.sqrt(v) + 1e-7), rtol=2e-7, atol=1e-6)
    for q in p:
        q.grad = torch.full_like(q, float('inf'))
    opt.step()
    assert all(torch.isnan(q).all() for q in p)


def test_group_numbers_of_other_types():
    """Any integers; floating-point columns as far as their type holds whole numbers exactly."""
    for t in (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64):
        assert sym.whole_numbers(torch.tensor([0, 7, 3], dtype=t)).tolist() == [0, 7, 3]
    for t, bits in ((torch.bfloat16, 8), (torch.float16, 11), (torch.float32, 24), (torch.float64, 53)):
        assert sym.whole_numbers(torch.tensor([2.0 ** bits], dtype=t)).tolist() == [2 ** bits]
        with pytest.raises(ValueError, match='2\\^%d are not exact' % bits):
            sym.whole_numbers(torch.tensor([2.0 ** (bits + 1)], dtype=t))


def test_a_table_looked_up_by_several_columns():
    """Its gradient is the sum over the uses, in the order of the uses whatever the device does with one index_add."""
    from bayes_vi_amd.model.model import _MappedLikelihood

    class Inner:
        device, group, sharded, logp_ref = torch.device('cpu'), None, False, None

        def logp_grad(self, theta, want_grad=True, relative=False):
            self.theta = theta
            return theta.sum(1), torch.tensor([[1.0, 2.0 ** 24, 3.0, 1.0, 7.0, 1.0, 9.0, 1.0]])

    feats = dict(a=torch.zeros(6), b=torch.zeros(6), c=torch.zeros(6))
    m = Model(_priors(u=2, scale=0), lambda u, scale, features: tfd.Normal(
        loc=sym.gather(u, features['a']) + sym.gather(u, features['b']) - sym.gather(u, features['c']), scale=scale))
    index = m.describe_likelihood(feats)['index']
    assert index == [-1, 2, 0, 1, 0, 1, 0, 1]
    lik = _MappedLikelihood(Inner(), index, 3)
    assert [cols.tolist() for cols, _ in lik.uses] == [[2, 0, 1], [0, 1], [0, 1]]
    lp, g = lik.logp_grad(torch.tensor([[4.0, 5.0, 6.0]]))
    assert lik.inner.theta.tolist() == [[0.0, 6.0, 4.0, 5.0, 4.0, 5.0, 4.0, 5.0]]
    assert g.tolist() == [[3.0 + 7.0 + 9.0, 3.0, 2.0 ** 24]]


def test_adam_step_refuses_lists_that_share_memory():
    """Nothing is launched: the status comes from the ranges alone.  Empty variables share nothing."""
    lib, at = _native.lib(), lambda *a: (ctypes.c_void_p * len(a))(*a)
    ws, big = ctypes.c_void_p(1 << 20), 1 << 30

    def status(x, g, m, v, sizes):
        return lib.bvi_adam_step(len(sizes), at(*x), at(*g), at(*m), at(*v), _native._int64s(sizes), ws, .1, .9, .999, 1e-7,
                                 1., 1., ws, big, None)
    base = [4096, 8192, 12288, 16384]
    for k in range(4):
        lists = [[b, b + 64] for b in base]
        lists[k][1] = lists[k][0] + 16                       # 5 floats from 0, 3 from the fourth of them
        assert status(*lists, [5, 3]) == -1
        lists[k][1] = lists[(k + 1) % 4][0]                  # one list's array in another's
        assert status(*lists, [5, 3]) == -1


def test_shapes_beyond_the_kernels_are_refused_at_recognition():
    """As other unsupported likelihoods are, not by the constructor or the C entry point once the data is there."""
    names = ['x%d' % k for k in range(65)]
    feats = {k: torch.zeros(6) for k in names + ['g', 'h']}

    def features_beside_a_table(count):
        priors = _priors(u=3, w=count, scale=0)
        return Model(priors, lambda u, w, scale, features: tfd.Normal(
            loc=sym.gather(u, features['g']) + sum(w[k] * features[names[k]] for k in range(count)), scale=scale))
    assert len(features_beside_a_table(64).describe_likelihood(feats)['columns']) == 64
    with pytest.raises(sym.UnsupportedLikelihood, match='64 feature columns'):
        features_beside_a_table(65).describe_likelihood(feats)
    m = Model(_priors(u=3, scale=0), lambda u, scale, features: tfd.Normal(
        loc=sym.gather(u, features['g']) + sym.gather(u, features['h']), scale=scale))
    m.block_sizes = [1 << 24, 1]
    assert m.describe_likelihood(feats)['family'] == 'grouped'
    m.block_sizes = [(1 << 24) + 1, 1]
    with pytest.raises(sym.UnsupportedLikelihood, match='entries together'):
        m.describe_likelihood(feats)


def test_gather_needs_a_vector_parameter():
    """tf.gather over the last axis of a [2, 3] parameter gives two values per row, of a scalar's draws values of other
    chains: neither is the table of six or of one entry that the flat layout would suggest."""
    feats = dict(g=torch.zeros(6))
    for prior, fine in ((tfd.Normal(torch.zeros(2, 3), torch.ones(2, 3)), False), (tfd.Normal(0., 1.), False),
                        (tfd.Normal(torch.zeros(1, 6), torch.ones(1, 6)), False),
                        (tfd.Normal(torch.zeros(1), torch.ones(1)), True), (tfd.Normal(torch.zeros(6), torch.ones(6)), True)):
        m = Model(collections.OrderedDict(u=prior, scale=tfd.HalfNormal(1.)),
                  lambda u, scale, features: tfd.Normal(loc=sym.gather(u, features['g']), scale=scale))
        if fine:
            assert m.describe_likelihood(feats)['family'] == 'grouped'
        else:
            with pytest.raises(sym.UnsupportedLikelihood, match='vector parameter'):
                m.describe_likelihood(feats)


def test_feature_lists_are_converted_straight_to_float32():
    """Whole numbers beyond 64 bits, and fractions under a default type of fewer bits, keep their float32 values."""
    feats = dict(g=[0, 2, 1], x=[10 ** 20, 1, -3], v=[1 + 2.0 ** -20, 2.5, 3.0])
    m = Model(_priors(u=3, w=2, scale=0), lambda u, w, scale, features: tfd.Normal(
        loc=w[0] * features['x'] + w[1] * features['v'] + sym.gather(u, features['g']) * features['v'], scale=scale))
    d = m.describe_likelihood(feats)
    want = torch.tensor([[1e20, 1 + 2.0 ** -20], [1., 2.5], [-3., 3.]])
    before = torch.get_default_dtype()
    try:
        for default in (torch.float32, torch.bfloat16):
            torch.set_default_dtype(default)
            X, y = m.design_matrix(d, feats, torch.zeros(3, dtype=torch.float32))
            (ids, z), = m.lookup_columns(d, feats)
            assert X.dtype == torch.float32 and torch.equal(X, want)
            assert ids.tolist() == [0, 2, 1] and torch.equal(z, want[:, 1])
    finally:
        torch.set_default_dtype(before)
