"""GPU: linear regression with group-level effects against its formulas in 64 bits, and its use from a model down:
log-density, NUTS / HMC, ADVI with the joint clip, posterior-predictive draws, row shards.

Tolerances, u = 2^-24.  A residual e = y - b - x.w - sum z t is D + 2 L + 3 roundings of partial results no larger than
M = |y| + |b| + sum |x w| + sum |z t|, so it is off by at most r = (D + 2 L + 3) u M.  Sums over k rows in float inside a
wave's stretch (double beyond) add at most k u sum |terms|; a stretch has at most max(128, N / 4096) rows."""
import collections
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make(rng, n, d, groups, chains, skew=1.0, columns=False, dev='cuda'):
    X = rng.normal(size=(n, d)).astype(np.float32)
    ids = [np.minimum((rng.random(n) ** skew * g).astype(np.int64), g - 1) for g in groups]
    z = [rng.normal(size=n).astype(np.float32) if columns and k % 2 == 0 else None for k in range(len(groups))]
    y = rng.normal(1.0, 2.0, n).astype(np.float32)
    theta = np.concatenate([rng.normal(size=(chains, 1 + d)), rng.uniform(0.7, 2.0, (chains, 1)),
                            rng.normal(size=(chains, sum(groups)))], 1).astype(np.float32)
    return X, y, ids, z, theta


def oracle(X, y, ids, z, theta, groups):
    """(logp, grad, their error bounds) in 64 bits."""
    n, d = X.shape
    X, y, theta = X.astype(np.float64), y.astype(np.float64), theta.astype(np.float64)
    at = np.cumsum([d + 2] + list(groups))
    span = max(128, n // 4096 + 1)
    out = []
    for th in theta:
        s = th[d + 1]
        e, M = y - th[0] - X @ th[1:d + 1], np.abs(y) + abs(th[0]) + np.abs(X) @ np.abs(th[1:d + 1])
        zs = [np.ones(n) if k is None else k.astype(np.float64) for k in z]
        for k, i in enumerate(ids):
            t = zs[k] * th[at[k]:at[k + 1]][i]
            e, M = e - t, M + np.abs(t)
        r = (d + 2 * len(ids) + 3) * U * M
        sq, esq = (e * e).sum(), (2 * np.abs(e) * r + r * r).sum() + (span + 2) * U * ((np.abs(e) + r) ** 2).sum()
        lp = -n * math.log(s) - n / 2 * math.log(2 * math.pi) - sq / (2 * s * s)
        es = lambda wgt: ((np.abs(wgt) * r).sum() + (span + 2) * U * (np.abs(wgt) * (np.abs(e) + r)).sum()) / s ** 2
        g, b = np.zeros(len(th)), np.zeros(len(th))
        g[0], b[0] = e.sum() / s ** 2, es(np.ones(n))
        for j in range(d):
            g[1 + j], b[1 + j] = (e * X[:, j]).sum() / s ** 2, es(X[:, j])
        g[d + 1], b[d + 1] = sq / s ** 3 - n / s, esq / s ** 3
        for k, i in enumerate(ids):
            g[at[k]:at[k + 1]] = np.bincount(i, zs[k] * e, groups[k]) / s ** 2
            b[at[k]:at[k + 1]] = np.bincount(i, np.abs(zs[k]) * (r + (span + 2) * U * (np.abs(e) + r)), groups[k]) / s ** 2
        out.append((lp, g, esq / (2 * s * s) + 2 * U * abs(lp), b + 4 * U * np.abs(g) + 1e-30))
    return [np.stack(k) for k in zip(*out)]


def likelihood(X, y, ids, z, groups, dev, id_type=torch.int64):
    from bayes_vi_amd.fused_target import GroupedRegression
    t = lambda a: None if a is None else torch.tensor(a, device=dev)
    return GroupedRegression(t(X), t(y), [t(i).to(id_type) for i in ids], groups, [t(k) for k in z])


def check(lik, X, y, ids, z, theta, groups, dev):
    lp, g = lik.logp_grad(torch.tensor(theta, device=dev))
    rlp, rg, blp, bg = oracle(X, y, ids, z, theta, groups)
    e = np.abs(lp.cpu().numpy() - rlp)
    assert (e <= blp).all(), (e / blp).max()
    e = np.abs(g.cpu().numpy() - rg)
    assert (e <= bg).all(), ((e / bg).max(), np.argwhere(e > bg)[:5])
    lp2, none = lik.logp_grad(torch.tensor(theta, device=dev), want_grad=False)
    assert none is None and (np.abs(lp2.cpu().numpy() - rlp) <= blp).all()
    lp3, g3 = lik.logp_grad(torch.tensor(theta, device=dev))
    assert torch.equal(lp, lp3) and torch.equal(g, g3)                       # the same bits again


@pytest.mark.parametrize('chains', [1, 2, 4, 5, 16, 17, 64, 67])
@pytest.mark.parametrize('n,d,groups', [(1, 0, [1]), (919, 1, [85]), (130, 3, [200]), (2000, 0, [7, 300]),
                                        (5003, 8, [3, 11, 2])], ids=str)
def test_value_and_gradient(gpu_device, n, d, groups, chains):
    rng = np.random.default_rng(n + chains)
    X, y, ids, z, theta = make(rng, n, d, groups, chains, skew=2.0, columns=d > 0)
    check(likelihood(X, y, ids, z, groups, gpu_device), X, y, ids, z, theta, groups, gpu_device)


@pytest.mark.parametrize('d', [2, 4, 5, 13, 16, 17, 33, 64])
def test_feature_counts(gpu_device, d):
    rng = np.random.default_rng(d)
    X, y, ids, z, theta = make(rng, 700, d, [40], 6)
    check(likelihood(X, y, ids, z, [40], gpu_device, torch.int32), X, y, ids, z, theta, [40], gpu_device)


@pytest.mark.parametrize('chains', [1, 4, 64])
@pytest.mark.parametrize('groups,skew', [([2], 1.0), ([60, 20000], 1.0), ([100000], 1.0), ([500], 8.0)], ids=str)
def test_large(gpu_device, groups, skew, chains):
    """Groups that span many waves, groups of a few rows, most rows in one group, empty groups."""
    rng = np.random.default_rng(chains)
    X, y, ids, z, theta = make(rng, 300_001, 2, groups, chains, skew=skew)
    lik = likelihood(X, y, ids, z, groups, gpu_device)
    if chains == 64:
        theta = theta[:, :]
        lp, g = lik.logp_grad(torch.tensor(theta, device=gpu_device))
        for c in (0, 31, 63):                                 # three of the chains against the formulas
            rlp, rg, blp, bg = oracle(X, y, ids, z, theta[c:c + 1], groups)
            assert abs(float(lp[c]) - rlp[0]) <= blp[0]
            assert (np.abs(g[c].cpu().numpy() - rg[0]) <= bg[0]).all()
    else:
        check(lik, X, y, ids, z, theta, groups, gpu_device)


def test_gradient_against_differences(gpu_device):
    rng = np.random.default_rng(3)
    X, y, ids, z, theta = make(rng, 400, 2, [9, 4], 1, columns=True)
    lik = likelihood(X, y, ids, z, [9, 4], gpu_device)
    _, g = lik.logp_grad(torch.tensor(theta, device=gpu_device))
    f = lambda th: oracle(X, y, ids, z, th[None], [9, 4])[0][0]
    scale = float(g.abs().max())
    for j in range(theta.shape[1]):
        h = 1e-4
        hi, lo = theta[0].astype(np.float64), theta[0].astype(np.float64)
        hi[j] += h
        lo[j] -= h
        # the oracle's own rounding (2^-52 of ~1e3) over 2h, and h^2 / 6 of the third derivative (~1e5 for the scale)
        assert abs((f(hi) - f(lo)) / (2 * h) - float(g[0, j])) <= 1e-5 * scale + 1e-3


def test_reduces_to_linear_regression(gpu_device):
    """With all effects zero the value and the shared gradients are those of the plain regression kernels."""
    from bayes_vi_amd.fused_target import LinearRegression
    rng = np.random.default_rng(4)
    X, y, ids, z, theta = make(rng, 3000, 6, [30], 5)
    theta[:, 8:] = 0
    lp, g = likelihood(X, y, ids, z, [30], gpu_device).logp_grad(torch.tensor(theta, device=gpu_device))
    plain = LinearRegression(torch.tensor(X, device=gpu_device), torch.tensor(y, device=gpu_device))
    lp2, g2 = plain.logp_grad(torch.tensor(theta[:, :8], device=gpu_device))
    _, _, blp, bg = oracle(X, y, ids, z, theta, [30])
    # both sides within the bound of the exact value
    assert (np.abs((lp - lp2).cpu().numpy()) <= 2 * blp).all()
    assert (np.abs((g[:, :8] - g2).cpu().numpy()) <= 2 * bg[:, :8] + 1e-5 * np.abs(g2.cpu().numpy()).max()).all()


def test_relative_level_and_non_finite_parameters(gpu_device):
    rng = np.random.default_rng(5)
    X, y, ids, z, theta = make(rng, 5000, 1, [12], 3)
    lik = likelihood(X, y, ids, z, [12], gpu_device)
    th = torch.tensor(theta, device=gpu_device)
    lp, g = lik.logp_grad(th)
    lik.logp_ref = torch.tensor([float(lp[0]), 0.0], dtype=torch.float64, device=gpu_device)
    rel, g2 = lik.logp_grad(th, relative=True)
    rlp, _, blp, _ = oracle(X, y, ids, z, theta, [12])
    assert (np.abs(rel.cpu().numpy() - (rlp - float(lp[0]))) <= blp).all() and torch.equal(g, g2)
    bad = th.clone()
    bad[0, 5] = float('nan')
    bad[1, 0] = float('inf')
    lp3, g3 = lik.logp_grad(bad)
    assert not torch.isfinite(lp3[:2]).any() and torch.equal(lp3[2], lp[2]) and torch.equal(g3[2], g[2])


def test_graphs_keep_their_scratch(gpu_device):
    """A captured evaluation replays correctly after the likelihood was used for more chains (more scratch) in between,
    and two graphs of one likelihood do not share any."""
    rng = np.random.default_rng(6)
    X, y, ids, z, theta = make(rng, 3000, 2, [40, 6], 40)
    lik = likelihood(X, y, ids, z, [40, 6], gpu_device)
    th = torch.tensor(theta, device=gpu_device)
    small = [th[:3].clone(), th[3:8].clone()]
    want = [lik.logp_grad(t) for t in small]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in small:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(lik.logp_grad(t))
    for k in range(4):
        big = lik.logp_grad(th)
        junk = torch.full((1 << 20,), float('nan'), device=gpu_device)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (lp, gr), (wl, wg) in zip(outs, want):
            assert torch.equal(lp, wl) and torch.equal(gr, wg)
        assert torch.isfinite(big[1]).all() and torch.isnan(junk).all()


def test_theta_is_checked(gpu_device):
    rng = np.random.default_rng(8)
    X, y, ids, z, theta = make(rng, 50, 1, [4], 2)
    lik = likelihood(X, y, ids, z, [4], gpu_device)
    th = torch.tensor(theta, device=gpu_device)
    for bad in (th[:, :-1], torch.cat([th, th], 1)):
        with pytest.raises(ValueError, match='theta must be'):
            lik.logp_grad(bad)
    from bayes_vi_amd._native import BviError
    for bad in (th.cpu(), th.double()):
        with pytest.raises(BviError):
            lik.logp_grad(bad)


def test_rows_without_a_group_have_no_effect(gpu_device):
    """The C entry point takes ids outside the table (the Python class refuses them): such rows have no effect of that
    lookup, wherever in a stretch of rows they fall."""
    import ctypes
    from bayes_vi_amd import _native as nat
    rng = np.random.default_rng(9)
    for chains in (1, 3, 16, 40):
        X, y, ids, z, theta = make(rng, 700, 1, [9, 5], chains)
        for i, rows in zip(ids, (9, 5)):
            out = rng.random(700) < 0.3
            i[out] = rng.choice([-1, rows, rows + 3, 2 ** 31 - 1, -2 ** 31], out.sum())
        dev = lambda a: torch.tensor(a, device=gpu_device)
        packed, mask = nat.grouped_pack(dev(X), dev(y), [dev(i.astype(np.int32)) for i in ids], [9, 5], [None, None])
        th = dev(theta)
        lp, g = torch.empty(chains, device=gpu_device), torch.empty_like(th)
        ws = nat._scratch(nat.grouped_ws_bytes(700, 1, [9, 5], chains), gpu_device)
        nat.check(nat.lib().bvi_grouped_logp_grad(packed.data_ptr(), 700, 1, 2, nat._int64s([9, 5]), mask, th.data_ptr(), chains,
                                                  lp.data_ptr(), g.data_ptr(), None, ws.data_ptr(), ws.numel(), nat._stream()),
                  'bvi_grouped_logp_grad')
        # the same with one more row in each table whose effect is zero
        ids2 = [np.where((i >= 0) & (i < r), i, r) for i, r in zip(ids, (9, 5))]
        th2 = np.concatenate([theta[:, :12], np.zeros((chains, 1)), theta[:, 12:], np.zeros((chains, 1))], 1).astype(np.float32)
        rlp, rg, blp, bg = oracle(X, y, ids2, z, th2, [10, 6])
        keep = [j for j in range(th2.shape[1]) if j not in (12, 18)]
        assert (np.abs(lp.cpu().numpy() - rlp) <= blp).all()
        assert (np.abs(g.cpu().numpy() - rg[:, keep]) <= bg[:, keep]).all()


@pytest.mark.parametrize('chains', [1, 3, 16, 40])
@pytest.mark.parametrize('n_lookups', [1, 2])
def test_columns_beside_no_group_are_not_used(gpu_device, n_lookups, chains):
    """What a multiplier holds in rows without a group of its lookup (here NaN and infinities) changes nothing."""
    from bayes_vi_amd import _native as nat
    rng, groups = np.random.default_rng(10), [9, 5][:n_lookups]
    X, y, ids, z, theta = make(rng, 700, 1, groups, chains)
    z = [rng.normal(size=700).astype(np.float32) for _ in groups]
    masked = []
    for i, k, rows in zip(ids, z, groups):
        out = rng.random(700) < 0.3
        i[out] = rng.choice([-1, rows, 2 ** 31 - 1], out.sum())
        masked.append(k.copy())
        masked[-1][out] = rng.choice([np.nan, np.inf, -np.inf], out.sum())
        k[out] = 0.0
    dev = lambda a: torch.tensor(a, device=gpu_device)
    th, got = dev(theta), []
    for columns in (z, masked):
        packed, mask = nat.grouped_pack(dev(X), dev(y), [dev(i.astype(np.int32)) for i in ids], groups, [dev(k) for k in columns])
        lp, g = torch.empty(chains, device=gpu_device), torch.empty_like(th)
        ws = nat._scratch(nat.grouped_ws_bytes(700, 1, groups, chains), gpu_device)
        nat.check(nat.lib().bvi_grouped_logp_grad(packed.data_ptr(), 700, 1, n_lookups, nat._int64s(groups), mask,
                                                  th.data_ptr(), chains, lp.data_ptr(), g.data_ptr(), None, ws.data_ptr(),
                                                  ws.numel(), nat._stream()), 'bvi_grouped_logp_grad')
        got.append((lp, g))
    assert torch.isfinite(got[0][0]).all() and torch.isfinite(got[0][1]).all()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_a_table_looked_up_three_times(gpu_device):
    """One table of a model read by three columns: the gradient is the sum over the uses, the same bits every time."""
    import bayes_vi_amd.distributions as tfd
    from bayes_vi_amd import symbolic as sym
    from bayes_vi_amd.model import Model
    rng, G, n = np.random.default_rng(11), 300, 5000
    ids = [rng.integers(0, G, n) for _ in range(3)]
    y = rng.normal(size=n).astype(np.float32)
    priors = collections.OrderedDict(u=tfd.Normal(torch.zeros(G), torch.ones(G)), scale=tfd.HalfNormal(2.))
    model = Model(priors, lambda u, scale, features: tfd.Normal(
        loc=sym.gather(u, features['a']) + sym.gather(u, features['b']) - sym.gather(u, features['c']), scale=scale))
    feats = {k: torch.tensor(i, device=gpu_device) for k, i in zip('abc', ids)}
    lik = model._build_likelihood(feats, torch.tensor(y, device=gpu_device))
    theta = np.concatenate([rng.normal(size=(4, G)), rng.uniform(0.7, 2.0, (4, 1))], 1).astype(np.float32)
    th = torch.tensor(theta, device=gpu_device)
    lp, g = lik.logp_grad(th)
    kernel_theta = np.concatenate([np.zeros((4, 1)), theta[:, G:]] + [theta[:, :G]] * 3, 1).astype(np.float32)
    z = [None, None, -np.ones(n, np.float32)]
    rlp, rg, blp, bg = oracle(np.zeros((n, 0), np.float32), y, ids, z, kernel_theta, [G] * 3)
    assert (np.abs(lp.cpu().numpy() - rlp) <= blp).all()
    fold = lambda a: np.concatenate([a[:, 2:].reshape(4, 3, G).sum(1), a[:, 1:2]], 1)
    e, b = np.abs(g.cpu().numpy() - fold(rg)), fold(bg)
    b += 3 * U * fold(np.abs(rg))                             # two additions of the three uses
    assert (e <= b).all()
    for _ in range(5):
        assert torch.equal(lik.logp_grad(th)[1], g)


def test_refusals(gpu_device):
    from bayes_vi_amd.fused_target import GroupedRegression
    y = torch.zeros(5, device=gpu_device)
    i = torch.tensor([0, 1, 2, 1, 0], device=gpu_device)
    for bad in (lambda: GroupedRegression(None, y, [i], [2]), lambda: GroupedRegression(None, y, [i - 1], [3]),
                lambda: GroupedRegression(None, y, [i[:4]], [3]), lambda: GroupedRegression(None, y, [i.float()], [3]),
                lambda: GroupedRegression(None, y, [i, i], [3]), lambda: GroupedRegression(None, y, [i] * 9, [3] * 9),
                lambda: GroupedRegression(torch.zeros(5, 65, device=gpu_device), y, [i], [3]),
                lambda: GroupedRegression(torch.zeros(10, device=gpu_device), y, [i], [3]),
                lambda: GroupedRegression(torch.zeros(5, 2), y, [i], [3]),
                lambda: GroupedRegression(None, y, [i], [3], [torch.zeros(4, device=gpu_device)])):
        with pytest.raises(ValueError):
            bad()
    lik = GroupedRegression(None, y, [i], [3])
    lp, g = lik.logp_grad(torch.tensor([[0., 1., 0., 0., 0.]], device=gpu_device))
    assert abs(float(lp) + 2.5 * math.log(2 * math.pi)) <= 4 * U * 5 and g[0].tolist() == [0., -5., 0., 0., 0.]


# ---- from the model down ----
def schools(dev, n=400, groups=8, seed=0):
    """y ~ Normal(mu + u[school] + w x, scale): data whose effects are known."""
    import bayes_vi_amd.distributions as tfd
    from bayes_vi_amd import symbolic as sym
    from bayes_vi_amd.model import Model
    from bayes_vi_amd.utils.datasets import TensorDataset
    rng = np.random.default_rng(seed)
    x, g = rng.normal(size=n).astype(np.float32), rng.integers(0, groups, n)
    u = np.linspace(-2, 2, groups)
    y = (0.5 + u[g] + 0.8 * x + 0.5 * rng.normal(size=n)).astype(np.float32)
    priors = collections.OrderedDict(u=tfd.Normal(torch.zeros(groups), 3.0 * torch.ones(groups)), w=tfd.Normal(0., 5.),
                                     scale=tfd.HalfNormal(2.))
    model = Model(priors, lambda u, w, scale, features: tfd.Normal(
        loc=0.5 + w * features['x'] + sym.gather(u, features['school']), scale=scale))
    t = lambda a: torch.tensor(a, dtype=torch.float32, device=dev)
    return model, TensorDataset(dict(school=t(g), x=t(x)), t(y)), (x, g, y, u)


def test_model_log_prob(gpu_device):
    model, ds, (x, g, y, _) = schools(gpu_device)
    post = model.get_joint_distribution(features=ds.features).posterior(ds.targets)
    rng = np.random.default_rng(1)
    u, w, s = rng.normal(size=(3, 8)), rng.normal(size=3), rng.uniform(.4, 1., 3)
    theta = torch.tensor(np.concatenate([u, w[:, None], s[:, None]], 1), dtype=torch.float32, device=gpu_device)
    ll, gl = post.likelihood.logp_grad(theta)
    kernel = np.concatenate([np.zeros((3, 1)), w[:, None], s[:, None], u], 1).astype(np.float32)
    rlp, rg, blp, bg = oracle(x[:, None], (y - np.float32(.5)), [g], [None], kernel, [8])
    assert (np.abs(ll.cpu().numpy() - rlp) <= blp).all()
    got = gl.cpu().numpy()
    assert (np.abs(got[:, :8] - rg[:, 3:]) <= bg[:, 3:]).all() and (np.abs(got[:, 8:10] - rg[:, 1:3]) <= bg[:, 1:3]).all()


def exact_effects(x, g, y, scale, groups=8):
    """Posterior mean and deviation of (u, w) for a known scale: a Gaussian."""
    A = np.concatenate([np.eye(groups)[g], x[:, None]], 1).astype(np.float64)
    prec = A.T @ A / scale ** 2 + np.diag([1 / 9.] * groups + [1 / 25.])
    cov = np.linalg.inv(prec)
    return cov @ (A.T @ (y.astype(np.float64) - 0.5)) / scale ** 2, np.sqrt(np.diag(cov))


def test_nuts_recovers_the_effects(gpu_device):
    from bayes_vi_amd.inference.mcmc import MCMC
    from bayes_vi_amd.inference.mcmc.stepsize_adaptation_kernels import DualAveragingStepSizeAdaptation
    from bayes_vi_amd.inference.mcmc.transition_kernels import NoUTurnSampler
    model, ds, (x, g, y, _) = schools(gpu_device)
    adapt = DualAveragingStepSizeAdaptation(num_adaptation_steps=400)
    res = MCMC(model, ds, transition_kernel=NoUTurnSampler(stepsize_adaptation_kernel=adapt)).fit(
        num_chains=8, num_samples=400, num_burnin_steps=500, progress_bar=False, seed=3)
    u = res.samples[0].reshape(-1, 8).double().cpu().numpy()
    mean, sd = exact_effects(x, g, y, float(res.samples[2].mean()))
    # 3200 draws with an effective size of 200 at the very least: the mean within 5 standard errors, the deviation 30 %
    assert (np.abs(u.mean(0) - mean[:8]) < 5 * sd[:8] / math.sqrt(200)).all()
    assert (np.abs(u.std(0) / sd[:8] - 1) < 0.3).all()


@pytest.mark.parametrize('capture', [False, True])
@pytest.mark.parametrize('mean_field', [False, True])
def test_a_training_run_uses_all_of_them_together(gpu_device, mean_field, capture):
    """ADVI of the grouped model with the joint clip: the lookups' gradient, the global norm and the Adam step in one
    optimisation step.  The fused step against the same step by autograd and the host formulas of the optimiser, on
    injected noise."""
    from bayes_vi_amd.inference.vi import VI
    from bayes_vi_amd.inference.vi.surrogate_posteriors import ADVI
    from bayes_vi_amd.inference.vi.vi import Adam
    runs = []
    for fused in (True, False):
        model, ds, _ = schools(gpu_device)
        gen = torch.Generator(); gen.manual_seed(11)
        sur = ADVI(model, mean_field=mean_field, generator=gen)
        noise = torch.randn(12, 4, 10, generator=gen).to(gpu_device)
        count = torch.zeros((), dtype=torch.long, device=gpu_device)

        def base_noise(n, dim, noise=noise, count=count):
            e = noise.index_select(0, count.reshape(1))[0]
            count += 1
            return e
        vi = VI(model, ds, sur)
        sur.base_noise = base_noise
        vi.fused_advi = fused
        sur.approx_joint_marginal_posteriors = lambda k: None
        _, losses = vi.fit(Adam(learning_rate=0.05, global_clipnorm=0.3), num_steps=12, sample_size=4, progress_bar=False,
                           capture_graph=capture)
        runs.append((losses, [p.detach().clone() for p in sur.parameters()]))
    # gradients agree to ~1e-5 of their norm (parity of the two routes), an Adam step moves by lr x a ratio of moments
    np.testing.assert_allclose(runs[0][0], runs[1][0], rtol=2e-4)
    for a, b in zip(runs[0][1], runs[1][1]):
        assert float((a - b).abs().max()) <= 12 * 0.05 * 2e-3


def test_posterior_predictive_uses_the_lookup(gpu_device):
    model, ds, (x, g, y, u) = schools(gpu_device)
    draws = [torch.tensor(np.tile(u, (500, 1)), dtype=torch.float32, device=gpu_device),
             torch.full((500,), 0.8, device=gpu_device), torch.full((500,), 0.5, device=gpu_device)]
    pred = model.get_posterior_predictive_distribution(posterior_samples=draws, features=ds.features).sample((300,))
    assert pred['y'].shape == (300, 400)
    want = 0.5 + u[g] + 0.8 * x
    # 300 draws of deviation 0.5: five standard errors over 400 rows
    assert np.abs(pred['y'].double().mean(0).cpu().numpy() - want).max() < 5 * 0.5 / math.sqrt(300)


def test_row_shards_add_up(gpu_device):
    rng = np.random.default_rng(7)
    X, y, ids, z, theta = make(rng, 2001, 3, [20, 5], 4, columns=True)
    whole = likelihood(X, y, ids, z, [20, 5], gpu_device)
    th = torch.tensor(theta, device=gpu_device)
    lp, g = whole.logp_grad(th)
    parts = []
    for a, b in ((0, 700), (700, 701), (701, 2001)):
        cut = lambda k: None if k is None else k[a:b]
        parts.append(likelihood(X[a:b], y[a:b], [i[a:b] for i in ids], [cut(k) for k in z], [20, 5], gpu_device).logp_grad(th))
    rlp, rg, blp, bg = oracle(X, y, ids, z, theta, [20, 5])
    assert (np.abs(sum(p[0].double() for p in parts).cpu().numpy() - rlp) <= 2 * blp).all()
    assert (np.abs(sum(p[1].double() for p in parts).cpu().numpy() - rg) <= 2 * bg).all()


@pytest.mark.parametrize('chains', [16, 17, 64])
def test_sums_over_many_rows_do_not_lose_bits(gpu_device, chains):
    """Log-densities, and their differences between chains, at 9M rows in two groups.  y, the effects and the weights are
    multiples of 2^-8 and the features -1, 0 or 1, so every residual is exact, |e| < 4, and e^2 a multiple of 2^-16 below 16:
    a float holds the sum of 16 of them exactly, not that of a thousand.  Sums that move to double every 32 rows or sooner
    therefore leave nothing but the roundings of the results (2 u each; the double arithmetic is off by 2^-52 of ~1e7),
    however many rows there are.  Sums of e and e x are multiples of 2^-8 below 2^13 within 2048 rows: exact as well."""
    from bayes_vi_amd.fused_target import GroupedRegression
    n, d = 9_000_001, 2
    gen = torch.Generator(device=gpu_device); gen.manual_seed(chains)
    grid = lambda t: torch.round(t * 256) / 256
    X = torch.randint(-1, 2, (n, d), generator=gen, device=gpu_device).float()
    ids = (torch.rand(n, generator=gen, device=gpu_device) < 0.3).long()
    e0 = grid(torch.randn(n, generator=gen, device=gpu_device).clamp_(-3, 3))
    w, u = torch.tensor([0.25, -0.5], device=gpu_device), torch.tensor([1.5, -0.75], device=gpu_device)
    y = 0.5 + X @ w + u[ids] + e0
    off = grid(0.15 * torch.rand(chains, 5, generator=gen, device=gpu_device))       # |e - e0| <= 0.6 < 1
    th = torch.cat([0.5 + off[:, :1], w + off[:, 1:3], 1 + off[:, :1], u + off[:, 3:]], 1)
    lik = GroupedRegression(X, y, [ids], [2])
    y64, X64 = y.double(), X.double()
    want, grads = [], []
    for t in th.double():
        e = y64 - t[0] - X64 @ t[1:3] - t[4:][ids]
        s, sq = float(t[3]), float((e * e).sum())
        want.append(-n * math.log(s) - n / 2 * math.log(2 * math.pi) - sq / (2 * s * s))
        back = torch.stack([(e * (1 - ids)).sum(), (e * ids).sum()])
        grads.append(torch.cat([e.sum()[None], e @ X64, torch.tensor([sq / s - n * s], device=gpu_device), back]).cpu() / s ** 2)
    want, grads = np.array(want), torch.stack(grads).numpy()
    lik.logp_ref = torch.tensor([want[0], 0.0], dtype=torch.float64, device=gpu_device)
    rel, g = lik.logp_grad(th, relative=True)
    err = np.abs(rel.double().cpu().numpy() - (want - want[0]))
    assert (err <= 2 * U * np.abs(want - want[0]) + 1e-7).all(), err.max()
    # d s is a difference of two terms of the size n / s
    assert (np.abs(g.double().cpu().numpy() - grads) <= 2 * U * np.abs(grads) + 1e-7).all()
    value, none = lik.logp_grad(th, want_grad=False, relative=True)
    assert none is None and (np.abs(value.double().cpu().numpy() - (want - want[0])) <= 2 * U * np.abs(want - want[0]) + 1e-7).all()


def test_the_table_sizes_are_checked_before_the_ids(gpu_device):
    from bayes_vi_amd.fused_target import GroupedRegression
    y, i = torch.zeros(5, device=gpu_device), torch.full((5,), 7, device=gpu_device)
    for rows in ([1 << 24, (1 << 24) + 1], [0, 3]):
        with pytest.raises(ValueError, match='at least one row each and at most'):
            GroupedRegression(None, y, [i, i], rows)


def test_gather_of_draws(gpu_device):
    """Any leading shape, none and no draws among them, as indexing gives it; group numbers of another type or device."""
    from bayes_vi_amd import symbolic as sym
    gen = torch.Generator(device=gpu_device); gen.manual_seed(3)
    ids = torch.tensor([4, 0, 0, 2, 1], device=gpu_device)
    for lead in ((), (1,), (7,), (3, 5), (0,), (2, 0)):
        u = torch.randn(*lead, 5, generator=gen, device=gpu_device)
        for i in (ids, ids.float(), ids.cpu(), ids[:0]):
            got = sym.gather(u, i)
            assert torch.equal(got, u[..., i.long().to(gpu_device)]) and got.device == u.device
