"""`VI`: variational inference (mirror of bayes_vi/inference/vi/vi.py)."""
import numpy as np
import torch

from ... import _native
from ...fused_target import differentiable_log_prob, replicate_from_rank0
from ..inference import Inference


def kl_reverse(logu):
    """Reverse KL in log space: f(log u) = -log u (tfp.vi.kl_reverse)."""
    return -logu


# elements of a variable up to which bvi_clip_adam_step (one workgroup) is used: 4.7 us at 1024 elements, 8.9 at 4096 and
# 95 at 65536, where bvi_adam_step takes 6.4, 6.9 and 11.7
ONE_WORKGROUP_MAX = 4096
# unconstrained parameters up to which the gradients of the ADVI surrogates are taken in closed form on the device: every
# workgroup of those kernels looks through all of them.  us a step, closed form / autograd, for 1 and 64 samples: mean-field
# 256 parameters 213 / 237 and 232 / 276, 300 parameters 246 / 240 and 273 / 284, 512 parameters 375 / 243 and 406 / 285;
# full-rank 256 parameters 271 / 280 and 288 / 329, 300 parameters 354 / 280 and 345 / 308, 512 parameters 520 / 281
FUSED_ADVI_MAX = 256


def _graph_is_alive(params):
    """Whether an autograd graph that leads to one of these leaves is alive: it holds the leaf's gradient accumulator, which
    is otherwise made anew for every graph and would not know what was noted on the one before."""
    def accumulator(p):
        with torch.enable_grad():
            return p.view_as(p).grad_fn.next_functions[0][0]

    for p in params:
        accumulator(p).metadata['bvi_seen'] = True
        if accumulator(p).metadata.pop('bvi_seen', False):
            return True
    return False


class _AdamState:
    """The update of tf.optimizers.Adam (the optimizer `VI.fit` defaults to, vi.py:77) on torch parameters:
        m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g^2
        lr_t = lr sqrt(1 - b2^t) / (1 - b1^t);  x <- x - lr_t m / (sqrt(v) + epsilon)
    (epsilon sits outside the bias correction, unlike torch.optim.Adam), after all gradients together were clipped to
    `global_clipnorm`, if given (tf.clip_by_global_norm).  The step counter lives on the parameters' device and nothing
    here reads it back, so a step can be recorded in a HIP graph."""

    def __init__(self, params, lr, betas, eps, global_clipnorm=None):
        self.params = list(params)
        self.lr, (self.b1, self.b2), self.eps = lr, betas, eps
        if global_clipnorm is not None and not float(global_clipnorm) > 0.0:
            raise ValueError('global_clipnorm must be positive, got %r' % global_clipnorm)
        self.global_clipnorm = None if global_clipnorm is None else float(global_clipnorm)
        dev = self.params[0].device if self.params else torch.device('cpu')
        self.t = torch.zeros((), dtype=torch.float64, device=dev)
        self.m = [torch.zeros_like(p) for p in self.params]
        self.v = [torch.zeros_like(p) for p in self.params]

    def zero_grad(self, set_to_none=False):
        for p in self.params:
            if p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.zero_()

    @torch.no_grad()
    def step(self):
        if self.global_clipnorm is not None:
            grads = [p.grad for p in self.params if p.grad is not None]
            if grads:
                norm = torch.sqrt(sum((g.double() * g.double()).sum() for g in grads))
                factor = torch.clamp(self.global_clipnorm / norm, max=1.0) + (norm - norm)    # NaN if norm is not finite
                for g in grads:
                    g.mul_(factor.to(g.dtype))
        self.t += 1
        lr_t = (self.lr * torch.sqrt(1.0 - self.b2 ** self.t) / (1.0 - self.b1 ** self.t)).to(torch.float32)
        for p, m, v in zip(self.params, self.m, self.v):
            if p.grad is None:
                continue
            g = p.grad
            m.mul_(self.b1).add_(g, alpha=1.0 - self.b1)
            v.mul_(self.b2).addcmul_(g, g, value=1.0 - self.b2)
            p.sub_(lr_t * m / (v.sqrt() + self.eps))

    def clip_and_step(self, clip_norm=1.0):
        """tf.clip_by_norm(grad, clip_norm) per variable (vi.py:70) followed by `step`.  On the GPU each variable is
        one launch of bvi_clip_adam_step (norm, clip, moments, update) instead of some seven element-wise kernels,
        which is most of a step's launches for a flow with a few dozen small variables.  With `global_clipnorm`, or a
        variable too large for one workgroup, all variables go through bvi_adam_step together."""
        live = [(p, g, m, v) for p, g, m, v in zip(self.params, [p.grad for p in self.params], self.m, self.v)
                if g is not None]
        on_device = bool(live) and all(p.is_cuda and p.dtype == torch.float32 and p.is_contiguous()
                                       and g.is_contiguous() and g.dtype == torch.float32 for p, g, _, _ in live)
        if not on_device:
            with torch.no_grad():
                for _, g, _, _ in live:     # without a host sync
                    g.mul_(torch.clamp(clip_norm / (g.norm() + 1e-30), max=1.0))
            self.step()
            return
        listed = self.global_clipnorm is not None or any(p.numel() > ONE_WORKGROUP_MAX for p, _, _, _ in live)
        if listed and self.global_clipnorm is None and _native.share_memory([t for row in live for t in row]):
            listed = False        # a variable twice, or one gradient for two: one after the other, as their order says
        if listed:
            if len({id(p) for p, _, _, _ in live}) != len(live):
                raise ValueError('a variable is in the optimiser twice: the step over the list would write it twice at once')
            hyper = (self.lr, self.b1, self.b2, self.eps)
            if self.global_clipnorm is None:      # the constants that bvi_clip_adam_step takes: same results to rounding
                hyper = tuple(float(np.float32(h)) for h in hyper)
            _native.adam_step(*zip(*live), self.t, *hyper, float(clip_norm), self.global_clipnorm or 0.0)
            return
        lib, ptr, st = _native.lib(), _native._ptr, _native._stream()
        with torch.no_grad():
            for i, (p, g, m, v) in enumerate(live):
                _native.check(lib.bvi_clip_adam_step(p.numel(), ptr(p), ptr(g), ptr(m), ptr(v), ptr(self.t),
                                                     1 if i == 0 else 0, self.lr, self.b1, self.b2, self.eps,
                                                     float(clip_norm), st), 'bvi_clip_adam_step')


class Adam:
    """Optimizer description with the reference's spelling, tf.optimizers.Adam(learning_rate=...);
    bound to the surrogate's parameters when `VI.fit` starts.  `global_clipnorm`: the step first clips all gradients
    together to this norm (they come clipped to norm 1 per variable from `VI.fit`, vi.py:70)."""

    def __init__(self, learning_rate=0.001, beta_1=0.9, beta_2=0.999, epsilon=1e-7, global_clipnorm=None):
        self.learning_rate, self.betas, self.eps = learning_rate, (beta_1, beta_2), epsilon
        if global_clipnorm is not None and not float(global_clipnorm) > 0.0:
            raise ValueError('global_clipnorm must be positive, got %r' % global_clipnorm)
        self.global_clipnorm = global_clipnorm

    def bind(self, params, capturable=False):
        return _AdamState(params, self.learning_rate, self.betas, self.eps, self.global_clipnorm)


class VI(Inference):
    """Same construction and `fit` signature as the reference (vi.py:37, 77-78).

    The whole dataset is one batch on the GPU (vi.py:40); `target_log_prob` is the closure of
    vi.py:46-52 on flat constrained samples [S, P(+extra)], evaluated -- value AND gradient in the
    same pass -- by the fused kernels and exposed to autograd as a single node.
    """

    def __init__(self, model, dataset, surrogate_posterior, discrepancy_fn=kl_reverse, group=None, precision=None):
        super().__init__(model=model, dataset=dataset)
        self.features, self.targets = dataset.full_batch()
        self.distribution = model.get_joint_distribution(num_samples=self.targets.shape[0], features=self.features,
                                                         group=group, precision=precision)
        self.posterior = self.distribution.posterior(self.targets)
        self.device = self.posterior.likelihood.device
        self.surrogate_posterior = surrogate_posterior.to(self.device)
        self.group = group
        # rows sharded over ranks: every rank optimises the same surrogate on the same Monte-Carlo samples, so the
        # parameters and the device's random stream are taken from rank 0
        for p in self.surrogate_posterior.parameters():
            replicate_from_rank0(p.data, group)
        if getattr(self.posterior.likelihood, 'sharded', False) or \
                getattr(getattr(self.posterior.likelihood, 'inner', None), 'sharded', False):
            seed = replicate_from_rank0(torch.tensor([torch.initial_seed() % (1 << 62)], dtype=torch.int64), group)
            torch.manual_seed(int(seed[0]))
        p = self.model.flat_param_event_ndims
        base = lambda sample: differentiable_log_prob(self.posterior, sample[:, :p].contiguous())
        self.target_log_prob = self.surrogate_posterior.get_corrected_target_log_prob_fn(base)
        self.discrepancy_fn = discrepancy_fn

    def safe_discrepancy_fn(self, logu):
        """Discrepancy with non-finite entries dropped before the mean (vi.py:55-58)."""
        d = self.discrepancy_fn(logu)
        return d[torch.isfinite(d)]

    def loss(self, sample_size):
        """Monte-Carlo variational loss with reparameterised samples
        (tfp.vi.monte_carlo_variational_loss as called at vi.py:109-116).  The mean over the finite
        discrepancies (vi.py:55-58) is taken as a masked mean: same value and gradient as
        `safe_discrepancy_fn(logu).mean()`, without the data-dependent shape (and host round trip)
        of boolean indexing."""
        q, logq = self.surrogate_posterior.sample_and_log_prob(sample_size)
        logu = self.target_log_prob(q) - logq
        d = self.discrepancy_fn(logu)
        finite = torch.isfinite(d)
        return torch.where(finite, d, torch.zeros_like(d)).sum() / finite.sum()

    # ---- ADVI (mean-field or full-rank) with the built-in priors / bijectors: the whole step on the device, no autograd ----
    def _fused_advi_eligible(self, opt):
        from .surrogate_posteriors import ADVI
        sur = self.surrogate_posterior
        if not (getattr(self, 'fused_advi', True) and isinstance(sur, ADVI) and sur.extra_ndims == 0
                and sur.unconstrained_event_ndims <= FUSED_ADVI_MAX
                and self.discrepancy_fn is kl_reverse and isinstance(opt, _AdamState) and self.device.type == 'cuda'
                and self.posterior.device_blocks() is not None):
            return False
        scale = sur.raw_scale if sur.mean_field else sur.raw_tril
        return (sur.loc.requires_grad and scale.requires_grad and scale.is_contiguous()
                and [id(p) for p in opt.params] == [id(sur.loc), id(scale)])

    def _step_fused_advi(self, opt, sample_size):
        """One step of `_step` for the ADVI surrogates (mean-field, full-rank) when the model's priors and bijectors are the
        device-side ones: sample -> constrain -> fused data pass -> assemble -> closed-form ELBO gradients ->
        per-variable clip + Adam, eight launches (surrogate_posteriors.py:113-123, vi.py:55-75, 109-116).  Same
        loss, clipped gradients (left in `.grad`) and parameters as autograd over the same formulas."""
        lib, ptr, st = _native.lib(), _native._ptr, _native._stream()
        sur, post = self.surrogate_posterior, self.posterior
        s, pu = int(sample_size), sur.unconstrained_event_ndims
        eps = sur.base_noise(s, pu).contiguous()
        b = getattr(self, '_advi_bufs', None)
        if b is None or b['z'].shape != (s, pu):
            f = lambda *shape: torch.empty(*shape, dtype=torch.float32, device=self.device)
            b = self._advi_bufs = dict(z=f(s, pu), loss=f(()))
        scale = sur.raw_scale if sur.mean_field else sur.raw_tril
        sample, grads = ((lib.bvi_advi_meanfield_sample, lib.bvi_advi_meanfield_grads) if sur.mean_field
                         else (lib.bvi_advi_fullrank_sample, lib.bvi_advi_fullrank_grads))
        for prm in (sur.loc, scale):
            if prm.grad is None:
                prm.grad = torch.zeros_like(prm)
        with torch.no_grad():
            _native.check(sample(s, pu, ptr(eps), ptr(sur.loc), ptr(scale), ptr(b['z']), st), 'bvi_advi_*_sample')
            lp, gz = post.unconstrained_log_prob_and_grad(b['z'], True)
            _native.check(grads(s, pu, ptr(lp), ptr(gz), ptr(eps), ptr(scale), ptr(b['loss']), ptr(sur.loc.grad),
                                ptr(scale.grad), st), 'bvi_advi_*_grads')
        opt.clip_and_step(1.0)
        return b['loss'].clone()

    def _step(self, opt, params, sample_size):
        if self._fused_advi_eligible(opt):
            return self._step_fused_advi(opt, sample_size)
        opt.zero_grad(set_to_none=False)
        loss = self.loss(sample_size)
        loss.backward()
        if isinstance(opt, _AdamState):
            opt.clip_and_step(1.0)
        else:
            for p in params:
                if p.grad is not None:     # tf.clip_by_norm(grad, 1.0), without a host sync
                    p.grad.mul_(torch.clamp(1.0 / (p.grad.norm() + 1e-30), max=1.0))
            opt.step()
        return loss.detach()

    def fit(self, optimizer=None, num_steps=10000, sample_size=1, num_samples_to_approx_marginals=10000,
            progress_bar=True, capture_graph=None):
        """Returns (approx_posterior, losses[num_steps]) (vi.py:77-127).  Every gradient is clipped
        to norm 1 per variable, not globally (vi.py:70).

        `capture_graph` (default: on for GPU runs with the built-in `Adam`): after three eager steps
        the whole step -- sampling, fused log-posterior pass, backward, clipping, optimizer update -- is
        captured once as a HIP graph and replayed, which removes the per-kernel launch cost that
        dominates on small datasets.  The steps and their results are the same either way.  A loss that the caller
        evaluated beforehand and still holds keeps the parameters' gradient accumulators on the stream it ran on, and a
        captured backward pass that waits for that stream ends the process: by default the steps then stay eager (of the
        surrogates whose step takes a backward pass), and `capture_graph=True` raises."""
        optimizer = optimizer if optimizer is not None else Adam()
        params = [p for p in self.surrogate_posterior.parameters() if p.requires_grad]
        on_gpu, asked = self.device.type == 'cuda', bool(capture_graph)
        if capture_graph is None:
            # a row-sharded likelihood has a collective inside the step: that stays eager unless asked for
            lik = self.posterior.likelihood
            sharded = getattr(lik, 'sharded', False) or getattr(getattr(lik, 'inner', None), 'sharded', False)
            capture_graph = on_gpu and hasattr(optimizer, 'bind') and num_steps > 8 and not sharded
        if capture_graph and not (on_gpu and hasattr(optimizer, 'bind')):
            raise ValueError('capture_graph needs a GPU run and the built-in Adam description')
        if hasattr(optimizer, 'bind'):
            opt = optimizer.bind(params, capturable=True) if capture_graph else optimizer.bind(params)
        else:
            opt = optimizer(params)
        if capture_graph and not self._fused_advi_eligible(opt) and _graph_is_alive(params):
            if asked:
                raise ValueError('capture_graph: an autograd graph of the surrogate\'s parameters is still alive (a loss that '
                                 'was evaluated before and is held somewhere); drop it, or fit without capture')
            capture_graph = False
        losses_dev = torch.zeros(num_steps, dtype=torch.float32, device=self.device)
        bar = None
        if progress_bar:
            try:
                from tqdm import tqdm
                bar = tqdm(total=num_steps, leave=False)
            except Exception:
                bar = None
        n_eager = min(num_steps, 3) if capture_graph else num_steps
        for i in range(n_eager):
            losses_dev[i] = self._step(opt, params, sample_size)
            if bar is not None:
                bar.update(1)
        if capture_graph and num_steps > n_eager:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                static_loss = self._step(opt, params, sample_size)
            for i in range(n_eager, num_steps):
                graph.replay()
                losses_dev[i] = static_loss
                if bar is not None and (i & 63) == 0:
                    bar.update(64)
        if bar is not None:
            bar.close()
        losses = losses_dev.cpu().numpy().astype(np.float64)
        approx_posterior = self.surrogate_posterior.approx_joint_marginal_posteriors(num_samples_to_approx_marginals)
        return approx_posterior, losses

    def stochastic_fit(self, *args, **kwargs):
        raise NotImplementedError('minibatch fitting is outside the fused full-batch hot path')
