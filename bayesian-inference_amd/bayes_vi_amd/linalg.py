"""The handful of `tf.linalg` functions the reference's likelihood callables use
(exploratory_experiments/multivariate-gaussian-test.ipynb cell 15: `cholesky_solve`, `eye`), on torch tensors and on
the symbolic stand-ins a likelihood is recognised with (`bayes_vi_amd.symbolic`); and, for training, `global_norm` and
`clip_by_global_norm` (tf.linalg.global_norm, tf.clip_by_global_norm) over lists of gradients, on the gfx950 kernels."""
from __future__ import annotations

import torch

from . import _native
from . import symbolic as sym


class Eye:
    """tf.linalg.eye(d) as written inside a likelihood callable."""

    def __init__(self, d):
        self.d = int(d)

    def tensor(self, like):
        return torch.eye(self.d, dtype=like.dtype, device=like.device)


def eye(num_rows):
    return Eye(num_rows)


def cholesky_solve(chol, rhs):
    """tf.linalg.cholesky_solve(chol, rhs): X with (chol chol^T) X = rhs.  With a symbolic parameter and `eye` as
    right-hand side it returns the description `CholeskySolveIdentity` (the full inverse (chol chol^T)^-1); with
    tensors, the solution [..., D, M] (only the lower triangle of `chol` is read)."""
    if isinstance(chol, sym.ParamSym):
        d = int(round(chol.size ** 0.5))
        if chol.index is not None or d * d != chol.size or not isinstance(rhs, Eye) or rhs.d != d:
            raise sym.UnsupportedLikelihood('cholesky_solve is fused for a whole [D, D] parameter and eye(D) only')
        return sym.CholeskySolveIdentity(chol)
    chol = torch.as_tensor(chol)
    b = rhs.tensor(chol) if isinstance(rhs, Eye) else torch.as_tensor(rhs, dtype=chol.dtype, device=chol.device)
    return torch.cholesky_solve(b.expand(chol.shape[:-2] + b.shape[-2:]), torch.tril(chol))


def _listed(t_list, what):
    if not isinstance(t_list, (list, tuple)):
        raise TypeError('%s takes a list of tensors, got %s' % (what, type(t_list).__name__))
    live = [t for t in t_list if t is not None]
    if not live:
        raise ValueError('%s: no tensor in the list' % what)
    return live, _native.tensor_list(live, what)


def global_norm(t_list):
    """tf.linalg.global_norm: sqrt of the sum of all squares of a list of GPU tensors (float32, bfloat16, float16, mixed;
    None entries are skipped), a float32 scalar on the device.  Squares are summed in double.  Not differentiable."""
    live, device = _listed(t_list, 'global_norm')
    with torch.no_grad():
        return _native.global_norm([t.contiguous() for t in live], device)


def clip_by_global_norm(t_list, clip_norm, use_norm=None, inplace=False):
    """tf.clip_by_global_norm: (the tensors times min(1, clip_norm / norm), norm).  `use_norm`: a float32 scalar on the
    device to use instead of the list's own norm (for instance one reduced over ranks).  Where the norm is not finite
    every entry becomes NaN, as in tf.  None entries stay None.  `inplace=True` writes the tensors themselves (contiguous
    ones, no two of them overlapping) and returns them; nothing is written where nothing has to be clipped.  Nothing
    synchronises.  Not differentiable."""
    live, device = _listed(t_list, 'clip_by_global_norm')
    clip_norm = float(clip_norm)
    if not clip_norm > 0.0:
        raise ValueError('clip_norm must be positive, got %r' % clip_norm)
    if use_norm is not None:
        if not (isinstance(use_norm, torch.Tensor) and use_norm.dtype == torch.float32 and use_norm.numel() == 1
                and use_norm.device == device):
            raise ValueError('use_norm must be one float32 on %s' % device)
    if inplace:
        if not all(t.is_contiguous() for t in live):
            raise ValueError('clip_by_global_norm(inplace=True) needs contiguous tensors')
        if _native.share_memory(live):
            raise ValueError('clip_by_global_norm(inplace=True): two tensors of the list overlap')
        if use_norm is not None and any(_native.share_memory([t, use_norm]) for t in live):
            raise ValueError('clip_by_global_norm(inplace=True): use_norm lies in a tensor of the list, which is written')
        src = out = live
    else:
        with torch.no_grad():
            src = [t.contiguous() for t in live]
            out = [torch.empty_like(t) for t in src]
    norm = _native.clip_by_global_norm(src, out, clip_norm, use_norm, device)
    if inplace:
        torch.autograd.graph.increment_version(live)
        return list(t_list), norm
    if len(live) == len(t_list):
        return out, norm
    result = iter(out)
    return [None if t is None else next(result) for t in t_list], norm
