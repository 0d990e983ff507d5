"""Operators over rows of vocabulary logits ``[N, V]`` (fp32 or bf16, unit stride along the
vocabulary, any row stride, V up to 262144, on the GPU fewer than 2^22 rows), beside the
cross-entropy and the sampling step:

* :func:`top_logits` -- what a teacher records of its answer: the k largest logits of a row and
  the log-sum-exp at a temperature;
* :func:`distill_xent` / :func:`distill_loss` -- a student's loss against such a record, with
  its gradient in the same pass, or through autograd;
* :func:`sample_logits` -- one id a row from one uniform number a row, under temperature, top-k,
  top-p and min-p.

GPU tensors take the HIP kernels (csrc/topk.hip, distill.hip, filter.hip), CPU tensors the plain
forms at the end.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import native

MAX_V = 262144  # csrc/kernels.h kRowMaxV
MAX_K = 256     # csrc/kernels.h kRowMaxK: recorded entries a row

Opt = Optional[torch.Tensor]
Setting = Union[float, torch.Tensor]


class Distill(NamedTuple):
    """What a training step is given of a teacher (``CharRNN.train_step``): its record of the
    batch, time-major, and how the loss weighs it (see :func:`distill_xent`)."""

    values: torch.Tensor   # [T, B, k] fp32
    indices: torch.Tensor  # [T, B, k] int32
    lse: Opt               # [T, B] fp32, at `temperature`
    alpha: float
    temperature: float

    def check(self, T: int, B: int) -> None:
        """Raises unless the record is one of a batch of ``B`` sequences of ``T``: a batch-major one
        has as many rows, in another order."""
        v, want = self.values, (T, B)
        if v.dim() != 3 or tuple(v.shape[:2]) != want:
            raise ValueError(f"a record's values must be [T, B, k] = [{T}, {B}, k], "
                             f"got {list(v.shape)}")
        if self.indices.shape != v.shape:
            raise ValueError(f"a record's indices must be {list(v.shape)} as its values, "
                             f"got {list(self.indices.shape)}")
        if self.lse is not None and tuple(self.lse.shape) != want:
            raise ValueError(f"a record's lse must be [T, B] = [{T}, {B}], "
                             f"got {list(self.lse.shape)}")


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(values [N, k] fp32, indices [N, k] int32, lse [N] fp32)``: the ``k`` (at most 256)
    largest logits of each row, largest first and the lowest index first among equals, and
    ``log sum exp(logits / temperature)`` over the whole row.  NaN counts as -inf in the order
    and makes the row's ``lse`` NaN."""
    if logits.is_cuda:
        return native.op("top_logits")(logits, k, temperature)
    _check_logits(logits)
    torch._check(1 <= k <= min(MAX_K, logits.shape[1]), lambda: f"k must be 1 to {MAX_K} and V")
    _check_temperature(temperature)
    z = logits.float()
    lse = torch.logsumexp(z / temperature, 1)
    z = torch.where(z.isnan(), -math.inf, z)
    values, indices = torch.sort(z, dim=1, descending=True, stable=True)
    return values[:, :k].contiguous(), indices[:, :k].to(torch.int32).contiguous(), lse


def distill_xent(logits: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, *,
                 top_lse: Opt = None, targets: Opt = None, alpha: float = 1.0,
                 temperature: float = 1.0, scale: Optional[float] = None,
                 grad_dtype: Optional[torch.dtype] = None, grad: Opt = None
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss, row losses [N], gradient [N, V])`` of a student's ``logits`` against a teacher's
    recorded entries ``values`` / ``indices`` ``[N, k]`` (:func:`top_logits`), in one pass:

        row  = alpha T^2 KL(q || softmax(logits / T)) + (1 - alpha) xent(logits, target)
        loss = scale * sum of the rows                       (scale: 1 / N by default)

    ``top_lse`` (the teacher's log-sum-exp at the same temperature T) makes ``q`` the teacher's
    own probabilities, and what they leave of 1 is held against what the student gives to all
    other tokens together.  Without it ``q`` is the softmax over the entries alone.

    An entry whose index is not in ``[0, V)`` is none (rows with fewer than k entries are padded
    with -1); a token recorded twice counts with both values.  A row whose target is not in
    ``[0, V)`` is padding, as is one whose logits are all -inf: loss and gradient are zero there.
    A record that holds nothing -- all values -inf, and ``top_lse`` too where it is given, as
    :func:`top_logits` answers to a row of nothing but -inf -- has no divergence.

    The gradient is written in ``grad_dtype`` (the logits' by default) or into ``grad``, which may
    be the logits themselves, but else shares no memory with them."""
    if scale is None:
        scale = 1.0 / max(1, logits.shape[0])
    if not logits.is_cuda:
        return _cpu_distill_xent(logits, values, indices, top_lse, targets, alpha, temperature,
                                 scale, grad_dtype, grad)
    if grad is None:
        return native.op("distill_xent")(logits, values, indices, top_lse, targets, alpha,
                                         temperature, scale, grad_dtype)
    row, loss = _outputs(logits)
    native.op("distill")(logits, values, indices, top_lse, targets, alpha, temperature, scale,
                         None, row, grad, loss)
    return loss, row, grad


def distill_loss(logits: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, *,
                 top_lse: Opt = None, targets: Opt = None, alpha: float = 1.0,
                 temperature: float = 1.0, scale: Optional[float] = None) -> torch.Tensor:
    """The loss of :func:`distill_xent`, differentiable (once) in ``logits``."""
    return distill_loss_rows(logits, values, indices, top_lse=top_lse, targets=targets,
                             alpha=alpha, temperature=temperature, scale=scale)[0]


def distill_loss_rows(logits, values, indices, *, top_lse=None, targets=None, alpha=1.0,
                      temperature=1.0, scale=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`distill_loss` and the row losses (without a gradient of their own)."""
    if scale is None:
        scale = 1.0 / max(1, logits.shape[0])
    return _DistillLoss.apply(logits, values, indices, top_lse, targets, alpha, temperature,
                              scale)


class _DistillLoss(torch.autograd.Function):
    """The backward runs the same pass with the incoming gradient as a factor: it reads the
    logits a second time instead of keeping a gradient of their size from the forward."""

    @staticmethod
    def forward(ctx, logits, values, indices, lse, targets, alpha, temperature, scale):
        ctx.save_for_backward(logits, values, indices, lse, targets)
        ctx.args = (alpha, temperature, scale)
        if not logits.is_cuda:
            loss, row, _ = _cpu_distill_xent(logits, values, indices, lse, targets, alpha,
                                             temperature, scale, None, None)
        else:
            row, loss = _outputs(logits)
            native.op("distill")(logits, values, indices, lse, targets, alpha, temperature,
                                 scale, None, row, None, loss)
        ctx.mark_non_differentiable(row)
        return loss, row

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        logits, values, indices, lse, targets = ctx.saved_tensors
        alpha, temperature, scale = ctx.args
        if not logits.is_cuda:
            grad = _cpu_distill_xent(logits, values, indices, lse, targets, alpha, temperature,
                                     scale, torch.float32, None)[2]
            grad = (grad * g).to(logits.dtype)
        else:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            row = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
            native.op("distill")(logits, values, indices, lse, targets, alpha, temperature, scale,
                                 g, row, grad, None)
        return (grad,) + (None,) * 7


def sample_logits(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Setting = 1.0,
                  min_p: Setting = 0.0) -> torch.Tensor:
    """One id a row (int32 ``[N]``) from uniform numbers ``u`` (fp32 ``[N]`` in [0, 1)).

    Tokens are ordered by logit, the lowest index first among equals, and weigh
    ``exp((logit - max) / temperature)``.  Kept are the first ``top_k`` of the order (0: all); of
    these the tokens in front of which less than ``top_p`` of their weight lies (1: all); of
    these the ones that weigh at least ``min_p`` times the first.  The first of the order is
    always kept.  Drawn is, in the order of the indices, the first kept token at which the
    running weight passes ``u`` times the whole.  Temperature 0 gives the first of the order.

    Every setting is a number, or a tensor with one per row (fp32; ``top_k`` int32), where
    ``top_k`` below 1 and NaN mean no filter, ``top_p`` below 0 counts as 0, ``min_p`` above 1 as
    1, and a temperature below 0 or NaN as 0.  NaN logits count as -inf; a row of nothing else
    gives 0.  Weights are added as whole numbers of 2^-44 of the first's, so the answer does not
    depend on the order of any sum; a token that weighs less than half of that is never drawn."""
    if not logits.is_cuda:
        return _cpu_sample(logits, u, temperature, top_k, top_p, min_p)
    t, ts = _setting(temperature, 1.0)
    k, ks = _setting(top_k, 0)
    p, ps = _setting(top_p, 1.0)
    q, qs = _setting(min_p, 0.0)
    return native.op("filter_sample")(logits, u, t, k, p, q, ts, ks, ps, qs)


def _setting(v, default):
    return (default, v) if isinstance(v, torch.Tensor) else (v, None)


def _outputs(logits):
    f32 = dict(dtype=torch.float32, device=logits.device)
    return torch.empty(logits.shape[0], **f32), torch.empty((), **f32)


# ---- plain forms (CPU) -----------------------------------------------------------------------
def _check_logits(logits):
    ok = torch._check
    ok(logits.dim() == 2, lambda: "logits must be [N, V]")
    ok(logits.dtype in (torch.float32, torch.bfloat16), lambda: "logits must be float32 or bfloat16")
    ok(1 <= logits.shape[1] <= MAX_V, lambda: f"vocabularies of 1 to {MAX_V} entries")
    ok(logits.shape[1] == 1 or logits.stride(1) == 1,
       lambda: "logits need unit stride along the vocabulary")


def _check_temperature(t):
    both = torch.tensor([t, 1.0 / t if t > 0 else 0.0], dtype=torch.float64).float()  # as used
    torch._check(bool((both > 0).all() and both.isfinite().all()),
                 lambda: f"the temperature must be positive and finite, got {t}")


def _check_rows(t, logits, dtype, shape, name):
    torch._check(t.shape == shape and t.dtype == dtype and t.device == logits.device
                 and t.is_contiguous(), lambda: f"{name} must be {tuple(shape)} {dtype}, contiguous")


def _cpu_distill_xent(logits, values, indices, lse, targets, alpha, tau, scale, grad_dtype, grad):
    _check_logits(logits)
    n, v = logits.shape
    ok = torch._check
    ok(values.dim() == 2 and 1 <= values.shape[1] <= MAX_K, lambda: f"1 to {MAX_K} entries a row")
    shape = (n, values.shape[1])
    _check_rows(values, logits, torch.float32, shape, "values")
    _check_rows(indices, logits, torch.int32, shape, "indices")
    _check_temperature(tau)
    ok(0 <= alpha <= 1, lambda: "alpha must be in [0, 1]")
    ok(alpha == 1 or targets is not None, lambda: "alpha < 1 needs targets")
    ok(math.isfinite(scale), lambda: "scale must be finite")
    kind = (grad_dtype or logits.dtype) if grad is None else grad.dtype
    ok(kind in (torch.float32, torch.bfloat16), lambda: "grad must be float32 or bfloat16")
    if grad is not None:
        ok(grad.device == logits.device and grad.shape == logits.shape
           and (v == 1 or grad.stride(1) == 1) and (n <= 1 or grad.stride(0) >= v),
           lambda: "grad must be [N, V] on the logits' device, unit stride along the vocabulary, "
                   "rows apart")
    z = logits.float()
    idx = indices.long()
    here = (idx >= 0) & (idx < v)
    idx = idx.clamp(0, v - 1)
    skip = torch.isneginf(z).all(1)
    if lse is not None:
        _check_rows(lse, logits, torch.float32, (n,), "top_lse")
    if targets is not None:
        _check_rows(targets, logits, torch.int32, (n,), "targets")
        skip = skip | (targets < 0) | (targets >= v)
    z = torch.where(skip[:, None], 0.0, z)
    z = z - torch.where(skip[:, None], 0.0, z.max(1, keepdim=True).values)
    logp = torch.log_softmax(z / tau, 1)
    t = torch.where(here, values / tau, -math.inf)
    some = ~torch.isneginf(t).all(1)
    if lse is not None:
        some = some | ~torch.isneginf(lse)
    base = torch.logsumexp(t, 1) if lse is None else lse
    logq = t - torch.where(some, base, 0.0)[:, None]
    q = logq.exp()
    kl = torch.where(q > 0, q * (logq - logp.gather(1, idx)), 0.0).sum(1)
    g = logp.exp()
    if lse is not None:
        entry = torch.zeros(n, v + 1).scatter_(
            1, torch.where(here, idx, v), 1.0)[:, :v].bool()
        rest = (1.0 - q.sum(1)).clamp_min(0.0)
        out = torch.logsumexp(torch.where(entry, -math.inf, logp), 1)
        left = (rest > 0) & ~torch.isneginf(out)
        kl = kl + torch.where(left, rest * (rest.log() - out), 0.0)
        gone = torch.where(left, rest.log() - out, -math.inf)[:, None]
        g = torch.where(entry, g, g - torch.where(left[:, None], (logp + gone).exp(), 0.0))
    kl = torch.where(some, kl, 0.0)
    g = (g.scatter_add(1, idx, -torch.where(here, q, 0.0))) * (alpha * tau) * some.float()[:, None]
    row = alpha * tau * tau * kl
    if targets is not None and alpha < 1:
        y = targets.long().clamp(0, v - 1)[:, None]
        lp = torch.log_softmax(z, 1)
        row = row - (1 - alpha) * lp.gather(1, y)[:, 0]
        g = g + (1 - alpha) * lp.exp().scatter_add(1, y, -torch.ones(n, 1))
    row = torch.where(skip, 0.0, row)
    g = torch.where(skip[:, None], 0.0, g * scale).to(grad_dtype or logits.dtype)
    if grad is not None:
        grad.copy_(g)
        g = grad
    return row.sum() * scale, row, g


def _cpu_sample(logits, u, temperature, top_k, top_p, min_p):
    _check_logits(logits)
    n, v = logits.shape
    ok = torch._check
    _check_rows(u, logits, torch.float32, (n,), "u")

    def row(x, dtype, good, name):
        if isinstance(x, torch.Tensor):
            _check_rows(x, logits, dtype, (n,), name)
            return x.double()[:, None]
        ok(good(x), lambda: f"{name} is out of range: {x}")
        return torch.full((n, 1), x, dtype=dtype).double()

    f32 = torch.float32
    temp = row(temperature, f32, lambda x: x >= 0 and math.isfinite(x), "temperature")
    k = row(top_k if isinstance(top_k, torch.Tensor) else min(top_k, v), torch.int32,
            lambda x: x >= 0, "top_k")
    p = row(top_p, f32, lambda x: 0 <= x <= 1, "top_p")
    q = row(min_p, f32, lambda x: 0 <= x <= 1, "min_p").clamp_max(1.0)
    z = logits.double()
    z = torch.where(z.isnan(), -math.inf, z)
    zs, order = torch.sort(z, dim=1, descending=True, stable=True)
    top = zs[:, :1]
    first = ~(temp > 0) | torch.isneginf(top)
    w = torch.exp((zs - top) / torch.where(temp > 0, temp, 1.0))
    w = torch.where(zs == top, 1.0, torch.where(torch.isneginf(zs) | torch.isposinf(top), 0.0, w))
    rank = torch.arange(v)[None]
    units = torch.round(w * 2.0 ** 44).long()
    units = torch.where((k <= 0) | (rank < k), units, 0)
    before = torch.cumsum(units, 1) - units
    share = torch.ceil(torch.where(p < 1, p, 1.0).clamp_min(0.0) * units.sum(1, keepdim=True).double())
    keep = ~(p < 1) | (rank == 0) | (before < share.long())
    keep &= ~(w < q) | (rank == 0)
    units = torch.zeros_like(units).scatter_(1, order, torch.where(keep, units, 0))
    cdf = torch.cumsum(units, 1)
    total = cdf[:, -1:].contiguous()
    r = u.double()[:, None]
    r = torch.minimum((torch.where(r > 0, r, 0.0).clamp_max(1.0) * total.double()).long(), total - 1)
    pick = torch.searchsorted(cdf, r, right=True)
    return torch.where(first, order[:, :1], pick)[:, 0].to(torch.int32)
