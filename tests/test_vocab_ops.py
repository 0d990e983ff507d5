"""Operators over vocabulary rows (ops/vocab.py; csrc/topk.hip, distill.hip, filter.hip) against
plain float64 forms, on the CPU and on the GPU.

Tolerances.  u = 2^-24.  A log-sum-exp of numbers up to L is off by its own rounding, that of the
scaled logits (2 u L), and some 16 u of the sum.  A probability has the relative error of its
exponent, (2 L + 32) u with L the largest |logit| / T; the teacher's rest 1 - sum q adds k u.
Gradients are sums of probabilities times alpha T, 1 - alpha and the scale; losses are
probabilities times log-probabilities, bounded with the largest of them.  A bf16 gradient adds
half a step, 2^-8 relative.  Whole numbers are equal."""
import math

import pytest
import torch

from distributed_char_rnn_amd.ops import vocab as O

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
INF, NAN = math.inf, math.nan


def rows(N, V, dtype, dev, seed=0, spread=2.5, pad=0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(N, V + pad, generator=g) * spread).to(dtype).to(dev)
    return z[:, :V]


# ---- top_logits ------------------------------------------------------------------------------
def check_top(z, k, t=1.0):
    values, indices, lse = O.top_logits(z, k, t)
    d = z.double().cpu()
    clean = torch.where(d.isnan(), -INF, d)
    want = torch.sort(clean, dim=1, descending=True, stable=True)
    assert torch.equal(values.double().cpu(), want.values[:, :k])
    assert torch.equal(indices.long().cpu(), want.indices[:, :k])
    assert values.dtype == F32 and indices.dtype == torch.int32
    ref = torch.logsumexp(d / t, 1)
    got = lse.double().cpu()
    same = (got == ref) | (got.isnan() & ref.isnan())
    L = torch.where(clean.isinf(), 0.0, clean).abs().max() / t
    assert (same | ((got - ref).abs() <= (4 * L + 32) * U)).all(), (got, ref)


TOP = [(1, 1, 1), (3, 2, 2), (5, 65, 1), (50, 65, 16), (7, 65, 65), (4, 256, 256), (3, 257, 33),
       (2, 1000, 256), (3, 1024, 7), (3, 1025, 64), (2, 4099, 200), (2, 8192, 64), (2, 8193, 9)]
TOP_GPU = [(3, 32001, 50), (2, 65536, 256), (2, 65537, 3), (2, 131072, 100), (1, 262144, 256),
           (3000, 300, 20)]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,V,k", TOP)
def test_top(N, V, k, dtype, dev):
    check_top(rows(N, V, dtype, dev), k, 0.7)
    check_top(rows(N, V, dtype, dev, seed=1, pad=3), k, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,V,k", TOP_GPU)
def test_top_large(N, V, k, dtype):
    check_top(rows(N, V, dtype, "cuda", pad=1), k, 2.0)


def hard_rows(V, dtype, dev):
    """Rows of equal values, few values, masks, infinities, NaN and signed zeros."""
    g = torch.Generator().manual_seed(3)
    z = torch.randn(11, V, generator=g)
    z[0] = 1.25
    z[1] = torch.randint(0, 3, (V,), generator=g).float()
    z[2] = -INF
    z[3, torch.rand(V, generator=g) < 0.8] = -INF
    z[4] = torch.finfo(torch.bfloat16).min
    z[5, V // 2:] = NAN
    z[6, V // 3] = INF
    z[7] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
    z[8] = NAN
    z[9] = torch.arange(V).float() / V
    z[10] = 0.0
    z[10, -1] = 1.0
    return z.to(dtype).to(dev)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [5, 65, 300, 1500, 5000])
def test_top_hard_rows(V, dtype, dev):
    for k in sorted({1, min(V, 4), min(V, 60), min(V, 256)}):
        check_top(hard_rows(V, dtype, dev), k)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [20000, 40001, 70001])
def test_top_hard_rows_large(V):
    check_top(hard_rows(V, F32, "cuda"), 256)
    check_top(hard_rows(V, BF16, "cuda"), 19)


# ---- distillation ----------------------------------------------------------------------------
def reference_distill(z, values, indices, lse, targets, alpha, tau, scale):
    """float64 from log-probabilities, the gradient by automatic differentiation; row by row."""
    z = z.detach().double().cpu()
    V = z.shape[1]
    loss, grads = [], []
    for n in range(z.shape[0]):
        zn = z[n].clone().requires_grad_(True)
        y = None if targets is None else int(targets[n])
        if (y is not None and not 0 <= y < V) or bool(torch.isneginf(z[n]).all()):
            loss.append(torch.zeros((), dtype=torch.float64))
            grads.append(torch.zeros(V, dtype=torch.float64))
            continue
        lp = torch.log_softmax(zn / tau, 0)
        idx = indices[n].long().cpu()
        ok = (idx >= 0) & (idx < V)
        idx, t = idx[ok], values[n].double().cpu()[ok] / tau
        row = torch.zeros((), dtype=torch.float64)
        if lse is not None:
            lq = t - float(lse[n])
            rest = 1.0 - lq.exp().sum()
            others = torch.ones(V, dtype=torch.bool)
            others[idx] = False
            out = lp[others & ~torch.isneginf(z[n])]
            if rest > 0 and out.numel():
                row = row + rest * (rest.log() - torch.logsumexp(out, 0))
        else:
            lq = torch.log_softmax(t, 0) if idx.numel() and not torch.isneginf(t).all() else None
        if lq is not None:
            some = lq > -INF
            row = row + (lq[some].exp() * (lq[some] - lp[idx[some]])).sum()
        row = alpha * tau * tau * row
        if y is not None and alpha < 1:
            row = row - (1 - alpha) * torch.log_softmax(zn, 0)[y]
        g = torch.autograd.grad(row, zn)[0] if row.requires_grad else torch.zeros_like(z[n])
        loss.append(row.detach())
        grads.append(g * scale)
    return torch.stack(loss), torch.stack(grads)


def record(z, k, tau, seed=5):
    g = torch.Generator().manual_seed(seed)
    t = z.float().cpu() + torch.randn(z.shape, generator=g)
    top = torch.topk(t, k, dim=1)
    return (top.values.to(z.device), top.indices.int().to(z.device),
            torch.logsumexp(t / tau, 1).to(z.device))


def check_distill(z, values, indices, lse, targets, alpha, tau, gtype=None):
    N, V = z.shape
    loss, row, grad = O.distill_xent(z, values, indices, top_lse=lse, targets=targets, alpha=alpha,
                                     temperature=tau, grad_dtype=gtype)
    want, gwant = reference_distill(z, values, indices, lse, targets, alpha, tau, 1.0 / N)
    k = values.shape[1]
    fine = torch.where(z.isinf(), 0.0, z.float()).abs().max().item()
    L = max(fine, values[~values.isinf()].abs().max().item() if (~values.isinf()).any() else 0)
    L = max(L, L / tau)
    top = 2 * L + math.log(V) + 20  # the largest log-probability or log of the rest
    bound = (2 * L + 64 + 2 * k) * U
    assert row.dtype == F32 and grad.dtype == (gtype or z.dtype)
    assert ((row.double().cpu() - want).abs() <= bound * (alpha * tau * tau + 1) * top).all(), \
        (row.cpu(), want)
    assert abs(loss.item() - want.sum().item() / N) <= bound * (alpha * tau * tau + 1) * top
    half = 2.0 ** -8 if grad.dtype == BF16 else 0.0
    err = (grad.double().cpu() - gwant).abs()
    allowed = bound * (alpha * tau + 1) / N
    assert (err <= allowed + half * (gwant.abs() + allowed)).all(), (err.max(), allowed)
    return loss, row, grad


DISTILL = [(1, 1, 1), (2, 2, 1), (3, 65, 8), (50, 65, 65), (7, 256, 16), (5, 257, 256),
           (3, 1000, 3), (2, 1024, 64), (3, 1030, 40), (2, 4097, 100), (2, 8192, 64)]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype,gtype", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("N,V,k", DISTILL)
def test_distill(N, V, k, dtype, gtype, dev):
    z = rows(N, V, dtype, dev, pad=N % 3)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(1)).int().to(dev)
    for tau, alpha, tail in ((1.0, 1.0, True), (2.0, 0.6, True), (0.5, 0.3, False),
                             (1.0, 0.5, False), (3.0, 1.0, False), (1.0, 0.0, True)):
        values, indices, lse = record(z, k, tau)
        check_distill(z, values, indices, lse if tail else None, y if alpha < 1 else None, alpha,
                      tau, gtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gtype", [(F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("N,V,k", [(3, 32001, 32), (2, 65536, 256), (2, 70001, 64), (1, 262144, 9),
                                   (5000, 65, 8)])
def test_distill_large(N, V, k, dtype, gtype):
    z = rows(N, V, dtype, "cuda")
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(1)).int().cuda()
    values, indices, lse = record(z, k, 2.0)
    check_distill(z, values, indices, lse, y, 0.7, 2.0, gtype)
    check_distill(z, values, indices, None, None, 1.0, 2.0, gtype)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [65, 1500])
def test_distill_odd_records(V, dev):
    """Padded entries, entries recorded twice, values of -inf, padded rows, masked students."""
    N, k = 9, 12
    z = rows(N, V, F32, dev)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(1)).int().to(dev)
    values, indices, lse = record(z, k, 2.0)
    lse = lse + 0.5
    indices[0, 5:] = -1
    indices[1] = -1
    indices[2, 3:] = V
    indices[3, 4] = indices[3, 1]
    indices[3, 9] = indices[3, 1]
    indices[4] = indices[4, 0]
    values[5, 2:] = -INF
    values[6] = -INF
    y[7] = -1
    z[8] = -INF
    for lz in (lse, None):
        for alpha in (0.4, 1.0):
            _, row, grad = check_distill(z, values, indices, lz, y, alpha, 2.0)
            assert row[7] == 0 and row[8] == 0
            assert (grad[7] == 0).all() and (grad[8] == 0).all()
    # masked columns of the student that nobody asks for have no part and no gradient
    z = rows(N, V, F32, dev, seed=4)
    values, indices, lse = record(z, k, 1.0)
    masked = torch.ones(N, V, dtype=torch.bool, device=dev)
    masked.scatter_(1, indices.long(), False)
    masked.scatter_(1, y.clamp_min(0).long()[:, None], False)
    masked &= (torch.rand(N, V, generator=torch.Generator().manual_seed(2)) < 0.5).to(dev)
    z.masked_fill_(masked, -INF)
    _, _, grad = check_distill(z, values, indices, lse + 0.1, y, 0.5, 1.0)
    assert (grad[masked] == 0).all()
    # a student sure of the recorded tokens: the rest's share keeps its digits
    z = torch.full((2, V), -40.0, device=dev)
    z[:, :2] = 40.0
    values = torch.tensor([[2.0, 1.0]] * 2, device=dev)
    indices = torch.tensor([[0, 1]] * 2, dtype=torch.int32, device=dev)
    check_distill(z, values, indices, torch.full((2,), 2.6, device=dev), None, 1.0, 1.0)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [65, 1500, 40001])
@pytest.mark.parametrize("alpha", [0.4, 1.0])
def test_distill_teacher_row_without_tokens(V, alpha, dev):
    """A teacher's row that its mask leaves empty records -inf throughout: it says nothing, and the
    target's part of the loss stays."""
    N, k, tau = 4, 7, 2.0
    t, z = rows(N, V, F32, dev, seed=1), rows(N, V, F32, dev, seed=2)
    t[1] = -INF
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(1)).int().to(dev)
    y[3] = -1
    values, indices, lse = O.top_logits(t, k, tau)
    assert lse[1] == -INF and (values[1] == -INF).all()
    for record_of in ((values, indices), (values, torch.where(values > -INF, indices, -1))):
        _, row, grad = O.distill_xent(z, *record_of, top_lse=lse, targets=y, alpha=alpha,
                                      temperature=tau)
        # a finite log-sum-exp and the other rows: as they were
        want, gwant = reference_distill(z, values, indices, torch.where(lse > -INF, lse, 0.0), y,
                                        alpha, tau, 1.0 / N)
        lp = torch.log_softmax(z[1].double().cpu(), 0)
        want[1] = -(1 - alpha) * lp[int(y[1])]
        gwant[1] = (1 - alpha) / N * lp.exp()
        gwant[1, int(y[1])] -= (1 - alpha) / N
        # as check_distill's bound, with logits and log-probabilities up to 40
        bound = (2 * 20 + 64 + 2 * k) * U
        assert ((row.double().cpu() - want).abs() <= bound * (alpha * tau * tau + 1) * 40).all()
        assert ((grad.double().cpu() - gwant).abs() <= bound * (alpha * tau + 1) / N).all()
        assert row[3] == 0 and (grad[3] == 0).all()
        if alpha == 1.0:
            assert row[1] == 0 and (grad[1] == 0).all()
    leaf = z.clone().requires_grad_(True)
    O.distill_loss(leaf, values, indices, top_lse=lse, targets=y, alpha=alpha,
                   temperature=tau).backward()
    assert torch.allclose(leaf.grad, grad, atol=1e-9, rtol=1e-6)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tau", [0.5, 2.0])
def test_distill_lowest_values(tau, dtype, dev):
    """Masks of the type's lowest value, and rows of nothing else: those are uniform."""
    N, V, k = 3, 300, 4
    low = torch.finfo(dtype).min
    z = rows(N, V, dtype, dev)
    values, indices, lse = record(z, k, tau)
    z[0] = low
    masked = torch.ones(V, dtype=torch.bool, device=dev)
    masked[indices[1].long()] = False
    z[1, masked] = low
    y = indices[:, 0].contiguous()
    loss, row, grad = O.distill_xent(z, values, indices, top_lse=None, targets=y, alpha=0.5,
                                     temperature=tau)
    half = 2.0 ** -8 if dtype == BF16 else 0.0
    zs = z.double().cpu()
    zs[0] = 0.0  # the same distribution
    want, gwant = reference_distill(zs, values, indices, None, y, 0.5, tau, 1.0 / N)
    assert ((row.double().cpu() - want).abs() <= 256 * U * 30 * (tau * tau + 1)).all(), (row, want)
    tol = 256 * U * (tau + 1)
    assert ((grad.double().cpu() - gwant).abs() <= tol + half * (gwant.abs() + tol)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N,V,k,tau", [(12, 2136, 1, 3.278), (306, 1909, 63, 2.844),
                                       (8, 151, 77, 0.929), (4, 9000, 4, 5.0), (4, 70000, 2, 4.0)])
def test_distill_small_divergences_keep_their_digits(N, V, k, tau):
    """A student near its teacher, few recorded tokens: the divergence is some 1e-3 of its terms.
    It is a sum of q (d - 1 + exp(-d)), d = log(q / p), none negative and each with a relative error
    of 2 err(d) / |d|; the weighted |d| is sqrt(2 KL), err(d) under 32 u.  The gradient's error is that
    of p and q, 128 u of p each (q < 2 p).  Off the entries it is T p (1 - r / s) with r = 1 - sum q: where
    the entries hold most, r has the absolute error of that sum, 32 u of sum q <= 1 and k u from
    adding, and the gradient p / s of it; where they hold little, 1 - r / s = sum (q - p) / s has
    64 u of sum (q + p) <= 1.5, over s > 1/4."""
    z = rows(N, V, F32, "cuda")
    g = torch.Generator().manual_seed(5)
    t = z.cpu() + 0.1 * torch.randn(z.shape, generator=g)
    top = torch.topk(t, k, dim=1)
    values, indices = top.values.cuda(), top.indices.int().cuda()
    lse = torch.logsumexp(t.double() / tau, 1).float().cuda()
    _, row, grad = O.distill_xent(z, values, indices, top_lse=lse, temperature=tau)
    want, gwant = reference_distill(z, values, indices, lse, None, 1.0, tau, 1.0 / N)
    kl = want / tau ** 2
    assert (kl < 0.05).all()
    err = (row.double().cpu() - want).abs() / tau ** 2
    assert (err <= 64 * U * (2 * kl).sqrt() + 64 * U * kl).all(), (err / kl).max()
    p = torch.softmax(z.double().cpu() / tau, 1)
    off = torch.ones_like(p).scatter(1, indices.long().cpu(), 0.0)
    s = (p * off).sum(1, keepdim=True)
    allowed = 256 * U * p + off * p / s * (k + 96) * U
    assert ((grad.double().cpu() - gwant).abs() <= allowed * tau / N + 1e-12).all()


@pytest.mark.parametrize("dev", DEVS)
def test_distill_sure_students(dev):
    """The student's mass off the entries is too small for fp32: the divergence is still a number."""
    V = 500
    z = torch.full((2, V), -60.0, device=dev)
    z[:, 3:5] = 60.0
    values = torch.tensor([[2.0, 1.0], [-3.0, -3.5]], device=dev)
    indices = torch.tensor([[3, 4]] * 2, dtype=torch.int32, device=dev)
    check_distill(z, values, indices, torch.tensor([2.6, 2.0], device=dev), None, 1.0, 1.0)


@pytest.mark.parametrize("dev", DEVS)
def test_distill_infinite_and_nan(dev):
    z = rows(4, 70, F32, dev)
    values, indices, lse = record(z, 4, 1.0)
    z[0, indices[0, 0].item()] = -INF  # the teacher wants what the student has ruled out
    z[1, 3] = NAN
    loss, row, grad = O.distill_xent(z, values, indices, top_lse=lse)
    assert row[0] == INF and row[1].isnan() and row[2:].isfinite().all()
    assert grad[0].isfinite().all() and grad[1].isnan().any() and grad[2:].isfinite().all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_autograd_and_differences(dtype, dev):
    N, V, k = 6, 90, 5
    z = rows(N, V, dtype, dev)
    y = torch.arange(N, dtype=torch.int32, device=dev)
    values, indices, lse = record(z, k, 2.0)
    kw = dict(top_lse=lse, targets=y, alpha=0.7, temperature=2.0)
    leaf = z.clone().requires_grad_(True)
    loss = O.distill_loss(leaf, values, indices, **kw)
    (loss * 3.0).backward()
    one, _, grad = O.distill_xent(z, values, indices, scale=3.0 / N, **kw)
    assert torch.allclose(loss.detach() * 3.0, one, rtol=1e-6)
    tol = 1e-6 if dtype == F32 else 2.0 ** -7
    assert torch.allclose(leaf.grad.float(), grad.float(), rtol=tol, atol=1e-8)
    if dtype == F32:
        # the row's loss moves by its gradient; step 2^-7, truncation ~ step^2
        for i in range(0, V, 17):
            up, dn = z.clone(), z.clone()
            up[:, i] += 2.0 ** -7
            dn[:, i] -= 2.0 ** -7
            a = O.distill_xent(up, values, indices, **kw)[1]
            b = O.distill_xent(dn, values, indices, **kw)[1]
            assert torch.allclose((a - b) * 64, grad[:, i] * N / 3.0, atol=2e-3)
    # into a caller's buffer, wider than the row
    buf = torch.full((N, V + 5), 7.0, dtype=dtype, device=dev)
    out = O.distill_xent(z, values, indices, grad=buf[:, :V], scale=3.0 / N, **kw)[2]
    assert torch.equal(out, grad) and (buf[:, V:] == 7.0).all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,V", [(5, 65), (4, 1500), (1100, 1500), (3, 9000), (1100, 9000), (3, 40001)])
def test_distill_gradient_over_the_logits(N, V, dtype, dev):
    """The gradient written over the logits, with entries and targets everywhere in the row, and beside
    them in the rows of one buffer."""
    k = 9
    buf = rows(N, 2 * V + 3, dtype, dev)
    z = buf[:, 1:V + 1]
    g = torch.Generator().manual_seed(6)
    y = torch.randint(0, V, (N,), generator=g).int().to(dev)
    indices = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(N)]).int().to(dev)
    values = torch.randn(N, k, generator=g).to(dev)
    kw = dict(targets=y, alpha=0.6, temperature=2.0)
    want = O.distill_xent(z, values, indices, **kw)
    beside = O.distill_xent(z, values, indices, grad=buf[:, V + 1:2 * V + 1], **kw)
    over = O.distill_xent(z, values, indices, grad=z, **kw)
    for got in (beside, over):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert over[2].data_ptr() == z.data_ptr()


@pytest.mark.gpu
def test_distill_refuses_a_gradient_across_the_logits():
    N, V, k = 4, 65, 3
    buf = rows(N, 3 * V, F32, "cuda")
    flat = torch.zeros(4 * N * V, device="cuda")
    z = buf[:, V:2 * V]
    values, indices, _ = O.top_logits(z.contiguous(), k)
    for grad in (buf[:, V + 1:2 * V + 1], buf[:, 1:V + 1], buf[:, V - 3:2 * V - 3]):
        with pytest.raises(RuntimeError, match="memory"):
            O.distill_xent(z, values, indices, grad=grad)
    a = flat[:N * V].view(N, V)
    for off, ok in ((0, True), (1, False), (N * V - 1, False), (N * V, True), (V, False)):
        b = flat[off:off + N * V].view(N, V)
        for p, q in ((a, b), (b, a)):
            if ok:
                O.distill_xent(p, values, indices, grad=q)
            else:
                with pytest.raises(RuntimeError, match="memory"):
                    O.distill_xent(p, values, indices, grad=q)
    half = flat.view(BF16)[:N * V].view(N, V)  # the same place in another type
    with pytest.raises(RuntimeError, match="memory"):
        O.distill_xent(a, values, indices, grad=half)
    with pytest.raises(RuntimeError, match="memory"):
        O.distill_xent(a[:1].expand(N, V), values, indices, grad=a)


@pytest.mark.parametrize("dev", DEVS)
def test_distill_agrees_with_cross_entropy(dev):
    """A record of one sure entry is a target: the loss is the plain cross-entropy."""
    N, V = 8, 65
    z = rows(N, V, F32, dev)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(1)).int().to(dev)
    _, row, grad = O.distill_xent(z, torch.zeros(N, 1, device=dev), y[:, None].contiguous())
    lp = torch.log_softmax(z.double(), 1)
    assert torch.allclose(row.double(), -lp.gather(1, y.long()[:, None])[:, 0], atol=2e-6)
    want = (lp.exp() - torch.nn.functional.one_hot(y.long(), V)) / N
    assert torch.allclose(grad.double(), want, atol=1e-7)


# ---- sampling --------------------------------------------------------------------------------
def reference_sample(z, u, temp, top_k, top_p, min_p):
    """float64, row by row."""
    out = []
    for n in range(z.shape[0]):
        x = z[n].double().cpu()
        x = torch.where(x.isnan(), -INF, x)
        V = x.numel()
        order = sorted(range(V), key=lambda i: (-x[i].item(), i))
        t, k, p, q = (float(s[n]) if isinstance(s, torch.Tensor) else
                      (s if i == 1 else float(torch.tensor(s, dtype=F32)))
                      for i, s in enumerate((temp, top_k, top_p, min_p)))
        top = x[order[0]].item()
        if not t > 0 or top == -INF:
            out.append(order[0])
            continue
        xs = x[order]
        w = torch.exp((xs - top) / t)
        w[torch.isneginf(xs)] = 0.0
        if top == INF:
            w = torch.zeros(V, dtype=torch.float64)
        w[xs == top] = 1.0
        if k >= 1:
            w[int(k):] = 0.0
        total, before = w.sum().item(), torch.cumsum(w, 0) - w
        keep = torch.ones(V, dtype=torch.bool)
        if p < 1:
            keep &= before < p * total
        if q == q:
            keep &= w >= min(q, 1.0)
        keep[0] = True
        full = torch.zeros(V, dtype=torch.float64)
        full[torch.tensor(order)] = torch.where(keep, w, 0.0)
        cdf = torch.cumsum(full, 0)
        r = float(u[n])
        r = (r if r > 0 else 0.0) * cdf[-1].item()
        hit = torch.nonzero(cdf > r)
        last = torch.nonzero(full)[-1].item()
        out.append(min(hit[0].item(), last) if hit.numel() else last)
    return torch.tensor(out, dtype=torch.int32)


def check_sample(z, seed=0, u=None, **kw):
    u = torch.rand(z.shape[0], generator=torch.Generator().manual_seed(seed)).to(z.device) \
        if u is None else u
    got = O.sample_logits(z, u, **kw)
    s = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw)
    want = reference_sample(z, u, s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), want), (got.cpu(), want, kw)


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=5), dict(top_p=0.8),
            dict(min_p=0.1), dict(temperature=1.3, top_k=40, top_p=0.9, min_p=0.02),
            dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0), dict(temperature=50.0, top_p=0.5),
            dict(temperature=1e-3, top_p=0.999), dict(top_k=700, top_p=0.95),
            dict(temperature=1e-30, top_k=3)]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,V", [(1, 1), (4, 2), (9, 65), (5, 256), (4, 257), (3, 1000), (3, 1025),
                                 (3, 4099), (3, 8200)])
def test_sample(N, V, dtype, dev):
    for i, kw in enumerate(SETTINGS):
        check_sample(rows(N, V, dtype, dev, seed=i, pad=i % 3), seed=i, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,V", [(2, 32001), (2, 65536), (2, 70001), (1, 262144)])
def test_sample_large(N, V, dtype):
    for i, kw in enumerate(SETTINGS):
        check_sample(rows(N, V, dtype, "cuda", seed=i), seed=i, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,V", [(3000, 65), (400, 700), (60, 9000)])
def test_sample_many_rows(N, V, dtype):
    """Many draws against the plain form on the CPU, itself held to the row-by-row one above."""
    for i, kw in enumerate(SETTINGS):
        z = rows(N, V, dtype, "cuda", seed=i)
        u = torch.rand(N, generator=torch.Generator().manual_seed(i))
        got = O.sample_logits(z, u.cuda(), **kw)
        assert torch.equal(got.cpu(), O.sample_logits(z.cpu(), u, **kw)), kw


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [3, 65, 700, 1500, 20000])
def test_sample_weights_that_round_to_nothing(V, dev):
    """The smallest u takes the first token that weighs anything: less than 2^-45 of the largest is
    nothing (exp(-40) = 2^-57.7), more is something (exp(-30) = 2^-43.3)."""
    z = torch.full((4, V), -40.0, device=dev)
    z[:, 2] = 0.0
    z[1, 1] = -30.0
    z[2, 0] = -30.0
    z[3, :2] = torch.tensor([-INF, -80.0])
    for kw in (dict(), dict(top_k=3), dict(top_k=V), dict(top_p=1 - 2.0 ** -24), dict(min_p=1e-20),
               dict(temperature=0.5)):
        got = O.sample_logits(z, torch.zeros(4, device=dev), **kw)
        if kw in (dict(temperature=0.5), dict(top_p=1 - 2.0 ** -24)):
            # exp(-60) is nothing; a share of 1 - 2^-24 leaves out what lies behind the first
            want = [2, 2, 2, 2]
        else:
            want = [2, 1, 0, 2]
        assert got.tolist() == want, kw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [257, 300, 511, 512, 513, 768, 769])
def test_sample_rows_that_leave_chunks_empty(V, dtype):
    """Rows of one wave that do not fill its last chunks: the draw's running weights have no part of
    them.  Between the draws other rows of the same kernel leave theirs behind in LDS."""
    N = 4000
    full = rows(N, 1024, dtype, "cuda", seed=V)
    u = torch.rand(N, generator=torch.Generator().manual_seed(V))
    for i, kw in enumerate([dict(), dict(min_p=0.01), dict(top_p=0.9), dict(temperature=30.0)]):
        z = rows(N, V, dtype, "cuda", seed=i, pad=i % 2)
        O.sample_logits(full, u.cuda())
        got = O.sample_logits(z, u.cuda(), **kw)
        assert torch.equal(got.cpu(), O.sample_logits(z.cpu(), u, **kw)), kw


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [5, 65, 300, 1500, 5000])
def test_sample_hard_rows(V, dev):
    for dtype in (F32, BF16):
        z = hard_rows(V, dtype, dev)
        for i, kw in enumerate(SETTINGS):
            check_sample(z, seed=i, **kw)
        for u in (0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, NAN):  # the last three: not uniform numbers
            check_sample(z, u=torch.full((z.shape[0],), u, device=dev), top_k=3)
            check_sample(z, u=torch.full((z.shape[0],), u, device=dev), top_p=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [20000, 70001])
def test_sample_hard_rows_large(V):
    z = hard_rows(V, F32, "cuda")
    for i, kw in enumerate(SETTINGS):
        u = torch.rand(z.shape[0], generator=torch.Generator().manual_seed(i))
        got = O.sample_logits(z, u.cuda(), **kw)
        assert torch.equal(got.cpu(), O.sample_logits(z.cpu(), u, **kw)), kw


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("V", [65, 1500])
def test_sample_per_row_settings(V, dev):
    N = 24
    z = rows(N, V, F32, dev)
    g = torch.Generator().manual_seed(8)
    temp, p, q = (torch.rand(N, generator=g) for _ in range(3))
    temp[0], temp[1], temp[2], temp[3] = 0.0, -1.0, NAN, INF
    p[4], p[5], p[6] = 1.5, -0.5, NAN
    q = q * 0.2
    q[7], q[8], q[9] = 2.0, -1.0, NAN
    k = torch.randint(0, 2 * V, (N,), generator=g, dtype=torch.int32)
    k[10], k[11] = -3, 1
    t = {n: v.to(dev) for n, v in dict(temperature=temp, top_k=k, top_p=p, min_p=q).items()}
    check_sample(z, **t)
    check_sample(z, temperature=t["temperature"], top_p=0.9)
    check_sample(z, top_k=t["top_k"], min_p=0.05)


@pytest.mark.gpu
def test_sample_follows_the_distribution():
    """200k draws of one row: each kept token's share within 5 standard deviations."""
    N, V = 200000, 65
    z = rows(1, V, F32, "cuda", seed=7, spread=1.5).expand(N, V)
    u = torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    ids = O.sample_logits(z, u, temperature=0.8, top_k=30, top_p=0.95)
    p = torch.softmax(z[0].double() / 0.8, 0)
    s = torch.sort(p, descending=True)
    w = torch.where(torch.arange(V, device="cuda") < 30, s.values, 0.0)
    w = torch.where(torch.cumsum(w, 0) - w < 0.95 * w.sum(), w, 0.0)
    want = torch.zeros_like(p).scatter(0, s.indices, w / w.sum())
    freq = torch.bincount(ids.long(), minlength=V).double() / N
    assert ((freq - want).abs() <= 5 * (want * (1 - want) / N).sqrt() + 1e-12).all()


# ---- refusals, streams, graphs ---------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVS)
def test_no_rows(dev):
    z = torch.zeros(0, 65, device=dev)
    v, i, lse = O.top_logits(z, 4)
    assert v.shape == (0, 4) and i.shape == (0, 4) and lse.shape == (0,)
    loss, row, grad = O.distill_xent(z, v, i, top_lse=lse)
    assert loss == 0 and row.shape == (0,) and grad.shape == (0, 65)
    assert O.sample_logits(z, torch.zeros(0, device=dev)).shape == (0,)


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    z = rows(4, 65, F32, dev)
    v, i, lse = O.top_logits(z, 4)
    u = torch.zeros(4, device=dev)
    y = torch.zeros(4, dtype=torch.int32, device=dev)
    bad = [
        lambda: O.top_logits(z[0], 4),
        lambda: O.top_logits(z.double(), 4),
        lambda: O.top_logits(z.half(), 4),
        lambda: O.top_logits(z.t().contiguous().t(), 4),
        lambda: O.top_logits(z, 0),
        lambda: O.top_logits(z, 66),
        lambda: O.top_logits(torch.zeros(1, 600, device=dev), 257),
        lambda: O.top_logits(z, 4, temperature=0.0),
        lambda: O.top_logits(z, 4, temperature=-1.0),
        lambda: O.top_logits(z, 4, temperature=INF),
        lambda: O.top_logits(torch.zeros(1, O.MAX_V + 1, device=dev), 4),
        lambda: O.top_logits(torch.zeros(1, 0, device=dev), 1),
        lambda: O.distill_xent(z, v[:2], i),
        lambda: O.distill_xent(z, v, i.long()),
        lambda: O.distill_xent(z, v, i[:, :3]),
        lambda: O.distill_xent(z, v.bfloat16(), i),
        lambda: O.distill_xent(z, v[:, :0], i[:, :0]),
        lambda: O.distill_xent(z, v.t().contiguous().t(), i),
        lambda: O.distill_xent(z, v, i, top_lse=lse[:2]),
        lambda: O.distill_xent(z, v, i, alpha=0.5),
        lambda: O.distill_xent(z, v, i, alpha=1.5),
        lambda: O.distill_xent(z, v, i, temperature=0.0),
        lambda: O.distill_xent(z, v, i, scale=INF),
        lambda: O.distill_xent(z, v, i, targets=y.long(), alpha=0.5),
        lambda: O.distill_xent(z, v, i, targets=y[:1], alpha=0.5),
        lambda: O.sample_logits(z, u[:2]),
        lambda: O.sample_logits(z, u.double()),
        lambda: O.sample_logits(z, u, temperature=-0.5),
        lambda: O.sample_logits(z, u, temperature=NAN),
        lambda: O.sample_logits(z, u, top_k=-1),
        lambda: O.sample_logits(z, u, top_p=1.5),
        lambda: O.sample_logits(z, u, min_p=-0.1),
        lambda: O.sample_logits(z, u, temperature=u[:1]),
        lambda: O.sample_logits(z, u, top_k=u),
        lambda: O.sample_logits(z.t().contiguous().t(), u),
    ]
    for n, fn in enumerate(bad):
        with pytest.raises(RuntimeError):
            fn()
            pytest.fail(f"call {n} was not refused")


@pytest.mark.parametrize("dev", DEVS)
def test_refusals_are_the_same_on_both_devices(dev):
    z = rows(4, 65, F32, dev)
    v, i, lse = O.top_logits(z, 4)
    wide = torch.zeros(4, 65, device=dev)
    for t in (1e-46, 1e-40, 1e39, 1e300, NAN):  # no number, or no reciprocal, in fp32
        for call in (lambda: O.top_logits(z, 4, t), lambda: O.distill_xent(z, v, i, temperature=t)):
            with pytest.raises(RuntimeError):
                call()
    for kw in (dict(grad_dtype=torch.float16), dict(grad_dtype=torch.float64),
               dict(grad=wide.half()), dict(grad=wide.double()), dict(grad=wide[:2]),
               dict(grad=wide[None]), dict(grad=wide[:, :64]), dict(grad=wide[:1].expand(4, 65)),
               dict(grad=torch.zeros(65, 4, device=dev).t())):
        with pytest.raises(RuntimeError):
            O.distill_xent(z, v, i, top_lse=lse, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [65, 1500, 9000, 70001])
def test_far_rows(V):
    """Rows more than 2^31 elements apart, logits and gradient."""
    N, far = 3, (1 << 30) + 7
    buf = torch.empty(2 * far + V, dtype=BF16, device="cuda")
    z = torch.as_strided(buf, (N, V), (far, 1))
    z.copy_(rows(N, V, BF16, "cuda"))
    near = z.contiguous()
    u = torch.rand(N, device="cuda")
    for a, b in zip(O.top_logits(z, 5), O.top_logits(near, 5)):
        assert torch.equal(a, b)
    values, indices, lse = record(near, 5, 1.0)
    out = torch.as_strided(torch.empty(2 * far + V, dtype=BF16, device="cuda"), (N, V), (far, 1))
    a = O.distill_xent(z, values, indices, top_lse=lse, grad=out)
    b = O.distill_xent(near, values, indices, top_lse=lse)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for kw in (dict(top_k=20), dict(top_p=0.9), dict()):
        assert torch.equal(O.sample_logits(z, u, **kw), O.sample_logits(near, u, **kw))


@pytest.mark.gpu
def test_refuses_more_rows_than_a_launch_holds():
    z = torch.zeros(1, 3, device="cuda").expand(1 << 22, 3)
    with pytest.raises(RuntimeError):
        O.top_logits(z, 2)
    with pytest.raises(RuntimeError):
        O.sample_logits(z, torch.zeros(1 << 22, device="cuda"))
    x = torch.zeros(1, 1, 1, device="cuda").expand(2, 1 << 15, (1 << 13) + 1)
    with pytest.raises(RuntimeError):
        torch.ops.dcr.linrec_fwd(x, x, None, None, None, False)


@pytest.mark.gpu
def test_refuses_mixed_devices():
    z = rows(4, 65, F32, "cuda")
    v, i, lse = O.top_logits(z, 4)
    with pytest.raises(RuntimeError):
        O.distill_xent(z, v.cpu(), i)
    with pytest.raises(RuntimeError):
        O.distill_xent(z, v, i, grad=torch.zeros(4, 65))
    with pytest.raises(RuntimeError):
        O.sample_logits(z, torch.zeros(4))


@pytest.mark.gpu
def test_streams_and_graph_replays():
    """Teacher's record, student's loss and a draw on another stream, then captured: every replay
    with new inputs equals the eager result, also with eager work in between."""
    N, V, k = 40, 1200, 16
    t, z = rows(N, V, F32, "cuda", seed=1), rows(N, V, F32, "cuda", seed=2)
    u = torch.rand(N, device="cuda")

    def run():
        v, i, lse = O.top_logits(t, k, 2.0)
        loss, row, grad = O.distill_xent(z, v, i, top_lse=lse, temperature=2.0)
        return v, i, lse, loss, row, grad, O.sample_logits(z, u, top_k=50, top_p=0.9)

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for s in range(4):
        t.copy_(rows(N, V, F32, "cuda", seed=10 + s))
        z.copy_(rows(N, V, F32, "cuda", seed=20 + s))
        u.copy_(torch.rand(N, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, run()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [300, 20000, 40001, 70001])
def test_wide_rows_in_a_graph(V, dtype):
    """The forms of wide rows (large LDS, rows read again), captured: record, loss with its gradient
    by autograd, draws; each replay with new inputs equals the eager calls."""
    N, k = 3, 9
    t, z = rows(N, V, dtype, "cuda", seed=1), rows(N, V, dtype, "cuda", seed=2)
    u = torch.rand(N, device="cuda")

    def run():
        v, i, lse = O.top_logits(t, k, 2.0)
        leaf = z.detach().requires_grad_(True)
        loss = O.distill_loss(leaf, v, i, top_lse=lse, temperature=2.0)
        (grad,) = torch.autograd.grad(loss * 3.0, leaf)
        return (v, i, lse, loss.detach(), grad, O.sample_logits(z, u, top_k=50),
                O.sample_logits(z, u, top_p=0.9), O.sample_logits(z, u))

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for s in range(3):
        t.copy_(rows(N, V, dtype, "cuda", seed=10 + s))
        z.copy_(rows(N, V, dtype, "cuda", seed=20 + s))
        u.copy_(torch.rand(N, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, run()))


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls in flight on two streams, one row kernel beside another, share nothing."""
    N, V, k = 300, 9000, 12
    z = [rows(N, V, F32, "cuda", seed=i) for i in range(2)]
    u = [torch.rand(N, device="cuda") for _ in range(2)]

    def run(i):
        v, ix, lse = O.top_logits(z[i], k, 2.0)
        return (v, ix, lse) + O.distill_xent(z[1 - i], v, ix, top_lse=lse, temperature=2.0) + (
            O.sample_logits(z[i], u[i], top_p=0.9),)

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(side[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))
