"""The gated linear recurrence (ops/recurrence.py, csrc/linrec.hip) against a step-by-step float64
form and its automatic derivative, on the CPU and on the GPU.

Tolerances.  A state is a convex combination of the inputs, so M = max(|x|, |h0|) bounds it; a
step adds at most 3 roundings of 2^-24 M and the gates' relative error (under 32 x 2^-24 for the
gates used here) times what they move, which the decay of the step itself pays back: after T steps
(3 T + 32) 2^-24 M.  The same holds for the gradient's recursion with its own bound, and their
products in df.  A bf16 output adds its half step, 2^-9 of the value's power of two (2^-8
relative)."""
import pytest
import torch

from distributed_char_rnn_amd.ops import recurrence as R

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, BF16 = torch.float32, torch.bfloat16


def reference(x, f, h0, lengths, starts):
    """float64, one step after the other; differentiable."""
    T, B, H = x.shape
    h, out = h0, []
    for t in range(T):
        a = torch.sigmoid(f[t])
        keep = a * h
        if starts is not None:
            keep = torch.where(starts[t][:, None], torch.zeros_like(h), keep)
        new = keep + (1 - a) * x[t]
        if lengths is not None:
            live = (t < lengths)[:, None]
            out.append(torch.where(live, new, torch.zeros_like(new)))
            h = torch.where(live, new, h)
        else:
            out.append(new)
            h = new
    return (torch.stack(out) if out else x.new_zeros(0, B, H)), h


def inputs(T, B, H, dtype, dev, seed=0, layout="tbh"):
    g = torch.Generator().manual_seed(seed)

    def seq(shift=0.0):
        v = (torch.randn(T, B, H, generator=g) + shift).to(dtype).to(dev)
        if layout == "bth":
            return v.transpose(0, 1).contiguous().transpose(0, 1)
        return v

    x, f, dh = seq(), seq(1.0), seq()
    if layout == "fused":  # both halves of one projection
        z = torch.cat([x, f], 2)
        x, f = z[..., :H], z[..., H:]
    if layout == "offset":  # rows that start at odd places
        buf = torch.zeros(2 * T * B * H + 7, dtype=dtype, device=dev)
        xv = buf[1:1 + T * B * H].view(T, B, H)
        fv = buf[T * B * H + 4:2 * T * B * H + 4].view(T, B, H)
        xv.copy_(x)
        fv.copy_(f)
        x, f = xv, fv
    h0 = torch.randn(B, H, generator=g).to(dev)
    dlast = torch.randn(B, H, generator=g).to(dev)
    return x, f, h0, dh, dlast


def marks(T, B, which, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    lengths = starts = None
    if "l" in which:
        lengths = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        lengths[0] = 0
        lengths[-1] = T
        if B > 2:
            lengths[1] = 1
        lengths = lengths.to(dev)
    if "s" in which:
        starts = torch.rand(T, B, generator=g) < 0.15
        starts[0, 0] = True
        starts[-1] = True
        starts = starts.to(dev)
    return lengths, starts


def close(got, want, bound, name):
    if want.numel() == 0:
        assert got.shape == want.shape
        return
    half = torch.finfo(got.dtype).eps / 2 if got.dtype == BF16 else 0.0
    err = (got.double().cpu() - want.cpu()).abs()
    allowed = bound + half * (want.abs().cpu() + bound)
    worst = (err - allowed).max().item()
    assert worst <= 0, f"{name}: {err.max().item()} off, {worst} over"


def check(x, f, h0, dh, dlast, lengths, starts):
    T = x.shape[0]
    d = [v.detach().double().cpu().requires_grad_(True) for v in (x, f, h0)]
    lc, sc = (None if v is None else v.cpu() for v in (lengths, starts))
    h_ref, last_ref = reference(*d, lc, sc)
    outs = [last_ref] + ([h_ref] if T else [])
    grads = [dlast.double().cpu()] + ([dh.double().cpu()] if T else [])
    want = [torch.zeros_like(v) if w is None else w for v, w in
            zip(d, torch.autograd.grad(outs, d, grads, allow_unused=True))]
    h, last, carry = R.linear_recurrence_fwd(x, f, h0, lengths=lengths, starts=starts)
    dx, df, dh0 = R.linear_recurrence_bwd(x, f, carry, dh, dlast=dlast, lengths=lengths,
                                          starts=starts)
    M = max([v.abs().max().item() for v in (d[0], d[2]) if v.numel()] + [0.0])
    unit = (3 * T + 32) * 2.0 ** -24
    close(h, h_ref.detach(), unit * M, "h")
    close(last, last_ref.detach(), unit * M, "last")
    # |g| <= |dh| + a |g'|: bounded by the largest sum, taken from the gradient with respect to b
    G = dlast.abs().max().item() + (dh.abs().max().item() if T else 0.0) * \
        (1 + sum(min(1.0, 0.999 ** i) for i in range(T)))
    G = min(G, 1e3)
    close(dx, want[0], unit * G, "dx")
    close(df, want[1], unit * G * (1 + M), "df")
    close(dh0, want[2], unit * G, "dh0")


SHAPES = [(1, 1, 1), (1, 3, 7), (2, 5, 33), (7, 2, 64), (8, 1, 6), (31, 3, 12), (32, 2, 128),
          (33, 4, 130), (50, 50, 128), (129, 3, 257), (300, 1, 512)]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", ["", "l", "s", "ls"])
@pytest.mark.parametrize("T,B,H", SHAPES)
def test_against_steps(T, B, H, which, dtype, dev):
    check(*inputs(T, B, H, dtype, dev), *marks(T, B, which, dev))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,B,H,which", [(1025, 1, 64, ""), (2500, 2, 40, "ls"), (700, 3, 1000, "l"),
                                         (40, 300, 512, "ls"), (4096, 1, 33, "s")])
def test_long_and_wide(T, B, H, which, dtype):
    """Time axes that are cut into segments, and grids of many workgroups."""
    check(*inputs(T, B, H, dtype, "cuda"), *marks(T, B, which, "cuda"))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("layout", ["bth", "fused", "offset"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H", [24, 25, 26])
def test_layouts(H, dtype, layout, dev):
    args = inputs(37, 5, H, dtype, dev, layout=layout)
    check(*args, *marks(37, 5, "ls", dev))
    h, _, _ = R.linear_recurrence_fwd(*args[:3])
    if layout == "bth":
        assert h.stride() == args[0].stride()


@pytest.mark.parametrize("dev", DEVS)
def test_no_steps_and_no_streams(dev):
    check(*inputs(0, 3, 8, F32, dev)[:5], None, None)
    for B, H in ((0, 8), (3, 0)):
        x = torch.zeros(4, B, H, device=dev)
        h, last, carry = R.linear_recurrence_fwd(x, x, None)
        assert h.shape == (4, B, H) and last.shape == (B, H)
        dx, df, dh0 = R.linear_recurrence_bwd(x, x, carry, x)
        assert dx.shape == df.shape == (4, B, H) and dh0.shape == (B, H)


@pytest.mark.parametrize("dev", DEVS)
def test_defaults_are_zeros(dev):
    x, f, h0, dh, dlast = inputs(20, 3, 16, F32, dev)
    z = torch.zeros_like(h0)
    a = R.linear_recurrence_fwd(x, f)
    b = R.linear_recurrence_fwd(x, f, z)
    assert all(torch.equal(p, q) for p, q in zip(a[:2], b[:2]))
    assert R.linear_recurrence_fwd(x, f, want_carry=False)[2].numel() == 0
    p = R.linear_recurrence_bwd(x, f, a[2], dh)
    q = R.linear_recurrence_bwd(x, f, a[2], dh, dlast=z)
    assert all(torch.equal(u, v) for u, v in zip(p, q))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padding_and_starts_let_nothing_through(dtype, dev):
    """NaN behind a sequence's end, and in a document before a start, stay there."""
    x, f, h0, dh, dlast = inputs(41, 4, 20, dtype, dev)
    lengths = torch.tensor([41, 17, 1, 0], dtype=torch.int32, device=dev)
    starts = torch.zeros(41, 4, dtype=torch.bool, device=dev)
    starts[9, 0] = True
    clean = R.linear_recurrence_fwd(x, f, h0, lengths=lengths, starts=starts)
    cg = R.linear_recurrence_bwd(x, f, clean[2], dh, dlast=dlast, lengths=lengths, starts=starts)
    bad = [v.clone() for v in (x, f, dh)]
    for b, n in enumerate(lengths.tolist()):
        for v in bad:
            v[n:, b] = float("nan")
    dirty = R.linear_recurrence_fwd(bad[0], bad[1], h0, lengths=lengths, starts=starts)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    dg = R.linear_recurrence_bwd(bad[0], bad[1], dirty[2], bad[2], dlast=dlast, lengths=lengths,
                                 starts=starts)
    assert all(torch.equal(u, v) for u, v in zip(cg, dg))
    x2 = x.clone()
    x2[3, 0] = float("nan")
    h2, last2, carry2 = R.linear_recurrence_fwd(x2, f, h0, lengths=lengths, starts=starts)
    assert torch.equal(h2[9:, 0], clean[0][9:, 0]) and h2[3:9, 0].isnan().all()
    assert torch.equal(last2, clean[1])
    g2 = R.linear_recurrence_bwd(x2, f, carry2, dh, dlast=dlast, lengths=lengths, starts=starts)
    assert torch.equal(g2[0][9:, 0], cg[0][9:, 0]) and torch.equal(g2[1][9:, 0], cg[1][9:, 0])


def documents(T, B, dev, every=37):
    """Starts at places that differ from stream to stream, in neighbouring steps too; the last stream
    begins in a document that goes on from before.  With the first and the last step of the document
    that each step belongs to, [T, B]."""
    starts = torch.zeros(T, B, dtype=torch.bool)
    for b in range(B):
        starts[b % 5::every + 4 * b, b] = True
        starts[min(b % 5 + 1, T - 1), b] = True
    starts[:every, B - 1] = False
    starts[T // 2, B - 1] = True
    first = torch.zeros(T, B, dtype=torch.long)
    last = torch.zeros(T, B, dtype=torch.long)
    for t in range(T):
        first[t] = torch.where(starts[t], t, first[max(t - 1, 0)])
    for t in reversed(range(T)):
        last[t] = T - 1 if t == T - 1 else torch.where(starts[t + 1], t, last[t + 1])
    return starts.to(dev), first, last


def check_nan_stays_in_its_document(T, B, H, dtype, dev, level, every=37):
    """One NaN a channel, next to a start and far from one.  What depends on it is NaN -- from there to
    the document's last step forward, to its first backward -- and all else as without it."""
    x, f, h0, dh, dlast = inputs(T, B, H, dtype, dev)
    f = f + level
    starts, first, last = documents(T, B, dev, every)
    clean = R.linear_recurrence_fwd(x, f, h0, starts=starts)
    cg = R.linear_recurrence_bwd(x, f, clean[2], dh, dlast=dlast, starts=starts)
    g = torch.Generator().manual_seed(9)
    at = torch.randint(0, T, (B, H), generator=g)
    marked = starts.cpu()
    for b in range(B):  # three channels of four within a step of a start
        near = marked[:, b].nonzero()[:, 0]
        pick = near[torch.randint(0, len(near), (H,), generator=g)] + torch.arange(H) % 4 - 1
        at[b] = torch.where(torch.arange(H) % 4 < 3, pick.clamp(0, T - 1), at[b])
    steps = torch.arange(T)[:, None, None]
    s = first.gather(0, at.t().reshape(-1, B).contiguous()).t()  # [B, H]: of the NaN's document
    e = last.gather(0, at.t().reshape(-1, B).contiguous()).t()
    after, until = (steps >= at) & (steps <= e), (steps >= s) & (steps <= at)
    inside, none = (steps >= s) & (steps <= e), torch.zeros(T, B, H, dtype=torch.bool)
    open_ = (s == 0) & ~marked[0][:, None]  # the document goes on from h0
    want = dict(x=(after, none, after), f=(after, until, inside), dh=(none, until, until))
    for what, (h_nan, dx_nan, df_nan) in want.items():
        v = dict(x=x, f=f, dh=dh)
        v[what] = v[what].clone()
        v[what].scatter_(0, at[None].to(dev), float("nan"))
        h, end, carry = R.linear_recurrence_fwd(v["x"], v["f"], h0, starts=starts)
        dx, df, dh0 = R.linear_recurrence_bwd(v["x"], v["f"], carry, v["dh"], dlast=dlast,
                                              starts=starts)
        for name, got, ref, nan in (("h", h, clean[0], h_nan), ("final", end, clean[1], h_nan[-1]),
                                    ("dx", dx, cg[0], dx_nan), ("df", df, cg[1], df_nan),
                                    ("dh0", dh0, cg[2], dx_nan[0] & open_)):
            nan = nan.to(dev)
            assert torch.equal(got.isnan(), nan), (what, name)
            assert torch.equal(got[~nan], ref[~nan]), (what, name)


NAN_SHAPES = [(9, 2, 16), (41, 4, 20), (200, 2, 33)]
# these are cut into segments, of one, two and four channels a lane
NAN_SHAPES_LONG = [(1100, 2, 24), (2100, 3, 1000), (4400, 3, 1000)]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("T,B,H", NAN_SHAPES)
def test_nan_gates_stay_in_their_document(T, B, H, dev):
    check_nan_stays_in_its_document(T, B, H, F32, dev, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,B,H", NAN_SHAPES_LONG)
def test_nan_gates_stay_in_their_document_long(T, B, H, dtype):
    check_nan_stays_in_its_document(T, B, H, dtype, "cuda", 0.0)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("T,B,H", NAN_SHAPES)
def test_nan_outlives_small_products(T, B, H, dev):
    """Gates whose product over eight steps is too small for fp32 (exp(-112)) are no starts."""
    check_nan_stays_in_its_document(T, B, H, F32, dev, -15.0)


@pytest.mark.gpu
@pytest.mark.parametrize("T,B,H,level", [s + (-15.0,) for s in NAN_SHAPES_LONG]
                         + [(40000, 1, 64, -1.0), (12000, 4, 360, -1.0)])
def test_nan_outlives_small_products_long(T, B, H, level):
    """Level -1: gates around a half, whose product over a segment's 200 steps or more is too small;
    documents of many segments."""
    check_nan_stays_in_its_document(T, B, H, F32, "cuda", level, every=max(37, T // 7))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("T,level", [(50, -14.0), (1300, -4.0)])
def test_marks_lose_no_bad_state(T, level, bad, dev):
    """A state or a gradient that is not finite stays so with lengths given, as it does without."""
    B, H = 2, 12
    x, f, h0, dh, dlast = inputs(T, B, H, F32, dev)
    f = torch.full_like(f, level)
    h0[0, 3], dlast[1, 5] = bad, bad
    lengths = torch.full((B,), T, dtype=torch.int32, device=dev)
    for n in (None, lengths):
        h, last, carry = R.linear_recurrence_fwd(x, f, h0, lengths=n)
        dx, df, dh0 = R.linear_recurrence_bwd(x, f, carry, dh, dlast=dlast, lengths=n)
        for got, at in ((h[:, 0, 3], True), (last[0, 3], True), (dx[:, 1, 5], True),
                        (df[:, 1, 5], True), (dh0[1, 5], True), (h[:, 1], False),
                        (last[1], False), (dx[:, 0], False), (dh0[0], False)):
            assert (got.isfinite() != at).all()


@pytest.mark.parametrize("dev", DEVS)
def test_saturated_gates(dev):
    """Gates at the ends of the range: the state is kept or replaced to the last digit."""
    T, B, H = 12, 2, 8
    x, _, h0, dh, dlast = inputs(T, B, H, F32, dev)
    keep = torch.full_like(x, 200.0)
    h, last, carry = R.linear_recurrence_fwd(x, keep, h0)
    assert torch.equal(last, h0) and torch.equal(h, h0.expand(T, B, H))
    dx, df, dh0 = R.linear_recurrence_bwd(x, keep, carry, dh, dlast=dlast)
    assert (dx == 0).all() and (df == 0).all()
    h, last, carry = R.linear_recurrence_fwd(x, -keep, h0)
    assert torch.equal(h, x) and torch.equal(last, x[-1])
    # a large gate's complement keeps its own digits: s(-30) = 9.4e-14
    far = torch.full_like(x, 30.0)
    _, last, _ = R.linear_recurrence_fwd(x, far, torch.zeros_like(h0))
    want = reference(x.double().cpu(), far.double().cpu(), torch.zeros(B, H).double(), None, None)
    want = (1 / (1 + torch.exp(far.double().cpu()))) * x.double().cpu()
    assert torch.allclose(last.double().cpu(), want.sum(0), rtol=1e-5, atol=0)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,H", [(1, 1), (3, 7), (5, 66), (256, 512)])
def test_step(B, H, dtype, dev):
    x, f, h0, _, _ = inputs(6, B, H, dtype, dev)
    starts = torch.rand(6, B, generator=torch.Generator().manual_seed(2)).to(dev) < 0.3
    h, last, _ = R.linear_recurrence_fwd(x, f, h0, starts=starts)
    s = h0.clone()
    M = max(x.abs().max().item(), h0.abs().max().item())
    for t in range(6):
        y = R.linear_recurrence_step(x[t], f[t], s, starts=starts[t])
        close(y, h[t].double(), 2 * (3 * 6 + 32) * 2.0 ** -24 * M
              + (2.0 ** -8 * M if dtype == BF16 else 0), "step")
    close(s, last.double(), 2 * (3 * 6 + 32) * 2.0 ** -24 * M, "state")


@pytest.mark.parametrize("dev", DEVS)
def test_autograd_matches_explicit_and_differences(dev):
    x, f, h0, dh, dlast = inputs(9, 2, 5, F32, dev)
    lengths, starts = marks(9, 2, "ls", dev)
    leaves = [v.clone().requires_grad_(True) for v in (x, f, h0)]
    h, last = R.linear_recurrence(*leaves, lengths=lengths, starts=starts)
    (h * dh).sum().backward(retain_graph=True)  # the final state unused
    (last * dlast).sum().backward()
    carry = R.linear_recurrence_fwd(x, f, h0, lengths=lengths, starts=starts)[2]
    want = R.linear_recurrence_bwd(x, f, carry, dh, dlast=dlast, lengths=lengths, starts=starts)
    for a, b in zip(leaves, want):
        assert torch.allclose(a.grad, b, rtol=1e-5, atol=1e-6)
    # central differences of step 2^-6 in fp32: truncation < 2^-12, rounding < 2^-24 * 64 * sum
    step = 2.0 ** -6
    for k, leaf in enumerate((x, f, h0)):
        flat = leaf.view(-1)
        for i in range(0, flat.numel(), 11):
            vals = []
            for s in (step, -step):
                moved = [v.clone() for v in (x, f, h0)]
                moved[k].view(-1)[i] += s
                hh, ll, _ = R.linear_recurrence_fwd(*moved, lengths=lengths, starts=starts)
                vals.append(((hh.double() * dh.double()).sum()
                             + (ll.double() * dlast.double()).sum()).item())
            got = want[k].reshape(-1)[i].item()
            assert abs((vals[0] - vals[1]) / (2 * step) - got) < 5e-3, (k, i)
    s = R.linear_recurrence(*leaves)[0].sum()  # an expanded gradient
    s.backward()


@pytest.mark.parametrize("dev", DEVS)
def test_lengths_are_clamped(dev):
    args = inputs(23, 4, 10, F32, dev)
    odd = torch.tensor([-5, 99, 23, 7], dtype=torch.int32, device=dev)
    a = R.linear_recurrence_fwd(*args[:3], lengths=odd)
    b = R.linear_recurrence_fwd(*args[:3], lengths=odd.clamp(0, 23))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = [R.linear_recurrence_bwd(*args[:2], a[2], args[3], dlast=args[4], lengths=n)
         for n in (odd, odd.clamp(0, 23))]
    assert all(torch.equal(p, q) for p, q in zip(*g))


@pytest.mark.gpu
def test_far_offsets():
    """Steps more than 2^31 elements apart."""
    T, B, H, far = 3, 2, 64, (1 << 30) + 64
    small = inputs(T, B, H, BF16, "cuda")
    bufs = [torch.empty(2 * far + B * H, dtype=BF16, device="cuda") for _ in range(3)]
    x, f, dh = (torch.as_strided(b, (T, B, H), (far, H, 1)) for b in bufs)
    for v, s in zip((x, f, dh), (small[0], small[1], small[3])):
        v.copy_(s)
    a = R.linear_recurrence_fwd(x, f, small[2])
    b = R.linear_recurrence_fwd(*small[:3])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = R.linear_recurrence_bwd(x, f, a[2], dh, dlast=small[4])
    w = R.linear_recurrence_bwd(small[0], small[1], b[2], small[3], dlast=small[4])
    assert all(torch.equal(p, q) for p, q in zip(g, w))


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    x = torch.zeros(4, 2, 6, device=dev)
    h0 = torch.zeros(2, 6, device=dev)
    i32 = torch.zeros(2, dtype=torch.int32, device=dev)
    st = torch.zeros(4, 2, dtype=torch.bool, device=dev)
    carry = R.linear_recurrence_fwd(x, x)[2]
    bad = [
        lambda: R.linear_recurrence_fwd(x[0], x[0]),
        lambda: R.linear_recurrence_fwd(x.half(), x.half()),
        lambda: R.linear_recurrence_fwd(x, x.bfloat16()),
        lambda: R.linear_recurrence_fwd(x, x[:3]),
        lambda: R.linear_recurrence_fwd(x.transpose(1, 2), x.transpose(1, 2)),
        lambda: R.linear_recurrence_fwd(x, x, h0[:1]),
        lambda: R.linear_recurrence_fwd(x, x, h0.double()),
        lambda: R.linear_recurrence_fwd(x, x, h0, lengths=i32.long()),
        lambda: R.linear_recurrence_fwd(x, x, h0, lengths=i32[:1]),
        lambda: R.linear_recurrence_fwd(x, x, h0, starts=st[:2]),
        lambda: R.linear_recurrence_fwd(x, x, h0, starts=st.int()),
        lambda: R.linear_recurrence_bwd(x, x, carry[:0], x),
        lambda: R.linear_recurrence_bwd(x, x, carry, x[:2]),
        lambda: R.linear_recurrence_bwd(x, x, carry, x, dlast=h0[:1]),
        lambda: R.linear_recurrence_step(x[0], x[0], h0[:1]),
        lambda: R.linear_recurrence_step(x[0], x[0], h0.t().contiguous().t()),
        lambda: R.linear_recurrence_step(x, x, h0),
    ]
    for fn in bad:
        with pytest.raises(RuntimeError):
            fn()


@pytest.mark.gpu
def test_refuses_mixed_devices():
    x = torch.zeros(4, 2, 6, device="cuda")
    with pytest.raises(RuntimeError):
        R.linear_recurrence_fwd(x, x, torch.zeros(2, 6))
    with pytest.raises(RuntimeError):
        R.linear_recurrence_fwd(x, x, lengths=torch.zeros(2, dtype=torch.int32))


@pytest.mark.gpu
def test_streams_and_graph_replays():
    """On another stream, and captured forward and backward replayed with new inputs: each replay
    equals the eager result, also with eager work in between."""
    x, f, h0, dh, dlast = inputs(600, 2, 96, BF16, "cuda")
    lengths, starts = marks(600, 2, "ls", "cuda")

    def both():
        h, last, carry = R.linear_recurrence_fwd(x, f, h0, lengths=lengths, starts=starts)
        return (h, last) + R.linear_recurrence_bwd(x, f, carry, dh, dlast=dlast, lengths=lengths,
                                                   starts=starts)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for k in range(4):
        n = inputs(600, 2, 96, BF16, "cuda", seed=10 + k)
        for a, b in zip((x, f, h0, dh, dlast), n):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, both()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,B,H", [(7, 3, 5), (40, 5, 36), (1100, 2, 24)])
def test_broadcast_inputs(T, B, H, dtype):
    """Candidates that are the same at every step, gates that are the same in every stream, starts in
    common: results as of copies, and the gradients of what was broadcast are the sums."""
    dev = "cuda"
    x, f, h0, dh, dlast = inputs(T, B, H, dtype, dev)
    starts = marks(T, 1, "s", dev)[1].expand(T, B)
    lengths = marks(T, B, "l", dev)[0]
    v, w = x[0].clone().requires_grad_(True), f[:, :1].clone().requires_grad_(True)
    xs, fs = v.expand(T, B, H), w.expand(T, B, H)
    h, last = R.linear_recurrence(xs, fs, h0, lengths=lengths, starts=starts)
    torch.autograd.backward([h, last], [dh, dlast])
    a, b = xs.detach().contiguous(), fs.detach().contiguous()
    want_h, want_last, carry = R.linear_recurrence_fwd(a, b, h0, lengths=lengths,
                                                       starts=starts.contiguous())
    assert torch.equal(h, want_h) and torch.equal(last, want_last)
    dx, df, _ = R.linear_recurrence_bwd(a, b, carry, dh, dlast=dlast, lengths=lengths,
                                        starts=starts.contiguous())
    assert torch.equal(v.grad, dx.sum(0)) and torch.equal(w.grad, df.sum(1, keepdim=True))
