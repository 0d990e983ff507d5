"""The gated linear recurrence (csrc/linrec.hip) against its formulas in float64, element by element
within a first-order bound of the rounding errors, at the sizes whose time axis is cut into segments.

The bound.  u = 2^-24; a step's gate s(f) is off by at most (2 |f| + 9) u of itself: the argument of the
exponential as rounded twice (2 |f| u), the exponential and the reciprocal (2 u each), the sum, the
products.  With |f| < 7 and a rounding each of a product and a sum, a value is off by less than C u of
itself for every step it goes through, C = 32 -- whether the steps are multiplied one after the other
or as pairs, which add a rounding in eight steps.  What goes in at step s and comes out at step t has
gone through t - s + 1 of them, so with

    S_t = a_t S_{t-1} + s(-f_t) |x_t|,  P_t = a_t P_{t-1} + S_t   (S_0 from |h0|, P_0 = 0)

the state is off by C u P_t; the same for the gradient's recursion, G_t = |dh_t| + E_{t+1},
E_t = a_t G_t, Q_t = a_t (Q_{t+1} + G_t):

    dx_t  s(-f) C u (Q_{t+1} + 2 G_t),      dh0  C u Q_0,
    df_t  s(f) s(-f) C u [(Q_{t+1} + 3 G_t) (S_{t-1} + |x_t|) + G_t P_{t-1}].

A bf16 output adds half its step."""
import os

import pytest
import torch

from distributed_char_rnn_amd.ops import recurrence as R

LIB = os.path.join(os.path.dirname(__file__), "..", "distributed_char_rnn_amd", "_C.so")
F32, BF16 = torch.float32, torch.bfloat16
C, U = 32, 2.0 ** -24
NAMES = ("h", "last", "dx", "df", "dh0")


def formulas(x, f, h0, dh, dlast, lengths, starts):
    """Values and bounds of (h, last, dx, df, dh0), float64 on the inputs' device."""
    x, f, h0, dh, dlast = (v.double() for v in (x, f, h0, dh, dlast))
    T = x.shape[0]
    on = [None] * T if lengths is None else [(t < lengths)[:, None] for t in range(T)]
    keep, take = torch.sigmoid(f), torch.sigmoid(-f)
    zero = torch.zeros_like(h0)
    outs = [torch.zeros_like(x) for _ in range(4)]  # h, its bound, then those in front of the step
    (hs, hb, prev, pb), sb = outs, torch.zeros_like(x)

    def only(t, new, old):
        return new if on[t] is None else torch.where(on[t], new, old)

    def cut(t, v):
        return v if starts is None else torch.where(starts[t][:, None], zero, v)

    h, S, P = h0, h0.abs(), zero
    for t in range(T):
        a = cut(t, keep[t])
        prev[t], sb[t], pb[t] = cut(t, h), cut(t, S), cut(t, P)
        new = a * prev[t] + take[t] * x[t]
        nS = a * sb[t] + take[t] * x[t].abs()
        nP = a * pb[t] + nS
        hs[t], hb[t] = only(t, new, zero), only(t, nP, zero)
        h, S, P = only(t, new, h), only(t, nS, S), only(t, nP, P)
    last, lastb = h, P
    dx, dxb, df, dfb = (torch.zeros_like(x) for _ in range(4))
    e, E, Q = dlast, dlast.abs(), zero
    for t in reversed(range(T)):
        a = cut(t, keep[t])
        g, G = dh[t] + e, dh[t].abs() + E
        dx[t], dxb[t] = only(t, take[t] * g, zero), only(t, take[t] * (Q + 2 * G), zero)
        kt = keep[t] * take[t]
        df[t] = only(t, kt * g * (prev[t] - x[t]), zero)
        dfb[t] = only(t, kt * ((Q + 3 * G) * (sb[t] + x[t].abs()) + G * pb[t]), zero)
        e, E, Q = only(t, a * g, e), only(t, a * G, E), only(t, a * (Q + G), Q)
    return (hs, last, dx, df, e), tuple(C * U * b for b in (hb, lastb, dxb, dfb, Q))


def run(x, f, h0, dh, dlast, lengths, starts):
    h, last, carry = R.linear_recurrence_fwd(x, f, h0, lengths=lengths, starts=starts)
    return (h, last) + R.linear_recurrence_bwd(x, f, carry, dh, dlast=dlast, lengths=lengths,
                                               starts=starts)


def misses(got, want, bounds):
    """The outputs that leave their bound."""
    out = []
    for name, g, w, b in zip(NAMES, got, want, bounds):
        half = torch.finfo(g.dtype).eps / 2 if g.dtype == BF16 else 0.0
        over = (g.double() - w).abs() - (b + half * (w.abs() + b) + 2.0 ** -126)
        if not (over <= 0).all():
            out.append(name)
    return out


def inputs(T, B, H, dtype, dev, which, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, shift=0.0):
        return torch.randn(*shape, device=dev, generator=g) + shift

    x, f, dh = normal(T, B, H).to(dtype), normal(T, B, H, shift=1.0).to(dtype), \
        normal(T, B, H).to(dtype)
    f = f.clamp(-7, 7)
    lengths = starts = None
    if "l" in which:
        lengths = torch.linspace(T, T // 3, B, device=dev).to(torch.int32)
    if "s" in which:
        starts = torch.rand(T, B, device=dev, generator=g) < 8.0 / T
    return x, f, normal(B, H), dh, normal(B, H), lengths, starts


@pytest.mark.parametrize("which", ["", "l", "s", "ls"])
def test_formulas_are_the_definitions_derivatives(which):
    """The float64 form above against automatic differentiation of the recurrence."""
    x, f, h0, dh, dlast, lengths, starts = inputs(40, 3, 5, F32, "cpu", which)
    (h, last, dx, df, dh0), _ = formulas(x, f, h0, dh, dlast, lengths, starts)
    leaves = [v.double().requires_grad_(True) for v in (x, f, h0)]
    s, rows = leaves[2], []
    for t in range(40):
        a = torch.sigmoid(leaves[1][t])
        p = s if starts is None else torch.where(starts[t][:, None], 0.0, s)
        new = a * p + (1 - a) * leaves[0][t]
        live = torch.ones(3, 1, dtype=torch.bool) if lengths is None else (t < lengths)[:, None]
        rows.append(torch.where(live, new, 0.0))
        s = torch.where(live, new, s)
    grads = torch.autograd.grad([torch.stack(rows), s], leaves, [dh.double(), dlast.double()])
    for a, b in zip((h, last, dx, df, dh0), (torch.stack(rows), s) + grads):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("which", ["", "ls"])
def test_bounds_hold_and_find_mistakes(which):
    """The CPU form keeps the bounds, and leaves them where the formulas are given a mistake: a
    gradient scaled, the state or the gradient dropped at one border of 64 steps."""
    T, B, H = 400, 2, 24
    args = inputs(T, B, H, F32, "cpu", which)
    got = run(*args)
    want, bounds = formulas(*args)
    assert misses(got, want, bounds) == []
    for i, factor in ((0, 1.001), (2, 0.999), (3, 0.5), (3, 1.001), (4, 0.99)):
        wrong = list(want)
        wrong[i] = want[i] * factor
        assert misses(got, wrong, bounds) == [NAMES[i]]
    starts = torch.zeros(T, B, dtype=torch.bool) if args[6] is None else args[6].clone()
    starts[64, 0] = True  # as if a segment's border let nothing through
    wrong, _ = formulas(*args[:6], starts)
    found = misses(got, wrong, bounds)
    assert "h" in found and "dx" in found and "df" in found


def plan(T, B, H, bf16):
    torch.ops.load_library(LIB)
    return tuple(torch.ops.dcr.linrec_plan(T, B, H, bf16))


@pytest.mark.skipif(not os.path.exists(LIB), reason="native library not built")
def test_plans_cover_the_steps():
    """Every tile in a segment, every segment with a tile, launches within their limits."""
    g = torch.Generator().manual_seed(0)

    def size(most):
        return int(torch.exp(torch.rand((), generator=g) * torch.log(torch.tensor(float(most)))))

    for i in range(3000):
        T, B, H = size(1 << 20), size(512), size(4096)
        vec, waves, tiles, segs, per = plan(T, B, H, i % 2 == 0)
        assert H % vec == 0 and vec in (1, 2, 4) and waves in (1, 2, 4, 8)
        assert waves * vec <= 16
        assert (tiles - 1) * waves * 8 < T <= tiles * waves * 8
        assert (segs - 1) * per < tiles <= segs * per and 1 <= segs <= 128
        assert -(-B * (H // vec) // 64) * 64 * waves < 1 << 32


# (T, B, H) and what its plan has to be: channels a lane, waves, tiles of a segment
SEGMENTED = [((4500, 3, 1000), (4, 4, 2)), ((9001, 3, 1000), (4, 4, 4)), ((4500, 2, 998), (2, 8, 3)),
             ((8211, 2, 66), (1, 8, 2))]


@pytest.mark.skipif(not os.path.exists(LIB), reason="native library not built")
@pytest.mark.parametrize("size,want", SEGMENTED)
@pytest.mark.parametrize("bf16", [False, True])
def test_segmented_sizes_reach_their_forms(size, want, bf16):
    vec, waves, tiles, segs, per = plan(*size, bf16)
    assert (vec, waves, per) == want and segs > 1
    assert tiles % per != 0  # the last segment is short


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", ["", "ls"])
@pytest.mark.parametrize("size", [s for s, _ in SEGMENTED])
def test_segments_against_the_formulas(size, which, dtype):
    args = inputs(*size, dtype, "cuda", which)
    assert misses(run(*args), *formulas(*args)) == []


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", ["", "l", "s"])
@pytest.mark.parametrize("size", [(1, 3, 7), (33, 4, 130), (129, 3, 257), (300, 1, 512),
                                  (1025, 1, 64), (700, 3, 1000), (40, 300, 512)])
def test_forms_against_the_formulas(size, which, dtype):
    args = inputs(*size, dtype, "cuda", which)
    assert misses(run(*args), *formulas(*args)) == []


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [(7, 3, 5), (40, 5, 36), (600, 2, 24)])
def test_broadcast_inputs_against_the_formulas(size, dtype, dev):
    """Inputs of stride zero: one step for all, one stream for all.  (On the CPU not bit by bit those of
    copies: its logistic function of a strided tensor is another of two forms.)"""
    T, B, H = size
    x, f, h0, dh, dlast, lengths, starts = inputs(T, B, H, dtype, dev, "ls")
    args = (x[:1].expand(T, B, H), f[:, :1].expand(T, B, H), h0, dh[:, :1].expand(T, B, H), dlast,
            lengths, starts[:, :1].expand(T, B))
    assert misses(run(*args), *formulas(*args)) == []
