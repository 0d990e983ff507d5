"""The gated linear recurrence over a sequence, beside the LSTM / GRU / BasicRNN cells:

    h_t = a_t h_{t-1} + s(-f_t) x_t,    a_t = s(f_t), or 0 where ``starts[t, b]``

with ``s`` the logistic function, ``x`` the candidates and ``f`` the gate pre-activations, both
``[T, B, H]`` (time-major, as everywhere in the framework; any strides along T and B, so a
transposed batch-first tensor or one half of a fused projection ``[T, B, 2H]`` is taken as it
is).  Nothing in the step depends on ``h_{t-1}`` but the state itself, so unlike the other cells
it needs no pass over the weights per step: the whole sequence is one or two launches.

``starts`` (bool ``[T, B]``) marks steps that begin a document: the state restarts there.
``lengths`` (int32 ``[B]``, clamped to ``[0, T]``) are the sequences' own lengths in a padded
batch: behind them output rows are zero, gradients are zero, the padding is never read into a
result, and the final state is the one after the sequence's last step (``h0`` for length 0).  A
NaN reaches what depends on it, to its document's last step (backward: its first), and nothing
else; an infinite state stays one or becomes NaN.

Inputs and outputs are fp32 or bf16; states (``h0``, the final state, their gradients and the
sums inside) are fp32.  GPU tensors take the HIP kernels (csrc/linrec.hip), CPU tensors the plain
form below.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import native

Opt = Optional[torch.Tensor]


def linear_recurrence_fwd(x: torch.Tensor, f: torch.Tensor, h0: Opt = None, *,
                          lengths: Opt = None, starts: Opt = None, want_carry: bool = True
                          ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(h [T, B, H], final state [B, H], carry)``.  ``carry`` holds the fp32 states that
    :func:`linear_recurrence_bwd` starts from; it is empty without ``want_carry``."""
    if x.is_cuda:
        return native.op("linrec_fwd")(x, f, h0, lengths, starts, want_carry)
    _check(x, f, h0, lengths, starts)
    return _cpu_fwd(x, f, h0, lengths, starts, want_carry)


def linear_recurrence_bwd(x: torch.Tensor, f: torch.Tensor, carry: torch.Tensor,
                          dh: torch.Tensor, *, dlast: Opt = None, lengths: Opt = None,
                          starts: Opt = None
                          ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dx, df, dh0)`` from the gradients of the outputs (``dh``, in ``x``'s type) and of the
    final state (``dlast`` fp32, absent: zero).  ``x``, ``f``, ``lengths`` and ``starts`` are the
    forward's, ``carry`` what it returned."""
    if x.is_cuda:
        return native.op("linrec_bwd")(x, f, carry, dh, dlast, lengths, starts)
    _check(x, f, dlast, lengths, starts)
    torch._check(dh.shape == x.shape and dh.dtype == x.dtype, lambda: "dh must be like x")
    torch._check(carry.shape == x.shape, lambda: "carry must be the forward's")
    return _cpu_bwd(x, f, carry, dh, dlast, lengths, starts)


def linear_recurrence_step(x: torch.Tensor, f: torch.Tensor, h: torch.Tensor, *,
                           starts: Opt = None) -> torch.Tensor:
    """One step of every stream: ``x``, ``f`` ``[B, H]``; the fp32 state ``h`` is updated in
    place and its copy in ``x``'s type returned.  ``starts``: bool ``[B]``."""
    if x.is_cuda:
        return native.op("linrec_step")(x, f, h, starts)
    torch._check(x.dim() == 2, lambda: "x and f must be [B, H]")
    torch._check(h.is_contiguous(), lambda: "h must be contiguous")
    st = None if starts is None else starts[None]
    _check(x[None], f[None], h, None, st)
    y, last, _ = _cpu_fwd(x[None], f[None], h, None, st, False)
    h.copy_(last)
    return y[0]


def linear_recurrence(x: torch.Tensor, f: torch.Tensor, h0: Opt = None, *, lengths: Opt = None,
                      starts: Opt = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(h, final state)``, differentiable (once) in ``x``, ``f`` and ``h0``."""
    return _LinearRecurrence.apply(x, f, h0, lengths, starts)


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, h0, lengths, starts):
        need = any(ctx.needs_input_grad[:3])
        h, last, carry = linear_recurrence_fwd(x, f, h0, lengths=lengths, starts=starts,
                                               want_carry=need)
        ctx.save_for_backward(x, f, carry, lengths, starts)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        x, f, carry, lengths, starts = ctx.saved_tensors
        if dh is None:
            dh = torch.zeros_like(x)
        elif x.shape[-1] > 1 and dh.stride(-1) != 1:  # e.g. the expanded gradient of a sum
            dh = dh.contiguous()
        if dlast is not None:
            dlast = dlast.contiguous()
        dx, df, dh0 = linear_recurrence_bwd(x, f, carry, dh, dlast=dlast, lengths=lengths,
                                            starts=starts)
        need = ctx.needs_input_grad
        return (dx if need[0] else None, df if need[1] else None, dh0 if need[2] else None,
                None, None)


# ---- plain form (CPU): the same arithmetic in fp32, one step after the other -----------------
def _check(x, f, state, lengths, starts):
    ok = torch._check
    ok(x.dim() == 3, lambda: "x must be [T, B, H]")
    ok(x.dtype in (torch.float32, torch.bfloat16), lambda: "x must be float32 or bfloat16")
    ok(f.shape == x.shape and f.dtype == x.dtype and f.device == x.device,
       lambda: "f must be like x")
    for t in (x, f):
        ok(t.shape[2] <= 1 or t.stride(2) == 1,
           lambda: "x and f need unit stride along their last dimension")
    if state is not None:
        ok(state.shape == x.shape[1:] and state.dtype == torch.float32
           and state.device == x.device and state.is_contiguous(),
           lambda: "states must be [B, H] float32, contiguous")
    if lengths is not None:
        ok(lengths.shape == x.shape[1:2] and lengths.dtype == torch.int32
           and lengths.device == x.device and lengths.is_contiguous(),
           lambda: "lengths must be [B] int32, contiguous")
    if starts is not None:
        ok(starts.shape == x.shape[:2] and starts.dtype == torch.bool
           and starts.device == x.device, lambda: "starts must be [T, B] bool")


def _live(t, B, lengths):
    return None if lengths is None else (t < lengths)[:, None]


def _cpu_fwd(x, f, h0, lengths, starts, want_carry):
    T, B, H = x.shape
    h = torch.zeros(B, H) if h0 is None else h0.clone()
    out, carry = torch.empty_like(x), torch.empty(T if want_carry else 0, B, H)
    for t in range(T):
        if want_carry:
            carry[t] = h
        ft = f[t].float()
        new = torch.sigmoid(ft) * h
        if starts is not None:
            new = torch.where(starts[t][:, None], 0.0, new)
        new = new + torch.sigmoid(-ft) * x[t].float()
        live = _live(t, B, lengths)
        out[t] = new if live is None else torch.where(live, new, 0.0)
        h = new if live is None else torch.where(live, new, h)
    return out, h, carry


def _cpu_bwd(x, f, carry, dh, dlast, lengths, starts):
    T, B, H = x.shape
    e = torch.zeros(B, H) if dlast is None else dlast.clone()
    dx, df = torch.empty_like(x), torch.empty_like(f)
    for t in reversed(range(T)):
        keep, take = torch.sigmoid(f[t].float()), torch.sigmoid(-f[t].float())
        prev, g = carry[t], dh[t].float() + e
        back = keep * g
        if starts is not None:
            cut = starts[t][:, None]
            prev, back = torch.where(cut, 0.0, prev), torch.where(cut, 0.0, back)
        ox, of = take * g, keep * take * g * (prev - x[t].float())
        live = _live(t, B, lengths)
        if live is not None:
            ox, of = torch.where(live, ox, 0.0), torch.where(live, of, 0.0)
            back = torch.where(live, back, e)
        dx[t], df[t], e = ox, of, back
    return dx, df, e
