"""Cases of the operators beside the recurrent cells and the softmax head: the gated linear
recurrence (training pass, forward pass, single-token step), a teacher's top logits, the
distillation loss with its gradient, and sampling with temperature, top-k, top-p and min-p.

Where ``own`` is false, :func:`run` computes them in their plain form (elementary torch
operations in 32 bits, 64 where a whole number depends on the value), otherwise it calls the
framework.  :func:`exact` gives the definition in 64 bits.
"""
import math

import torch

own = False

F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"fp32": F32, "bf16": BF16}
SIZE = {"fp32": 4, "bf16": 2}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _rec(mode, T, B, H, dtype, ragged=False, starts=False, batch_first=False):
    return dict(op="recurrence", mode=mode, T=T, B=B, H=H, dtype=dtype, ragged=ragged,
                starts=starts, batch_first=batch_first)


def _top(N, V, k, dtype, temperature):
    return dict(op="top", N=N, V=V, k=k, dtype=dtype, temperature=temperature)


def _distill(N, V, k, dtype, grad, alpha, temperature, tail):
    return dict(op="distill", N=N, V=V, k=k, dtype=dtype, grad=grad, alpha=alpha,
                temperature=temperature, tail=tail)


def _sample(N, V, dtype, per_row, temperature, top_k, top_p, min_p, masked):
    return dict(op="sample", N=N, V=V, dtype=dtype, per_row=per_row, temperature=temperature,
                top_k=top_k, top_p=top_p, min_p=min_p, masked=masked)


def listed():
    return [
        # the trainer's default shape (batch 50, sequence 50, rnn_size 128): launch-bound
        dict(_rec("train", 50, 50, 128, "fp32"), name="recurrence train default"),
        # the headline shape of the benchmark (seq 128, batch 256, rnn_size 512)
        dict(_rec("train", 128, 256, 512, "bf16"), name="recurrence train headline"),
        # a few long documents, packed and padded, with a size that is no power of two
        dict(_rec("train", 16384, 4, 1000, "bf16", ragged=True, starts=True),
             name="recurrence train long ragged"),
        # one stream's long prompt, batch-first, before sampling
        dict(_rec("forward", 4096, 1, 512, "bf16", batch_first=True),
             name="recurrence prompt"),
        # one token of 256 streams
        dict(_rec("step", 1, 256, 512, "bf16"), name="recurrence step"),
        # a teacher's record over one small batch of characters
        dict(_top(50, 65, 16, "fp32", 2.0), name="top small"),
        # a teacher's record over a whole training batch (256 x 128) of the 8k vocabulary
        dict(_top(32768, 8192, 64, "fp32", 1.0), name="top wide"),
        # a student's step at the trainer's default shape, characters
        dict(_distill(2500, 65, 8, "fp32", "fp32", 0.5, 2.0, True), name="distill default"),
        # a student's step over a whole training batch of the 8k vocabulary, as the head has it:
        # fp32 logits, bf16 gradient
        dict(_distill(32768, 8192, 64, "fp32", "bf16", 0.7, 2.0, True), name="distill wide"),
        # an odd vocabulary in bf16, teacher's entries alone
        dict(_distill(2047, 32001, 32, "bf16", "bf16", 1.0, 1.0, False), name="distill odd"),
        # one character of 16 streams
        dict(_sample(16, 65, "fp32", False, 0.8, 20, 0.95, 0.0, False), name="sample characters"),
        # a serving batch whose requests differ in every setting, some tokens masked
        dict(_sample(256, 32001, "bf16", True, 0.0, 0, 0.0, 0.0, True), name="sample mixed"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "top", "distill", "sample"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "recurrence":
        mode = rng.choice(["train", "train", "forward", "step"])
        B, H = _log(rng, 1, 256), _log(rng, 32, 2048)
        if rng.random() < 0.6:
            H = max(32, H // 32 * 32)
        most = (1 << 26) if dtype == "bf16" else (1 << 25)
        T = 1 if mode == "step" else _log(rng, 1, max(1, min(16384, most // (B * H))))
        plain = mode == "step"
        return _rec(mode, T, B, H, dtype, not plain and rng.random() < 0.4,
                    not plain and rng.random() < 0.4, not plain and rng.random() < 0.4)
    if op == "sample":
        V = _log(rng, 32, 131072)
        N = _log(rng, 1, max(1, min(4096, (1 << 23) // V)))
        per_row = rng.random() < 0.4
        return _sample(N, V, dtype, per_row, 0.0 if per_row else round(rng.uniform(0.3, 1.5), 3),
                       0 if per_row else rng.choice([0, 0, _log(rng, 1, V)]),
                       0.0 if per_row else rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                       0.0 if per_row else rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.3), 3)]),
                       rng.random() < 0.3)
    V = _log(rng, 32, 131072)
    N = _log(rng, 1, max(1, min(32768, (1 << 27) // V)))
    k = _log(rng, 1, min(V, 256))
    if op == "top":
        return _top(N, V, k, dtype, round(rng.uniform(0.5, 4.0), 3))
    tail = rng.random() < 0.5
    alpha = rng.choice([1.0, round(rng.uniform(0.1, 0.9), 3)])
    grad = "bf16" if dtype == "bf16" else rng.choice(["fp32", "bf16"])
    return _distill(N, V, k, dtype, grad, alpha, round(rng.uniform(0.5, 4.0), 3), tail)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, device="cuda", generator=g, dtype=torch.int32)

    dt = TYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "recurrence":
        T, B, H = case["T"], case["B"], case["H"]
        if case["mode"] == "step":
            # gates around +2: a state that remembers some eight tokens
            return dict(s, x=normal(B, H).to(dt), f=(normal(B, H) + 2.0).to(dt), h=normal(B, H))

        def seq(shift=0.0):  # [T, B, H]; batch-first programs hold it as a view of [B, T, H]
            if case["batch_first"]:
                return (normal(B, T, H) + shift).to(dt).transpose(0, 1)
            return (normal(T, B, H) + shift).to(dt)

        s.update(x=seq(), f=seq(2.0), h0=normal(B, H), lengths=None, start=None)
        if case["ragged"]:
            s["lengths"] = whole(0, T + 1, B)
        if case["starts"]:
            s["start"] = uniform(T, B) < min(0.5, 8.0 / T)
        if case["mode"] == "train":
            s.update(dh=seq(), dlast=normal(B, H))
        return s
    N, V = case["N"], case["V"]
    s["logits"] = (normal(N, V) * 2.5).to(dt)
    if case["op"] == "top":
        return s
    if case["op"] == "distill":
        # a teacher near the student: its logits are the student's and some more
        t = s["logits"].float() + normal(N, V)
        top = torch.topk(t, case["k"], dim=1)
        s.update(values=top.values, indices=top.indices.to(torch.int32), lse=None, targets=None)
        if case["tail"]:
            s["lse"] = torch.logsumexp(t / case["temperature"], 1)
        if case["alpha"] < 1.0:
            s["targets"] = whole(0, V, N)
        return s
    s["u"] = uniform(N)
    if case["masked"]:
        s["logits"].masked_fill_(uniform(N, V) < 0.3, -math.inf)
    if case["per_row"]:
        s.update(temperature=0.3 + 1.2 * uniform(N), top_p=0.3 + 0.8 * uniform(N),
                 min_p=torch.clamp(0.4 * uniform(N) - 0.2, min=0.0),
                 top_k=torch.exp(uniform(N) * math.log(2.0 * V)).to(torch.int32))
        s["temperature"][::7] = 0.0  # some requests are greedy
        s["top_k"][1::5] = 0         # some set no top-k
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    with torch.no_grad():
        return (_own if own else _plain)[state["op"]](state)


def _own_recurrence(s):
    from distributed_char_rnn_amd.ops import recurrence as rec

    if s["mode"] == "step":
        return rec.linear_recurrence_step(s["x"], s["f"], s["h"]), s["h"]
    h, last, carry = rec.linear_recurrence_fwd(s["x"], s["f"], s["h0"], lengths=s["lengths"],
                                               starts=s["start"], want_carry=s["mode"] == "train")
    if s["mode"] == "forward":
        return h, last
    dx, df, dh0 = rec.linear_recurrence_bwd(s["x"], s["f"], carry, s["dh"], dlast=s["dlast"],
                                            lengths=s["lengths"], starts=s["start"])
    return h, last, dx, df, dh0


def _own_top(s):
    from distributed_char_rnn_amd.ops import vocab

    return vocab.top_logits(s["logits"], s["k"], temperature=s["temperature"])


def _own_distill(s):
    from distributed_char_rnn_amd.ops import vocab

    return vocab.distill_xent(s["logits"], s["values"], s["indices"], top_lse=s["lse"],
                              targets=s["targets"], alpha=s["alpha"],
                              temperature=s["temperature"], grad_dtype=TYPES[s["grad"]])


def _own_sample(s):
    from distributed_char_rnn_amd.ops import vocab

    return vocab.sample_logits(s["logits"], s["u"], temperature=s["temperature"],
                               top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


_own = dict(recurrence=_own_recurrence, top=_own_top, distill=_own_distill, sample=_own_sample)


# ---------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 0, doubling the span combined in each round."""
    d, T = 1, a.shape[0]
    while d < T:
        b = torch.cat([b[:d], torch.addcmul(b[d:], a[d:], b[:-d])])
        if 2 * d < T:
            a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _plain_recurrence(s):
    dt = s["x"].dtype
    x, f = s["x"].float(), s["f"].float()
    keep, take = torch.sigmoid(f), torch.sigmoid(-f)
    if s["mode"] == "step":
        s["h"].copy_(keep * s["h"] + take * x)
        return s["h"].to(dt), s["h"]
    T, B, H = x.shape
    a, b = keep, take * x
    live = None
    if s["start"] is not None:
        a = torch.where(s["start"][:, :, None], torch.zeros_like(a), a)
    if s["lengths"] is not None:
        live = (torch.arange(T, device=x.device)[:, None] < s["lengths"][None, :])[:, :, None]
        a = torch.where(live, a, torch.ones_like(a))
        b = torch.where(live, b, torch.zeros_like(b))
    b = torch.cat([torch.addcmul(b[:1], a[:1], s["h0"][None]), b[1:]])
    h = _scan(a, b)
    last = h[-1]
    y = (h if live is None else torch.where(live, h, torch.zeros_like(h))).to(dt)
    if s["mode"] == "forward":
        return y, last
    dh = s["dh"].float()
    if live is not None:
        dh = torch.where(live, dh, torch.zeros_like(dh))
    # g_t = dh_t + a_{t+1} g_{t+1}, the last step's with the final state's gradient
    dh = torch.cat([dh[:-1], dh[-1:] + s["dlast"][None]])
    g = _scan(torch.cat([a[:1], a[1:].flip(0)]), dh.flip(0)).flip(0)
    prev = torch.cat([s["h0"][None], h[:-1]])
    if s["start"] is not None:
        prev = torch.where(s["start"][:, :, None], torch.zeros_like(prev), prev)
    dx, df = take * g, keep * take * g * (prev - x)
    if live is not None:
        dx, df = (torch.where(live, v, torch.zeros_like(v)) for v in (dx, df))
    return y, last, dx.to(dt), df.to(dt), a[0] * g[0]


def _plain_top(s):
    z = s["logits"].float()
    values, indices = torch.sort(z, dim=1, descending=True, stable=True)
    m = values[:, :1]
    lse = torch.exp((z - m) / s["temperature"]).sum(1).log() + m[:, 0] / s["temperature"]
    k = s["k"]
    return values[:, :k].contiguous(), indices[:, :k].to(torch.int32), lse


def _distill_terms(s, z):
    """Row losses and their gradient (times the number of rows) in ``z``'s type."""
    tau, alpha = s["temperature"], s["alpha"]
    idx = s["indices"].long()
    t = s["values"].to(z.dtype) / tau
    zt = z / tau
    m = zt.max(1, keepdim=True).values
    e = torch.exp(zt - m)
    p = e / e.sum(1, keepdim=True)
    logp = zt - m - e.sum(1, keepdim=True).log()
    lk = logp.gather(1, idx)
    rest = torch.ones_like(p).scatter_(1, idx, 0.0)
    if s["lse"] is not None:
        logq = t - s["lse"].to(z.dtype)[:, None]
        q = torch.exp(logq)
        r = (1.0 - q.sum(1, keepdim=True)).clamp_min(0.0)
        left = (p * rest).sum(1, keepdim=True)
        has = (r > 0) & (left > 0)
        tail = torch.where(has, r * (r.log() - left.log()), torch.zeros_like(r))
        share = torch.where(has, r / left, torch.zeros_like(r))
        kl = (q * (logq - lk)).sum(1) + tail[:, 0]
        grad = p - p * rest * share
    else:
        tm = t.max(1, keepdim=True).values
        logq = t - tm - torch.exp(t - tm).sum(1, keepdim=True).log()
        q = torch.exp(logq)
        kl = (q * (logq - lk)).sum(1)
        grad = p
    grad = grad.scatter_add(1, idx, -q) * (alpha * tau)
    loss = alpha * tau * tau * kl
    if alpha < 1.0:
        y = s["targets"].long()[:, None]
        m1 = z.max(1, keepdim=True).values
        e1 = torch.exp(z - m1)
        s1 = e1.sum(1, keepdim=True)
        p1 = e1 / s1
        loss = loss + (1 - alpha) * (s1.log() + m1 - z.gather(1, y))[:, 0]
        grad = grad + (1 - alpha) * p1.scatter_add(1, y, -torch.ones_like(p1[:, :1]))
    return loss, grad


def _plain_distill(s):
    n = s["logits"].shape[0]
    rows, grad = _distill_terms(s, s["logits"].float())
    return rows.sum() / n, rows, (grad / n).to(TYPES[s["grad"]])


def _plain_sample(s):
    # 64 bits: the answer is a whole number, and a value next to a border decides it
    z = s["logits"].double()
    n, v = z.shape

    def row(p):
        return p.double()[:, None] if isinstance(p, torch.Tensor) else torch.full(
            (n, 1), p, dtype=F32, device=z.device).double()

    tau, top_p, min_p, top_k = (row(s[k]) for k in ("temperature", "top_p", "min_p", "top_k"))
    zs, order = torch.sort(z, dim=1, descending=True, stable=True)
    greedy = ~(tau > 0)
    w = torch.exp((zs - zs[:, :1]) / torch.where(greedy, torch.ones_like(tau), tau))
    rank = torch.arange(v, device=z.device)[None, :]
    keep = (top_k <= 0) | (rank < top_k)
    w = torch.where(keep, w, torch.zeros_like(w))
    before = torch.cumsum(w, 1) - w
    keep &= (top_p >= 1) | (rank == 0) | (before < top_p * w.sum(1, keepdim=True))
    keep &= w >= min_p
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    cdf = torch.cumsum(w, 1)
    pick = torch.searchsorted(cdf, s["u"].double()[:, None] * cdf[:, -1:], right=True)
    last = torch.where(w > 0, rank, torch.zeros_like(order)).max(1, keepdim=True).values
    pick = torch.where(greedy, order[:, :1], torch.minimum(pick, last))
    return pick[:, 0].to(torch.int32)


_plain = dict(recurrence=_plain_recurrence, top=_plain_top, distill=_plain_distill,
              sample=_plain_sample)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "recurrence":
        n, st = case["T"] * case["B"] * case["H"], case["B"] * case["H"] * 4
        if case["mode"] == "step":
            return {"bytes": 3 * n * e + 2 * st, "flops": 8 * n}
        if case["mode"] == "forward":
            return {"bytes": 3 * n * e + 2 * st, "flops": 8 * n}
        return {"bytes": 6 * n * e + 4 * st, "flops": 20 * n}
    n = case["N"] * case["V"]
    if case["op"] == "top":
        return {"bytes": n * e + case["N"] * (8 * case["k"] + 4), "flops": 4 * n}
    if case["op"] == "distill":
        return {"bytes": n * (e + SIZE[case["grad"]]) + case["N"] * (8 * case["k"] + 12),
                "flops": 12 * n}
    return {"bytes": n * e + case["N"] * 8, "flops": 6 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "recurrence":
        return _exact_recurrence(s)
    if case["op"] == "sample":
        return None  # whole numbers
    z = s["logits"]
    if case["op"] == "top":
        at = _sorted_top(z, case["k"])
        lse = torch.stack([torch.logsumexp(r.double() / case["temperature"], 0) for r in z]) \
            if z.shape[0] <= 64 else torch.cat(
                [torch.logsumexp(r.double() / case["temperature"], 1) for r in z.split(1024)])
        return at, None, lse
    return _exact_distill(s)


def _sorted_top(z, k):
    return torch.cat([r.double().sort(1, descending=True).values[:, :k] for r in z.split(2048)])


def _exact_recurrence(s):
    x, f = s["x"].double(), s["f"].double()
    if s["mode"] == "step":
        h = torch.sigmoid(f) * s["h"].double() + torch.sigmoid(-f) * x
        return h, h
    T, B, H = x.shape
    h, rows, before = s["h0"].double(), [], []
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), T, device=x.device)
    for t in range(T):
        p = torch.sigmoid(f[t])
        old = h if s["start"] is None else torch.where(s["start"][t][:, None], 0.0, h)
        new = p * old + torch.sigmoid(-f[t]) * x[t]
        on = (t < n)[:, None]
        h = torch.where(on, new, h)
        rows.append(torch.where(on, new, 0.0))
        before.append(old)
    if s["mode"] == "forward":
        return torch.stack(rows), h
    last, g, dx, df = h, s["dlast"].double(), [None] * T, [None] * T
    for t in range(T - 1, -1, -1):
        on = (t < n)[:, None]
        p, c = torch.sigmoid(f[t]), torch.sigmoid(-f[t])
        q = s["dh"][t].double() + g
        dx[t] = torch.where(on, c * q, 0.0)
        df[t] = torch.where(on, p * c * q * (before[t] - x[t]), 0.0)
        back = p * q if s["start"] is None else torch.where(s["start"][t][:, None], 0.0, p * q)
        g = torch.where(on, back, g)
    return torch.stack(rows), last, torch.stack(dx), torch.stack(df), g


def _exact_distill(s):
    """The loss from log-probabilities in 64 bits, its gradient by automatic differentiation."""
    n, tau, alpha = s["logits"].shape[0], s["temperature"], s["alpha"]
    rows, grads = [], []
    step = max(1, (1 << 25) // s["logits"].shape[1])
    for i in range(0, n, step):
        part = slice(i, i + step)
        with torch.enable_grad():
            z = s["logits"][part].double().requires_grad_(True)
            logp = torch.log_softmax(z / tau, 1)
            idx = s["indices"][part].long()
            lk = logp.gather(1, idx)
            t = s["values"][part].double() / tau
            if s["lse"] is not None:
                logq = t - s["lse"][part].double()[:, None]
                r = 1.0 - logq.exp().sum(1)
                out = logp.scatter(1, idx, -math.inf)
                ok = (r > 0) & (s["logits"].shape[1] > idx.shape[1])
                safe = torch.where(ok, r, torch.ones_like(r))
                tail = torch.where(ok, safe * (safe.log() - torch.logsumexp(out, 1)), 0.0) \
                    if s["logits"].shape[1] > idx.shape[1] else torch.zeros_like(r)
            else:
                logq, tail = torch.log_softmax(t, 1), 0.0
            row = alpha * tau ** 2 * ((logq.exp() * (logq - lk)).sum(1) + tail)
            if alpha < 1.0:
                y = s["targets"][part].long()[:, None]
                row = row - (1 - alpha) * torch.log_softmax(z, 1).gather(1, y)[:, 0]
            grads.append(torch.autograd.grad(row.sum(), z)[0] / n)
        rows.append(row.detach())
    rows = torch.cat(rows)
    return rows.sum() / n, rows, torch.cat(grads)
