"""Distillation in training (``CharRNN.train_step(distill=...)``, ``train.py --teacher``) and the
filtered sampler (``sample.py --temperature/--top_k/--top_p/--min_p``) on the framework's own
paths; and the operators together as a student uses them: a recurrent layer trained on a
teacher's record, then run step by step to sample."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from distributed_char_rnn_amd.engine.distill import Teacher
from distributed_char_rnn_amd.engine.optim import TFAdam
from distributed_char_rnn_amd.engine.sampler import sample
from distributed_char_rnn_amd.models.char_rnn import CharRNN
from distributed_char_rnn_amd.models.params import ModelConfig
from distributed_char_rnn_amd.models.reference import ReferenceBackend, forward
from distributed_char_rnn_amd.ops import recurrence as R
from distributed_char_rnn_amd.ops import vocab as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def models(model, H, V, dev, L=2, **kw):
    t = CharRNN(ModelConfig(model="lstm", vocab_size=V, rnn_size=64, num_layers=1), device=dev,
                seed=11)
    with torch.no_grad():
        t.store.flat.mul_(3.0)  # answers that are not uniform
    t.params_changed()
    s = CharRNN(ModelConfig(model=model, vocab_size=V, rnn_size=H, num_layers=L, **kw), device=dev,
                seed=1)
    return t, s


def batch(B, T, V, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32)
    y = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32)
    return x.to(dev), y.to(dev)


@pytest.mark.parametrize("dev", DEVS)
def test_record_is_time_major(dev):
    t, _ = models("lstm", 32, 65, dev)
    x, _ = batch(3, 7, 65, dev)
    (values, indices, lse), state = t.record_top(x, t.zero_state(3), 5, 2.0)
    assert values.shape == (7, 3, 5) and lse.shape == (7, 3)
    st = t.zero_state(3)
    for i in range(7):
        logits, st = t.step_logits(x[:, i:i + 1], st)
        v, ix, ls = O.top_logits(logits.float().contiguous(), 5, 2.0)
        # the step and the sequence kernels round their bf16 operands alike, their sums differ
        assert torch.allclose(values[i], v, atol=2e-2, rtol=2e-2)
        assert torch.allclose(lse[i], ls, atol=2e-2, rtol=2e-2)
    for a, b in zip(st, state):
        for p, q in zip(a, b):
            assert torch.allclose(p, q, atol=2e-2)


def _plain_loss(cfg, params, x, y, state, d):
    """The definition with torch's own softmax and automatic differentiation."""
    logits, _, _ = forward(cfg, params, x, state, training=False)
    B, T = x.shape
    z = logits.view(B, T, -1).transpose(0, 1)  # [T, B, V]
    lp = torch.log_softmax(z / d.temperature, 2)
    lq = d.values / d.temperature - d.lse[..., None]
    idx = d.indices.long()
    out = lp.scatter(2, idx, float("-inf"))
    rest = (1 - lq.exp().sum(2)).clamp_min(1e-30)
    kl = (lq.exp() * (lq - lp.gather(2, idx))).sum(2) + rest * (
        rest.log() - torch.logsumexp(out, 2))
    ce = torch.nn.functional.cross_entropy(logits, y.reshape(-1).long())
    return d.alpha * d.temperature ** 2 * kl.mean() + (1 - d.alpha) * ce


def test_reference_step_matches_the_definition():
    t, s = models("gru", 16, 29, "cpu")
    x, y = batch(4, 6, 29, "cpu")
    d = Teacher(t, top_k=7, alpha=0.6, temperature=2.0).record(x)
    loss, _, extras = s.train_step(x, y, s.zero_state(4), distill=d)
    params = {n: s.store.view(n).detach().clone().requires_grad_(True) for n in s.store.names()}
    want = _plain_loss(s.cfg, params, x, y, s.zero_state(4), d)
    want.backward()
    assert abs(loss.item() - want.item()) < 1e-5 * max(1.0, want.item())
    assert abs(extras["loss"].mean().item() - loss.item()) < 1e-5
    for n in s.store.names():
        assert torch.allclose(s.store.gview(n), params[n].grad, atol=1e-6, rtol=1e-4), n


@pytest.mark.gpu
@pytest.mark.parametrize("model,H,V,B,T,kw", [
    ("lstm", 128, 65, 32, 16, {}), ("lstm", 96, 65, 5, 9, {}), ("gru", 128, 65, 16, 12, {}),
    ("rnn", 64, 65, 8, 6, {}), ("nas", 64, 65, 8, 6, {}), ("lstm", 72, 65, 8, 9, {}),
    ("lstm", 128, 2048, 32, 16, {}), ("lstm", 128, 300, 8, 10, {}),
    ("lstm", 128, 65, 32, 16, dict(clip_norm="dense"))])
def test_native_step_matches_oracle(model, H, V, B, T, kw):
    """Loss, every gradient and the following Adam steps against the fp32 oracle with the same
    record; tolerances as for the cross-entropy step (bf16 operands)."""
    t, s = models(model, H, V, "cuda", **kw)
    x, y = batch(B, T, V, "cuda")
    teacher = Teacher(t, top_k=16, alpha=0.7, temperature=2.0)
    d = teacher.record(x)
    ref = ReferenceBackend(s.store)
    want, _, _ = ref.train_step(x, y, s.zero_state(B), distill=d)
    g_ref = s.store.grad[: s.store.numel].clone()
    slot = s.store.norm_slot_view().clone()
    opt = TFAdam(s.store, guard=s.error_word())
    s.bind_optimizer(opt)
    loss, state, extras = s.train_step(x, y, s.zero_state(B), want_extras=True, distill=d)
    torch.cuda.synchronize()
    assert abs(loss.item() - want.item()) < 2e-2 * max(1.0, abs(want.item()))
    g = s.store.grad[: s.store.numel]
    for n in s.store.names():
        sp = s.store.by_name[n]
        a, b = g[sp.offset:sp.offset + sp.numel], g_ref[sp.offset:sp.offset + sp.numel]
        assert ((a - b).norm() / (b.norm() + 1e-12)).item() < 5e-2, n
    assert torch.allclose(s.store.norm_slot_view(), slot, rtol=5e-2)
    assert torch.allclose(extras["loss"].mean(), loss.view(()), rtol=1e-4)
    opt.step(1e-3)
    # a cross-entropy step after it, and another distillation step, on the same model
    s.train_step(x, y, state)
    opt.step(1e-3)
    again, _, _ = s.train_step(x, y, s.zero_state(B), distill=teacher.record(x))
    s.check_errors()
    assert torch.isfinite(again).all() and torch.isfinite(s.store.flat).all()


@pytest.mark.gpu
def test_cross_entropy_step_is_unchanged_by_a_distillation_step():
    _, s = models("lstm", 128, 65, "cuda")
    t, _ = models("lstm", 32, 65, "cuda")
    x, y = batch(16, 12, 65, "cuda")
    a, _, _ = s.train_step(x, y, s.zero_state(16))
    a, ga = a.clone(), s.store.grad.clone()
    s.train_step(x, y, s.zero_state(16), distill=Teacher(t).record(x))
    b, _, _ = s.train_step(x, y, s.zero_state(16))
    assert torch.equal(a, b) and torch.equal(ga, s.store.grad)


def test_teacher_refuses():
    t, _ = models("lstm", 32, 65, "cpu")
    for kw in (dict(top_k=0), dict(top_k=257), dict(alpha=-0.1), dict(alpha=1.1),
               dict(temperature=0.0), dict(temperature=float("inf"))):
        with pytest.raises(ValueError):
            Teacher(t, **kw)


@pytest.mark.parametrize("dev", DEVS)
def test_train_step_refuses_records_of_another_shape(dev):
    """Batch-major records, of another batch, or with parts of another: as many rows or not."""
    t, s = models("lstm", 32, 29, dev)
    x, y = batch(4, 6, 29, dev)
    d = Teacher(t, top_k=5).record(x)
    assert d.values.shape == (6, 4, 5)
    swap = {n: getattr(d, n).transpose(0, 1).contiguous() for n in ("values", "indices", "lse")}
    for bad in (d._replace(**swap), d._replace(values=swap["values"]),
                d._replace(indices=swap["indices"]), d._replace(lse=swap["lse"]),
                d._replace(values=d.values.view(24, 5), indices=d.indices.view(24, 5)),
                d._replace(indices=d.indices[..., :3]), d._replace(lse=d.lse.view(-1)),
                Teacher(t, top_k=5).record(x[:2])):
        with pytest.raises(ValueError, match="record"):
            s.train_step(x, y, s.zero_state(4), distill=bad)
    s.train_step(x, y, s.zero_state(4), distill=d._replace(lse=None))
    s.check_errors()


@pytest.mark.parametrize("dev", DEVS)
def test_resume_gives_the_teacher_its_state_back(tmp_path, dev, monkeypatch):
    """A run resumed in the middle of an epoch sees the records of the uninterrupted run."""
    from distributed_char_rnn_amd.engine import trainer
    from distributed_char_rnn_amd.utils.config import train_parser

    monkeypatch.chdir(tmp_path)
    common = ["--synthetic_text", "2000", "--batch_size", "4", "--seq_length", "20", "--num_epochs",
              "1", "--log_dir", "logs", "--summary_every", "0", "--device", dev, "--rnn_size", "32"]
    seen = []
    record = Teacher.record

    def spy(self, x):
        d = record(self, x)
        seen.append(d.values.float().cpu())
        return d

    def run(*args):
        seen.clear()
        assert trainer.train(train_parser().parse_args(common + list(args))) == 0
        return list(seen)

    run("--save_dir", "t", "--max_steps", "3")
    monkeypatch.setattr(Teacher, "record", spy)
    whole = run("--save_dir", "a", "--teacher", "t", "--max_steps", "6")
    run("--save_dir", "b", "--teacher", "t", "--max_steps", "3", "--save_state")
    rest = run("--save_dir", "c", "--teacher", "t", "--init_from", "b", "--resume_exact",
               "--max_steps", "3")
    assert len(whole) == 6 and len(rest) == 6  # three to catch up, three of its own
    for a, b in zip(whole, rest):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", ["auto", "fp32"])
def test_teacher_computes_in_the_students_type(tmp_path, dev, dtype, monkeypatch):
    """``--dtype`` holds for the teacher, too; in fp32 on a GPU its record is the oracle's."""
    from distributed_char_rnn_amd.engine import trainer
    from distributed_char_rnn_amd.utils.config import train_parser

    monkeypatch.chdir(tmp_path)
    common = ["--synthetic_text", "2000", "--batch_size", "4", "--seq_length", "20", "--num_epochs",
              "1", "--log_dir", "logs", "--summary_every", "0", "--device", dev, "--rnn_size", "64",
              "--max_steps", "3"]
    teachers, load = [], Teacher.load.__func__
    asked = []

    def spy(cls, save_dir, chars, device, dtype="auto", **kw):
        t = load(cls, save_dir, chars, device, dtype, **kw)
        asked.append(dtype)
        teachers.append(t)
        return t

    monkeypatch.setattr(Teacher, "load", classmethod(spy))
    assert trainer.train(train_parser().parse_args(common + ["--save_dir", "t"])) == 0
    assert trainer.train(train_parser().parse_args(
        common + ["--save_dir", "s", "--teacher", "t", "--dtype", dtype])) == 0
    (t,) = teachers
    assert asked == [dtype]
    want = {"cpu": {"auto": "reference", "fp32": "reference"},
            "cuda": {"auto": "native", "fp32": "native32"}}[dev][dtype]
    assert t.model.backend_name == want
    if dtype == "fp32":
        x, _ = batch(4, 20, t.model.cfg.vocab_size, dev)
        logits, _ = t.model.backend.sequence_logits(x, t.model.zero_state(4))
        oracle, _ = ReferenceBackend(t.model.store).sequence_logits(x, t.model.zero_state(4))
        assert torch.allclose(logits, oracle, rtol=1e-4, atol=1e-5)


# ---- sampling ---------------------------------------------------------------------------------
CHARS = [" "] + [chr(97 + i) for i in range(25)]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("model,H", [("lstm", 64), ("gru", 40), ("nas", 32)])
def test_sampler_filters(model, H, dev):
    m = CharRNN(ModelConfig(model=model, vocab_size=26, rnn_size=H, num_layers=1), device=dev,
                seed=2)
    with torch.no_grad():
        m.store.flat.mul_(4.0)
    m.params_changed()
    vocab = {c: i for i, c in enumerate(CHARS)}
    kw = dict(num=30, prime="ab c", num_samples=3, seed=5)
    plain = sample(m, CHARS, vocab, sampling_type=0, **kw)
    # always the likeliest: temperature 0, the top 1, nothing but the first of the order
    for f in (dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(temperature=1e-4)):
        assert sample(m, CHARS, vocab, sampling_type=1, **kw, **f) == plain, f
    assert sample(m, CHARS, vocab, sampling_type=0, **kw, top_k=5) == plain
    a = sample(m, CHARS, vocab, sampling_type=1, **kw, temperature=0.9, top_k=6, min_p=0.01)
    assert a == sample(m, CHARS, vocab, sampling_type=1, **kw, temperature=0.9, top_k=6, min_p=0.01)
    assert all(s.startswith("ab c") and len(s) == 34 for s in a) and len(set(a)) > 1
    b = sample(m, CHARS, vocab, sampling_type=2, **kw, temperature=0.9, top_k=6)
    assert all(len(s) == 34 for s in b)
    for f in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=1.5), dict(min_p=2.0)):
        with pytest.raises(ValueError):
            sample(m, CHARS, vocab, **kw, **f)


@pytest.mark.gpu
def test_sampler_graph_equals_eager_and_follows_the_rule():
    V, S, num = 65, 4, 25
    m = CharRNN(ModelConfig(model="lstm", vocab_size=V, rnn_size=128, num_layers=2), device="cuda",
                seed=2)
    with torch.no_grad():
        m.store.flat.mul_(4.0)
    m.params_changed()
    u = torch.rand(num, S, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for mode in (1, 2):
        args = ([3, 7, 1], num, mode, u, 0, 0.8, 20, 0.9, 0.01)
        ids = m.backend.sample_filtered(*args)
        assert ids == m.backend.sample_filtered(*args, use_graph=False)
        # teacher forcing: each pick follows from the logits after the picks before it
        st = m.zero_state(S)
        for c in (3, 7):
            _, st = m.step_logits(torch.full((S, 1), c, dtype=torch.int32, device="cuda"), st)
        cur = torch.full((S,), 1, dtype=torch.int32, device="cuda")
        for i in range(num):
            logits, st = m.step_logits(cur[:, None], st)
            temp = 0.8 if mode == 1 else (cur == 0).float() * 0.8
            cur = O.sample_logits(logits, u[i], temp, 20, 0.9, 0.01)
            assert cur.tolist() == [row[i] for row in ids], i


@pytest.mark.parametrize("dev", DEVS)
def test_cli_teacher_then_sample(tmp_path, dev):
    """train.py, train.py --teacher on its result, sample.py with filters."""
    w, env = str(tmp_path), dict(os.environ, PYTHONPATH=ROOT)

    def run(script, *args, ok=True):
        r = subprocess.run([sys.executable, os.path.join(ROOT, script), "--device", dev, *args],
                           cwd=w, env=env, capture_output=True, text=True, timeout=110)
        assert (r.returncode == 0) == ok, r.stdout[-2000:] + r.stderr[-2000:]
        return r.stdout + r.stderr

    common = ["--synthetic_text", "4000", "--batch_size", "4", "--seq_length", "20",
              "--num_epochs", "1", "--max_steps", "3", "--log_dir", "logs", "--summary_every", "2"]
    run("train.py", "--save_dir", "teacher", "--rnn_size", "32", *common)
    out = run("train.py", "--save_dir", "student", "--rnn_size", "32", "--model", "gru", "--teacher",
              "teacher", "--teacher_top_k", "20", "--distill_alpha", "0.8", *common)
    assert "distilling from teacher: top 20 logits" in out
    assert "distill_alpha" in run("train.py", "--save_dir", "x", "--teacher", "teacher",
                                  "--distill_alpha", "2", *common, ok=False)
    out = run("sample.py", "--save_dir", "student", "-n", "12", "--prime", "a", "--seed", "1",
              "--temperature", "0.7", "--top_k", "8", "--top_p", "0.9")
    assert out.strip()


# ---- the operators together -------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_student(dtype, dev):
    """A student whose layer is the linear recurrence (padded batch, documents), trained against a
    teacher's record through autograd; its gradients against float64 autograd of the definition;
    then the same layer, one token at a time, gives the sequence's logits and samples."""
    T, B, E, H, V, k = 12, 3, 8, 16, 37, 6
    g = torch.Generator().manual_seed(0)
    w = {n: (torch.randn(*s, generator=g) * 0.4).to(dtype).to(dev) for n, s in
         dict(emb=(V, E), win=(E, 2 * H), wout=(H, V)).items()}
    ids = torch.randint(0, V, (T, B), generator=g).to(dev)
    lengths = torch.tensor([T, 5, 0], dtype=torch.int32, device=dev)
    starts = (torch.rand(T, B, generator=g) < 0.2).to(dev)
    teacher = (torch.randn(T * B, V, generator=g) * 2).to(dev)
    values, indices, lse = O.top_logits(teacher, k, 2.0)
    y = torch.randint(0, V, (T, B), generator=g).int().to(dev)
    y[torch.arange(T, device=dev)[:, None] >= lengths[None]] = -1  # padding
    leaves = {n: v.clone().requires_grad_(True) for n, v in w.items()}

    def run(p, rec, dt):
        z = p["emb"][ids] @ p["win"]
        h, last = rec(z[..., :H], z[..., H:])
        return (h @ p["wout"]).reshape(T * B, V), last

    logits, last = run(leaves, lambda a, f: R.linear_recurrence(a, f, lengths=lengths,
                                                                starts=starts), dtype)
    loss = O.distill_loss(logits, values, indices, top_lse=lse, targets=y.reshape(-1), alpha=0.5,
                          temperature=2.0)
    loss.backward()
    # the definition, in float64 on the CPU
    ref = {n: v.detach().double().cpu().requires_grad_(True) for n, v in w.items()}
    ids, lc, sc = ids.cpu(), lengths.cpu(), starts.cpu()

    def steps(a, f):
        h, out = torch.zeros(B, H, dtype=torch.float64), []
        for t in range(T):
            s = torch.sigmoid(f[t])
            new = torch.where(sc[t][:, None], 0.0, s * h) + (1 - s) * a[t]
            live = (t < lc)[:, None]
            out.append(torch.where(live, new, 0.0))
            h = torch.where(live, new, h)
        return torch.stack(out), h

    rl, rlast = run(ref, steps, torch.float64)
    on = (y.reshape(-1) >= 0).cpu()
    idx = indices.long().cpu()
    lp = torch.log_softmax(rl / 2.0, 1)
    lq = values.double().cpu() / 2.0 - lse.double().cpu()[:, None]
    rest = 1 - lq.exp().sum(1)
    kl = (lq.exp() * (lq - lp.gather(1, idx))).sum(1) + rest * (
        rest.log() - torch.logsumexp(lp.scatter(1, idx, -np.inf), 1))
    ce = -torch.log_softmax(rl, 1).gather(1, y.reshape(-1).long().clamp_min(0).cpu()[:, None])[:, 0]
    want = (torch.where(on, 0.5 * 4.0 * kl + 0.5 * ce, 0.0)).sum() / (T * B)
    want.backward()
    # bf16: each of four products and two operators rounds its result by 2^-9, relative to what it
    # sums; fp32: 2^-24 through the same chain
    tol = 4e-2 if dtype == torch.bfloat16 else 2e-5
    assert abs(loss.item() - want.item()) <= tol * max(1.0, want.item())
    assert torch.allclose(last.double().cpu(), rlast.detach(), atol=tol, rtol=tol)
    for n in w:
        a, b = leaves[n].grad.double().cpu(), ref[n].grad
        assert ((a - b).norm() / b.norm()).item() <= tol, n
    # serving: one token at a time
    h = torch.zeros(B, H, device=dev)
    u = torch.rand(T, B, generator=g).to(dev)
    with torch.no_grad():
        full, _ = run(w, lambda a, f: R.linear_recurrence_fwd(a, f, starts=starts)[:2], dtype)
        ids = ids.to(dev)
        for t in range(T):
            z = w["emb"][ids[t]] @ w["win"]
            o = R.linear_recurrence_step(z[:, :H], z[:, H:], h, starts=starts[t]) @ w["wout"]
            assert torch.allclose(o.float(), full.view(T, B, V)[t].float(), atol=tol, rtol=tol)
            pick = O.sample_logits(o.float(), u[t], 0.8, 10, 0.9)
            assert ((pick >= 0) & (pick < V)).all()


# ---- modes of training with a teacher ---------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("model,H", [("lstm", 64), ("gru", 48), ("rnn", 32)])
def test_fp32_step_matches_oracle(model, H):
    """``--dtype fp32``: teacher and student on the fp32 kernels, loss and gradients at fp32 accuracy
    (as the cross-entropy step's, tests/test_fp32.py)."""
    V, B, T = 65, 6, 11
    t = CharRNN(ModelConfig(model="lstm", vocab_size=V, rnn_size=64, num_layers=1), device="cuda",
                seed=11, dtype="fp32")
    with torch.no_grad():
        t.store.flat.mul_(3.0)
    t.params_changed()
    s = CharRNN(ModelConfig(model=model, vocab_size=V, rnn_size=H, num_layers=2), device="cuda",
                seed=1, dtype="fp32")
    assert t.backend_name == s.backend_name == "native32"
    x, y = batch(B, T, V, "cuda")
    d = Teacher(t, top_k=12, alpha=0.7, temperature=2.0).record(x)
    want, want_state, _ = ReferenceBackend(s.store).train_step(x, y, s.zero_state(B), distill=d)
    g_ref = s.store.grad[: s.store.numel].clone()
    loss, state, _ = s.train_step(x, y, s.zero_state(B), distill=d)
    assert abs(loss.item() - want.item()) < 1e-4 * max(1.0, abs(want.item()))
    for n in s.store.names():
        sp = s.store.by_name[n]
        a, b = (v[sp.offset:sp.offset + sp.numel] for v in (s.store.grad, g_ref))
        assert ((a - b).norm() / (b.norm() + 1e-12)).item() < 1e-4, n
    for p, q in zip(state, want_state):
        for a, b in zip(p, q):
            assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dev", DEVS)
def test_teacher_carries_its_state_over_batches(dev):
    """Two batches in a row against one token at a time from the same start, and the start of an
    epoch back at zero."""
    V, B, T, k = 65, 5, 9, 6
    t, _ = models("lstm", 32, V, dev)
    x, _ = batch(B, 2 * T, V, dev, seed=3)
    teacher = Teacher(t, top_k=k, alpha=1.0, temperature=2.0)
    two = [teacher.record(x[:, :T]), teacher.record(x[:, T:])]
    st = t.zero_state(B)
    for i in range(2 * T):
        logits, st = t.step_logits(x[:, i:i + 1], st)
        values, _, lse = O.top_logits(logits.float().contiguous(), k, 2.0)
        d = two[i // T]
        # (as in test_record_is_time_major)
        assert torch.allclose(d.values[i % T], values, atol=2e-2, rtol=2e-2), i
        assert torch.allclose(d.lse[i % T], lse, atol=2e-2, rtol=2e-2), i
    fresh = Teacher(t, top_k=k, alpha=1.0, temperature=2.0).record(x[:, T:])
    assert not torch.allclose(fresh.values, two[1].values, atol=2e-2, rtol=2e-2)  # a state mattered
    teacher.reset(B)
    again = teacher.record(x[:, :T])
    assert torch.equal(again.values, two[0].values) and torch.equal(again.lse, two[0].lse)


def _rank(rank, world, port, sharded, out_q):
    import torch.distributed as dist

    from distributed_char_rnn_amd.parallel.grad_sync import GradSync
    from distributed_char_rnn_amd.parallel.zero import ShardedStep

    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        t, s = models("lstm", 16, 29, "cpu")
        opt = TFAdam(s.store, clip=0.5)
        sync = (ShardedStep(s.store, opt, world, rank) if sharded
                else GradSync(s.store, world, 8.0, "fp32"))
        losses = _steps(t, s, opt, lambda v: v[rank * 3:(rank + 1) * 3], sync, sharded)
        out_q.put((rank, s.store.flat.clone().numpy(), losses))
    finally:
        dist.destroy_process_group()


def _steps(t, s, opt, rows, sync=None, sharded=False):
    x, y = batch(6, 24, 29, "cpu", seed=4)
    x, y = rows(x), rows(y)
    teacher = Teacher(t, top_k=7, alpha=0.6, temperature=2.0)
    state, losses = s.zero_state(x.shape[0]), []
    for i in range(3):
        part = slice(8 * i, 8 * i + 8)
        told = teacher.record(x[:, part])
        if sync is not None:
            sync.reset()
        loss, state, _ = s.train_step(x[:, part], y[:, part], state, sync, distill=told)
        if sharded:
            sync.step(0.01)
        else:
            opt.step(0.01, grad_scale=1.0 if sync is None else sync.finish(defer_scale=True))
        losses.append(loss.item())
    return losses


@pytest.mark.parametrize("sharded", [False, True])
def test_two_ranks_with_a_teacher_equal_one_of_twice_the_batch(sharded):
    """Each rank's teacher reads its own rows and carries their states; replicated and sharded steps
    end at the parameters of one process with both ranks' rows."""
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as c:
        c.bind(("127.0.0.1", 0))
        port = c.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, sharded, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict((r, (flat, losses)) for r, flat, losses in (q.get(timeout=110) for _ in procs))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    t, s = models("lstm", 16, 29, "cpu")
    opt = TFAdam(s.store, clip=0.5)
    losses = _steps(t, s, opt, lambda v: v)
    np.testing.assert_array_equal(got[0][0], got[1][0])
    # (as test_distributed.py's cross-entropy steps)
    np.testing.assert_allclose(got[0][0], s.store.flat.numpy(), rtol=2e-4, atol=2e-6)
    np.testing.assert_allclose(np.mean([got[0][1], got[1][1]], 0), losses, rtol=1e-5)
