"""Text sampling from a trained model (reference: ``Model.sample``, model.py:105-140;
sample.py:27-46).

Semantics kept: zero state; feed ``prime[:-1]`` to warm the state; then ``num`` steps from
``prime[-1]``; ``sampling_type`` 0 = argmax, 1 = weighted pick (inverse CDF via cumsum +
searchsorted of ``rand * sum``), 2 = weighted pick only when the *previous* char is a space,
else argmax.  Beyond the reference, weighted picks can be drawn under a temperature, top-k,
top-p and min-p (ops/vocab.py ``sample_logits``).  Sampling is batched (``num_samples``
independent streams) and, on the GPU, the whole autoregressive loop runs device-side (one fused
kernel per generated char, no host sync until the end) via the native backend's
``sample_sequence``.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import numpy as np
import torch

from ..models.char_rnn import CharRNN
from ..ops.vocab import sample_logits


def weighted_pick(weights: np.ndarray, rng: np.random.Generator) -> int:
    t = np.cumsum(weights)
    s = np.sum(weights)
    return int(np.searchsorted(t, rng.random() * s))


def sample(model: CharRNN, chars: Sequence[str], vocab: Dict[str, int], num: int = 200,
           prime: str = "The ", sampling_type: int = 1, seed: Optional[int] = None,
           num_samples: int = 1, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
           min_p: float = 0.0) -> List[str]:
    if not prime:
        prime = chars[0]
    for ch in prime:
        if ch not in vocab:
            raise KeyError(f"prime character {ch!r} not in vocabulary")
    if (temperature, top_k, top_p, min_p) != (1.0, 0, 1.0, 0.0):
        ids = _sample_filtered(model, [vocab[c] for c in prime], num, sampling_type, seed,
                               num_samples, vocab.get(" ", -1), temperature, top_k, top_p, min_p)
        return [prime + "".join(chars[int(i)] for i in row) for row in ids]
    native = getattr(model.backend, "sample_sequence", None)
    if native is not None and model.device.type == "cuda":
        ids = native([vocab[c] for c in prime], num, sampling_type,
                     seed if seed is not None else int(np.random.SeedSequence().entropy % (1 << 62)),
                     num_samples, vocab.get(" ", -1))
        return [prime + "".join(chars[int(i)] for i in row) for row in ids]

    rng = np.random.default_rng(seed)
    S = num_samples
    state = model.zero_state(S)
    with torch.no_grad():
        for ch in prime[:-1]:
            x = np.full((S, 1), vocab[ch], dtype=np.int32)
            _, state = model.step_logits(x, state)
        outs = [prime for _ in range(S)]
        cur = [prime[-1]] * S
        for _ in range(num):
            x = np.array([[vocab[c]] for c in cur], dtype=np.int32)
            logits, state = model.step_logits(x, state)
            probs = torch.softmax(logits.float(), dim=-1).cpu().numpy()
            nxt = []
            for s in range(S):
                p = probs[s]
                if sampling_type == 0:
                    k = int(np.argmax(p))
                elif sampling_type == 2:
                    k = weighted_pick(p, rng) if cur[s] == " " else int(np.argmax(p))
                else:
                    k = weighted_pick(p, rng)
                k = min(k, len(chars) - 1)
                nxt.append(chars[k])
            cur = nxt
            outs = [o + c for o, c in zip(outs, cur)]
    return outs


def _sample_filtered(model: CharRNN, prime: Sequence[int], num: int, sampling_type: int,
                     seed: Optional[int], num_samples: int, space_id: int, temperature: float,
                     top_k: int, top_p: float, min_p: float) -> List[List[int]]:
    """Ids [S][num].  The uniform numbers come from the seed alone, so every device and backend
    draws with the same ones."""
    for name, v, ok in (("temperature", temperature, 0.0 <= temperature < float("inf")),
                        ("top_k", top_k, top_k >= 0), ("top_p", top_p, 0.0 <= top_p <= 1.0),
                        ("min_p", min_p, 0.0 <= min_p <= 1.0)):
        if not ok:
            raise ValueError(f"{name} is out of range: {v}")
    S = num_samples
    rng = np.random.default_rng(seed)
    u = torch.from_numpy(rng.random((num, S), dtype=np.float32)).to(model.device)
    native = getattr(model.backend, "sample_filtered", None)
    if native is not None and model.device.type == "cuda":
        return native(prime, num, sampling_type, u, space_id, temperature, top_k, top_p, min_p)
    state = model.zero_state(S)
    cur = torch.empty(S, dtype=torch.int32, device=model.device)
    out = torch.empty(S, num, dtype=torch.int32, device=model.device)
    with torch.no_grad():
        for cid in prime[:-1]:
            _, state = model.step_logits(cur.fill_(cid)[:, None], state)
        cur.fill_(prime[-1])
        for i in range(num):
            logits, state = model.step_logits(cur[:, None], state)
            t = 0.0 if sampling_type == 0 else temperature
            if sampling_type == 2:
                t = (cur == space_id).float() * temperature
            cur = sample_logits(logits, u[i], t, top_k, top_p, min_p)
            out[:, i] = cur
    return out.tolist()
