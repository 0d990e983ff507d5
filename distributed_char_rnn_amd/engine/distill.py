"""Distillation from a trained model (``train.py --teacher``): the teacher reads every batch beside
the student, carries its own TBPTT state, and hands the student's step its k largest logits per
position (ops/vocab.py).  Only those leave the teacher's forward: at k = 64 of 8192 tokens 0.5 KB
a position instead of 32 KB.
"""
from __future__ import annotations

from typing import Sequence

import torch

from ..models.char_rnn import CharRNN
from ..ops.vocab import MAX_K, Distill
from .sample_cli import load_for_inference


class Teacher:
    def __init__(self, model: CharRNN, top_k: int = 64, alpha: float = 0.5,
                 temperature: float = 2.0):
        if not 1 <= top_k <= MAX_K:
            raise ValueError(f"teacher_top_k must be 1 to {MAX_K}, got {top_k}")
        if not 0.0 <= alpha <= 1.0:
            raise ValueError(f"distill_alpha must be in [0, 1], got {alpha}")
        if not 0.0 < temperature < float("inf"):
            raise ValueError(f"distill_temperature must be positive and finite, got {temperature}")
        self.model = model
        self.k = min(top_k, model.cfg.vocab_size)
        self.alpha, self.temperature = float(alpha), float(temperature)
        self.state = None

    @classmethod
    def load(cls, save_dir: str, chars: Sequence[str], device, dtype: str = "auto",
             **kw) -> "Teacher":
        """The latest checkpoint of ``save_dir``, whose vocabulary must be the student's; it computes
        in ``dtype``, the student's."""
        model, saved, _, _ = load_for_inference(save_dir, device, dtype)
        if tuple(saved) != tuple(chars):
            raise ValueError(f"the teacher in {save_dir} was trained on another character set")
        return cls(model, **kw)

    def reset(self, batch: int) -> None:
        """The start of an epoch: the state the student starts from, too."""
        self.state = self.model.zero_state(batch)

    @torch.no_grad()
    def record(self, x) -> Distill:
        if self.state is None:
            self.reset(x.shape[0])
        (values, indices, lse), self.state = self.model.record_top(x, self.state, self.k,
                                                                   self.temperature)
        return Distill(values, indices, lse, self.alpha, self.temperature)
