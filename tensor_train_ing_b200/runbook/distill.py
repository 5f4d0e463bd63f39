"""Distil a conventional teacher into a tensor-network student, end to end on synthetic text.

    python -m tensor_train_ing_b200.runbook.distill --out runs/distill.json [--steps 60] [--top 16] [--device cuda]

A small control (softmax attention, SwiGLU, layer norms) is trained on sequences of a random order-1 Markov
source, then frozen.  For every student batch its logits go through ``top_logits`` (the k largest, their columns and the row's
log-sum-exp: all that a stored teacher keeps), and a polynomial-attention bilinear student is trained through
``TrainEngine.step(..., teacher=...)`` on the distillation loss alone.  The report gives both models' held-out
cross-entropy, the student's before and after, and the source's entropy rate, the best any model can do.
"""
from __future__ import annotations

import argparse
import json
import math
import sys
from pathlib import Path

import torch


class MarkovSource:
    """Sequences of a random order-1 Markov chain over ``vocab`` tokens (seeded, on the CPU)."""

    def __init__(self, vocab: int, seed: int, sharpness: float = 2.0):
        self.gen = torch.Generator().manual_seed(seed)
        self.table = torch.softmax(sharpness * torch.randn(vocab, vocab, generator=self.gen), 1)

    def batch(self, rows: int, length: int):
        """(inputs, document ids, targets), each (rows, length)."""
        tokens = torch.randint(0, self.table.shape[0], (rows, 1), generator=self.gen)
        for _ in range(length):
            nxt = torch.multinomial(self.table[tokens[:, -1]], 1, generator=self.gen)
            tokens = torch.cat([tokens, nxt], 1)
        return tokens[:, :-1].contiguous(), torch.zeros(rows, length, dtype=torch.long), tokens[:, 1:].contiguous()

    def entropy_rate(self) -> float:
        p = torch.full((self.table.shape[0],), 1.0 / self.table.shape[0], dtype=torch.float64)
        t = self.table.double()
        for _ in range(200):
            p = p @ t
        return float(-(p[:, None] * t * t.log()).sum())


def _config(vocab: int, teacher: bool, lr: float):
    from ..config import Config
    model = dict(vocab_size=vocab, padded_vocab=-(-vocab // 64) * 64, layers=2, d_model=128, heads=2, d_key=64,
                 d_value=64, d_mlp=256, loss_chunk_tokens=1024)
    if teacher:
        model.update(attention="softmax", mlp="swiglu", normalization="pre_ln", final_normalization="layer",
                     attention_backend="reference")
    return Config.from_dict({"model": model, "train": {"optimizer": "adamw", "lr": lr, "compile": False}})


@torch.no_grad()
def _cross_entropy(model, batch, device) -> float:
    model.eval()
    idx, doc, targets = (t.to(device) for t in batch)
    _, loss = model(idx, doc, targets)
    model.train()
    return float(loss)


def run_distill(*, steps: int = 60, teacher_steps: int = 120, rows: int = 16, length: int = 64, vocab: int = 200,
                top: int = 16, temperature: float = 2.0, lr: float = 3e-3, seed: int = 0, device: str = "cuda") -> dict:
    from ..engine import TrainEngine
    from ..ops import distill
    if steps < 1 or teacher_steps < 1:
        raise ValueError("the example trains both models for at least one step")
    source = MarkovSource(vocab, seed)
    held_out = source.batch(4 * rows, length)
    torch.manual_seed(seed)
    teacher = TrainEngine(_config(vocab, True, lr), device=device, micro_batch=rows)
    student = TrainEngine(_config(vocab, False, lr), device=device, micro_batch=rows)
    for _ in range(teacher_steps):
        teacher.step(*source.batch(rows, length))
    teacher.model.eval()
    before = _cross_entropy(student.model, held_out, device)
    top_logits = distill.top_logits if torch.device(device).type == "cuda" else distill.top_logits_reference
    losses = []
    for _ in range(steps):
        idx, doc, targets = source.batch(rows, length)
        with torch.no_grad():
            listed = top_logits(teacher.model(idx.to(device), doc.to(device)).float(), top, temperature=temperature)
        lists = distill.Teacher(listed.ids, listed.values, listed.lse, temperature=temperature)
        loss, count = student.step(idx, doc, targets, teacher=lists)
        losses.append(loss / count)
    report = {"device": device, "steps": steps, "teacher_steps": teacher_steps, "top": top, "temperature": temperature,
              "teacher_ce": _cross_entropy(teacher.model, held_out, device), "student_ce_before": before,
              "student_ce_after": _cross_entropy(student.model, held_out, device),
              "source_entropy": source.entropy_rate(), "uniform_ce": math.log(vocab),
              "distillation_losses": [float(x) for x in losses]}
    if torch.device(device).type == "cuda":
        from ..ops._ext import check_status
        check_status()
    return report


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--out")
    for name, kind, default in (("steps", int, 60), ("teacher-steps", int, 120), ("rows", int, 16), ("length", int, 64),
                                ("vocab", int, 200), ("top", int, 16), ("temperature", float, 2.0), ("seed", int, 0)):
        ap.add_argument(f"--{name}", type=kind, default=default)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    args = vars(ap.parse_args(argv))
    out = args.pop("out")
    report = run_distill(**args)
    text = json.dumps(report, indent=2) + "\n"
    if out:
        Path(out).write_text(text)
    print(text, end="")
    return 0


if __name__ == "__main__":
    sys.exit(main())
