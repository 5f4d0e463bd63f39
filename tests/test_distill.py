"""Distillation and layer norm off the GPU: the plain forms against independent formulas in 64 bits, the model,
engine and example paths that use them, and their refusals.

Tolerances: everything is fp64 unless it says otherwise, so 1e-10 bounds thousands of roundings of 1e-16; fp32
trajectories that must agree only up to summation order are held to 1e-5."""
import math

import pytest
import torch

from tensor_train_ing_b200.config import Config, ModelConfig
from tensor_train_ing_b200.engine import TrainEngine
from tensor_train_ing_b200.models.model import TensorLM
from tensor_train_ing_b200.models.normalization import LayerNorm
from tensor_train_ing_b200.models.shapes import count_params
from tensor_train_ing_b200.ops import distill


def _cfg(**kw):
    base = dict(layers=1, d_model=16, heads=2, d_key=8, d_value=8, d_mlp=24, vocab_size=30, padded_vocab=32,
                norm_groups=4, attention_backend="reference")
    return ModelConfig(**{**base, **kw})


# ------------------------------------------------------------------------------------ layer norm
@pytest.mark.parametrize("shape", [(5, 16), (2, 3, 16), (1, 1), (0, 16)])
def test_layer_norm_module_is_the_formula(shape):
    torch.manual_seed(0)
    norm = LayerNorm(shape[-1], 1e-5).double()
    with torch.no_grad():
        norm.weight.add_(torch.randn_like(norm.weight))
        norm.bias.add_(torch.randn_like(norm.bias))
    x = (torch.randn(shape, dtype=torch.float64) * 3 + 7).requires_grad_(True)
    want = torch.nn.functional.layer_norm(x, shape[-1:], norm.weight, norm.bias, 1e-5)
    torch.testing.assert_close(norm(x), want, rtol=1e-10, atol=1e-10)
    if x.numel():
        assert torch.autograd.gradcheck(norm, (x,))


def test_layer_norm_package_in_the_model():
    cfg = _cfg(normalization="pre_ln", final_normalization="layer")
    torch.manual_seed(1)
    model = TensorLM(cfg)
    names = set(model.state_dict())
    assert {"blocks.0.attn_in.bias", "blocks.0.mlp_in.weight", "final_norm.bias"} <= names
    assert count_params(cfg)["total"] == sum(p.numel() for p in model.parameters())
    assert model.operator_audit()["class"] == "N"
    idx = torch.randint(0, 30, (2, 6))
    _, loss = model(idx, targets=idx)
    loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    from tensor_train_ing_b200.models.init_stream import named_initial_tensors
    torch.manual_seed(1)
    streamed = dict(named_initial_tensors(cfg))
    torch.manual_seed(1)
    for name, t in TensorLM(cfg).state_dict().items():
        assert torch.equal(streamed[name], t)


def test_layer_norm_has_no_gain_to_fold():
    from tensor_train_ing_b200.analysis import gain
    with pytest.raises(ValueError, match="layer norm"):
        gain(LayerNorm(8, 1e-6), 8, "cpu")


# ------------------------------------------------------------------------------------ plain forms
def _brute(z, ids, t, lse, target, tau, kd, ce):
    """One row of the loss, entry by entry."""
    q = torch.softmax(z / tau, 0)
    listed = [int(i) for i in ids if i >= 0]
    a = [float(x) / tau for i, x in zip(ids, t) if i >= 0]
    if not listed:
        kl = z.sum() * 0
    else:
        L = float(lse) if lse is not None else math.log(sum(math.exp(x) for x in a))
        p = [math.exp(x - L) for x in a]
        kl = sum(pi * (math.log(pi) - torch.log(q[c])) for pi, c in zip(p, listed))
        m = 1 - sum(p) if lse is not None and len(listed) < len(z) else 0.0
        if m > 2.0 ** -20:
            rest = torch.stack([q[j] for j in range(len(z)) if j not in listed]).sum()
            kl = kl + m * (math.log(m) - torch.log(rest))
    return kd * tau ** 2 * kl - ce * torch.log_softmax(z, 0)[target]


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("v,k", [(1, 1), (5, 5), (9, 3), (40, 7)])
def test_reference_loss_row_by_row(v, k, rest):
    g = torch.Generator().manual_seed(v + k)
    z = torch.randn(6, v, dtype=torch.float64, generator=g).requires_grad_(True)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(6)])
    ids[1] = -1
    if k > 1:
        ids[2, 0] = -1
    t = torch.randn(6, k, dtype=torch.float64, generator=g)
    lse = torch.logsumexp(t / 1.5, 1) + 0.3 if rest else None
    y = torch.randint(0, v, (6,), generator=g)
    y[4] = -100
    rows = distill.distillation_loss_reference(z, ids, t, lse, y, 1.5, 0.8, 0.25, 2.0, "none")
    want = torch.stack([2.0 * _brute(z[i], ids[i], t[i], None if lse is None else lse[i], int(y[i]), 1.5, 0.8, 0.25)
                        if y[i] >= 0 else z[i].sum() * 0 for i in range(6)])
    torch.testing.assert_close(rows, want, rtol=1e-10, atol=1e-10)
    (got,) = torch.autograd.grad(rows.sum(), z, retain_graph=True)
    (grad,) = torch.autograd.grad(want.sum(), z)
    torch.testing.assert_close(got, grad, rtol=1e-10, atol=1e-10)
    if v > 1:
        f = lambda q: distill.distillation_loss_reference(q, ids, t, lse, y, 1.5, 0.8, 0.25)  # noqa: E731
        assert torch.autograd.gradcheck(f, (z,))


def test_reference_top_logits():
    z = torch.tensor([[1.0, 3.0, 3.0, -2.0], [0.0, 0.0, float("-inf"), 0.0]])
    got = distill.top_logits_reference(z, 3, temperature=2.0)
    assert got.ids.tolist() == [[1, 2, 0], [0, 1, 3]] and got.ids.dtype == torch.int32
    torch.testing.assert_close(got.lse, torch.logsumexp(z / 2, 1))


def test_a_student_equal_to_its_teacher_has_nothing_to_learn():
    z = torch.randn(4, 50, dtype=torch.float64, generator=torch.Generator().manual_seed(2)).requires_grad_(True)
    top = distill.top_logits_reference(z.detach(), 10)
    loss = distill.distillation_loss_reference(z, top.ids, top.values, top.lse)
    (g,) = torch.autograd.grad(loss, z)
    assert abs(float(loss)) < 1e-10 and g.abs().max() < 1e-10


# ------------------------------------------------------------------------------------ model, engine, example
def _lists(n_rows, T, vocab, k, seed=0, tau=2.0):
    g = torch.Generator().manual_seed(seed)
    top = distill.top_logits_reference(torch.randn(n_rows, T, vocab, generator=g) * 2, k, tau)
    return distill.Teacher(top.ids, top.values, top.lse, temperature=tau)


@pytest.mark.parametrize("chunk", [0, 5])
def test_model_returns_the_distillation_loss(chunk):
    torch.manual_seed(3)
    model = TensorLM(_cfg(loss_chunk_tokens=chunk))
    idx = torch.randint(0, 30, (2, 7))
    y = torch.roll(idx, -1, 1)
    y[0, -2:] = -100
    teacher = _lists(2, 7, 30, 4)._replace(ce_weight=0.3)
    _, loss, n = model(idx, targets=y, reduction="sum", teacher=teacher)
    want = distill.distillation_loss_reference(model(idx), teacher.ids, teacher.values, teacher.lse, y, 2.0, 1.0, 0.3)
    torch.testing.assert_close(loss, want)
    assert int(n) == 12
    _, mean = model(idx, targets=y, teacher=teacher)
    torch.testing.assert_close(mean, want / 12)
    _, scaled, _ = model(idx, targets=y, reduction="sum", teacher=teacher, scale=torch.tensor([0.5]))
    torch.testing.assert_close(scaled, want * 0.5)
    with pytest.raises(ValueError, match="targets"):
        model(idx, teacher=teacher)
    with pytest.raises(ValueError, match="teacher"):
        model(idx, targets=y, scale=torch.ones(1))


def test_engine_step_with_a_teacher_is_independent_of_the_micro_batch():
    after = []
    for micro in (1, 4):
        torch.manual_seed(4)
        cfg = Config.from_dict({"model": {k: v for k, v in vars(_cfg()).items()}, "train": {"optimizer": "adamw"}})
        engine = TrainEngine(cfg, device="cpu", micro_batch=micro)
        g = torch.Generator().manual_seed(5)
        idx = torch.randint(0, 30, (4, 6), generator=g)
        y = torch.roll(idx, -1, 1)
        y[2] = -100
        loss, count = engine.step(idx, torch.zeros_like(idx), y, teacher=_lists(4, 6, 30, 5))
        after.append((float(loss), int(count), [p.detach().clone() for p in engine.model.parameters()]))
    assert after[0][1] == after[1][1] == 18
    assert abs(after[0][0] - after[1][0]) <= 1e-5 * abs(after[1][0])
    for p, q in zip(after[0][2], after[1][2]):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-5)


def test_teacher_rows():
    t = _lists(4, 6, 30, 5)
    part = t.rows(1, 3)
    assert torch.equal(part.ids, t.ids[1:3]) and torch.equal(part.lse, t.lse[1:3]) and part.temperature == 2.0
    assert t._replace(lse=None).rows(0, 2).lse is None


def test_example_distils_on_the_cpu(tmp_path):
    from tensor_train_ing_b200.runbook import distill as example
    out = tmp_path / "report.json"
    assert example.main(["--out", str(out), "--steps", "12", "--teacher-steps", "20", "--rows", "4", "--length", "16",
                         "--vocab", "40", "--top", "8", "--device", "cpu"]) == 0
    import json
    report = json.loads(out.read_text())
    assert report["student_ce_after"] < report["student_ce_before"]
    assert len(report["distillation_losses"]) == 12
    with pytest.raises(ValueError, match="at least one step"):
        example.run_distill(steps=0, device="cpu")


def test_kernel_entry_points_refuse_cpu_tensors():
    from tensor_train_ing_b200.ops.layer_norm import layer_norm
    z = torch.randn(3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        distill.top_logits(z, 2)
    with pytest.raises(ValueError, match="CUDA"):
        distill.distillation_loss(z, torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 1))
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(z, torch.ones(8))
    with pytest.raises(ValueError, match="targets"):
        distill.distillation_loss_reference(z, torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 1), ce_weight=1.0)


def test_a_teacher_row_without_any_logit_has_no_divergence():
    """A row masked throughout gives a list of -inf and a log-sum-exp of -inf: nothing to learn from it but its target."""
    z = torch.randn(3, 30, dtype=torch.float64, generator=torch.Generator().manual_seed(6))
    teacher = torch.randn(3, 30, dtype=torch.float64, generator=torch.Generator().manual_seed(7))
    teacher[1] = -math.inf
    top = distill.top_logits_reference(teacher, 5)
    assert top.lse[1] == -math.inf
    y = torch.tensor([3, 4, 5])
    for ce, targets in ((0.0, None), (0.3, y)):
        zz = z.clone().requires_grad_(True)
        rows = distill.distillation_loss_reference(zz, top.ids, top.values, top.lse, targets, ce_weight=ce, reduction="none")
        (g,) = torch.autograd.grad(rows.sum(), zz)
        assert torch.isfinite(rows).all() and torch.isfinite(g).all()
        want = -ce * torch.log_softmax(z, 1)[1, 4]
        torch.testing.assert_close(rows[1], want)
        others = distill.distillation_loss_reference(z[::2], top.ids[::2], top.values[::2], top.lse[::2],
                                                     None if targets is None else targets[::2], ce_weight=ce, reduction="none")
        torch.testing.assert_close(rows[::2].detach(), others)
