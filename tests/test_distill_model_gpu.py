"""Distillation and layer norms inside the model on the sm_100a path (B200).

Tolerances, as in the model parity tests: the fused path rounds GEMM operands to bf16, so its losses agree with the fp32
module path to 2 % and its gradients to 5 % of their norm; paths that run the same kernels agree bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(seed=0, **kw):
    from tensor_train_ing_b200.config import ModelConfig
    from tensor_train_ing_b200.models.model import TensorLM
    torch.manual_seed(seed)
    base = dict(vocab_size=500, padded_vocab=512, d_model=256, layers=2, heads=4, d_key=64, d_value=64, d_mlp=512,
                loss_chunk_tokens=100)
    return TensorLM(ModelConfig(**{**base, **kw})).cuda()


def _batch(seed=1, B=2, T=96, k=12, tau=2.0):
    from tensor_train_ing_b200.ops import distill
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = torch.randint(0, 500, (B, T), device="cuda", generator=g)
    y = torch.roll(idx, -1, 1)
    y[:, -1] = -100
    top = distill.top_logits(torch.randn(B, T, 500, device="cuda", generator=g) * 2, k, tau)
    return idx, y, distill.Teacher(top.ids, top.values, top.lse, temperature=tau, ce_weight=0.25)


def _run(model, idx, y, teacher, scale=None):
    model.zero_grad(set_to_none=True)
    _, loss, n = model(idx, targets=y, reduction="sum", teacher=teacher, scale=scale)
    loss.backward()
    return loss.detach(), {k: p.grad.detach().clone() for k, p in model.named_parameters()}


@pytest.mark.parametrize("norms", [{}, dict(normalization="pre_ln", final_normalization="layer")])
def test_fused_distillation_against_the_module_path(norms):
    model = _model(**norms)
    idx, y, teacher = _batch()
    assert model.uses_fused_path(idx)
    loss, grads = _run(model, idx, y, teacher)
    model._force_reference = True
    want, ref = _run(model, idx, y, teacher)
    assert abs(loss - want) <= 0.02 * abs(want)
    for name, g in grads.items():
        assert (g - ref[name]).norm() <= 0.05 * ref[name].norm() + 1e-7, name
    from tensor_train_ing_b200.ops._ext import check_status
    check_status()


def test_recomputing_the_gradient_gives_the_same_bits(monkeypatch):
    from tensor_train_ing_b200.ops.fused import LinearDistillFn
    model = _model()
    idx, y, teacher = _batch()
    loss, grads = _run(model, idx, y, teacher)
    monkeypatch.setattr(LinearDistillFn, "KEEP_BYTES", 0)
    again, ref = _run(model, idx, y, teacher)
    assert torch.equal(loss, again)
    for name, g in grads.items():
        assert torch.equal(g, ref[name]), name


def test_scale_is_the_factor_of_the_loss():
    model = _model()
    idx, y, teacher = _batch()
    loss, grads = _run(model, idx, y, teacher)
    half, ref = _run(model, idx, y, teacher, torch.tensor([0.5], device="cuda"))
    torch.testing.assert_close(half, 0.5 * loss)
    for name, g in grads.items():  # a power of two commutes with every rounding
        torch.testing.assert_close(ref[name], 0.5 * g, rtol=1e-6, atol=0)
    with torch.no_grad():
        _, evaluated, _ = model(idx, targets=y, reduction="sum", teacher=teacher)
    torch.testing.assert_close(evaluated, loss)


def test_layer_norm_module_runs_its_kernel():
    from tensor_train_ing_b200.models.normalization import LayerNorm
    from tensor_train_ing_b200.ops._ext import launch_counter
    norm = LayerNorm(640, 1e-6).cuda()
    with torch.no_grad():
        norm.weight.add_(0.3 * torch.randn_like(norm.weight))
        norm.bias.add_(0.3 * torch.randn_like(norm.bias))
    x = torch.randn(3, 50, 640, device="cuda", requires_grad=True)
    with launch_counter() as c:
        y = norm(x)
        dx = torch.autograd.grad(y.square().sum(), x)[0]
    assert c.by_name["layer_norm"] == 1 and c.by_name["autograd"] == 2
    x64 = x.detach().double().requires_grad_(True)
    wide = LayerNorm(640, 1e-6).cuda().double()
    wide.load_state_dict(norm.state_dict())
    want = wide(x64)
    torch.testing.assert_close(y.double(), want, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(dx.double(), torch.autograd.grad(want.square().sum(), x64)[0], rtol=1e-4, atol=1e-4)


def test_kernels_agree_with_the_plain_forms():
    from tensor_train_ing_b200.ops import distill
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn(30, 1000, device="cuda", generator=g, requires_grad=True)
    top = distill.top_logits(torch.randn(30, 1000, device="cuda", generator=g) * 3, 20, 1.5)
    y = torch.randint(-1, 1000, (30,), device="cuda", generator=g)
    args = (top.ids, top.values, top.lse, y, 1.5, 0.7, 0.2, 0.5)
    loss = distill.distillation_loss(z, *args)
    (grad,) = torch.autograd.grad(loss, z)
    z64 = z.detach().double().requires_grad_(True)
    want = distill.distillation_loss_reference(z64, *args)
    (ref,) = torch.autograd.grad(want, z64)
    torch.testing.assert_close(loss.double(), want, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(grad.double(), ref, rtol=1e-4, atol=1e-7)


def test_example_distils_on_the_gpu():
    from tensor_train_ing_b200.ops._ext import launch_counter
    from tensor_train_ing_b200.runbook.distill import run_distill
    with launch_counter() as c:
        report = run_distill(steps=25, teacher_steps=40, rows=8, device="cuda")
    assert report["student_ce_after"] < report["student_ce_before"] - 0.2
    assert {"layer_norm", "top_logits", "distill_loss", "autograd"} <= set(c.by_name)


def test_evaluation_forms_no_gradient():
    """Without recorded gradients the loss needs its logits chunk and little else: 2 x 2000 rows of 4096 columns would be
    33 MB of 16-bit gradients."""
    model = _model(vocab_size=4000, padded_vocab=4096, loss_chunk_tokens=100)
    idx, y, teacher = _batch(B=2, T=2000)
    with torch.no_grad():
        model(idx, targets=y, reduction="sum", teacher=teacher)  # caches of the weights
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        x = torch.randn(4000, 256, device="cuda").bfloat16()
        from tensor_train_ing_b200.ops import fused
        from tensor_train_ing_b200.ops.weights import group_for
        group = group_for(model, "unembed", [model.unembed.weight])
        torch.cuda.reset_peak_memory_stats()
        loss = fused.linear_distillation(x, y.reshape(-1), group, 4000, teacher, 1.0, 100)
        peak = torch.cuda.max_memory_allocated() - base
    assert peak < 12 << 20, peak
    x.requires_grad_(True)
    again = fused.linear_distillation(x, y.reshape(-1), group, 4000, teacher, 1.0, 100)
    assert torch.equal(loss, again.detach())
    (dx,) = torch.autograd.grad(again, x)
    assert dx.shape == x.shape and dx.any()


@pytest.mark.parametrize("fused", [True, False])
def test_the_mean_is_the_sum_with_its_factor_inside(fused):
    """reduction="mean" hands one over the count to the loss kernel, which rounds the gradient once, after it."""
    model = _model()
    model._force_reference = not fused
    idx, y, teacher = _batch()
    assert model.uses_fused_path(idx) == fused
    for factor in (None, torch.tensor([0.7], device="cuda")):
        n = (y != -100).sum().float().reshape(1)
        loss, want = _run(model, idx, y, teacher, (1 if factor is None else factor) / n)
        model.zero_grad(set_to_none=True)
        _, mean = model(idx, targets=y, teacher=teacher, scale=factor)
        mean.backward()
        assert torch.equal(mean.detach(), loss)
        for name, p in model.named_parameters():
            assert torch.equal(p.grad, want[name]), name
    _, none = model(idx, targets=torch.full_like(y, -100), teacher=teacher)
    assert none == 0


@pytest.mark.parametrize("keep", [8 << 30, 0])
def test_lists_from_inference_mode_train_the_fused_path(keep, monkeypatch):
    from tensor_train_ing_b200.ops.fused import LinearDistillFn
    monkeypatch.setattr(LinearDistillFn, "KEEP_BYTES", keep)
    model = _model()
    idx, y, teacher = _batch()
    loss, grads = _run(model, idx, y, teacher)
    with torch.inference_mode():
        made = teacher._replace(ids=teacher.ids.clone(), values=teacher.values.clone(), lse=teacher.lse.clone())
    again, ref = _run(model, idx, y, made)
    assert torch.equal(loss, again)
    for name, g in grads.items():
        assert torch.equal(g, ref[name]), name
