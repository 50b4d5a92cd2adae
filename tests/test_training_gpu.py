"""The training loop with the multi-tensor AdamW and the losses on logits: its steps run, its gradients are those of the same
losses in torch operations, and its update is that of torch.optim.AdamW behind clip_grad_norm_."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

SMALL = dict(vocab=199, dim=64, layers=3, heads=4, seq=32, global_batch=8, micro_batch=4, total_steps=20)


def _trainer(**kw):
    from nvfp4_sm120_b200 import quant
    from nvfp4_sm120_b200.train import Trainer
    quant._SEED[0] = 0
    return Trainer(torch.device("cuda", 0), **{**SMALL, **kw})


@pytest.mark.parametrize("backend", ["bf16", "fp4"])
@pytest.mark.parametrize("optimizer", ["torch", "adamw", "adamw8"])
@pytest.mark.parametrize("objective", ["lm", "preference", "policy"])
def test_steps_run(backend, optimizer, objective):
    tr = _trainer(backend=backend, optimizer=optimizer, objective=objective)
    before = [p.detach().clone() for p in tr.params]
    for step in (1, 2, 3):
        loss = tr.step(step)
        assert torch.isfinite(loss)
    assert all(torch.isfinite(p).all() and not torch.equal(p, b) for p, b in zip(tr.params, before))
    if tr.reference is not None:                              # it stays what it was
        assert all(torch.equal(p, b) and p.grad is None for p, b in zip(tr.reference.parameters(), before))


@pytest.mark.parametrize("objective", ["preference", "policy"])
def test_gradients_are_those_of_torch_operations(objective, monkeypatch):
    from nvfp4_sm120_b200 import losses

    def logps(logits, labels, ignore=-100):
        lp = logits.float().log_softmax(-1).gather(-1, labels.clamp(min=0)[..., None])[..., 0]
        return torch.where(labels == ignore, 0.0, lp)

    def preference(logits, labels, ref, beta=0.1):
        c, r = (beta * (logps(logits, labels).double().sum(1) - ref)).chunk(2)
        return -F.logsigmoid(c - r).mean().float(), c, r

    def policy(logits, labels, old, adv, ref, kl_coef):
        lp = logps(logits, labels)
        rho, d, a, live = (lp - old).exp(), ref - lp, adv[:, None], labels != -100
        t = torch.minimum(rho * a, rho.clamp(0.8, 1.2) * a) - kl_coef * (d.expm1() - d)
        return -torch.where(live, t, 0.0).sum() / live.sum(), {}

    def gradients(plain):
        tr = _trainer(backend="bf16", objective=objective)
        with torch.no_grad():                                 # away from the reference model, where the losses are flat
            gen = torch.Generator(device="cuda").manual_seed(1)
            for p in tr.params:
                p.add_(0.01 * torch.randn(p.shape, device="cuda", generator=gen))
        with monkeypatch.context() as m:
            if plain:
                m.setattr(losses, "token_logprobs", logps)
                m.setattr(losses, "preference_loss", preference)
                m.setattr(losses, "policy_loss", policy)
            loss = getattr(tr, "_" + objective)()
            loss.backward()
        return loss.detach(), [p.grad.double() for p in tr.params]

    (a, ga), (b, gb) = gradients(False), gradients(True)
    # (tokens whose ratio lies at 1 within a rounding count the same on both sides: the clamp is far)
    assert abs(a.item() - b.item()) <= 1e-5 * (1 + abs(b.item()))
    # the gradients of the logits are one rounding to bf16 apart, and go through the same backward pass
    for x, y in zip(ga, gb):
        assert (x - y).norm() <= 2.0 ** -7 * y.norm()


def test_first_step_is_that_of_torchs_optimizer():
    """At the first step the update is lr g / (|g| + eps): rounding apart, the sign of the gradient, clipped or not."""
    from nvfp4_sm120_b200.train import lr_at
    a, b = _trainer(backend="bf16"), _trainer(backend="bf16", optimizer="adamw")
    la, lb = a.step(1), b.step(1)
    assert torch.equal(la, lb)
    lr = lr_at(1, a.lr, a.warmup, a.total_steps)
    for p, q in zip(a.params, b.params):
        # the embedding's gradient is summed by atomics: elements near eps may differ in all their digits
        assert (p - q).abs().max() <= 2.0 ** -22 * p.abs().max() + 2 * lr
        assert ((p - q).abs() > 2.0 ** -22 * p.abs() + 2.0 ** -10 * lr).float().mean() < 1e-2
    assert math.isfinite(float(b.opt.grad_norm)) and float(b.opt.grad_norm) > 0


def test_model_scores_are_its_cross_entropy():
    tr = _trainer(backend="fp4")
    x, y = tr.sample(4, 32)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        _, loss = tr.model(x, y)
        lp = tr.model.token_logprobs(x, y)
    assert lp.shape == y.shape and lp.dtype == torch.float32
    assert abs(float(-lp.mean()) - float(loss)) <= 1e-5 * float(loss)


def test_bad_choices_are_refused():
    for kw in (dict(optimizer="sgd"), dict(objective="score")):
        with pytest.raises(ValueError):
            _trainer(**kw)
