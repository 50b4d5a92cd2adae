"""The losses and the optimizer as the models and the training loop use them."""
import json
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _gpt(cls=None, **kw):
    from nvfp4_sm120_b200.models import GPT, GPTConfig
    torch.manual_seed(0)
    return (cls or GPT)(GPTConfig(vocab=61, dim=64, n_layers=2, n_heads=4, n_kv_heads=4, use_fp4=False, **kw), DEV)


def _tokens(shape=(3, 16), vocab=61):
    gen = torch.Generator(device=DEV).manual_seed(1)
    return (torch.randint(0, vocab, shape, device=DEV, generator=gen) for _ in range(2))


def test_scores_go_through_the_models_call():
    """Hooks on the model and a subclass's own forward count in its scores, as they do in its training step."""
    from nvfp4_sm120_b200 import losses
    from nvfp4_sm120_b200.models import GPT, LM
    x, y = _tokens()
    model = _gpt()
    want = model.token_logprobs(x, y)
    assert torch.equal(want, losses.token_logprobs(model(x)[0], y))
    seen = []
    pre = model.register_forward_pre_hook(lambda m, args: seen.append(args[0].shape))
    post = model.register_forward_hook(lambda m, args, out: (out[0] * 0.5, out[1]))
    got = model.token_logprobs(x, y)
    pre.remove()
    post.remove()
    assert seen == [x.shape] and torch.equal(got, losses.token_logprobs(model(x)[0] * 0.5, y))

    class Warm(GPT):
        def forward(self, idx, targets=None):
            logits, loss = super().forward(idx, targets)
            return logits / 2.0, loss

    assert torch.equal(_gpt(Warm).token_logprobs(x, y), got)
    torch.manual_seed(0)
    lm = LM(61, 64, 2, 4, 4, 16, 128, False)
    assert torch.equal(lm.token_logprobs(x, y), losses.token_logprobs(lm(x), y))


@pytest.mark.parametrize("objective,per_count", [("lm", 1), ("preference", 2), ("policy", 1)])
def test_reported_tokens_are_those_trained_on(objective, per_count, monkeypatch, tmp_path):
    from nvfp4_sm120_b200 import train
    trained = []
    step = train.Trainer.step

    def counted(self, n):
        hook = self.model.register_forward_pre_hook(lambda m, args: trained.append(args[0].numel()) if torch.is_grad_enabled() else None)
        loss = step(self, n)
        hook.remove()
        return loss

    monkeypatch.setattr(train.Trainer, "step", counted)
    out = tmp_path / "log.jsonl"
    monkeypatch.setattr(sys, "argv", ["train", "--steps", "4", "--backend", "bf16", "--vocab", "199", "--dim", "64", "--layers", "2", "--heads", "4",
                                      "--seq", "32", "--global-batch", "8", "--micro-batch", "4", "--objective", objective, "--out", str(out)])
    train.main()
    log = [json.loads(line) for line in open(out)]
    start, done = log[0], log[-1]
    assert start["tokens_per_step"] * 4 == sum(trained) == 4 * 8 * 32 * per_count
    assert abs(done["tokens_per_s"] * done["ms_per_step"] * 1e-3 - start["tokens_per_step"]) <= 1e-6 * start["tokens_per_step"]
