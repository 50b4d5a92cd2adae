"""Losses on logits (losses.py) as nodes of an autograd graph: hooks on saved tensors, second derivatives, what may have changed
between the forward and the backward pass."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

IGNORE = -100


@pytest.fixture(scope="module")
def losses():
    from nvfp4_sm120_b200 import losses as module
    return module


def _randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=torch.Generator(device="cuda").manual_seed(seed))


def _data(shape=(4, 6, 83), seed=1):
    """logits, labels, a vector of a value for each sequence and one for each label"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    y = torch.randint(0, shape[-1], shape[:-1], device="cuda", generator=gen)
    y[torch.rand(shape[:-1], device="cuda", generator=gen) < 0.3] = IGNORE
    return _randn(shape, seed), y, _randn(shape[:1], seed + 1), -4 + 0.3 * _randn(shape[:-1], seed + 2)


def _calls(losses, y, per_sequence, per_label):
    """Each loss as a function of the logits alone, with a gradient that all of its elements count in."""
    w = _randn(y.shape, 9)
    return {"logprobs": lambda x: (losses.token_logprobs(x, y) * w).sum(),
            "preference": lambda x: losses.preference_loss(x, y, per_sequence)[0],
            "policy": lambda x: losses.policy_loss(x, y, per_label, per_sequence, per_label + 0.1, kl_coef=0.1)[0]}


NAMES = ["logprobs", "preference", "policy"]


# ---- what was saved -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_that_come_back_changed_are_refused(losses, name):
    x, y, a, b = _data()
    call = _calls(losses, y, a, b)[name]
    x.requires_grad_(True)
    (want,) = torch.autograd.grad(call(x), x)
    same = lambda t: t
    vector = lambda t: t.dim() == 1 and t.is_floating_point()
    for unpack in (lambda t: t.half() if vector(t) else t, lambda t: t[:-1] if vector(t) else t, lambda t: t[:0] if vector(t) else t,
                   lambda t: t.cpu(), lambda t: t.cpu() if vector(t) else t, lambda t: t.cpu() if t.dim() == 2 else t,
                   lambda t: t.half() if t.dim() == 3 else t, lambda t: torch.cat((t, t), -1) if t.dim() == 3 else t, lambda t: t.float() if t.dim() == 2 else t,
                   lambda t: t[:, :-1] if t.dim() == 3 else t, lambda t: t[:, :-1] if t.dim() > 1 else t,
                   lambda t: torch.cat((t, t)) if t.dim() > 1 else t, lambda t: t[:1].expand(t.shape) if vector(t) else t):
        with torch.autograd.graph.saved_tensors_hooks(same, unpack):
            loss = call(x)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(3 * loss, x)           # (a factor: the policy loss has to write its gradient again)
    assert torch.equal(torch.autograd.grad(call(x), x)[0], want)
    with torch.autograd.graph.save_on_cpu():
        loss = call(x)
    assert torch.equal(torch.autograd.grad(loss, x)[0], want)


@pytest.mark.parametrize("name", NAMES)
def test_logits_swapped_behind_autograds_back_are_refused(losses, name):
    for other in (lambda x: x[:, :3].clone(), lambda x: torch.cat((x, x)), lambda x: torch.cat((x, x), -1), lambda x: x.bfloat16(), lambda x: x.double(), lambda x: x[0, 0].clone()):
        x, y, a, b = _data()
        leaf = x.requires_grad_(True)
        loss = _calls(losses, y, a, b)[name](leaf)
        leaf.data = other(leaf.detach())
        with pytest.raises(RuntimeError):
            torch.autograd.grad(3 * loss, leaf)        # (a factor: the policy loss has to write its gradient again)


# ---- second derivatives -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused_not_lost(losses, name):
    """A penalty on the gradient, added to something that is differentiable: its part must not be left out in silence."""
    h, y, a, b = _data()
    call = _calls(losses, y, a, b)[name]
    head = torch.nn.Parameter(1 + 0.1 * _randn(h.shape[-1:], 5))
    scale = torch.nn.Parameter(torch.ones((), device="cuda"))
    for factor in (1.0, scale):
        x = h * head
        loss = factor * call(x)
        (plain,) = torch.autograd.grad(loss, x, retain_graph=True)
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        assert torch.equal(g, plain) and g.requires_grad
        penalty = g.square().sum()
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(head.sum() + penalty, head, retain_graph=True)
        if factor is scale:                            # (the other penalty does not depend on it)
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(head.sum() + scale + penalty, scale, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            (loss + penalty).backward()
    head.grad = None                                   # without a second derivative such a graph is as good as any
    (call(h * head) + 0.0).backward(create_graph=True)
    first = head.grad.detach().clone()
    head.grad = None
    call(h * head).backward()
    assert torch.equal(first, head.grad)
    head.grad = None


# ---- the policy loss's gradient between its passes ----------------------------------------------------------------------
def test_hooks_on_saved_tensors_see_the_waiting_gradient(losses):
    """The gradient that the policy loss's forward pass leaves is as large as the logits: it can be moved away until it is needed."""
    x, y, a, b = _data((4, 64, 5003))
    x.requires_grad_(True)
    call = _calls(losses, y, a, b)["policy"]
    size = x.numel() * x.element_size()
    for factor in (1.0, 3.0):
        (want,) = torch.autograd.grad(factor * call(x), x)
        shapes = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: shapes.append(t.shape) or t, lambda t: t):
            loss = factor * call(x)
        assert shapes.count(x.shape) == 2              # the logits and their gradient
        assert torch.equal(torch.autograd.grad(loss, x, retain_graph=True)[0], want)
        assert torch.equal(torch.autograd.grad(loss, x)[0], want)          # written anew
        before = torch.cuda.memory_allocated()
        with torch.autograd.graph.save_on_cpu():
            loss = factor * call(x)
        assert torch.cuda.memory_allocated() - before < size // 2
        assert torch.equal(torch.autograd.grad(loss, x, retain_graph=True)[0], want)
        assert torch.equal(torch.autograd.grad(loss, x)[0], want)
    for back in (lambda t: t.half(), lambda t: t.cpu(), lambda t: t[:1], lambda t: t[..., :-1], lambda t: t.cpu() if t.dtype == torch.float32 else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: back(t) if t.shape == x.shape and t is not x else t):
            loss = call(x)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(3 * loss, x)
    # rows that come back in another order of memory
    def transposed(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2) if t.shape == x.shape else t
    for move in (transposed, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.shape == x.shape else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, move):
            loss = 3.0 * call(x)
        assert torch.equal(torch.autograd.grad(loss, x)[0], want)


def test_losses_inside_a_checkpoint(losses):
    from torch.utils.checkpoint import checkpoint
    x, y, a, b = _data()
    for name, call in _calls(losses, y, a, b).items():
        x.requires_grad_(True)
        (want,) = torch.autograd.grad(call(x * 1.5), x)
        loss = checkpoint(lambda t: call(t * 1.5), x, use_reentrant=False)
        assert torch.equal(torch.autograd.grad(loss, x)[0], want), name
