"""State of the multi-tensor AdamW (optim.py): hooks around loading, layouts, what a program may do to it between steps."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 256
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module")
def optim():
    from nvfp4_sm120_b200 import optim as module
    return module


def _params(shapes, dtype=torch.float32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for s in shapes:
        p = torch.nn.Parameter((0.02 * torch.randn(s, device="cuda", generator=gen)).to(dtype))
        p.grad = (1e-3 * torch.randn(s, device="cuda", generator=gen)).to(dtype)
        out.append(p)
    return out


def _same(a, b):
    return a == b if not isinstance(a, torch.Tensor) else torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---- hooks --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_hooks_around_loading(optim, bits):
    """What pre-hooks make of the saved dict is what is loaded, and post-hooks find it in place."""
    p, q = _params([(33, 7), (300,)]), _params([(33, 7), (300,)])
    x, y = optim.AdamW(p, **HYPER, state_bits=bits), optim.AdamW(q, **HYPER, state_bits=bits)
    x.step()
    x.step()
    seen = []

    def forget_the_second(opt, saved):
        seen.append("before")
        state = {0: {**saved["state"][0], "step": 7}}
        return {"state": state, "param_groups": [{**g, "lr": 0.5} for g in saved["param_groups"]]}

    def look(opt):
        assert len(opt.state) == 1 and opt.state[q[0]]["step"] == 7 and opt.param_groups[0]["lr"] == 0.5
        for name, t in x.state[p[0]].items():
            assert name == "step" or _same(opt.state[q[0]][name], t)
        seen.append("after")

    y.register_load_state_dict_pre_hook(forget_the_second)
    y.register_load_state_dict_post_hook(look)
    y.load_state_dict(x.state_dict())
    assert seen == ["before", "after"]
    y.load_state_dict(x.state_dict())                  # nothing of the first call is left behind
    assert seen == ["before", "after"] * 2
    y.step()
    assert y.state[q[0]]["step"] == 8 and y.state[q[1]]["step"] == 1
    # a pre-hook that spoils the state is refused before anything changes, and leaves no hook either
    z = optim.AdamW(q, **HYPER, state_bits=bits)
    spoil = z.register_load_state_dict_pre_hook(lambda opt, saved: {**saved, "state": {0: {"step": 1}}})
    with pytest.raises(ValueError, match=f"{bits}-bit"):
        z.load_state_dict(x.state_dict())
    assert not z.state
    spoil.remove()
    z.load_state_dict(x.state_dict())
    assert z.state[q[1]]["step"] == 2


# ---- layouts ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_strides_of_sizes_of_one_do_not_count(optim, bits):
    """A [1, n] parameter may have any stride along its first dimension: the step takes it, and so does loading."""
    a = _params([(1, 300), (5, 1, 7)])
    x = optim.AdamW(a, **HYPER, state_bits=bits)
    x.step()
    b = [torch.nn.Parameter(a[0].detach().clone().as_strided((1, 300), (1, 1))),
         torch.nn.Parameter(a[1].detach().clone().as_strided((5, 1, 7), (7, 1, 1)))]
    for p, q in zip(a, b):
        assert p.stride() != q.stride()
        q.grad = p.grad.clone()
    y = optim.AdamW(b, **HYPER, state_bits=bits)
    y.load_state_dict(x.state_dict())
    for _ in range(2):
        x.step()
        y.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    if bits == 8:                                      # an order that matters is refused as ever, whatever its number of sizes
        t = torch.nn.Parameter(torch.ones(5, 1, 7, device="cuda").permute(2, 1, 0).contiguous().permute(2, 1, 0))
        for other in (t, torch.nn.Parameter(torch.ones(35, device="cuda"))):
            with pytest.raises(ValueError, match="order"):
                optim.AdamW([b[0], other], state_bits=8).load_state_dict(x.state_dict())


# ---- what a program does between steps ----------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_looking_up_a_parameter_before_its_first_step(optim, bits):
    """`opt.state[p]` puts an empty dict there, which the first step takes for no state, as torch's optimizers do."""
    a, b = _params([(33, 7), (300,)]), _params([(33, 7), (300,)])
    x, y = optim.AdamW(a, **HYPER, state_bits=bits), optim.AdamW(b, **HYPER, state_bits=bits)
    assert all(len(x.state[p]) == 0 for p in a)
    saved = x.state_dict()
    assert len(saved["state"]) == 2
    x.load_state_dict(saved)                           # there is nothing in it
    assert not x.state and all(len(x.state[p]) == 0 for p in a)
    late, a[1].grad = a[1].grad, None
    x.step()
    assert x.state[a[0]]["step"] == 1
    a[1].grad = late
    for _ in range(2):
        x.step()
    b[1].grad = None
    y.step()
    b[1].grad = late
    for _ in range(2):
        y.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_norm_without_gradients_is_fp32_whatever_the_default(optim):
    p = torch.nn.Parameter(torch.ones(3, device="cuda"))
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.float64)
        got = optim.grad_norm([p])
    finally:
        torch.set_default_dtype(before)
    assert got.dtype == torch.float32 and got.device == p.device and float(got) == 0.0
    opt = optim.AdamW([p], max_norm=1.0)
    p.grad = torch.ones_like(p)
    opt.step(grad_norm=got)                            # and so it can be handed on


# ---- layouts and sizes of the 32-bit step -------------------------------------------------------------------------------
def _operations(p, g, m, v, t, lr, b1, b2, eps, wd):
    """One step in fp32, one torch operation for each."""
    g, pf = g.float(), p.float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    ratio = m / (v.sqrt() * (1 / math.sqrt(1 - b2 ** t)) + eps)
    return (pf * (1 - lr * wd) - ratio * (lr / (1 - b1 ** t))).to(p.dtype), m, v


def test_both_moments_in_every_layout_and_what_lies_around(optim):
    """Another memory order, no vector alignment, channels last, missing gradients: weights and both moments have the bits of the torch
    operations, and nothing around a parameter that is a part of a buffer is written."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    buf = rand(5001)
    around = buf.clone()
    params = [torch.nn.Parameter(rand(40, 70).t()), torch.nn.Parameter(buf[1:4097]), torch.nn.Parameter(rand(300)),
              torch.nn.Parameter(rand(6, 5, 4, 3).to(memory_format=torch.channels_last))]
    opt = optim.AdamW(params, **HYPER)
    model = [[p.detach().clone(), torch.zeros_like(p), torch.zeros_like(p), 0] for p in params]
    for k in range(4):
        for i, p in enumerate(params):
            p.grad = None
            if (k + i) % 3 != 0:
                g = rand(*p.shape)
                p.grad = g.contiguous()
                w, m, v, t = model[i]
                model[i] = [*_operations(w, g, m, v, t + 1, 3e-3, 0.9, 0.95, 1e-8, 0.1), t + 1]
        opt.step()
    for p, (w, m, v, t) in zip(params, model):
        st = opt.state[p]
        assert torch.equal(p.detach(), w) and torch.equal(st["exp_avg"], m) and torch.equal(st["exp_avg_sq"], v) and st["step"] == t
    assert torch.equal(buf[:1], around[:1]) and torch.equal(buf[4097:], around[4097:]) and not torch.equal(buf[1:4097], around[1:4097])


def test_more_elements_than_32_bits_count_with_32_bit_moments(optim):
    n = 2 ** 31 + 300
    p = torch.nn.Parameter(torch.ones(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    ends = torch.tensor([0, 255, 256, n // 2, n - 301, n - 45, n - 1], device="cuda")
    p.grad[ends] = 2.0
    opt = optim.AdamW([p], lr=0.5, weight_decay=0.0, max_norm=1e9)
    opt.step()
    # the gradient's sign at the first step, within the roundings of the update and of bf16 (0.5 is a bf16 number)
    assert ((p.detach()[ends].float() - 0.5).abs() <= 2.0 ** -8).all() and int((p.detach() != 1).sum()) == len(ends)
    st = opt.state[p]
    for name, want in (("exp_avg", 0.1 * 2), ("exp_avg_sq", 0.001 * 4)):
        assert (st[name][ends] - want).abs().max() <= 4 * 2.0 ** -24 * want and int(torch.count_nonzero(st[name])) == len(ends)
    del p, opt, st
    torch.cuda.empty_cache()


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_state_loads_with_torch_loads_defaults(optim, bits, tmp_path):
    """Tensors, numbers and tuples alone: no pickled code."""
    a = _params([(33, 77), (1, 5)])
    x = optim.AdamW(a, **HYPER, state_bits=bits, max_norm=1.0)
    x.step()
    torch.save(x.state_dict(), tmp_path / "state.pt")
    y = optim.AdamW(a, **HYPER, state_bits=bits, max_norm=1.0)
    y.load_state_dict(torch.load(tmp_path / "state.pt"))
    for p in a:
        assert all(_same(t, y.state[p][name]) for name, t in x.state[p].items())


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_made_in_inference_mode(optim, bits):
    """Refused outside that mode before anything changes, as torch's optimizers refuse them; stepped inside it."""
    with torch.inference_mode():
        p = torch.ones(300, device="cuda")
        p.grad = torch.ones_like(p)
    (q,) = _params([(300,)])
    w = q.detach().clone()
    opt = optim.AdamW([q, p], **HYPER, state_bits=bits)
    with pytest.raises(ValueError, match="inference"):
        opt.step()
    assert torch.equal(q.detach(), w) and torch.equal(p, torch.ones_like(p))
    assert all(st["step"] == 0 for st in opt.state.values())
    with torch.inference_mode():
        opt.step()
    assert opt.state[p]["step"] == 1 and (p != 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copied_optimizer_loads_state(optim, bits):
    import copy
    a = _params([(33, 7), (300,)])
    x = optim.AdamW(a, **HYPER, state_bits=bits)
    x.step()
    b, y = copy.deepcopy((a, x))
    x.step()
    y.load_state_dict(x.state_dict())
    for p, q in zip(a, b):
        assert y.state[q]["step"] == 2 and all(_same(t, y.state[q][name]) for name, t in x.state[p].items())
