"""Refusals of the optimizer and the losses that need no GPU, and argument checks of their C entry points."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nvfp4_sm120_b200 import build, _lib
    build.build()
    return _lib


def test_hyperparameters_are_checked():
    from nvfp4_sm120_b200.optim import AdamW
    p = torch.nn.Parameter(torch.ones(4))
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(weight_decay=-1.0),
                dict(state_bits=16), dict(max_norm=0.0), dict(max_norm=float("nan")), dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    with pytest.raises(ValueError):
        AdamW([])


def test_cpu_tensors_are_refused(lib):
    from nvfp4_sm120_b200 import losses
    from nvfp4_sm120_b200.optim import AdamW, grad_norm
    p = torch.nn.Parameter(torch.ones(4))
    assert AdamW([p]).step() is None                         # no gradient: nothing to do
    p.grad = torch.ones(4)
    with pytest.raises(lib.NVFP4Error):
        AdamW([p]).step()
    with pytest.raises(lib.NVFP4Error):
        grad_norm([p])
    x, y = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long)
    for call in (lambda: losses.token_logprobs(x, y), lambda: losses.preference_loss(x, y, torch.zeros(2)),
                 lambda: losses.policy_loss(x, y, torch.zeros(2, 3), torch.zeros(2))):
        with pytest.raises(lib.NVFP4Error):
            call()


def test_loss_arguments_are_checked():
    from nvfp4_sm120_b200 import losses
    x, y, z = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2)
    with pytest.raises(ValueError, match="label_smoothing"):
        losses.preference_loss(x, y, z, label_smoothing=1.5)
    for bad in (dict(clip=-0.1), dict(clip=1.5), dict(clip_high=-1.0), dict(kl_coef=0.1), dict(clip=float("nan"))):
        with pytest.raises(ValueError):
            losses.policy_loss(x, y, torch.zeros(2, 3), z, **bad)
    for logits, labels in ((torch.zeros(5), torch.zeros((), dtype=torch.long)), (x, y[:1]), (x.half(), y), (x, y.float()),
                           (torch.zeros(2, 3, 0), y), (torch.zeros(0, 3, 5), y[:0])):
        with pytest.raises(ValueError):
            losses.token_logprobs(logits, labels)


def test_c_entry_points_check_their_arguments(lib):
    L, c = lib.lib(), ctypes

    class Tensor(c.Structure):
        _fields_ = [(n, c.c_void_p) for n in ("param", "grad", "first", "second", "first_scale", "second_scale")] + \
                   [("n", c.c_int64), ("counter_base", c.c_uint64), ("hyper", c.c_int32)]

    class Hyper(c.Structure):
        _fields_ = [(n, c.c_float) for n in "abcdefgh"] + [("offset", c.c_uint64)]

    class Rows(c.Structure):
        _fields_ = [("logits", c.c_void_p), ("is_f32", c.c_int)] + \
                   [(n, c.c_int64) for n in ("batch", "seq", "vocab", "stride_b", "stride_t")] + \
                   [("labels", c.c_void_p), ("ignore", c.c_int64)]

    buf = c.create_string_buffer(1 << 16)
    p = (c.addressof(buf) + 255) & ~255                        # host memory: only argument checks run
    h = Hyper()

    def adamw(t, count=1, hypers=1, f32=1, bits=32, parts=None, n_parts=0, norm=None):
        return L.nvfp4_adamw(c.byref(t), count, c.byref(h), hypers, f32, bits, 0, parts, n_parts, norm, 1.0, None, None)

    good = dict(param=p, grad=p, first=p, second=p, n=4)
    assert adamw(Tensor(**good), count=0) == -2
    assert adamw(Tensor(**{**good, "n": 0})) == -2
    assert adamw(Tensor(**{**good, "grad": None})) == -1
    assert adamw(Tensor(**good), bits=8) == -1                 # no scales
    assert adamw(Tensor(**good), bits=4) == -4
    assert adamw(Tensor(**good), hypers=9) == -8
    assert adamw(Tensor(**good, hyper=1)) == -4
    assert adamw(Tensor(**{**good, "param": p + 2})) == -3
    assert adamw(Tensor(**good), parts=p, n_parts=0) == -4
    assert adamw(Tensor(**good), parts=p, n_parts=1, norm=p) == -4
    one = (c.c_int64 * 1)(4)
    ptr = (c.c_void_p * 1)(p + 1)
    assert L.nvfp4_sumsq_parts(1, one) == 1 and L.nvfp4_sumsq_parts(0, None) == 0
    assert L.nvfp4_sumsq_parts(1, (c.c_int64 * 1)(0)) == -2
    assert L.nvfp4_sumsq(ptr, one, 1, 1, p, None) == -3
    assert L.nvfp4_sumsq(None, one, 1, 1, p, None) == -1
    assert L.nvfp4_norm_of_sumsq(p, 0, p, None) == -2
    rows = dict(logits=p, is_f32=1, batch=2, seq=3, vocab=5, stride_b=15, stride_t=5, labels=p, ignore=-100)
    fwd = lambda r: L.nvfp4_logprob_fwd(c.byref(r), p, p, None)
    assert L.nvfp4_logprob_fwd(None, p, p, None) == -1
    assert fwd(Rows(**{**rows, "labels": None})) == -1
    assert fwd(Rows(**{**rows, "vocab": 0})) == -2
    assert fwd(Rows(**{**rows, "vocab": 1 << 40})) == -8
    assert fwd(Rows(**{**rows, "batch": 1 << 60})) == -8
    assert fwd(Rows(**{**rows, "logits": p + 2})) == -3
    r = Rows(**rows)
    assert L.nvfp4_logprob_bwd(c.byref(r), p, p, 0, None, 0, p, 15, 5, None) == -2
    assert L.nvfp4_logprob_bwd(c.byref(r), p, p, 1, None, 1, p, 15, 5, None) == -1       # nothing to compare with 1
    pref = lambda r, ws: L.nvfp4_preference_fwd(c.byref(r), p, 0.1, 0.0, p, p, p, p, p, p, ws, None)
    assert pref(Rows(**{**rows, "batch": 3}), 1 << 20) == -2 and pref(r, 16) == -7
    assert L.nvfp4_policy_fwd(c.byref(r), p, p, 3, None, 0.2, 0.2, 0.0, p, p, p, p, p, p, None, 0, 0, p, 16, None) == -7
    assert L.nvfp4_policy_fwd(c.byref(r), p, p, 0, None, 0.2, 0.2, 0.0, p, p, p, p, p, p, None, 0, 0, p, 1 << 20, None) == -2


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate parameters")
def test_a_parameter_stands_once():
    from nvfp4_sm120_b200.optim import AdamW
    p, q = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError, match="twice"):
        AdamW([p, q, p])
    opt = AdamW([p])
    for again in ([q, q], [p], [q, p]):
        with pytest.raises(ValueError):
            opt.add_param_group({"params": again})
    assert [g["params"] for g in opt.param_groups] == [[p]]
    opt.add_param_group({"params": q, "lr": 0.5})
    assert len(opt.param_groups) == 2 and opt.param_groups[1]["lr"] == 0.5


def test_state_of_coupled_weight_decay_is_refused():
    from nvfp4_sm120_b200.optim import AdamW
    p = torch.nn.Parameter(torch.ones(4))
    p.grad = torch.ones(4)
    other = torch.optim.Adam([p], weight_decay=0.1)
    other.step()
    with pytest.raises(ValueError, match="weight decay"):
        AdamW([p]).load_state_dict(other.state_dict())
