"""The multi-tensor AdamW (csrc/adamw.cu, optim.py) against its formula in 64 bits and, bit for bit, against the same
operations in fp32; 8-bit moments against a model of their code; clipping, state, refusals."""
import copy
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 256


@pytest.fixture(scope="module")
def optim():
    from nvfp4_sm120_b200 import optim as module
    return module


def _params(shapes, dtype=torch.float32, seed=0, scale=0.02):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for s in shapes:
        p = torch.nn.Parameter((scale * torch.randn(s, device="cuda", generator=gen)).to(dtype))
        p.grad = (1e-3 * torch.randn(s, device="cuda", generator=gen)).to(dtype)
        out.append(p)
    return out


def _formula(p, g, m, v, t, lr, b1, b2, eps, wd, c=1.0):
    """One step in 64 bits."""
    p, g, m, v = p.double(), g.double() * c, m.double(), v.double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps), m, v


def _operations(p, g, m, v, t, lr, b1, b2, eps, wd):
    """The same in fp32, one torch operation for each."""
    g, pf = g.float(), p.float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    ratio = m / (v.sqrt() * (1 / math.sqrt(1 - b2 ** t)) + eps)
    return (pf * (1 - lr * wd) - ratio * (lr / (1 - b1 ** t))).to(p.dtype), m, v


HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
ODD = [(1,), (7,), (8,), (255,), (256,), (257,), (2047,), (2049,), (33, 77), (129, 513), (50257, 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_follow_the_formula(optim, dtype):
    params = _params(ODD, dtype)
    opt = optim.AdamW(params, **HYPER)
    for t in range(1, 5):
        before = [p.detach().clone() for p in params]
        state = [(opt.state[p]["exp_avg"].clone(), opt.state[p]["exp_avg_sq"].clone()) if t > 1 else
                 (torch.zeros_like(p, dtype=torch.float32),) * 2 for p in params]
        version = params[0]._version
        opt.step()
        assert params[0]._version > version
        for p, b, (m, v) in zip(params, before, state):
            args = (b, p.grad, m, v, t, 3e-3, 0.9, 0.95, 1e-8, 0.1)
            pe, me, ve = _formula(*args)
            st = opt.state[p]
            assert st["step"] == t
            # roundings to fp32 (2^-24 each, constants among them): m 3 on each of its terms, v 4; then root, product, sum,
            # quotient, product on the update with theirs halved by the root, and two on the weight
            u = 2.0 ** -24
            gd = p.grad.double().abs()
            assert ((st["exp_avg"].double() - me).abs() <= 3.01 * u * (0.9 * m.double().abs() + 0.1 * gd) + 1e-44).all()
            assert ((st["exp_avg_sq"].double() - ve).abs() <= 4.01 * u * ve + 1e-44).all()
            size = 3e-3 / (1 - 0.9 ** t) * (0.9 * m.double().abs() + 0.1 * gd) / (ve.sqrt() / math.sqrt(1 - 0.95 ** t) + 1e-8)
            own = torch.finfo(dtype).eps / 2 * pe.abs()                   # the rounding of the result
            assert ((p.detach().double() - pe).abs() <= own * 1.001 + u * (3.01 * b.double().abs() + 12 * size)).all()
            po, mo, vo = _operations(*args)
            assert torch.equal(p.detach(), po) and torch.equal(st["exp_avg"], mo) and torch.equal(st["exp_avg_sq"], vo)


def test_groups_missing_gradients_and_layouts(optim):
    gen = torch.Generator(device="cuda").manual_seed(3)
    buf = torch.randn(5001, device="cuda", generator=gen)
    params = [torch.nn.Parameter(torch.randn(40, 70, device="cuda", generator=gen).t()),       # another memory order
              torch.nn.Parameter(buf[1:4097]),                                                 # no vector alignment
              torch.nn.Parameter(torch.randn(300, device="cuda", generator=gen)),
              torch.nn.Parameter(torch.randn(6, 5, 4, 3, device="cuda", generator=gen).to(memory_format=torch.channels_last)),
              torch.nn.Parameter(torch.empty(0, device="cuda")),
              torch.nn.Parameter(torch.randn(3, device="cuda", generator=gen), requires_grad=False)]
    groups = [dict(params=params[:2]), dict(params=params[2:], lr=1e-2, weight_decay=0.0, betas=(0.8, 0.9))]
    opt = optim.AdamW(groups, **HYPER)
    model = {i: [p.detach().clone(), torch.zeros_like(p), torch.zeros_like(p), 0] for i, p in enumerate(params)}
    for k in range(4):
        for i, p in enumerate(params[:4]):
            p.grad = None
            if (k + i) % 3 != 0:                                                               # steps of their own
                g = torch.randn(p.shape, device="cuda", generator=gen)
                p.grad = g if i != 3 else g.contiguous()                                       # not always p's strides
                lr, wd, b1, b2 = (3e-3, 0.1, 0.9, 0.95) if i < 2 else (1e-2, 0.0, 0.8, 0.9)
                w, m, v, t = model[i]
                model[i] = [*_operations(w, g, m, v, t + 1, lr, b1, b2, 1e-8, wd), t + 1]
        opt.step()
    for i, p in enumerate(params[:4]):
        assert torch.equal(p.detach(), model[i][0]) and opt.state[p]["step"] == model[i][3]
        assert torch.equal(opt.state[p]["exp_avg"], model[i][1])
    assert torch.equal(buf[0], buf[0]) and params[4] not in opt.state and params[5] not in opt.state


def test_neighbours_of_a_parameter_stay(optim):
    """A parameter that is a slice of a buffer: nothing outside it is written, in either form of the moments."""
    for bits in (32, 8):
        for start, n in ((1, 4096), (8, 1000), (256, 257)):
            buf = torch.full((5000,), 7.0, device="cuda")
            p = torch.nn.Parameter(buf[start:start + n])
            p.grad = torch.ones_like(p)
            optim.AdamW([p], **HYPER, state_bits=bits).step()
            assert (buf[:start] == 7).all() and (buf[start + n:] == 7).all() and (p != 7).all()


def test_more_tensors_than_a_table_and_more_steps_than_a_launch_holds(optim):
    params = _params([(i % 13 + 1, 17) for i in range(900)])
    opt = optim.AdamW(params, **HYPER, max_norm=0.01)
    for k in range(11):                                       # eleven different step counts in the last step
        for i, p in enumerate(params):
            p.grad = torch.full_like(p, 1e-3 * (i % 5 + 1)) if i % 11 <= k else None
        opt.step()
    assert [opt.state[p]["step"] for p in params[:11]] == list(range(11, 0, -1))
    want = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
    assert abs(float(opt.grad_norm) - want) <= 2.0 ** -23 * want


# ---- gradient norm and clipping -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 1e30, 1e-30])
def test_grad_norm(optim, dtype, scale):
    params = _params(ODD + [(300, 1000)], dtype)
    for p in params:
        p.grad = (p.grad.double() * scale).to(dtype)
    got = optim.grad_norm(params)
    want = torch.sqrt(sum(p.grad.double().square().sum() for p in params))
    assert got.dtype == torch.float32 and got.shape == ()
    # squares and sums in 64 bits, one rounding to fp32
    assert abs(float(got) - float(want)) <= 1.001 * 2.0 ** -24 * float(want)
    assert torch.equal(got, optim.grad_norm(iter(params)))
    for p in params:
        p.grad = None
    assert float(optim.grad_norm(params)) == 0.0
    params[3].grad = torch.full_like(params[3], math.inf)
    assert float(optim.grad_norm(params)) == math.inf


def test_clipping_is_that_of_clip_grad_norm(optim):
    a, b = _params(ODD), _params(ODD)
    b[2].data = b[2].data.clone()
    mine = optim.AdamW(a, **HYPER, max_norm=0.01)
    theirs = torch.optim.AdamW(b, **HYPER)
    for _ in range(3):
        grads = [p.grad.clone() for p in b]
        mine.step()
        norm = torch.nn.utils.clip_grad_norm_(b, 0.01)
        theirs.step()
        assert abs(float(mine.grad_norm) - float(norm)) <= 1e-6 * float(norm) and float(norm) > 0.01
        for p, q, g in zip(a, b, grads):
            # the update is at most lr / (1 - b1) / sqrt(1 - b2) times a few roundings; weights two more
            assert (p - q).abs().max() <= 2.0 ** -22 * q.abs().max() + 3e-3 * 45 * 2.0 ** -20
            assert torch.equal(p.grad, g)                     # left as it was
            q.grad = g
    for p in a:
        p.grad = p.grad * 1e-6                                # below the limit: no factor
    before = [(p.detach().clone(), mine.state[p]["exp_avg"].clone(), mine.state[p]["exp_avg_sq"].clone()) for p in a]
    mine.step()
    for p, (w, m, v) in zip(a, before):
        assert torch.equal(p.detach(), _operations(w, p.grad, m, v, 4, 3e-3, 0.9, 0.95, 1e-8, 0.1)[0])


def test_norm_given_by_the_caller(optim):
    a, b = _params(ODD), _params(ODD)
    x, y = optim.AdamW(a, **HYPER, max_norm=0.01), optim.AdamW(b, **HYPER, max_norm=0.01)
    x.step()
    y.step(grad_norm=optim.grad_norm(b))
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(x.grad_norm, y.grad_norm)


# ---- 8-bit moments ------------------------------------------------------------------------------------------------------
def _dither(groups, step, seed, base=0):
    """16 bits for each of eight elements from one Philox4x32-10 call."""
    m32 = np.uint64(0xffffffff)
    c = np.arange(groups, dtype=np.uint64) + np.uint64(base)
    x = [c & m32, c >> np.uint64(32), np.full_like(c, step), np.zeros_like(c)]
    k = [seed & 0xffffffff, seed >> 32]
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> np.uint64(32)) ^ x[1] ^ np.uint64(k[0]), b & m32, (a >> np.uint64(32)) ^ x[3] ^ np.uint64(k[1]), a & m32]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    w = np.stack(x, 1)
    return torch.from_numpy(np.stack([w & np.uint64(0xffff), w >> np.uint64(16)], 2).reshape(-1).astype(np.int64)).cuda()


def _reversed16(b):
    return sum(((b >> k) & 1) << (15 - k) for k in range(16))


def _codes(x, dither):
    """Values of the E4M3 codes and the scales that fp32 x [blocks, 256] becomes, by its definition in 64 bits."""
    x = x.double()
    top = x.abs().amax(1)
    e = torch.frexp(top.clamp(min=2.0 ** -100)).exponent.double() - 1
    nan = ~(top < 2.0 ** 51)
    e = torch.where(nan, 0.0, e)
    y = x.abs() * torch.exp2(7 - e)[:, None]
    grid = torch.exp2((torch.frexp(y).exponent.double() - 1).clamp(min=-6) - 3)
    grid = torch.where(y == 0, 2.0 ** -9, grid)
    y = torch.floor(y / grid + dither.view_as(y) / 65536.0) * grid * torch.sign(x)
    scale = torch.where(nan, math.nan, torch.exp2(e - 7))
    return y, scale, nan


@pytest.mark.parametrize("n", [1, 7, 255, 256, 257, 2048, 5000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eight_bit_moments(optim, n, dtype):
    seed = 0x123456789abcdef
    gen = torch.Generator(device="cuda").manual_seed(n)
    first = torch.nn.Parameter(torch.ones(300, device="cuda", dtype=dtype))                 # moves the counters
    p = torch.nn.Parameter((0.02 * torch.randn(n, device="cuda", generator=gen)).to(dtype))
    opt = optim.AdamW([first, p], **HYPER, state_bits=8, seed=seed)
    blocks = -(-n // BLOCK)
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for t in range(1, 6):
        # gradients over twelve decades, some zero, whole blocks of zeros
        g = torch.randn(n, device="cuda", generator=gen) * 10.0 ** (12 * torch.rand(n, device="cuda", generator=gen) - 10)
        g[torch.rand(n, device="cuda", generator=gen) < 0.2] = 0
        g[512:768] = 0
        p.grad = g.to(dtype)
        first.grad = torch.ones_like(first)
        before = p.detach().clone()
        opt.step()
        args = (before, p.grad, m, v, t, 3e-3, 0.9, 0.95, 1e-8, 0.1)
        (po, _, _), (_, mo, vo) = _formula(*args), _operations(*args)
        # approximate root and reciprocal (2^-23 and 2^-22.5) and a dozen roundings on the update, two on the weight, the
        # rounding to its dtype; the update is at most lr / (1 - b1^t) times (root / sqrt(1 - b2^t))^-1 of the terms of m
        update = 3e-3 / (1 - 0.9 ** t) * (0.9 * m.double().abs() + 0.1 * p.grad.double().abs()) / (
            vo.double().sqrt() / math.sqrt(1 - 0.95 ** t) + 1e-8)
        assert ((p.detach().double() - po).abs() <= torch.finfo(dtype).eps / 2 * 1.001 * po.abs()
                + 2.0 ** -24 * 3 * before.double().abs() + 2.0 ** -20 * update).all()
        st = opt.state[p]
        bits = _dither(blocks * 32, t, seed, base=2 * 32)
        pad = lambda x: torch.cat([x, x.new_zeros(blocks * BLOCK - n)]).view(blocks, BLOCK)
        for x, d, name in ((mo, bits, "exp_avg"), (vo.sqrt(), _reversed16(bits), "exp_avg_root")):
            value, scale, _ = _codes(pad(x), d)
            assert st[name].dtype == torch.float8_e4m3fn and torch.equal(st[name + "_scale"].double(), scale)
            got = st[name].double().view(blocks, BLOCK)
            # below 2^-20 of a code step the kernel's own scaling rounds: there the neighbouring code is as good
            assert (got != value).double().mean() < 1e-4 and (got - value).abs().max() <= 16
        decode = lambda name: (st[name].float().view(blocks, BLOCK) * st[name + "_scale"].float()[:, None]).view(-1)[:n]
        m, v = decode("exp_avg"), decode("exp_avg_root").square()


def test_rounding_of_moments_has_no_bias(optim):
    """65536 equal values between two codes: their mean is the value, within five standard deviations of the mean."""
    n = 1 << 16
    for value in (1.0625 * 0.7, 0.3, 1e-3):
        p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
        p.grad = torch.full((n,), value, device="cuda")
        p.grad[::BLOCK] = 1.9                                    # the block's maximum, so that the codes are small ones too
        opt = optim.AdamW([p], lr=1e-3, betas=(0.0, 0.0), state_bits=8, seed=5)
        opt.step()
        for name in ("exp_avg", "exp_avg_root"):
            st = opt.state[p]
            got = (st[name].double().view(-1, BLOCK) * st[name + "_scale"].double()[:, None])[:, 1:]
            low = got.min()
            step = float(got.max() - low)
            assert step > 0 and float(low) < value < float(low) + step
            # 2^-16: the dither has 16 bits; 2^-22: fp32 gradient and root
            assert abs(float(got.mean()) - value) <= 5 * step / 2 / math.sqrt(got.numel()) + step * 2.0 ** -16 + value * 2.0 ** -22


def test_what_is_no_number_stays_in_its_block(optim):
    for bad in (math.nan, math.inf, -math.inf, 1e38):
        p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
        opt = optim.AdamW([p], **HYPER, state_bits=8)
        p.grad = torch.ones(1024, device="cuda")
        p.grad[300] = bad
        opt.step()
        scale = opt.state[p]["exp_avg_scale"].float()
        assert torch.isnan(scale[1]) and torch.isfinite(scale[[0, 2, 3]]).all()
        p.grad = torch.ones(1024, device="cuda")
        opt.step()
        ok = torch.ones(1024, dtype=torch.bool, device="cuda")
        ok[256:512] = False
        assert torch.isfinite(p[ok]).all() and torch.isnan(p[~ok]).all()


def test_zero_gradients_and_extreme_scales(optim):
    p = torch.nn.Parameter(torch.ones(600, device="cuda"))
    for g in (0.0, 1e-38, 1e-45, 1e-25, 1e14):
        opt = optim.AdamW([p], lr=0.0, weight_decay=0.0, state_bits=8)
        p.grad = torch.full_like(p, g)
        opt.step()
        opt.step()
        assert torch.equal(p.detach(), torch.ones_like(p))
        for name in ("exp_avg_scale", "exp_avg_root_scale"):
            assert torch.isfinite(opt.state[p][name].float()).all()


def test_eight_bit_training_follows_thirty_two(optim):
    """A quadratic bowl: both reach the bottom, which they could not if small changes of the moments were lost."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    goal = torch.randn(4096, device="cuda", generator=gen)
    left = {}
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.zeros(4096, device="cuda"))
        opt = optim.AdamW([p], lr=2e-2, betas=(0.9, 0.999), weight_decay=0.0, state_bits=bits)
        for _ in range(400):
            p.grad = (p.detach() - goal)
            opt.step()
        left[bits] = float((p.detach() - goal).square().mean())
    assert left[32] < 1e-2 and left[8] < 1e-2


# ---- state --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_loaded_runs_go_on_the_same(optim, bits):
    shapes = [(33, 77), (257,), (12, 300)]
    a = _params(shapes)
    kw = dict(**HYPER, state_bits=bits, max_norm=0.05, seed=9)
    x = optim.AdamW(a, **kw)
    grads = [[1e-3 * torch.randn(p.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(100 * k + i))
              for i, p in enumerate(a)] for k in range(5)]

    def go(opt, params, ks):
        for k in ks:
            for p, g in zip(params, grads[k]):
                p.grad = g.clone()
            opt.step()

    go(x, a, (0, 1, 2))
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    y = optim.AdamW(b, **{**kw, "lr": 1.0})
    saved = x.state_dict()
    y.load_state_dict(copy.deepcopy(saved))
    c, z = copy.deepcopy((a, x))
    go(x, a, (3, 4))
    go(y, b, (3, 4))
    go(z, c, (3, 4))
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, r)
        for name, t in x.state[p].items():
            if name not in ("step", "layout"):
                assert torch.equal(t.view(torch.uint8), y.state[q][name].view(torch.uint8))
    assert y.state[b[0]]["step"] == 5 and y.param_groups[0]["lr"] == HYPER["lr"]
    flat = x.flat_state()[0]
    assert flat["exp_avg"].data_ptr() == x.state[a[0]]["exp_avg"].data_ptr()
    assert flat["exp_avg"].numel() == sum(-(-p.numel() // BLOCK) * BLOCK for p in a)
    # a parameter that joins later
    late = torch.nn.Parameter(torch.ones(10, device="cuda"))
    late.grad = torch.ones_like(late)
    x.add_param_group(dict(params=[late]))
    x.step()
    assert len(x.flat_state()) == 2 and x.state[late]["step"] == 1


def test_state_of_torchs_adamw_loads(optim):
    a, b = _params(ODD), _params(ODD)
    theirs = torch.optim.AdamW(a, **HYPER)
    theirs.step()
    mine = optim.AdamW(b, **HYPER)
    mine.load_state_dict(theirs.state_dict())
    for p, q in zip(a, b):
        q.data.copy_(p)
        assert torch.equal(mine.state[q]["exp_avg"], theirs.state[p]["exp_avg"]) and mine.state[q]["step"] == 1
    mine.step()
    theirs.step()
    for p, q in zip(a, b):
        assert (p - q).abs().max() <= 2.0 ** -22 * q.abs().max() + 3e-3 * 45 * 2.0 ** -20
    with pytest.raises(ValueError, match="8-bit"):
        optim.AdamW(b, **HYPER, state_bits=8).load_state_dict(theirs.state_dict())
    with pytest.raises(ValueError, match="amsgrad"):
        mine.load_state_dict(torch.optim.AdamW(a, **HYPER, amsgrad=True).state_dict())


def test_steps_are_the_same_every_time_and_on_another_stream(optim):
    def go(stream):
        with torch.cuda.stream(stream):
            params = _params(ODD, seed=4)
            opt = optim.AdamW(params, **HYPER, state_bits=8, max_norm=0.01, seed=3)
            for _ in range(3):
                opt.step()
        stream.synchronize()
        return params

    a, b = go(torch.cuda.current_stream()), go(torch.cuda.Stream())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_schedulers_and_closures(optim):
    p = _params([(64,)])[0]
    opt = optim.AdamW([p], **HYPER)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5 ** k)
    w = p.detach().clone()
    assert opt.step(lambda: torch.tensor(3.0)) == 3.0
    assert torch.equal(p.detach(), _operations(w, p.grad, 0 * w, 0 * w, 1, 3e-3, 0.9, 0.95, 1e-8, 0.1)[0])
    sched.step()
    w, m, v = p.detach().clone(), opt.state[p]["exp_avg"].clone(), opt.state[p]["exp_avg_sq"].clone()
    opt.step()
    assert torch.equal(p.detach(), _operations(w, p.grad, m, v, 2, 1.5e-3, 0.9, 0.95, 1e-8, 0.1)[0])


# ---- refusals -----------------------------------------------------------------------------------------------------------
def test_refusals(optim):
    from nvfp4_sm120_b200._lib import NVFP4Error
    p = _params([(64,)])[0]
    half = torch.nn.Parameter(torch.ones(8, device="cuda", dtype=torch.float16))
    half.grad = torch.ones_like(half)
    with pytest.raises(ValueError, match="fp32 or bf16"):
        optim.AdamW([half]).step()
    gaps = torch.nn.Parameter(torch.ones(8, 8, device="cuda")[:, :4])
    gaps.grad = torch.ones_like(gaps)
    with pytest.raises(ValueError, match="gaps"):
        optim.AdamW([gaps]).step()
    table = torch.nn.Parameter(torch.ones(8, 8, device="cuda"))
    table.grad = torch.ones(8, 8, device="cuda").to_sparse()
    with pytest.raises(ValueError, match="sparse"):
        optim.AdamW([table]).step()
    with pytest.raises(ValueError, match="max_norm"):
        optim.AdamW([p]).step(grad_norm=torch.ones((), device="cuda"))
    opt = optim.AdamW([p], max_norm=1.0)
    with pytest.raises(NVFP4Error):
        opt.step(grad_norm=torch.ones(()))
    with pytest.raises(ValueError, match="one fp32"):
        opt.step(grad_norm=torch.ones(2, device="cuda"))
    opt.step()
    opt.state[p]["exp_avg"] = torch.zeros(63, device="cuda")
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()
    assert opt.state[p]["step"] == 1
    opt = optim.AdamW([p])
    opt.step()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    w = p.detach().clone()
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            with pytest.raises(NVFP4Error, match="captured"):
                opt.step()
        finally:
            graph.capture_end()
    assert torch.equal(p.detach(), w)


def test_more_elements_than_32_bits_count(optim):
    n = 2 ** 31 + 300
    p = torch.nn.Parameter(torch.ones(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    ends = torch.tensor([0, 255, 256, n // 2, n - 301, n - 45, n - 1], device="cuda")
    p.grad[ends] = 2.0
    opt = optim.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8, max_norm=1e9)
    opt.step()
    # sign of the gradient at the first step, within the roundings of the update and of bf16 (0.5 is a bf16 number)
    assert ((p.detach()[ends].float() - 0.5).abs() <= 2.0 ** -8).all()
    assert int((p.detach() != 1).sum()) == len(ends)
    assert abs(float(opt.grad_norm) - 2 * math.sqrt(len(ends))) <= 1e-6 * 2 * math.sqrt(len(ends))
    st = opt.state[p]
    codes = st["exp_avg"].view(torch.uint8)
    assert int((codes != 0).sum()) == len(ends) and codes.numel() == -(-n // BLOCK) * BLOCK
    del p, opt, st, codes
    torch.cuda.empty_cache()


def test_reordered_parameters_are_noticed(optim):
    for bits in (8, 32):
        p = torch.nn.Parameter(torch.ones(4, 6, 5, 3, device="cuda"))
        p.grad = torch.ones_like(p)
        opt = optim.AdamW([p], state_bits=bits)
        opt.step()
        saved = opt.state_dict()
        p.data = p.data.to(memory_format=torch.channels_last)
        p.grad = torch.ones_like(p)
        w = p.detach().clone()
        with pytest.raises(ValueError, match="strides"):
            opt.step()
        assert torch.equal(p.detach(), w) and opt.state[p]["step"] == 1
        other = optim.AdamW([p], state_bits=bits)
        if bits == 8:
            with pytest.raises(ValueError, match="order"):
                other.load_state_dict(saved)
        else:
            other.load_state_dict(saved)               # element by element
            assert torch.equal(other.state[p]["exp_avg"], opt.state[p]["exp_avg"])


@pytest.mark.parametrize("bits", [32, 8])
def test_state_saved_to_a_file_loads_on_any_device(optim, bits, tmp_path):
    a = _params([(33, 77), (257,), (5,)])
    x = optim.AdamW(a, **HYPER, state_bits=bits)
    x.step()
    torch.save(x.state_dict(), tmp_path / "state.pt")
    saved = torch.load(tmp_path / "state.pt", map_location="cpu", weights_only=False)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    y = optim.AdamW(b, **HYPER, state_bits=bits)
    y.load_state_dict(saved)
    x.step()
    y.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # what does not fit is refused before anything is touched
    c = _params([(33, 78), (257,), (5,)])
    z = optim.AdamW(c, **HYPER, state_bits=bits)
    z.step()
    before = z.state[c[1]]["exp_avg"]
    with pytest.raises(ValueError):
        z.load_state_dict(saved)
    assert z.state[c[1]]["exp_avg"] is before and z.state[c[0]]["step"] == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_capture_leaves_no_state(optim, bits):
    """The first step would make the state, in memory that belongs to the graph."""
    from nvfp4_sm120_b200._lib import NVFP4Error
    p, q = _params([(64, 3)]), _params([(64, 3)])
    for a, b in zip(p, q):
        b.data.copy_(a.data)
        b.grad.copy_(a.grad)
    opt, plain = (optim.AdamW(x, max_norm=1.0, state_bits=bits) for x in (p, q))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            with pytest.raises(NVFP4Error, match="captured"):
                opt.step()
        finally:
            graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    assert not opt.state and not opt.flat_state()
    opt.step()
    plain.step()
    assert torch.equal(p[0], q[0])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("large", [1000, 6_500_003])
def test_the_norm_is_the_same_wherever_it_is_found(optim, bits, large):
    """Both dtypes and more tensors than a launch takes: every launch clips by the norm of all gradients."""
    sets = []
    for _ in range(2):
        sets.append(_params([(large,), (large + 5, 2)] + [(37,)] * 420) + _params([(large // 7,), (300,)], torch.bfloat16, 1))
    p, q = sets
    norm = optim.grad_norm(q)
    limit = 0.37 * float(norm)
    ours, given = (optim.AdamW(x, max_norm=limit, state_bits=bits, **HYPER) for x in (p, q))
    ours.step()
    given.step(grad_norm=norm)
    assert torch.equal(ours.grad_norm, norm)
    # (one rounding of the norm is two of them in its square; the sums are in 64 bits)
    assert abs(float(norm) ** 2 - sum(float(x.grad.double().square().sum()) for x in q)) <= 3 * 2.0 ** -24 * float(norm) ** 2
    for a, b in zip(p, q):
        assert torch.equal(a, b)
        for name in ours.state[a]:
            x, y = ours.state[a][name], given.state[b][name]
            assert x == y if not isinstance(x, torch.Tensor) else torch.equal(x.view(torch.uint8), y.view(torch.uint8))
