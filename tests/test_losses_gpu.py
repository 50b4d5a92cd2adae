"""Losses on logits (csrc/logprob.cu, losses.py) against their formulas in 64 bits, and their gradients against the
formulas' and against differences: sizes around the row kernels' borders, strides, masks, values that are no numbers."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

IGNORE = -100
U = 2.0 ** -24                                     # half a step of fp32


@pytest.fixture(scope="module")
def losses():
    from nvfp4_sm120_b200 import losses as module
    return module


def _logits(shape, dtype, seed, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, device="cuda", generator=gen)).to(dtype)


def _labels(shape, vocab, seed, masked=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed + 1000)
    y = torch.randint(0, vocab, shape, device="cuda", generator=gen)
    y[torch.rand(shape, device="cuda", generator=gen) < masked] = IGNORE
    return y


def _reference(x, y):
    """(log-probabilities, logsumexp) in 64 bits."""
    lse = torch.logsumexp(x.double(), -1)
    lp = x.double().gather(-1, y.clamp(min=0)[..., None])[..., 0] - lse
    return torch.where(y == IGNORE, 0.0, lp), lse


def _gradient(x, y, w):
    """w (onehot - softmax) in 64 bits; w: dloss / dlogp."""
    w = torch.where(y == IGNORE, 0.0, w.double())[..., None]
    d = -w * torch.softmax(x.double(), -1)
    return d.scatter_add(-1, y.clamp(min=0)[..., None], w)


def _lse_error(x):
    """Bound on the error of a row's logsumexp in fp32: the exponents are off by 3 roundings of at most the row's span,
    ex2 by 2^-22 and its flush to zero by 2^-126 a term; a thread adds at most vocab / 32 terms and joins 15 times;
    logf 2 ulp of at most ln(vocab), one rounding for its sum with the maximum."""
    vocab = x.shape[-1]
    top, low = x.double().amax(-1), x.double().amin(-1)
    rel = 3 * 1.45 * (top - low).clamp(max=100) * U + 2.0 ** -22 + (vocab / 32 + 15 * 4) * U
    return rel + 4 * U * math.log(max(vocab, 2)) + U * (top.abs() + math.log(vocab) + 1)


def _check_logp(got, x, y):
    want, _ = _reference(x, y)
    tol = _lse_error(x) + U * want.abs()
    assert got.dtype == torch.float32 and got.shape == y.shape
    assert ((got.double() - want).abs() <= tol).all()
    assert (got[y == IGNORE] == 0).all()


def _check_grad(got, x, y, w, w_error=0.0):
    """w_error: relative error that w itself may have."""
    want = _gradient(x, y, w)
    assert got.dtype == x.dtype and got.shape == x.shape
    _, lse = _reference(x, y)
    far = (x.double() - lse[..., None]).abs().clamp(max=150)
    rel = _lse_error(x)[..., None] + 4 * 1.45 * U * far + 2.0 ** -22 + 3 * U + w_error
    p = torch.softmax(x.double(), -1)
    w = torch.where(y == IGNORE, 0.0, w.double()).abs()[..., None]
    hot = torch.zeros_like(p).scatter_(-1, y.clamp(min=0)[..., None], 1.0)
    tol = w * (p * rel + hot * (w_error + 2 * U)) + torch.finfo(x.dtype).eps / 2 * want.abs() * 1.001 + 2.0 ** -126 * (1 + w)
    assert ((got.double() - want).abs() <= tol).all()


VOCABS = [1, 2, 7, 13, 64, 257, 2047, 2048, 2049, 5003, 50257, 131073]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprobs_and_gradient(losses, vocab, dtype):
    for shape in ((1, 1), (3, 5), (2, 37)):
        x = _logits((*shape, vocab), dtype, vocab + shape[1]).requires_grad_(True)
        y = _labels(shape, vocab, vocab)
        lp = losses.token_logprobs(x, y)
        _check_logp(lp.detach(), x.detach(), y)
        w = _logits(shape, torch.float32, 5)
        (g,) = torch.autograd.grad(lp, x, w)
        _check_grad(g, x.detach(), y, w)
        with torch.no_grad():
            assert torch.equal(losses.token_logprobs(x, y), lp)


def test_many_rows(losses):
    """More rows than the grid has groups, of a warp and of a CTA."""
    for rows, vocab in ((20011, 13), (2500, 2051)):
        x = _logits((rows, vocab), torch.bfloat16, 1).requires_grad_(True)
        y = _labels((rows,), vocab, 2)
        lp = losses.token_logprobs(x, y)
        _check_logp(lp.detach(), x.detach(), y)
        w = _logits((rows,), torch.float32, 3)
        (g,) = torch.autograd.grad(lp, x, w)
        _check_grad(g, x.detach(), y, w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [13, 5003])
def test_strides(losses, dtype, vocab):
    base = _logits((4, 9, vocab + 3), dtype, 8)
    views = {"shifted": base[:, :-1, :vocab], "offset": base[:, :, 1:vocab + 1], "time first": base.transpose(0, 1)[..., :vocab],
             "expanded": base[:1, :, :vocab].expand(4, 9, vocab), "vocab first": _logits((vocab, 4, 9), dtype, 9).permute(1, 2, 0),
             "rows": base[0, ::2, 2:vocab + 2]}
    for name, x in views.items():
        y = _labels(x.shape[:-1], vocab, 4)
        x = x.detach().requires_grad_(True)
        lp = losses.token_logprobs(x, y)
        _check_logp(lp.detach(), x.detach(), y)
        w = _logits(y.shape, torch.float32, 3)
        (g,) = torch.autograd.grad(lp, x, w)
        _check_grad(g, x.detach(), y, w)
        yt = y.t().contiguous().t() if y.dim() == 2 else y
        for other in (yt, y.int()):
            assert torch.equal(losses.token_logprobs(x, other), lp), name


def test_gradient_against_differences(losses):
    """d(sum of w lp) along random directions, by central differences in 64 bits of the formula and by the kernel's gradient."""
    x = _logits((2, 6, 301), torch.float32, 11).requires_grad_(True)
    y, w = _labels((2, 6), 301, 3), _logits((2, 6), torch.float32, 4)
    (g,) = torch.autograd.grad(losses.token_logprobs(x, y), x, w)
    for k in range(8):
        d = _logits(x.shape, torch.float64, 20 + k, 1.0)
        f = lambda h: float((_reference(x.detach().double() + h * d, y)[0] * w.double()).sum())
        slope = (f(1e-4) - f(-1e-4)) / 2e-4
        assert abs(float((g.double() * d).sum()) - slope) <= 1e-5 * float((g.double().abs() * d.abs()).sum()) + 1e-6


# ---- masks and values ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [13, 2049])
def test_masked_logits(losses, dtype, vocab):
    x = _logits((6, vocab), dtype, 5)
    y = torch.full((6,), 3, device="cuda")
    low = torch.finfo(dtype).min
    x[0, 5:] = -math.inf                               # most of the vocabulary masked
    x[1, :] = low                                      # the type's lowest value everywhere
    x[2, 5:] = low
    x[3, :] = -math.inf
    x[3, 3] = 2.0                                      # one token left
    x[4, :] = torch.finfo(dtype).max
    x[5, 3] = -math.inf                                # the label itself
    x.requires_grad_(True)
    out = losses.token_logprobs(x, y)
    lp = out.detach()
    want, _ = _reference(x.detach(), y)
    tol = 2.0 ** -20
    assert abs(float(lp[0]) - float(want[0])) < tol and abs(float(lp[2]) - float(want[2])) < tol
    # the rows of one huge value: log(vocab) is lost beside it in the rounding of the logsumexp, as in any fp32 sum
    assert float(lp[1]) == 0.0 and float(lp[4]) == 0.0 and float(lp[3]) == 0.0 and float(lp[5]) == -math.inf
    (g,) = torch.autograd.grad(out[[0, 2, 3]].sum(), x)
    assert torch.isfinite(g).all() and (g[0, 5:] == 0).all() and (g[2, 5:] == 0).all() and (g[3] == 0).all()
    assert (g[[1, 4, 5]] == 0).all()                   # nothing was asked of these


@pytest.mark.parametrize("vocab", [13, 2049])
def test_what_is_no_number_shows_in_its_row_only(losses, vocab):
    x = _logits((5, vocab), torch.float32, 5)
    y = torch.full((5,), 3, device="cuda")
    x[0, 7] = math.nan
    x[1, 7] = math.inf
    x[2, :] = -math.inf
    y[3] = vocab                                       # no index
    x.requires_grad_(True)
    lp = losses.token_logprobs(x, y)
    assert torch.isnan(lp[:4]).all() and torch.isfinite(lp[4])
    (g,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    assert torch.isnan(g[:4]).any(1).all() and torch.isfinite(g[4]).all()
    for bad in (-1, 2 ** 40, -2 ** 62):
        y[3] = bad
        assert torch.isnan(losses.token_logprobs(x, y)[3])
    y[:4] = IGNORE                                     # ignored rows are not looked at
    lp = losses.token_logprobs(x, y)
    (g,) = torch.autograd.grad(lp.sum(), x)
    assert (lp[:4] == 0).all() and (g[:4] == 0).all() and torch.isfinite(g).all()
    assert torch.equal(losses.token_logprobs(x, torch.where(y == IGNORE, 7, y), ignore_index=7), lp)


# ---- preference loss ----------------------------------------------------------------------------------------------------
def _preference(x, y, ref, beta, smooth):
    lp = _reference(x, y)[0].sum(1)
    r = beta * (lp - ref.double())
    c, j = r.chunk(2)
    f = torch.nn.functional.logsigmoid
    return (-(1 - smooth) * f(c - j) - smooth * f(j - c)).mean(), c, j, lp


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pairs,seq,vocab", [(1, 1, 13), (3, 5, 13), (40, 12, 13), (2, 300, 257), (3, 33, 2051), (1, 9, 50257)])
@pytest.mark.parametrize("smooth", [0.0, 0.1])
def test_preference(losses, dtype, pairs, seq, vocab, smooth):
    x = _logits((2 * pairs, seq, vocab), dtype, pairs + seq)
    y = _labels((2 * pairs, seq), vocab, 1)
    y[0] = IGNORE                                      # a sequence without a token
    ref = (_reference(x, y)[0].sum(1) + 5 * torch.randn(2 * pairs, device="cuda", dtype=torch.float64,
                                                        generator=torch.Generator(device="cuda").manual_seed(seq))).float()
    x.requires_grad_(True)
    loss, chosen, rejected = losses.preference_loss(x, y, ref, beta=0.3, label_smoothing=smooth)
    leaf = x.detach().double().requires_grad_(True)
    want, c, j, lp = _preference(leaf, y, ref, 0.3, smooth)
    err = 0.3 * ((_lse_error(x.detach()) * (y != IGNORE)).sum(1) + seq * U * 20 + U * lp.detach().abs())
    both = torch.cat((c, j)).detach()
    assert ((torch.cat((chosen, rejected)).double() - both).abs() <= err + U * both.abs()).all()
    assert abs(loss.item() - want.item()) <= float(err.max()) * 2 + 2 * U * abs(want.item())
    assert not chosen.requires_grad and loss.shape == ()
    (g,) = torch.autograd.grad(loss, x)
    # dloss / dL_i = +- beta / pairs s(h), whose error is that of h
    h = (c - j).detach()
    w = 0.3 / pairs * (smooth * torch.sigmoid(h) - (1 - smooth) * torch.sigmoid(-h))
    w = -torch.cat((w, -w))
    (exact,) = torch.autograd.grad(want, leaf)
    assert torch.allclose(_gradient(x.detach(), y, -w[:, None].expand_as(y)), exact, rtol=1e-9, atol=1e-15)
    off = float(err.max()) * 2 * 0.3 / pairs / float(w.abs().min()) + 4 * U
    _check_grad(g, x.detach(), y, -w[:, None].expand_as(y), off)


def test_preference_far_margins(losses):
    """Margins of hundreds: the loss is linear on one side and 0 on the other, its gradient beta or 0."""
    y = torch.full((2, 1), 0, device="cuda")
    x = torch.zeros(2, 1, 2, device="cuda", requires_grad=True)
    for far, want in ((500.0, 0.0), (-500.0, 500.0)):
        ref = torch.tensor([-far, 0.0], device="cuda")
        loss, _, _ = losses.preference_loss(x, y, ref, beta=1.0)
        (g,) = torch.autograd.grad(loss, x)
        assert abs(loss.item() - want) <= 1e-4 and torch.isfinite(g).all()
        assert abs(float(g[0, 0, 0]) - (0.0 if far > 0 else -0.5)) < 1e-6 and abs(float(g[1, 0, 0]) + float(g[0, 0, 0])) < 1e-6
    x = torch.full((2, 1, 2), math.nan, device="cuda", requires_grad=True)
    assert math.isnan(float(losses.preference_loss(x, y, torch.zeros(2, device="cuda"))[0]))


# ---- policy loss --------------------------------------------------------------------------------------------------------
def _policy(lp, y, old, adv, ref, lo, hi, kl):
    live = y != IGNORE
    n = max(1, int(live.sum()))
    a = adv.double() if adv.dim() == lp.dim() else adv.double()[:, None]
    rho = torch.exp(lp - old.double())
    kept = torch.minimum(rho * a, rho.clamp(1 - lo, 1 + hi) * a)
    k = torch.zeros_like(lp)
    if ref is not None:
        d = ref.double() - lp
        k = torch.expm1(d) - d
    return (torch.where(live, kl * k - kept, 0.0).sum() / n, torch.where(live, k, 0.0).sum() / n,
            (live & (rho * a > kept)).sum() / n, rho)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,seq,vocab", [(1, 1, 13), (3, 5, 1), (64, 12, 13), (2, 300, 257), (3, 33, 2051), (2, 9, 50257)])
@pytest.mark.parametrize("form", ["plain", "kl", "token"])
def test_policy(losses, dtype, batch, seq, vocab, form):
    gen = torch.Generator(device="cuda").manual_seed(batch + seq)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=gen)
    x, y = _logits((batch, seq, vocab), dtype, batch), _labels((batch, seq), vocab, 1)
    lp, _ = _reference(x, y)
    # ratios on both sides of both borders, none within a rounding of one
    old = (lp - torch.where(rand(batch, seq) < 0.5, 0.15, 0.6) * (2 * rand(batch, seq).round() - 1) * (0.9 + 0.1 * rand(batch, seq))).float()
    adv = torch.randn(batch, seq, device="cuda", generator=gen) if form == "token" else torch.randn(batch, device="cuda", generator=gen)
    ref = None if form == "plain" else (lp + 0.3 * rand(batch, seq)).float()
    kw = dict(clip=0.2, clip_high=0.3, kl_coef=0.0 if form == "plain" else 0.05)
    x.requires_grad_(True)
    loss, stats = losses.policy_loss(x, y, old, adv, ref, **kw)
    leaf = lp.clone().requires_grad_(True)
    want, k, cut, rho = _policy(leaf, y, old, adv, ref, 0.2, 0.3, kw["kl_coef"])
    (w,) = torch.autograd.grad(want, leaf)
    _check_logp(stats["logps"], x.detach(), y)
    err = _lse_error(x.detach()).max() + U * float(lp.abs().max()) + 4 * U * (float(old.abs().max()) + 1)
    top = float(adv.abs().max()) * float(rho.max()) + 1
    assert abs(loss.item() - want.item()) <= float(err) * top * 2 + 8 * U * top
    assert abs(float(stats["kl"]) - float(k)) <= float(err) + 8 * U
    assert abs(float(stats["clip_fraction"]) - float(cut)) <= U
    (g,) = torch.autograd.grad(loss, x, retain_graph=True)
    # w = -rho A + kl (1 - exp d), each with the relative error that its exponent's absolute one gives
    n = max(1, int((y != IGNORE).sum()))
    parts = (rho.detach() * (adv if form == "token" else adv[:, None])).abs() + kw["kl_coef"] * (1 if ref is None else (ref - lp).exp())
    off = (float(err) * 1.5 + 8 * U) * parts / n
    want_g = _gradient(x.detach(), y, w)
    p = torch.softmax(x.detach().double(), -1)
    _check_grad_with(g, x.detach(), y, w, off, want_g, p)
    # a factor in front of the loss, a second backward, both
    (g3,) = torch.autograd.grad(3.0 * loss, x, retain_graph=True)
    _check_grad_with(g3, x.detach(), y, 3 * w, 3 * off + 3 * w.abs() * U, 3 * want_g, p)
    (again,) = torch.autograd.grad(loss, x)
    assert torch.equal(again, g)
    loss2, _ = losses.policy_loss(x, y, old, adv, ref, **kw)
    (h3,) = torch.autograd.grad(3.0 * loss2, x)
    assert torch.equal(h3, g3)
    with torch.no_grad():
        assert torch.equal(losses.policy_loss(x, y, old, adv, ref, **kw)[0], loss)


def _check_grad_with(got, x, y, w, w_off, want, p):
    """_check_grad with an absolute error of w."""
    _, lse = _reference(x, y)
    far = (x.double() - lse[..., None]).abs().clamp(max=150)
    rel = _lse_error(x)[..., None] + 4 * 1.45 * U * far + 2.0 ** -22 + 3 * U
    hot = torch.zeros_like(p).scatter_(-1, y.clamp(min=0)[..., None], 1.0)
    live = (y != IGNORE)[..., None]
    w, w_off = w.abs()[..., None], w_off[..., None]
    tol = live * (w * (p * rel + hot * 2 * U) + w_off * (p + hot)) + torch.finfo(x.dtype).eps / 2 * want.abs() * 1.01 + 2.0 ** -126 * (1 + w)
    assert ((got.double() - want).abs() <= tol).all()


def test_policy_without_any_token(losses):
    x = _logits((2, 3, 13), torch.float32, 1).requires_grad_(True)
    y = torch.full((2, 3), IGNORE, device="cuda")
    loss, stats = losses.policy_loss(x, y, torch.zeros(2, 3, device="cuda"), torch.ones(2, device="cuda"))
    (g,) = torch.autograd.grad(loss, x)
    assert float(loss) == 0.0 and (g == 0).all() and float(stats["clip_fraction"]) == 0.0


def test_policy_values_that_are_no_numbers_show(losses):
    x = _logits((2, 3, 13), torch.float32, 1).requires_grad_(True)
    y = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    for old, adv in ((math.nan, 1.0), (0.0, math.nan)):
        loss, _ = losses.policy_loss(x, y, torch.full((2, 3), old, device="cuda"), torch.full((2,), adv, device="cuda"))
        (g,) = torch.autograd.grad(loss, x)
        assert math.isnan(float(loss)) and torch.isnan(g).any()


# ---- use ----------------------------------------------------------------------------------------------------------------
def test_gradient_reaches_what_made_the_logits(losses):
    """Logits that a linear head makes under autocast, the shifted view of them, a loss divided for accumulation."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    head = torch.nn.Linear(32, 77, bias=False, device="cuda")
    h = torch.randn(4, 9, 32, device="cuda", generator=gen)
    y, ref = _labels((4, 8), 77, 3), torch.zeros(4, device="cuda")
    grads = []
    for plain in (False, True):
        head.weight.grad = None
        with torch.autocast("cuda", dtype=torch.bfloat16):
            x = head(h)[:, :-1]
        if plain:
            c, j = (0.1 * (torch.where(y == IGNORE, 0.0, x.double().log_softmax(-1).gather(-1, y.clamp(min=0)[..., None])[..., 0]).sum(1) - ref)).chunk(2)
            loss = -torch.nn.functional.logsigmoid(c - j).mean()
        else:
            loss = losses.preference_loss(x, y, ref)[0]
        (loss / 4).backward()
        grads.append(head.weight.grad.double())
    # the gradients of the logits are the same numbers rounded to bf16 once; a few land on the other side
    assert ((grads[0] - grads[1]).norm() <= 2.0 ** -8 * grads[1].norm())


def test_capture_replay_and_streams(losses):
    x = _logits((4, 12, 2051), torch.bfloat16, 1).requires_grad_(True)
    y = _labels((4, 12), 2051, 2)
    old, adv, ref = _reference(x.detach(), y)[0].float() - 0.1, torch.randn(4, device="cuda"), torch.zeros(4, 12, device="cuda")

    def all_three():
        lp = losses.token_logprobs(x, y)
        a = torch.autograd.grad(lp.sum(), x)
        b = losses.preference_loss(x, y, lp.detach().sum(1) * 0.9)
        c = losses.policy_loss(x, y, old, adv, ref, kl_coef=0.1)
        return [lp, *a, b[0], *torch.autograd.grad(b[0], x), c[0], *torch.autograd.grad(c[0] / 3, x)]

    want = [t.detach().clone() for t in all_three()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_three()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(all_three())
        graphs.append(g)
    with torch.no_grad():
        x.mul_(-1)
    new = [t.detach().clone() for t in all_three()]
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):                                   # both graphs at once: they share nothing
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, new))
    assert not torch.equal(new[0], want[0])


def test_argument_checks(losses):
    from nvfp4_sm120_b200._lib import NVFP4Error
    x, y = _logits((4, 3, 13), torch.float32, 1), _labels((4, 3), 13, 1)
    cu = lambda *s: torch.zeros(*s, device="cuda")
    for call in (lambda: losses.preference_loss(x[:3], y[:3], cu(3)), lambda: losses.preference_loss(x, y, cu(2)),
                 lambda: losses.preference_loss(x[0], y[0], cu(2)), lambda: losses.policy_loss(x, y, cu(4, 2), cu(4)),
                 lambda: losses.policy_loss(x, y, cu(4, 3), cu(3)), lambda: losses.policy_loss(x, y, cu(4, 3), cu(4), cu(4))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: losses.token_logprobs(x, y.cpu()), lambda: losses.preference_loss(x, y, torch.zeros(4)),
                 lambda: losses.policy_loss(x, y, torch.zeros(4, 3), cu(4))):
        with pytest.raises(NVFP4Error):
            call()
    x.requires_grad_(True)
    lp = losses.token_logprobs(x, y)
    (g,) = torch.autograd.grad(lp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):                    # no second derivative
        g.sum().backward()


def test_more_logits_than_32_bits_count(losses):
    rows, vocab = 42800, 50257                           # 2^31 + 3.5 million
    assert rows * vocab > 2 ** 31
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 17, rows // 2, rows - 2, rows - 1], device="cuda")
    x[some] = _logits((5, vocab), torch.bfloat16, 7)
    x.requires_grad_(True)
    y = torch.full((rows,), IGNORE, device="cuda")
    y[some] = torch.tensor([0, 5, vocab - 1, 9, vocab - 1], device="cuda")
    lp = losses.token_logprobs(x, y)
    part = x.detach()[some]
    _check_logp(lp.detach()[some], part, y[some])
    w = torch.randn(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    (g,) = torch.autograd.grad(lp, x, w)
    _check_grad(g[some], part, y[some], w[some])
    assert torch.count_nonzero(g[1:17]) == 0 and torch.count_nonzero(g[rows - 100:rows - 2]) == 0


def test_gradients_lie_as_their_logits_do(losses):
    """Shifted and offset views: the gradient has the view's strides, its neighbours in memory belong to nobody."""
    base = _logits((3, 8, 2051), torch.bfloat16, 3)
    for x in (base[:, :-1], base[:, 1:], base[:, :, 1:], base[:1, :, :7], base[:, :1], base.transpose(0, 1)):
        x = x.detach().requires_grad_(True)
        y = _labels(x.shape[:-1], x.shape[-1], 5)
        w = _logits(y.shape, torch.float32, 6)
        (g,) = torch.autograd.grad(losses.token_logprobs(x, y), x, w)
        _check_grad(g, x.detach(), y, w)
        c = x.detach().contiguous().requires_grad_(True)
        (h,) = torch.autograd.grad(losses.token_logprobs(c, y), c, w)
        assert torch.allclose(g.float(), h.float(), rtol=2.0 ** -7, atol=1e-30)
    # through the view, into the whole tensor
    base = base.requires_grad_(True)
    y = _labels((3, 7), 2051, 5)
    losses.token_logprobs(base[:, :-1], y).sum().backward()
    assert torch.count_nonzero(base.grad[:, -1]) == 0 and torch.isfinite(base.grad).all()


def test_inference_mode(losses):
    with torch.inference_mode():
        x, y = _logits((2, 3, 50), torch.float32, 1), _labels((2, 3), 50, 2, 0.0)
        lp = losses.token_logprobs(x, y)
        loss, chosen, _ = losses.preference_loss(x, y, lp.sum(1))
        # the sums in fp32 here, in 64 bits there: three roundings of some ten
        assert abs(loss.item() - math.log(2)) <= 1e-5 and abs(chosen.item()) <= 1e-5
        loss, stats = losses.policy_loss(x, y, lp, torch.ones(2, device="cuda"))
        assert abs(loss.item() + 1) <= 4 * U and stats["clip_fraction"].item() == 0.0


@pytest.mark.parametrize("rows,vocab,dtype", [(4100, 7001, torch.bfloat16), (600, 7001, torch.bfloat16), (600, 20011, torch.bfloat16),
                                              (600, 40009, torch.float32), (30, 5003, torch.bfloat16), (30, 40009, torch.float32)])
def test_every_number_of_threads_a_row(losses, rows, vocab, dtype):
    """Warps, and CTAs of 128, 256 and 512 threads, for many rows and for few."""
    x, y = _logits((rows, vocab), dtype, rows), _labels((rows,), vocab, 3)
    lp64, _ = _reference(x, y)
    w = torch.randn(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    x.requires_grad_(True)
    lp = losses.token_logprobs(x, y)
    _check_logp(lp.detach(), x.detach(), y)
    _check_grad(torch.autograd.grad(lp, x, w)[0], x.detach(), y, w)
    # a policy loss whose ratios are 1.1: w = -1.1 A / n, with the error of the exponent on top
    loss, stats = losses.policy_loss(x, y, (lp64 - math.log(1.1)).float(), w)
    _check_logp(stats["logps"], x.detach(), y)
    n = int((y != IGNORE).sum())
    off = float(_lse_error(x.detach()).max()) * 1.5 + 4 * U * (float(lp64.abs().max()) + 4)
    _check_grad(torch.autograd.grad(loss, x)[0], x.detach(), y, -1.1 * w / n, off)


def test_no_gradient_from_behind_gives_none(losses):
    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            return None

    x, y = _logits((2, 3, 17), torch.float32, 1), _labels((2, 3), 17, 1, 0.0)
    old = torch.zeros(2, 3, device="cuda")
    for call in (lambda t: losses.token_logprobs(t, y).sum(), lambda t: losses.preference_loss(t, y, old[:, 0])[0],
                 lambda t: losses.policy_loss(t, y, old, old[:, 0] + 1)[0]):
        t = x.clone().requires_grad_()
        Nothing.apply(call(t)).backward()
        assert t.grad is None or not t.grad.any()
        call(t).backward()
        assert t.grad.any()
