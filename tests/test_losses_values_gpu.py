"""Losses on logits (csrc/logprob.cu, losses.py) at values where a formula that is right for ordinary numbers goes wrong: rows of
one mask value, common offsets, infinite margins, long sums, arguments of other precision or layout."""
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


def _randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=torch.Generator(device="cuda").manual_seed(seed))


def _labels(shape, vocab, seed, masked=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 1000)
    y = torch.randint(0, vocab, shape, device="cuda", generator=gen)
    y[torch.rand(shape, device="cuda", generator=gen) < masked] = IGNORE
    return y


# ---- rows far from zero -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("vocab", [13, 301, 2051, 50257])
@pytest.mark.parametrize("dtype,step,offsets", [(torch.float32, 1 / 16, (1e4, -1e4, 1e6, -1e6)), (torch.bfloat16, 4.0, (512.0, -512.0))])
def test_a_common_offset_changes_nothing(losses, vocab, dtype, step, offsets):
    """Logits on a grid that the offset leaves exact: x - M are the same numbers, and with them every result and gradient."""
    base = step * torch.randint(-40, 41, (4, 6, vocab), device="cuda", generator=torch.Generator(device="cuda").manual_seed(vocab)).float()
    y, adv, w = _labels((4, 6), vocab, 1, 0.2), _randn((4,), 2), _randn((4, 6), 3)

    def results(x):
        x = x.to(dtype).requires_grad_(True)
        lp = losses.token_logprobs(x, y)
        pref = losses.preference_loss(x, y, lp.detach().sum(1) + adv)
        pol = losses.policy_loss(x, y, lp.detach() - 0.05, adv, lp.detach() + 0.1, kl_coef=0.1)
        grads = [torch.autograd.grad(o, x, g)[0] for o, g in ((lp, w), (pref[0], None), (pol[0], None))]
        return [lp, *pref, pol[0], *pol[1].values(), *grads]

    want = results(base)
    for c in offsets:
        assert ((base + c).to(dtype).double() == base.double() + c).all()
        assert all(torch.equal(a, b) for a, b in zip(results(base + c), want))


@pytest.mark.parametrize("vocab", [1, 13, 2049, 50257])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_one_value(losses, dtype, vocab):
    """Every logit the same, the type's lowest value (a row whose mask leaves nothing) to its highest: the softmax is 1 / vocab."""
    info = torch.finfo(dtype)
    values = torch.tensor([info.min, -1e9, -1e4, 0.0, 1e9, info.max], device="cuda")
    x = values[:, None].expand(6, vocab).to(dtype).contiguous().requires_grad_(True)
    y, w = _labels((6,), vocab, 1), _randn((6,), 2)
    log_v = math.log(vocab)
    # the sum is exact; logf 2 steps of at most ln 2, the rest of the logarithm in 64 bits, one rounding of the result
    tol = 2 * U + U * log_v
    lp = losses.token_logprobs(x, y)
    assert (lp.double() + log_v).abs().max() <= tol
    # p: the logarithm's error, its rounding to fp32 in base 2 (times ln 2), ex2.approx 2^-22, two roundings; one to the dtype
    p = 1 / vocab
    rel = 2 * U + U * log_v + 2.0 ** -22 + 2 * U
    hot = torch.zeros(6, vocab, device="cuda", dtype=torch.float64).scatter_(1, y[:, None], 1.0)

    def right(g, w, w_rel=0.0):
        """w_rel: relative error that w itself may have."""
        want = w.double()[:, None] * (hot - p)
        off = w.double().abs()[:, None] * (p * rel + U + w_rel) + info.eps / 2 * 1.001 * want.abs()
        return ((g.double() - want).abs() <= off).all()

    assert right(torch.autograd.grad(lp, x, w)[0], w)
    # ratios of 1 and no KL term: dloss / dlogp = -A times a rounded 1 / 6
    loss, stats = losses.policy_loss(x, y, lp.detach(), w)
    assert torch.equal(stats["logps"], lp)
    assert right(torch.autograd.grad(loss, x)[0], -w / 6, 3 * U)
    # reward margins of 0: dloss / dL = -+ beta / 2 / pairs, and the sigmoid moves by half of itself times the margin's error
    ref = torch.full((6,), -log_v, device="cuda")
    off = 2 * (tol + U * log_v)
    loss, chosen, rejected = losses.preference_loss(x[:, None], y[:, None], ref, beta=1.0)
    assert torch.cat((chosen, rejected)).abs().max() <= off
    half = torch.tensor([-1 / 6] * 3 + [1 / 6] * 3, device="cuda")
    assert right(torch.autograd.grad(loss, x)[0], half, off + 2 * U)
    assert abs(loss.item() - math.log(2)) <= off + U


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [13, 2049])
def test_masked_rows(losses, dtype, vocab):
    """Rows with masked entries, rows whose mask leaves one entry or nothing, a masked label."""
    x = (3 * _randn((6, vocab), 5)).to(dtype)
    y = torch.full((6,), 3, device="cuda")
    low = torch.finfo(dtype).min
    x[0, 5:] = -math.inf
    x[1, :] = low
    x[2, 5:] = low
    x[3, :] = -math.inf
    x[3, 3] = 2.0
    x[4, :] = torch.finfo(dtype).max
    x[5, 3] = -math.inf
    x.requires_grad_(True)
    out = losses.token_logprobs(x, y)
    lp = out.detach()
    want = torch.log_softmax(x.detach()[[0, 2]].double(), 1)[:, 3]
    assert (lp[[0, 2]].double() - want).abs().max() < 2.0 ** -20
    assert (lp[[1, 4]].double() + math.log(vocab)).abs().max() <= 2 * U + U * math.log(vocab)
    assert float(lp[3]) == 0.0 and float(lp[5]) == -math.inf
    (g,) = torch.autograd.grad(out[[0, 2, 3]].sum(), x, retain_graph=True)
    assert torch.isfinite(g).all() and (g[0, 5:] == 0).all() and (g[2, 5:] == 0).all() and (g[3] == 0).all()
    assert (g[[1, 4, 5]] == 0).all()                   # nothing was asked of these
    (g,) = torch.autograd.grad(out[[1, 4]].sum(), x)
    want = torch.nn.functional.one_hot(y[[1, 4]], vocab).double() - 1 / vocab
    assert ((g[[1, 4]].double() - want).abs() <= (torch.finfo(dtype).eps + 2.0 ** -20) * want.abs()).all()


# ---- long sums ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("vocab,spread", [(1000, 2.0), (50257, 4.0), (150000, 4.0)])
def test_rows_of_a_sequence_are_not_off_the_same_way(losses, vocab, spread):
    """Most terms of a wide row are below 2^-24 of its sum, and must not vanish from it: a reward adds up a thousand such rows.
    The mean error of a row, from sequences whose reference is their own sum: ex2.approx is off by 2^-22 at most, the rest are roundings
    without a sign; those of a row are some 4 U (exponents of the few largest terms, three or so, and the logarithm), so the mean of n
    rows lies within five times that over sqrt(n)."""
    n = 640                                          # enough of them that a row gets the fewest threads
    x = spread * _randn((2, n // 2, vocab), vocab)
    y = _labels((2, n // 2), vocab, 1)
    want = torch.stack([torch.log_softmax(s.double(), 1).gather(1, t[:, None]).sum() for s, t in zip(x, y)])
    ref = want.float()
    _, chosen, rejected = losses.preference_loss(x, y, ref, beta=1.0)
    off = (torch.cat((chosen, rejected)).double() + ref.double() - want).sum() / n
    assert abs(float(off)) <= 2.0 ** -22 + 5 * 4 * U / math.sqrt(n)


# ---- infinite margins ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("smooth", [0.0, 0.1, 1.0])
def test_preference_with_an_impossible_token(losses, dtype, smooth):
    """A label whose logit is -inf makes its sequence's sum -inf: in a rejected sequence h = inf, where -logsigmoid(h) is 0, in a chosen
    one h = -inf, where it is inf.  The other pairs count as ever."""
    P, T, V = 3, 5, 17
    y, ref = _labels((2 * P, T), V, 2), _randn((2 * P,), 3) - T * math.log(V)
    for impossible in (P + 1, 1):                      # of the middle pair: the rejected sequence, the chosen one
        x = (0.3 * _randn((2 * P, T, V), 4)).to(dtype)
        x[impossible, 2, y[impossible, 2]] = -math.inf
        x.requires_grad_(True)
        loss, chosen, rejected = losses.preference_loss(x, y, ref, beta=0.5, label_smoothing=smooth)
        L = torch.log_softmax(x.detach().double(), 2).gather(2, y[..., None])[..., 0].sum(1)
        c, r = (0.5 * (L - ref.double())).chunk(2)
        h = c - r
        softplus = lambda t: torch.nn.functional.softplus(t.double())
        terms = torch.zeros_like(h)
        if smooth < 1:
            terms += (1 - smooth) * softplus(-h)
        if smooth > 0:
            terms += smooth * softplus(h)
        want = terms.mean().item()
        assert torch.equal(torch.isinf(torch.cat((chosen, rejected))), torch.isinf(torch.cat((c, r))))
        # five log-probabilities of some 3, their rewards, the loss: a few dozen roundings
        assert loss.item() == want if math.isinf(want) else abs(loss.item() - want) <= 64 * U * (1 + want)
        (g,) = torch.autograd.grad(loss, x)
        assert torch.isfinite(g).all()
        # dloss / dL: beta / P (s sigmoid(h) - (1 - s) sigmoid(-h)), 0 or a constant where h is infinite
        w = 0.5 / P * (smooth * torch.sigmoid(h) - (1 - smooth) * torch.sigmoid(-h))
        w = torch.cat((w, -w))[:, None, None]
        hot = torch.nn.functional.one_hot(y, V).double()
        exact = w * (hot - torch.softmax(x.detach().double(), 2))
        assert ((g.double() - exact).abs() <= (torch.finfo(dtype).eps / 2 + 64 * U) * exact.abs() + 64 * U * w.abs()).all()


# ---- a reference that is only looked at ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reference_without_a_coefficient_leaves_the_loss_alone(losses, dtype):
    """kl_coef 0: `kl` is measured, and the loss and its gradient are those of a call without a reference, however far that lies."""
    x = (2 * _randn((3, 4, 19), 1)).to(dtype).requires_grad_(True)
    y, adv = _labels((3, 4), 19, 2, 0.2), _randn((3,), 3)
    y[0, 0] = 3
    lp = losses.token_logprobs(x, y).detach()
    old = lp - 0.1
    plain, without = losses.policy_loss(x, y, old, adv)
    (g,) = torch.autograd.grad(plain, x)
    for far, kl in ((0.3, math.exp(0.3) - 1.3), (200.0, math.inf), (math.inf, math.inf)):
        loss, stats = losses.policy_loss(x, y, old, adv, lp + far)
        (h,) = torch.autograd.grad(loss, x)
        assert torch.equal(loss, plain) and torch.equal(h, g) and torch.equal(stats["clip_fraction"], without["clip_fraction"])
        # ref - logp is off by a rounding of ref, some 2^-21, and its term by that times exp(0.3) - 1
        assert float(stats["kl"]) == kl if math.isinf(kl) else abs(float(stats["kl"]) - kl) <= 2.0 ** -21


# ---- references in 64 bits ----------------------------------------------------------------------------------------------
def test_reference_sums_keep_their_precision(losses):
    """The reference of sequences of thousands of nats, in 64 bits: rewards are the small differences they are made of."""
    x = 2 * _randn((4, 1500, 301), 1)
    y = _labels((4, 1500), 301, 2)
    ref = losses.token_logprobs(x, y).double().sum(1)
    assert ref.abs().min() > 8192
    for shift in (0.0, 2.0 ** -13):                    # an eighth of an fp32 step there
        _, chosen, rejected = losses.preference_loss(x, y, ref + shift, beta=1.0)
        got = torch.cat((chosen, rejected)).double()
        # the same log-probabilities before and behind their rounding to fp32, of at most 2^-20 (under 32) and without a sign: five
        # standard deviations of the sum of 1500
        assert (got + shift).abs().max() <= 5 * 2.0 ** -20 / math.sqrt(3 / 1500)
    ints = torch.arange(4, device="cuda")
    with pytest.raises(ValueError, match="floating"):
        losses.preference_loss(x, y, ints)


# ---- layouts of the other arguments -------------------------------------------------------------------------------------
def test_lazily_negated_arguments(losses):
    """Views that torch negates when they are read (the imaginary part of a conjugate, say) count with their sign."""
    from nvfp4_sm120_b200 import optim
    x, y = _randn((2, 5, 31), 1).requires_grad_(True), _labels((2, 5), 31, 2, 0.3)
    w, adv = _randn((2, 5), 3), _randn((2,), 4)
    lp = losses.token_logprobs(x, y).detach()
    neg = lambda t: torch._neg_view(-t)
    assert neg(w).is_neg() and torch.equal(neg(w), w)

    def results(f):
        a = losses.token_logprobs(x, f(y))
        b = losses.preference_loss(x, y, f(adv - 20))
        c = losses.policy_loss(x, y, f(lp - 0.1), f(adv), f(lp + 0.1), kl_coef=0.1)
        grads = [torch.autograd.grad(o, x, f(g), retain_graph=True)[0] for o, g in ((a, w), (b[0], adv[0]), (c[0], adv[1]))]
        return [a, *b, c[0], *c[1].values(), *grads]

    assert all(torch.equal(a, b) for a, b in zip(results(neg), results(lambda t: t)))
    factor = torch.view_as_complex(torch.tensor([1.0, -2.5], device="cuda")).conj().imag
    assert factor.is_neg() and torch.equal(torch.autograd.grad(losses.preference_loss(x, y, adv)[0], x, factor)[0],
                                           torch.autograd.grad(losses.preference_loss(x, y, adv)[0], x, factor.clone().resolve_neg())[0])
    weights = []
    for norm in (neg(torch.full((), 10.0, device="cuda")), torch.full((), 10.0, device="cuda")):
        p = torch.nn.Parameter(torch.ones(5, device="cuda"))
        p.grad = torch.ones_like(p)
        optim.AdamW([p], max_norm=1e-7, eps=1e-3).step(grad_norm=norm)
        weights.append(p.detach())
    assert torch.equal(*weights)
    p = torch.nn.Parameter(neg(torch.ones(5, device="cuda")))
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="negated"):
        optim.AdamW([p]).step()


def test_vectors_of_another_shape_are_refused(losses):
    """As many values as there should be, in another order."""
    x, y = _randn((6, 4, 31), 1), _labels((6, 4), 31, 2, 0.3)
    per_label, per_sequence = _randn((6, 4), 3), _randn((6,), 4)
    want = losses.policy_loss(x, y, per_label, per_sequence, per_label, kl_coef=0.1)[0]
    token = losses.policy_loss(x, y, per_label, per_label)[0]
    for bad in (per_label.t(), per_label.view(4, 6), per_label.view(2, 3, 4), per_label.view(3, 8)):
        for call in (lambda: losses.policy_loss(x, y, bad, per_sequence), lambda: losses.policy_loss(x, y, per_label, bad),
                     lambda: losses.policy_loss(x, y, per_label, per_sequence, bad, kl_coef=0.1)):
            with pytest.raises(ValueError, match="must hold 24"):
                call()
    for good in (per_label[..., None], per_label[None], per_label.flatten(), per_label.double(), per_label.t().contiguous().t()):
        assert torch.equal(losses.policy_loss(x, y, good, per_sequence, good, kl_coef=0.1)[0], want)
    assert torch.equal(losses.policy_loss(x, y, per_label, per_label[..., None])[0], token)
    assert torch.equal(losses.policy_loss(x.flatten(0, 1), y.flatten(), per_label.flatten(), per_label.flatten())[0], token)
    loss = losses.preference_loss(x, y, per_sequence)[0]
    for bad in (per_sequence.view(3, 2), per_sequence.view(2, 3).t()):
        with pytest.raises(ValueError, match="must hold 6"):
            losses.preference_loss(x, y, bad)
    for good in (per_sequence[:, None], per_sequence[None], per_sequence.view(2, 3), per_sequence.bfloat16().double()):
        assert torch.equal(losses.preference_loss(x, y, good)[0], loss) or good.dtype == torch.float64
    one, label = _randn((2, 1, 31), 5), _labels((2, 1), 31, 6)
    assert torch.isfinite(losses.preference_loss(one, label, per_sequence[:2])[0])
    assert torch.isfinite(losses.policy_loss(one[:1], label[:1], per_label[:1, :1], per_sequence[:1], per_label[:1, 0])[0])


# ---- sizes --------------------------------------------------------------------------------------------------------------
def _softmax_gradient(x, y, w, rows=64):
    """w (onehot - softmax) of [rows, vocab] logits in 64 bits, in pieces: (index of the first row, gradient, softmax)."""
    for i in range(0, x.shape[0], rows):
        p = torch.softmax(x[i:i + rows].double(), 1)
        d = torch.where(y[i:i + rows] == IGNORE, 0.0, w[i:i + rows].double())[:, None]
        yield i, (-d * p).scatter_add(1, y[i:i + rows].clamp(min=0)[:, None], d), d.abs() * p


@pytest.mark.parametrize("rows,vocab,dtype", [(600, 131073, torch.float32), (400, 250007, torch.bfloat16)])
def test_policy_with_rows_that_the_cache_cannot_hold(losses, rows, vocab, dtype):
    """All rows in flight are more than the L2 holds: the second read of a row comes from memory."""
    x, y = (2 * _randn((rows, vocab), 1)).to(dtype), _labels((rows,), vocab, 2, 0.3)
    lp = torch.cat([torch.log_softmax(x[i:i + 64].double(), 1).gather(1, y[i:i + 64].clamp(min=0)[:, None]) for i in range(0, rows, 64)])[:, 0]
    adv = _randn((rows,), 3)
    x.requires_grad_(True)
    loss, stats = losses.policy_loss(x, y, (lp - math.log(1.1)).float(), adv)
    n = int((y != IGNORE).sum())
    live = y != IGNORE
    # logp: sums of 64 terms a thread, joined 13 times, 2^-22 of ex2.approx; its rounding of some 20.  Ratio 1.1 within the clamp.
    err = (64 + 13 + 4 + 8) * U + 2.0 ** -22 + 20 * U
    assert ((stats["logps"] - lp).abs()[live] <= err).all() and (stats["logps"][~live] == 0).all()
    assert abs(loss.item() + 1.1 * (adv.double() * live).sum().item() / n) <= 2 * 1.1 * float(adv.abs().max()) * (err + 20 * U)
    (g,) = torch.autograd.grad(loss, x)
    w = -1.1 * adv / n
    rel = err + 2.0 ** -22 + 40 * U + err + 20 * U        # of p: the sum's, ex2's, the exponents'; of w: the ratio's
    for i, want, size in _softmax_gradient(x.detach(), y, w):
        got = g[i:i + 64].double()
        off = size * rel + torch.finfo(dtype).eps / 2 * 1.001 * want.abs() + (err + 20 * U) * want.abs() + 2.0 ** -126
        assert ((got - want).abs() <= off).all()


@pytest.mark.parametrize("name", ["preference", "policy"])
def test_more_logits_than_32_bits_count_in_a_loss(losses, name):
    seq, vocab = 21400, 50257
    assert 2 * seq * vocab > 2 ** 31
    x = torch.zeros(2, seq, vocab, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 17, seq // 2, seq - 2, seq - 1], device="cuda")
    x[1, some] = (3 * _randn((5, vocab), 7)).bfloat16()
    x.requires_grad_(True)
    y = torch.full((2, seq), IGNORE, device="cuda")
    y[1, some] = torch.tensor([0, 5, vocab - 1, 9, vocab - 1], device="cuda")
    part = x.detach()[1, some]
    lp = torch.log_softmax(part.double(), 1).gather(1, y[1, some][:, None])[:, 0]
    if name == "preference":
        # L_0 = 0, h = beta (0 - (L_1 - ref)); dloss / dL_1 = beta sigmoid(-h)
        ref = torch.stack((torch.zeros_like(lp[0]), lp.sum() - 0.3))
        loss, chosen, rejected = losses.preference_loss(x, y, ref, beta=1.0)
        assert abs(float(rejected) - 0.3) <= 2.0 ** -18 and float(chosen) == 0.0
        w = torch.full((5,), 1 / (1 + math.exp(-0.3)), device="cuda")
    else:
        old, adv = torch.zeros(2, seq, device="cuda"), torch.tensor([0.0, 1.5], device="cuda")
        old[1, some] = (lp + 0.1).float()
        loss, stats = losses.policy_loss(x, y, old, adv)
        w = torch.full((5,), -1.5 * math.exp(-0.1) / 5, device="cuda")
    (g,) = torch.autograd.grad(loss, x)
    ((_, want, size),) = _softmax_gradient(part, y[1, some], w)
    # bf16's rounding, and 2^-18 for sums, exponents and w together
    assert ((g[1, some].double() - want).abs() <= 2.0 ** -18 * (size + want.abs()) + 2.0 ** -9 * 1.001 * 2 * want.abs() + 2.0 ** -126).all()
    assert torch.count_nonzero(g[0]) == 0 and torch.count_nonzero(g[1, 18:seq // 2]) == 0 and torch.count_nonzero(g[1, 1:17]) == 0
    assert torch.count_nonzero(g[1, seq // 2 + 1:seq - 2]) == 0
    del x, g
    torch.cuda.empty_cache()
