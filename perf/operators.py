"""Performance cases of the two ends of a training step: the loss on the logits and the optimizer.

  adamw       optim.AdamW.step over all parameters of a model, moments in 32 bits or in 8
  logprobs    losses.token_logprobs: log-probabilities of the labels, forward alone or with its gradient
  preference  losses.preference_loss, forward and backward
  policy      losses.policy_loss, forward and backward

Where `own` is false the same operators run as elementary torch operations.  `listed()` names fixed cases, `draw(rng)`
takes one more from the same ranges, `exact` gives the results in 64 bits.  Sizes are those of this repository's models
and benchmark configurations, or generic ones."""
import math

import torch

own = False

IGNORE = -100
BLOCK = 256            # elements of a moment tensor that share a scale when it is held in 8 bits
BETA1, BETA2, EPS, DECAY = 0.9, 0.95, 1e-8, 0.1
LR = 6e-5              # the end of the training schedule
STEPS = 100            # optimizer steps behind the state that a case starts from
SEED = 1234            # of the stochastic rounding of 8-bit moments
MARGIN = 0.1           # the preference loss's beta
CLIP, KL = 0.2, 0.04


def _adamw(bits, dtype, dim, kv, hidden, layers, vocab, gated, clip):
    return dict(op="adamw", bits=bits, dtype=dtype, dim=dim, kv=kv, hidden=hidden, layers=layers, vocab=vocab, gated=gated,
                clip=clip)


def _loss(op, batch, seq, vocab, dtype, prompt, grad=True):
    """batch: sequences (pairs for the preference loss); prompt: up to this share of each sequence is masked, and the
    padding behind its end too."""
    return dict(op=op, batch=batch, seq=seq, vocab=vocab, dtype=dtype, prompt=prompt, grad=grad)


def listed():
    return [
        # the addition-task model, as its trainer steps it: fifty tensors, 3.5M parameters, launches count
        dict(name="adamw32_lm", **_adamw(32, "f32", 256, 128, 768, 6, 13, False, 1.0)),
        # the GPT benchmark model with clipping, one optimizer step
        dict(name="adamw32_gpt", **_adamw(32, "f32", 768, 768, 4 * 768, 12, 50257, False, 1.0)),
        # bf16 weights with sizes that no vector width divides, no clipping
        dict(name="adamw32_odd", **_adamw(32, "bf16", 321, 107, 1111, 5, 5003, False, 0.0)),
        dict(name="adamw8_lm", **_adamw(8, "f32", 256, 128, 768, 6, 13, False, 1.0)),
        dict(name="adamw8_gpt", **_adamw(8, "f32", 768, 768, 4 * 768, 12, 50257, False, 1.0)),
        # bf16 weights of one wide layer (the feed-forward benchmark's sizes, grouped key heads)
        dict(name="adamw8_wide", **_adamw(8, "bf16", 4096, 1024, 14336, 1, 1000, True, 0.0)),
        # the frozen reference model's scores of a training microbatch: 16 x 1024 tokens, forward alone
        dict(name="logprobs_ref", **_loss("logprobs", 16, 1024, 50257, "bf16", 0.0, False)),
        # a short batch with fp32 logits (a model run without autocast), with its gradient
        dict(name="logprobs_grad", **_loss("logprobs", 3, 77, 50257, "f32", 0.5)),
        # pairs of the addition task: 13 logits a row, launches count
        dict(name="preference_lm", **_loss("preference", 256, 12, 13, "bf16", 0.5)),
        # four pairs at the training length
        dict(name="preference_gpt", **_loss("preference", 4, 1024, 50257, "bf16", 0.5)),
        # sampled answers of the addition task
        dict(name="policy_lm", **_loss("policy", 512, 12, 13, "bf16", 0.5)),
        # eight sampled sequences at the training length
        dict(name="policy_gpt", **_loss("policy", 8, 1024, 50257, "bf16", 0.25)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.4:
        dim = _log_int(rng, 64, 1200)
        return _adamw(rng.choice((32, 8)), rng.choice(("f32", "bf16")), dim, rng.randint(1, dim),
                      rng.randint(dim, 4 * dim), rng.randint(1, 8), _log_int(rng, 13, 30000), rng.random() < 0.5,
                      rng.choice((0.0, 1.0)))
    op = rng.choice(("logprobs", "preference", "policy"))
    vocab, dtype = _log_int(rng, 13, 160000), rng.choice(("bf16", "f32"))
    rows = 200_000_000 // vocab                 # under half of the largest listed case
    seq = _log_int(rng, 1, min(1500, rows))
    batch = _log_int(rng, 1, max(1, min(500, rows // (2 * seq))))
    return _loss(op, batch, seq, vocab, dtype, rng.choice((0.0, 0.3, 0.8)), op != "logprobs" or rng.random() < 0.5)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _shapes(case):
    d, k, h = case["dim"], case["kv"], case["hidden"]
    block = [(d,), (d, d), (k, d), (k, d), (d, d), (d,), (h, d), (d, h)] + ([(h, d)] if case["gated"] else [])
    return [(case["vocab"], d)] + block * case["layers"] + [(d,)]


def _segments(case):
    """(shape, first element, elements) of each tensor in a flat buffer whose tensors begin at multiples of BLOCK."""
    out, at = [], 0
    for s in _shapes(case):
        n = math.prod(s)
        out.append((s, at, n))
        at += -(-n // BLOCK) * BLOCK
    return out, at


def _used(segments, total):
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    for _, at, n in segments:
        used[at:at + n] = True
    return used


def _nearest8(x):
    """x [blocks, BLOCK] -> codes and scale bytes, nearest: the state that earlier steps left."""
    top = x.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
    e = torch.floor(torch.log2(top))
    codes = (x * torch.exp2(7 - e)).to(torch.float8_e4m3fn)
    return codes, (e[:, 0] - 7 + 127).to(torch.uint8)


def _prepare_adamw(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    segments, total = _segments(case)
    used = _used(segments, total)
    rand = lambda: torch.randn(total, device="cuda", generator=gen)
    grad = torch.zeros(total, device="cuda")
    for i, (_, at, n) in enumerate(segments):               # gradients of different tensors differ in size
        grad[at:at + n] = 1e-3 * 4.0 ** (i % 4 - 2)
    size = grad.clone()
    grad = (grad * rand()).to(_dtype(case))
    m = 0.3 * size * rand()
    root = size * (0.5 + 0.5 * torch.rand(total, device="cuda", generator=gen)) * used
    weight = (0.02 * rand() * used).to(_dtype(case))
    st = dict(case=case, weight=weight, grad=grad, step=STEPS, segments=segments)
    if case["bits"] == 32:
        st.update(m=m, v=root * root)
    else:
        (cm, sm), (cr, sr) = _nearest8(m.view(-1, BLOCK)), _nearest8(root.view(-1, BLOCK))
        st.update(cm=cm.view(-1), sm=sm, cr=cr.view(-1), sr=sr)
    if own:
        st["optimizer"] = _optimizer(st)
    return st


def _optimizer(st):
    """The optimizer object that a program keeps, with the state of its earlier steps loaded."""
    from nvfp4_sm120_b200.optim import AdamW
    case, params = st["case"], []
    for shape, at, n in st["segments"]:
        p = torch.nn.Parameter(st["weight"][at:at + n].view(shape))
        p.grad = st["grad"][at:at + n].view(shape)
        params.append(p)
    opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                max_norm=case["clip"] or None, seed=SEED)
    state = {}
    for i, (shape, at, n) in enumerate(st["segments"]):
        if case["bits"] == 32:
            state[i] = dict(step=STEPS, exp_avg=st["m"][at:at + n].view(shape), exp_avg_sq=st["v"][at:at + n].view(shape))
        else:
            to = at + -(-n // BLOCK) * BLOCK
            e8 = lambda s: s[at // BLOCK:to // BLOCK].view(torch.float8_e8m0fnu)
            state[i] = dict(step=STEPS, exp_avg=st["cm"][at:to], exp_avg_scale=e8(st["sm"]),
                            exp_avg_root=st["cr"][at:to], exp_avg_root_scale=e8(st["sr"]))
    saved = opt.state_dict()
    opt.load_state_dict(dict(state=state, param_groups=saved["param_groups"]))
    return opt


def _prepare_loss(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    b, t, v = case["batch"] * (2 if case["op"] == "preference" else 1), case["seq"], case["vocab"]
    logits = torch.empty(b, t, v, dtype=_dtype(case), device="cuda")
    labels = torch.randint(0, v, (b, t), device="cuda", generator=gen)
    logp = torch.empty(b, t, device="cuda")
    step = max(1, 200_000_000 // (t * v))
    for i in range(0, b, step):                             # (in pieces: the fp32 copies of a large batch are large)
        x = 2.0 * torch.randn(labels[i:i + step].shape + (v,), device="cuda", generator=gen)
        x.scatter_add_(2, labels[i:i + step, :, None], torch.full_like(x[..., :1], 6.0))
        logits[i:i + step] = x
        x = logits[i:i + step].float()
        logp[i:i + step] = x.gather(2, labels[i:i + step, :, None])[..., 0] - x.logsumexp(2)
        del x
    # the prompt in front and the padding behind are masked; a sequence may keep nothing
    start = (torch.rand(b, generator=host) * case["prompt"] * t).long()
    end = t - (torch.rand(b, generator=host) * 0.3 * t * (case["prompt"] > 0)).long()
    at = torch.arange(t)
    keep = ((at >= start[:, None]) & (at < end[:, None])).cuda()
    labels[~keep] = IGNORE
    logp = logp * keep
    noise = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    st = dict(case=case, logits=logits, labels=labels)
    if case["op"] == "logprobs":
        st["dlogp"] = noise(b, t)
    elif case["op"] == "preference":
        st["ref"] = (logp.double().sum(1) + 0.3 * math.sqrt(t) * noise(b)).float()
    else:
        # most tokens drifted little since they were sampled, some far; none lies within a rounding of the borders
        # ln 0.8 and ln 1.2, where the gradient has a step
        u = 2 * torch.rand(b, t, device="cuda", generator=gen) - 1
        far = torch.rand(b, t, device="cuda", generator=gen) < 0.15
        drift = torch.where(far, 0.3 * torch.sign(u) + 0.2 * u, 0.15 * u)
        st.update(old=logp - drift, ref=logp + 0.2 * noise(b, t), advantages=noise(b))
    logits.requires_grad_(case["grad"])
    return st


def prepare(case, seed):
    return _prepare_adamw(case, seed) if case["op"] == "adamw" else _prepare_loss(case, seed)


# ---- the operators in elementary operations --------------------------------------------------------------------------
def _power_of_two(e):
    """2^(e - 127) of exponent bytes held as int32."""
    return (e << 23).view(torch.float32)


def _bits16(groups, step):
    """16 random bits per element from Philox4x32-10: one call for eight elements, counter (group, step), key SEED."""
    low = 0xffffffff
    c0 = torch.arange(groups, device="cuda")
    c1, c2, c3 = torch.zeros_like(c0), torch.full_like(c0, step), torch.zeros_like(c0)
    k0, k1 = SEED & low, SEED >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), 1)
    return torch.stack((words & 0xffff, words >> 16), 2).view(-1).to(torch.int32)


def _reverse16(b):
    for s, mask in ((1, 0x5555), (2, 0x3333), (4, 0x0f0f), (8, 0x00ff)):
        b = ((b >> s) & mask) | ((b & mask) << s)
    return b


def _decode(codes, scale):
    """E4M3 codes and E8M0 scale bytes -> fp32 (every product is exact)."""
    return (codes.float().view(-1, BLOCK) * _power_of_two(scale.to(torch.int32))[:, None]).view(-1)


def _encode(x, dither):
    """Stochastic rounding to E4M3 under a power of two per block.  |x| times a power of two has E4M3's fields in its
    upper bits, so that adding the dither below them and cutting them off rounds, subnormal codes included."""
    x = x.view(-1, BLOCK)
    e = (x.abs().amax(1).view(torch.int32) >> 23).clamp(27, 177)
    y = (x.abs() * _power_of_two(205 - e)[:, None]) * 2.0 ** -64
    code = (y.view(torch.int32) + (dither.view(-1, BLOCK) << 4)) >> 20
    code = torch.where(x < 0, code | 0x80, code)
    return code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1), (e - 7).to(torch.uint8)


def _run_adamw(st):
    case = st["case"]
    st["step"] += 1
    t, g, out = st["step"], st["grad"].float(), {}
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * (torch.full_like(norm, case["clip"]) / (norm + 1e-6)).clamp(max=1.0)
        out["grad_norm"] = norm
    if case["bits"] == 32:
        m, v = st["m"], st["v"]
    else:
        m, root = _decode(st["cm"], st["sm"]), _decode(st["cr"], st["sr"])
        v = root * root
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * (1 - BETA2)) * g
    root = v.sqrt()
    ratio = m / (root * (1 / math.sqrt(1 - BETA2 ** t)) + EPS)
    p = st["weight"].float() * (1 - LR * DECAY) - ratio * (LR / (1 - BETA1 ** t))
    st["weight"] = out["weight"] = p.to(st["weight"].dtype)
    if case["bits"] == 32:
        st["m"], st["v"] = out["exp_avg"], out["exp_avg_sq"] = m, v
    else:
        bits = _bits16(m.numel() // 8, t)
        st["cm"], st["sm"] = _encode(m, bits)
        st["cr"], st["sr"] = _encode(root, _reverse16(bits))
        e8 = lambda s: s.view(torch.float8_e8m0fnu)
        out.update(exp_avg=st["cm"], exp_avg_scale=e8(st["sm"]), exp_avg_root=st["cr"], exp_avg_root_scale=e8(st["sr"]))
    return out


def _logprobs(x, labels):
    """(log-probabilities of the labels, 0 where ignored; logsumexp) of fp32 logits."""
    top = x.amax(2, keepdim=True)
    lse = top + (x - top).exp().sum(2, keepdim=True).log()
    at = labels.clamp(min=0)[..., None]
    return torch.where(labels == IGNORE, 0.0, (x.gather(2, at) - lse)[..., 0]), lse


def _dlogits(x, lse, labels, dlogp):
    d = torch.where(labels == IGNORE, 0.0, dlogp)[..., None]
    return ((x - lse).exp() * -d).scatter_add(2, labels.clamp(min=0)[..., None], d)


def _run_loss(st):
    case, logits, labels = st["case"], st["logits"].detach(), st["labels"]
    x = logits.float()
    logp, lse = _logprobs(x, labels)
    if case["op"] == "logprobs":
        if not case["grad"]:
            return logp
        return logp, _dlogits(x, lse, labels, st["dlogp"]).to(logits.dtype)
    if case["op"] == "preference":
        reward = MARGIN * (logp.double().sum(1) - st["ref"])
        chosen, rejected = reward.chunk(2)
        h = chosen - rejected
        loss = (1 + (-h).exp()).log().mean()
        d = -MARGIN / h.numel() / (1 + h.exp())
        dlogp = torch.cat((d, -d)).float()[:, None].expand_as(logp)
        return loss.float(), chosen.float(), rejected.float(), _dlogits(x, lse, labels, dlogp).to(logits.dtype)
    keep = (labels != IGNORE).float()
    count = keep.sum().clamp(min=1)
    adv = st["advantages"][:, None]
    ratio, far = (logp - st["old"]).exp(), st["ref"] - logp
    cut = ratio.clamp(1 - CLIP, 1 + CLIP)
    kl = far.exp() - far - 1
    free = ratio * adv <= cut * adv
    loss = ((KL * kl - torch.where(free, ratio, cut) * adv) * keep).sum() / count
    dlogp = (KL * (1 - far.exp()) - torch.where(free, ratio * adv, 0.0)) / count
    clipped = ((~free).float() * keep).sum() / count
    return loss, logp, (kl * keep).sum() / count, clipped, _dlogits(x, lse, labels, dlogp).to(logits.dtype)


# ---- the framework's calls -------------------------------------------------------------------------------------------
def _own_adamw(st):
    opt = st["optimizer"]
    opt.step()
    out = dict(weight=st["weight"], **opt.flat_state()[0])
    if st["case"]["clip"]:
        out["grad_norm"] = opt.grad_norm
    return out


def _own_loss(st):
    from nvfp4_sm120_b200 import losses
    case, logits, labels = st["case"], st["logits"], st["labels"]
    if case["op"] == "logprobs":
        logp = losses.token_logprobs(logits, labels)
        return (logp, *torch.autograd.grad(logp, logits, st["dlogp"])) if case["grad"] else logp
    if case["op"] == "preference":
        loss, chosen, rejected = losses.preference_loss(logits, labels, st["ref"], beta=MARGIN)
        return loss, chosen, rejected, *torch.autograd.grad(loss, logits)
    loss, stats = losses.policy_loss(logits, labels, st["old"], st["advantages"], st["ref"], clip=CLIP, kl_coef=KL)
    return loss, stats["logps"], stats["kl"], stats["clip_fraction"], *torch.autograd.grad(loss, logits)


def run(state):
    if state["case"]["op"] == "adamw":
        return _own_adamw(state) if own else _run_adamw(state)
    return _own_loss(state) if own else _run_loss(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        moments = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
        return dict(bytes=n * (3 * size + moments), flops=(15 if case["bits"] == 32 else 30) * n)
    rows = case["batch"] * case["seq"] * (2 if case["op"] == "preference" else 1)
    # a masked row is not read; on average half of `prompt` and 0.15 behind the end are masked
    read = rows * (1 - (case["prompt"] / 2 + 0.15 if case["prompt"] else 0)) * case["vocab"]
    small = rows * (8 + 4 + (4 * 4 if case["op"] == "policy" else 0))
    return dict(bytes=size * (read + (rows * case["vocab"] if case["grad"] else 0)) + small,
                flops=(8 if case["grad"] else 4) * read)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _philox_word(counter, offset, word):
    """One 32-bit word of Philox4x32-10 (Salmon et al. 2011) for each counter, key SEED."""
    m32 = 2 ** 32 - 1
    x = [counter.clone(), torch.zeros_like(counter), torch.zeros_like(counter) + offset, torch.zeros_like(counter)]
    key = [SEED % 2 ** 32, SEED // 2 ** 32]
    for r in range(10):
        ka, kb = (key[0] + r * 0x9E3779B9) & m32, (key[1] + r * 0xBB67AE85) & m32
        pa, pb = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [((pb >> 32) & m32) ^ x[1] ^ ka, pb & m32, ((pa >> 32) & m32) ^ x[3] ^ kb, pa & m32]
    return x[word]


def _rounded8(x, share):
    """x (64 bits) as E4M3 codes under the block's power of two, up where `share` (0 to 1) of a code step carries over."""
    x = x.view(-1, BLOCK)
    e = torch.frexp(x.abs().amax(1)).exponent.double() - 1
    e = torch.where(x.abs().amax(1) == 0, -100.0, e).clamp(-100, 50)
    y = x.abs() * torch.exp2(7 - e)[:, None]
    grid = torch.exp2(torch.where(y == 0, -6.0, torch.frexp(y).exponent.double() - 1).clamp(min=-6) - 3)
    y = torch.floor(y / grid + share.view(-1, BLOCK)) * grid * torch.sign(x)
    return y.float().to(torch.float8_e4m3fn).view(-1), torch.exp2(e - 7).float().to(torch.float8_e8m0fnu)


def _exact_adamw(case, seed):
    st = prepare(case, seed)
    t = st["step"] + 1
    g = st["grad"].double()
    out = {}
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        out["grad_norm"] = norm
        g = g * min(1.0, case["clip"] / (float(norm) + 1e-6))
    if case["bits"] == 32:
        m, v = st["m"].double(), st["v"].double()
    else:
        value = lambda c, s: (c.double().view(-1, BLOCK) * torch.exp2(s.double() - 127)[:, None]).view(-1)
        m, v = value(st["cm"], st["sm"]), value(st["cr"], st["sr"]) ** 2
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g * g, v, BETA2)
    out["weight"] = (st["weight"].double() * (1 - LR * DECAY)
                     - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS))
    if case["bits"] == 32:
        out.update(exp_avg=m, exp_avg_sq=v)
        return out
    place = torch.arange(m.numel(), device="cuda")
    word = torch.empty_like(place)
    for k in range(4):                                      # elements 2k and 2k + 1 of eight share word k
        word.view(-1, 8)[:, 2 * k:2 * k + 2] = _philox_word(place[:m.numel() // 8], t, k)[:, None]
    bits = torch.where(place % 2 == 0, word % 65536, word // 65536)
    turned = sum(((bits >> k) & 1) << (15 - k) for k in range(16))
    out["exp_avg"], out["exp_avg_scale"] = _rounded8(m, bits / 65536)
    out["exp_avg_root"], out["exp_avg_root_scale"] = _rounded8(v ** 0.5, turned / 65536)
    return out


def _exact_loss(case, seed):
    st = prepare(case, seed)
    logits, labels = st["logits"].detach(), st["labels"]
    live = labels != IGNORE
    label = torch.where(live, labels, 0)
    pieces = range(0, labels.shape[0], max(1, 50_000_000 // (labels.shape[1] * case["vocab"])))
    step = pieces.step
    log_softmax = lambda i: torch.log_softmax(logits[i:i + step].double(), -1)
    lp = torch.cat([log_softmax(i).gather(2, label[i:i + step, :, None])[..., 0] for i in pieces]) * live
    leaf = lp.clone().requires_grad_(True)                  # the losses' gradients by differentiation, the rows' by hand
    if case["op"] == "logprobs":
        head, slope = [lp], st["dlogp"].double()
    elif case["op"] == "preference":
        reward = MARGIN * ((leaf * live).sum(1) - st["ref"].double())
        chosen, rejected = reward[:case["batch"]], reward[case["batch"]:]
        loss = -torch.nn.functional.logsigmoid(chosen - rejected).mean()
        head, slope = [loss.detach(), chosen.detach(), rejected.detach()], torch.autograd.grad(loss, leaf)[0]
    else:
        n = max(1, int(live.sum()))
        a = st["advantages"].double()[:, None]
        rho = torch.exp(leaf - st["old"].double())
        kept = torch.minimum(rho * a, rho.clamp(1 - CLIP, 1 + CLIP) * a)
        off = st["ref"].double() - leaf
        kl = torch.expm1(off) - off
        loss = torch.where(live, KL * kl - kept, 0.0).sum() / n
        clipped = (live & (rho * a > kept)).sum() / n
        head = [loss.detach(), lp, torch.where(live, kl, 0.0).detach().sum() / n, clipped.double()]
        slope = torch.autograd.grad(loss, leaf)[0]
    if not case["grad"]:
        return head[0]
    slope = torch.where(live, slope, 0.0)
    grad = torch.empty_like(logits, dtype=torch.float64)
    for i in pieces:
        d = slope[i:i + step, :, None]
        grad[i:i + step] = -d * torch.exp(log_softmax(i))
        grad[i:i + step].scatter_add_(2, label[i:i + step, :, None], d)
    return (*head, grad)


def exact(case, seed):
    return _exact_adamw(case, seed) if case["op"] == "adamw" else _exact_loss(case, seed)
