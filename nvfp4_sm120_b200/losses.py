"""Losses on a model's logits that never hold a second copy of them (csrc/logprob.cu): log-probabilities of labels, a
preference loss over pairs of sequences and a clipped policy loss with a KL term, each with its gradient.

All take logits [batch, seq, vocab] (or [rows, vocab]; fp32 or bf16, any strides with contiguous rows) and integer labels of
the leading shape, already shifted: labels[b, t] is the token that logits[b, t] predict, as in models.GPT.forward(idx,
targets).  A position whose label is `ignore_index` (prompt, padding) has no part in the result and is not read; any other
label outside the vocabulary gives NaN.  Empty logits are refused.  Arithmetic is fp32, sums over tokens are 64 bits, the
gradient is rounded once to the logits' dtype.  Logits may lie anywhere: a common offset changes nothing, and a row of one finite
value, whatever it is, has the uniform distribution.  Gradients are those of the logits: every other argument is a constant.
Differentiable once: a second derivative raises.

All can be captured into a CUDA graph, backward pass included, while no eager graph of the same leaves lives: torch adds up a leaf's
gradient on the stream that its first living graph was made on.

The reference trains with cross-entropy alone (nvfp4_train.py:159-185)."""
from __future__ import annotations

from . import _lib

IGNORE_INDEX = -100


def token_logprobs(logits, labels, ignore_index=IGNORE_INDEX):
    """log softmax(logits)[label] in fp32, of the labels' shape; 0 where the label is ignored."""
    return _lib.host().token_logprobs(logits, labels, int(ignore_index))


def preference_loss(logits, labels, ref_logps, beta=0.1, label_smoothing=0.0, ignore_index=IGNORE_INDEX):
    """Loss over pairs of sequences, (loss, chosen rewards [pairs], rejected rewards [pairs]).

    logits [2 pairs, seq, vocab]: sequence i was preferred to sequence pairs + i.  ref_logps [2 pairs]: the sums of the
    sequences' log-probabilities under the reference model, best in 64 bits (token_logprobs(...).double().sum(1)): a reward is a
    small difference of long sums, and fp32 alone rounds a sum of 5000 by 2e-4.  With L_i the sum of sequence i's log-probabilities,
    reward_i = beta (L_i - ref_i) and h = reward_chosen - reward_rejected, the loss is the mean over the pairs of
    -(1 - label_smoothing) logsigmoid(h) - label_smoothing logsigmoid(-h)."""
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must lie in [0, 1], got {label_smoothing}")
    return _lib.host().preference_loss(logits, labels, ref_logps, float(beta), float(label_smoothing), int(ignore_index))


def policy_loss(logits, labels, old_logps, advantages, ref_logps=None, clip=0.2, clip_high=None, kl_coef=0.0,
                ignore_index=IGNORE_INDEX):
    """Clipped policy loss with a KL term, (loss, stats).

    old_logps: log-probabilities of the labels when they were sampled; advantages: one per sequence [batch] or one per
    label; ref_logps: log-probabilities under the reference model, for the KL term (with kl_coef 0 for `kl` alone).  With rho = exp(logp - old) and
    d = ref - logp, the loss is the mean over all labels that are not ignored (0 if there are none) of
    -min(rho A, clamp(rho, 1 - clip, 1 + clip_high) A) + kl_coef (exp(d) - d - 1); clip_high None means clip.
    stats: `logps` (of the labels' shape, 0 where ignored), `kl` (mean of exp(d) - d - 1) and `clip_fraction`.

    With gradients on, the forward pass writes the gradient of the logits too and keeps it until the backward pass, which
    is then free when the loss is differentiated as it is.  A loss that is scaled first (loss / accumulation steps) costs one
    more read and write of the logits: scale the advantages and kl_coef instead."""
    clip_high = clip if clip_high is None else clip_high
    if not (0.0 <= clip <= 1.0 and clip_high >= 0.0):
        raise ValueError(f"clip must lie in [0, 1] and clip_high must not be negative, got {clip} and {clip_high}")
    if kl_coef and ref_logps is None:
        raise ValueError("kl_coef needs ref_logps")
    loss, logps, kl, fraction = _lib.host().policy_loss(logits, labels, old_logps, advantages, ref_logps, float(clip),
                                                        float(clip_high), float(kl_coef), int(ignore_index))
    return loss, {"logps": logps, "kl": kl, "clip_fraction": fraction}
