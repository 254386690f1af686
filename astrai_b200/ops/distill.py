"""Distillation from a teacher's top logits: taking them, and the loss of a student's logits with their gradient.

The reference trains on hard labels, preferences and rewards (astrai/trainer/strategy.py) and has no distillation. Here
a teacher is given as :class:`TopLogits`: for each position the ids and logits of its most likely tokens and, if wanted,
the log-sum-exp of all its other logits, a few hundred bytes where its whole row takes ``vocab`` numbers.

* :func:`top_logits`   a teacher's rows of logits as :class:`TopLogits`
* :func:`distill_loss` the mean over positions of ``(1 - hard_weight) * temperature**2 * KL(teacher | student)``
  ``+ hard_weight * cross_entropy(target)``

On CUDA the kernels of ``csrc/distill.cu`` and ``csrc/top_logits.cu`` run (bfloat16, float16 and float32 logits): the
logits are read once, and the loss writes their gradient in the same pass. CPU tensors take the plain PyTorch functions below.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from astrai_b200.ops._ext import native


class TopLogits(NamedTuple):
    """A teacher's most likely tokens at each position, and what it leaves to the others."""

    ids: torch.Tensor                     # int32 or int64 [..., k]; an id outside the vocabulary: no entry
    values: torch.Tensor                  # their logits [..., k], bfloat16, float16 or float32
    rest: Optional[torch.Tensor] = None   # fp32 [...]: log sum exp(logit / temperature) over all other tokens


# ----------------------------------------------------------------------------- the teacher's side
def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The ``k`` (at most 256) largest of each row of ``logits [..., vocab]`` in descending order, of equal ones the
    lowest id first, and ``rest``: log sum exp(logit / temperature) over all others (-inf where there are none).

    A NaN counts as larger than every number. There is no gradient: under grad mode logits that require one are refused.
    """
    if logits.is_cuda:
        return TopLogits(*native().top_logits(logits, int(k), float(temperature)))
    if logits.dim() < 1 or not 1 <= k <= min(256, logits.shape[-1]):
        raise ValueError(f"top_logits: k must be in 1 .. min(256, vocab), got {k}")
    if not 0 < temperature < math.inf:
        raise ValueError("top_logits: temperature must be positive")
    if torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("top_logits has no gradient: call it under no_grad")
    values, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    rest = torch.logsumexp(values[..., k:].float() / temperature, -1)
    return TopLogits(ids[..., :k].int(), values[..., :k].contiguous(), rest)


# ----------------------------------------------------------------------------- loss
def _loss_reference(logits, teacher: TopLogits, tau, target, hard, ignore) -> torch.Tensor:
    V = logits.shape[-1]
    x = logits.reshape(-1, V).float()
    ids = teacher.ids.reshape(x.shape[0], -1).long()
    entry = (ids >= 0) & (ids < V)
    at = torch.where(entry, ids, 0)
    t = (teacher.values.detach().reshape(x.shape[0], -1).float() / tau).masked_fill(~entry, -math.inf)
    rest = torch.full_like(x[:, 0], -math.inf) if teacher.rest is None else teacher.rest.detach().reshape(-1).float()
    t = torch.cat([t, rest[:, None]], -1)
    none = (t == -math.inf).all(-1, keepdim=True)  # a position without any mass of the teacher adds nothing
    logp = torch.log_softmax(t.masked_fill(none, 0.0), -1)
    p = torch.where(none, 0.0, logp.exp())
    z = x / tau
    lse = torch.logsumexp(z, -1, keepdim=True)
    outside = torch.ones_like(z, dtype=torch.int32).scatter_reduce(1, at, 1 - entry.int(), "amin").bool()
    others = torch.where(outside, z, -math.inf)
    empty = ~outside.any(-1, keepdim=True)
    others = torch.logsumexp(torch.where(empty, 0.0, others), -1, keepdim=True)
    logq = torch.cat([z.gather(1, at), torch.where(empty, -math.inf, others)], -1) - lse
    live = p != 0  # what the teacher gives no mass adds nothing, whatever the student gives it
    row = (1 - hard) * tau ** 2 * (p * (torch.where(live, logp, 0.0) - torch.where(live, logq, 0.0))).sum(-1)
    n = x.shape[0]
    if target is not None:
        y = target.reshape(-1).long()
        counted = (y != ignore) & (y >= 0) & (y < V)
        if hard:
            label = torch.where(counted, y, 0)[:, None]
            row = row + hard * (torch.logsumexp(x, -1) - x.gather(1, label)[:, 0])
        row = torch.where(counted, row, 0.0)
        n = counted.sum().clamp(min=1)
    return row.sum() / max(n, 1) if isinstance(n, int) else row.sum() / n


def distill_loss(logits: torch.Tensor, teacher: TopLogits, temperature: float = 1.0,
                 target: Optional[torch.Tensor] = None, hard_weight: float = 0.0, ignore_index: int = -100,
                 expected_grad: float = 1.0) -> torch.Tensor:
    """Loss of a student's logits ``[..., vocab]`` against a teacher's top logits, a mean over the positions.

    With ``q`` the softmax of the student's logits over the temperature and ``p`` that of the teacher's ``values``
    over it, together with ``rest`` as one more entry that stands for all other tokens (given: the student's mass on
    them is one entry too; not given: ``p`` is normalised over the k entries)::

        (1 - hard_weight) * temperature**2 * sum_k p_k (log p_k - log q_k) + hard_weight * (logsumexp(x) - x[target])

    ``target [...]`` holds the labels; positions whose target is ``ignore_index`` or outside the vocabulary do not
    count, and without a target all do. A position without any mass of the teacher adds only its label's part. An id
    that comes twice stands for the sum of its entries' mass.

    On CUDA ``k`` is at most 1024 and the vocabulary at most 557048 (16-bit types) or 278524 (float32). The forward
    pass also writes the gradient of the logits, for an upstream gradient of ``expected_grad`` (what ``loss *
    expected_grad`` or a division by the accumulation steps will send back); any other one costs the backward
    another pass over the logits, with the same result, and so does a backward that is not in the forward's capture
    of a CUDA graph. There is no forward-mode and no second derivative: each is refused. CPU tensors take plain
    operations of PyTorch, which refuse neither, at any ``k``. There is no gradient of the teacher on either: under
    grad mode it is refused.
    """
    if logits.is_cuda:
        return native().distill_loss(logits, teacher.ids, teacher.values, teacher.rest, float(temperature), target,
                                     float(hard_weight), int(ignore_index), float(expected_grad))
    lead = logits.shape[:-1]
    if logits.dim() < 1 or teacher.ids.shape != teacher.values.shape or teacher.ids.shape[:-1] != lead:
        raise ValueError("distill_loss: the teacher's ids and values must be [..., k] with the logits' leading sizes")
    for name, t in (("rest", teacher.rest), ("target", target)):
        if t is not None and t.shape != lead:
            raise ValueError(f"distill_loss: {name} must have the logits' leading sizes")
    if not 0 < temperature < math.inf:
        raise ValueError("distill_loss: temperature must be positive")
    if not 0 <= hard_weight <= 1 or (hard_weight and target is None):
        raise ValueError("distill_loss: hard_weight must be in [0, 1] and needs a target")
    if torch.is_grad_enabled() and (teacher.values.requires_grad or (teacher.rest is not None
                                                                     and teacher.rest.requires_grad)):
        raise RuntimeError("distill_loss has no gradient of the teacher")
    return _loss_reference(logits, teacher, float(temperature), target, float(hard_weight), ignore_index)
