"""Loss terms of a training step beside its cross-entropy: distillation from a teacher's top logits, and the balance of a layer's experts.

No counterpart in the reference, whose training step is the cross-entropy alone (src/convlogic/model.py:137-152).  A network of gates is
often the small student of a larger one, and a layer's gates are experts of 16 operations each: ``residual_init`` starts all of them at one
operation, and training may leave them there.

    top = top_logits(teacher(x), 32, temperature=2.0)            # what a file of lists holds, 12 bytes per class listed
    loss = cross_entropy(scores, labels) + DistillationLoss(temperature=2.0)(scores, top)
    for layer in flat_layers:
        loss = loss + 0.01 * BalanceLoss()(layer.weights)[0]
"""

from typing import NamedTuple, Optional

import torch

from ._lib import native


class TopLogits(NamedTuple):
    """A teacher's lists: the largest logits of every row, where they are, and the logarithm of the mass of all others,
    ``logsumexp(unlisted / temperature)`` (``None``: not known)."""

    values: torch.Tensor
    indices: torch.Tensor
    rest: Optional[torch.Tensor] = None
    temperature: Optional[float] = None


def top_logits(logits, k, temperature=1.0):
    """The ``k`` largest of every row of ``logits`` [..., classes] as ``TopLogits``: values float32 [..., k] in descending order, indices int64
    [..., k], rest float32 [...].  Equal values are listed by index, NaN before every number; ``rest`` is -inf where nothing is left.

    float32, float16 or bfloat16 (not float64), any distance between rows; 1 <= k <= min(classes, 128).  No gradient."""
    return TopLogits(*native().top_logits(logits, k, float(temperature)), float(temperature))


def distillation_loss(scores, top, temperature=1.0, weight=None, reduction="mean"):
    """``temperature**2 * KL(teacher || softmax(scores / temperature))`` for a teacher that is known by lists of its top logits.

    ``top``: ``TopLogits`` or (values, indices[, rest]) with values and int64 indices [..., k], k <= 128, and rest [...].  With ``rest`` all unlisted
    classes of a row are one class, whose probability the student has to meet as a whole; without it the teacher's probabilities are those
    of the listed classes among themselves.  An entry whose index is outside [0, classes) does not exist (lists of unequal lengths); a class that is
    listed twice has both entries' probability.  The lists and the weight get no gradient.

    ``weight`` [...]: a factor for each row; a row of weight zero adds nothing and gets a gradient of zero whatever it holds, as does one without
    teacher mass (values and rest all -inf) or with scores that are all -inf.  ``reduction``: "none" (one loss for each row), "sum", or
    "mean", which divides by the number of rows, weighted or not (over the rows kept: ``weight=keep / keep.sum()`` with "sum").  No rows: 0.

    scores [..., classes] float32, float16 or bfloat16 (not float64: ``scores.float()``); the loss is float32, the gradient has the scores' type.

    The forward call writes the gradient for an upstream gradient of one, beside the loss (not for float16, nor with "none"); any other is computed by
    the backward call, which reads the scores again: ``0.5 * loss`` takes about 1.8 times as long as ``loss`` on long rows.  A coefficient within
    ``weight`` (``torch.full([rows], 0.5)``) costs nothing.  Under ``no_grad`` only the loss is computed."""
    if isinstance(top, TopLogits):
        made = top.temperature  # (one for each sample where a data loader has put samples' lists together)
        if made is not None and ((made != temperature).any() if isinstance(made, torch.Tensor) else made != temperature):
            raise ValueError(f"the lists were made at temperature {made}, the loss is taken at {temperature}")
        values, indices, rest = top[:3]
    else:
        if len(top) not in (2, 3):
            raise ValueError(f"the lists are (values, indices) or (values, indices, rest), got {len(top)} tensors")
        values, indices, rest = (*top, None)[:3]
    return native().distillation_loss(scores, values, indices, rest, weight, float(temperature), reduction)


def balance_loss(logits, top_k=1, keep=None):
    """(loss, counts) of rows of ``logits`` [..., experts] that choose their ``top_k`` largest (equal ones by index; never a logit of -inf; NaN counts as +inf and
    makes the loss and its row's gradient NaN):

    counts int64 [experts]: the rows that choose an expert; loss = experts / (rows * top_k) * sum_e counts[e] * mean probability of e, which is 1
    where choices and probabilities are even.  The gradient goes through the probabilities, the counts have none.

    ``keep`` bool [...]: the rows that count (a padded batch); rows without a logit above -inf never do.  No rows: 0.  float32, float16 or
    bfloat16 (not float64: ``logits.float()``); at most 1024 experts, top_k at most 32.

    For a layer's gates pass its ``weights`` ([..., 16]): the counts are then the operations of the discretised layer.  Not with
    ``GradBucket.direct()``, where a parameter's gradient is written by one backward call alone: that raises."""
    return native().balance_loss(logits, top_k, keep)


class DistillationLoss(torch.nn.Module):
    """``distillation_loss`` as a module: ``DistillationLoss(temperature)(scores, top, weight=None)``."""

    def __init__(self, temperature=1.0, reduction="mean"):
        super().__init__()
        if reduction not in ("none", "mean", "sum"):
            raise ValueError(f'reduction must be "none", "mean" or "sum", got {reduction!r}')
        self.temperature, self.reduction = float(temperature), reduction

    def forward(self, scores, top, weight=None):
        return distillation_loss(scores, top, self.temperature, weight, self.reduction)

    def extra_repr(self):
        return f"temperature={self.temperature}, reduction={self.reduction}"


class BalanceLoss(torch.nn.Module):
    """``balance_loss`` as a module: ``BalanceLoss(top_k)(logits, keep=None)`` is (loss, counts)."""

    def __init__(self, top_k=1):
        super().__init__()
        self.top_k = top_k

    def forward(self, logits, keep=None):
        return balance_loss(logits, self.top_k, keep)

    def extra_repr(self):
        return f"top_k={self.top_k}"
