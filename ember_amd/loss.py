"""Losses (``ember/loss/losses.py``)."""

from __future__ import annotations

import math
from abc import ABC, abstractmethod
from typing import NamedTuple

import numpy as np

from ember_amd import _core as C
from ember_amd import random as _random
from ember_amd.tensor import Tensor, _need_tensor, amax, exp, log, sum as _sum


class Loss(ABC):
    """Base class (``ember/loss/base.py:6-22``): ``forward`` returns the scalar
    loss and keeps what ``backward`` needs; ``backward`` returns the gradient
    with respect to ``pred``."""

    def __call__(self, pred: Tensor, target: Tensor) -> float:
        return self.forward(pred, target)

    @abstractmethod
    def forward(self, pred: Tensor, target: Tensor) -> float: ...

    @abstractmethod
    def backward(self) -> Tensor: ...


class MSELoss(Loss):
    """Mean squared error over all elements (``losses.py:9-26``):
    forward returns mean((pred - target)^2), backward (2/n)*(pred - target).

    Equal shapes take one fused pass (``_mse_loss``) that returns the same
    float sum as ``sum(diff * diff)`` and the gradient ``(2/n) * diff`` bit
    for bit; broadcasting shapes compose the operators as the reference.  That
    gradient is handed out once, and a further ``backward`` forms another:
    callers may write into what they get."""

    def __init__(self) -> None:
        self.diff: Tensor | None = None
        self.grad: Tensor | None = None
        self.pair: tuple | None = None
        self.n = 0

    def forward(self, pred: Tensor, target: Tensor) -> float:
        self.n = math.prod(pred.shape)
        if isinstance(pred, Tensor) and isinstance(target, Tensor) and pred.shape == target.shape:
            total, g = C._mse_loss(pred._core, target._core, 2.0 / self.n if self.n else 0.0)
            self.diff, self.grad = None, Tensor._from_core(g, pred.shape)
            self.pair = tuple(Tensor._from_core(x._core, x.shape) for x in (pred, target))
            return total / self.n
        self.grad = self.pair = None
        self.diff = pred - target
        return _sum(self.diff * self.diff) / self.n

    def backward(self) -> Tensor:
        if self.grad is not None:
            grad, self.grad = self.grad, None
            return grad
        if self.diff is None:
            if self.pair is None:
                raise RuntimeError("forward() must run before backward()")
            self.diff = self.pair[0] - self.pair[1]
        return (2.0 / self.n) * self.diff


class CrossEntropyLoss(Loss):
    """Softmax cross-entropy over (batch, classes) logits against one-hot (or
    probability) targets, averaged over the batch (``losses.py:29-56``):
    forward -sum(target * log_softmax(pred)) / batch with the log-sum-exp
    shift; backward (softmax(pred) - target) / batch.

    Equal shapes take one fused pass (``_cross_entropy_loss``) that forms the
    gradient with the probabilities, handed out once as MSELoss's is;
    broadcasting shapes compose the operators as the reference."""

    def __init__(self) -> None:
        self.probs: Tensor | None = None
        self.target: Tensor | None = None
        self.grad: Tensor | None = None
        self.n = 0

    def forward(self, pred: Tensor, target: Tensor) -> float:
        self.n = pred.shape[0]
        self.target = target
        self.grad = None
        if isinstance(pred, Tensor) and isinstance(target, Tensor) and pred.shape == target.shape and math.prod(pred.shape):
            rows = math.prod(pred.shape[:-1])
            total, p, g = C._cross_entropy_loss(pred._core, target._core, rows, self.n)
            self.probs, self.grad = Tensor._from_core(p, pred.shape), Tensor._from_core(g, pred.shape)
            return -total / self.n
        shifted = pred - amax(pred, axis=-1, keepdims=True)
        log_probs = shifted - log(_sum(exp(shifted), axis=-1, keepdims=True))
        self.probs = exp(log_probs)
        return -_sum(target * log_probs) / self.n

    def backward(self) -> Tensor:
        if self.probs is None or self.target is None:
            raise RuntimeError("forward() must run before backward()")
        if self.grad is not None:
            grad, self.grad = self.grad, None
            return grad
        return (self.probs - self.target) / self.n


class TokenLogProbs(NamedTuple):
    """What ``token_logprobs`` gives; ``top_tokens`` is a NumPy int32 array."""

    logp: Tensor
    entropy: Tensor
    lse: Tensor
    top_tokens: np.ndarray | None
    top_logp: Tensor | None


def _token_ids(logits: Tensor, tokens) -> np.ndarray:
    _need_tensor(logits, "token_logprobs() logits")
    ids = np.asarray(tokens)
    if not logits.shape or ids.dtype.kind not in "iu" or ids.shape != logits.shape[:-1]:
        raise ValueError(f"tokens must be integers shaped like logits {logits.shape} without the last "
                         f"dimension, got {ids.dtype} {ids.shape}")
    if logits.shape[-1] < 1:
        raise ValueError("logits need at least one class")
    classes = logits.shape[-1]
    known = ((ids >= 0) & (ids < classes)).reshape(-1)
    out = np.full(ids.size, -1, np.int32)
    out[known] = ids.reshape(-1)[known]
    return out


def _upload(ids: np.ndarray):
    return C._from_numpy(np.ascontiguousarray(ids, np.int32).view(np.float32))


def token_logprobs(logits: Tensor, tokens, top: int = 0) -> TokenLogProbs:
    """Log probabilities of ``tokens`` (integers, a NumPy array or nested lists,
    shaped like ``logits`` without its last dimension) under softmax(logits),
    with the entropy and logsumexp of each row, in one pass over the logits.
    A token outside the classes is a padded place: its log probability is 0.
    ``top`` (at most 64, and at most the classes) asks for that many of the
    likeliest tokens of each row, likeliest first and of equal ones the lowest
    id first, and their log probabilities; the ids come to the host, which
    waits for the device."""
    ids = _token_ids(logits, tokens)
    if not 0 <= top <= min(64, logits.shape[-1]):
        raise ValueError(f"top must be from 0 to {min(64, logits.shape[-1])}, not {top}")
    lead = logits.shape[:-1]
    logp, lse, _, entropy, ids_core, best = C._token_logprobs(logits._core, _upload(ids), ids.size, logits.shape[-1], top)
    rows = [Tensor._from_core(x, lead) for x in (logp, entropy, lse)]
    if not top:
        return TokenLogProbs(*rows, None, None)
    shape = (*lead, top)
    return TokenLogProbs(*rows, ids_core._to_np().view(np.int32).reshape(shape), Tensor._from_core(best, shape))


class TokenLoss(Loss):
    """Cross-entropy against token ids: forward -mean(log softmax(pred)[token])
    over the tokens within the classes (others are padded places), less
    ``entropy_bonus`` times their rows' mean entropy; backward its gradient with
    respect to ``pred`` (..., classes).  CrossEntropyLoss with one-hot targets,
    without the targets: ``tokens`` are integers, shaped as in
    ``token_logprobs``."""

    def __init__(self, entropy_bonus: float = 0.0) -> None:
        self.entropy_bonus = entropy_bonus
        self.saved: tuple | None = None

    def forward(self, pred: Tensor, target) -> float:
        ids = _token_ids(pred, target)
        tokens, known = _upload(ids), ids >= 0
        n = int(known.sum())
        logp, lse, rest, entropy, _, _ = C._token_logprobs(pred._core, tokens, ids.size, pred.shape[-1], 0)
        # The caller's Tensor may adopt another buffer before backward().
        self.saved = (Tensor._from_core(pred._core, pred.shape), tokens, known, n, lse, rest, entropy)
        if n == 0:
            return 0.0
        loss = -_sum(Tensor._from_core(logp, (ids.size,))) / n
        if self.entropy_bonus:
            loss -= self.entropy_bonus * float(entropy._to_np()[known].mean(dtype=np.float64))
        return loss

    def backward(self) -> Tensor:
        if self.saved is None:
            raise RuntimeError("forward() must run before backward()")
        pred, tokens, known, n, lse, rest, entropy = self.saved
        if n == 0:
            return _random.zeros(pred.shape)
        d_logp = _random.constant(-1.0 / n, (known.size,))
        d_entropy = Tensor(np.where(known, -self.entropy_bonus / n, 0.0)) if self.entropy_bonus else None
        grad = C._token_logprobs_bwd(pred._core, tokens, lse, rest, entropy, d_logp._core,
                                     None if d_entropy is None else d_entropy._core, known.size, pred.shape[-1])
        return Tensor._from_core(grad, pred.shape)


__all__ = ["Loss", "MSELoss", "CrossEntropyLoss", "TokenLoss", "TokenLogProbs", "token_logprobs"]
