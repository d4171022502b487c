"""Layers with manual backward, in the reference's ``ember.nn`` style.

``Layer`` has the interface of the reference's ABC (``ember/nn/base.py:7-35``):
``__call__(x, training)`` stores the input and output and calls ``forward``;
``backward(grad_y)`` returns the gradient with respect to the input and keeps
parameter gradients for ``gradients()``.

``Attention`` is the layer the reference lacks: fused scaled-dot-product
attention on the MI355X kernels.  Its input is the tuple ``(q, k, v)`` of
same-shaped Tensors ((S, D), (H, S, D) or (B, H, S, D)); ``backward`` returns
``(dq, dk, dv)``, recomputing the attention matrix from the forward's
logsumexp instead of storing it.
"""

from __future__ import annotations

import math
from abc import ABC, abstractmethod
from collections.abc import Sequence
from itertools import chain

from ember_amd import _core as C
from ember_amd import random as _random
from ember_amd.kv_cache import KVCache
from ember_amd.rows8 import activation_code, gated8, linear8, quantize8, rms_norm8
from ember_amd.tensor import Tensor, attention_backward, attention_forward


class Layer(ABC):
    x: object
    y: object

    def __call__(self, x, training: bool = True):
        self.x = x
        self._training = training
        self.y = self.forward(x, training)
        return self.y

    @abstractmethod
    def reset(self) -> None: ...

    @abstractmethod
    def parameters(self) -> list[Tensor]: ...

    @abstractmethod
    def gradients(self) -> list[Tensor | None]: ...

    @abstractmethod
    def forward(self, x, training: bool): ...

    @abstractmethod
    def backward(self, grad_y): ...


class Sequential(Layer):
    """Layers applied in order; backward runs them in reverse
    (``ember/nn/base.py:50-75``)."""

    def __init__(self, *layers: Layer):
        self.layers = layers
        self.x = self.y = None

    def reset(self) -> None:
        self.x = self.y = None
        for layer in self.layers:
            layer.reset()

    def forward(self, x, training: bool):
        for layer in self.layers:
            x = layer(x, training)
        return x

    def backward(self, grad_y):
        for layer in reversed(self.layers):
            grad_y = layer.backward(grad_y)
        return grad_y

    def parameters(self) -> list[Tensor]:
        return list(chain.from_iterable(layer.parameters() for layer in self.layers))

    def gradients(self) -> list[Tensor | None]:
        return list(chain.from_iterable(layer.gradients() for layer in self.layers))


class Attention(Layer):
    """softmax(q k^T * scale + mask) v; no parameters.  ``causal`` masks key
    j for query i unless j <= i; ``scale`` defaults to 1/sqrt(D)."""

    def __init__(self, causal: bool = False, scale: float | None = None):
        self.causal = causal
        self.scale = scale
        self.reset()

    def reset(self) -> None:
        self.x = self.y = None
        self.lse: Tensor | None = None

    def parameters(self) -> list[Tensor]:
        return []

    def gradients(self) -> list[Tensor | None]:
        return []

    def forward(self, x, training: bool) -> Tensor:
        q, k, v = x
        o, self.lse = attention_forward(q, k, v, self.causal, self.scale)
        return o

    def backward(self, grad_y: Tensor):
        if self.x is None or self.lse is None:
            raise RuntimeError("forward() must run before backward()")
        q, k, v = self.x
        return attention_backward(q, k, v, self.y, self.lse, grad_y, self.causal, self.scale)


def _rows(x: Tensor) -> tuple[int, int]:
    if len(x.shape) != 2:
        raise ValueError(f"expected a 2-D (rows, features) Tensor, got {x.shape}")
    return x.shape


def linear(x: Tensor, w: Tensor, b: Tensor | None = None, residual: Tensor | None = None,
           gelu: bool = False) -> tuple[Tensor, Tensor | None]:
    """``act(x @ w + b) + residual`` in one GEMM with a fused epilogue; returns
    (y, pre) where pre = x @ w + b is kept only when ``gelu`` (its backward
    needs it)."""
    n, k = _rows(x)
    k2, m = _rows(w)
    if k != k2:
        raise ValueError(f"Shape mismatch: {x.shape} cannot multiply {w.shape}")
    y, pre = C._linear(x._core, w._core, None if b is None else b._core,
                       None if residual is None else residual._core, n, m, k, 1 if gelu else 0, gelu)
    return Tensor._from_core(y, (n, m)), (Tensor._from_core(pre, (n, m)) if pre is not None else None)


def weight_grad(x: Tensor, grad_y: Tensor) -> Tensor:
    """x^T @ grad_y (in x out) for x (rows, in), grad_y (rows, out), reading x
    transposed in place (Ember's ``em.T(x) @ grad_y``, ``layers.py:53``)."""
    rows, n = _rows(x)
    rows2, m = _rows(grad_y)
    if rows != rows2:
        raise ValueError(f"Shape mismatch: {x.shape} and {grad_y.shape}")
    return Tensor._from_core(C._gemm(x._core, grad_y._core, 1, n, m, rows, True, False, None, None),
                             (n, m))


def input_grad(grad_y: Tensor, w: Tensor, residual: Tensor | None = None) -> Tensor:
    """grad_y @ w^T (+ residual) for w (in, out), reading w transposed in place
    (Ember's ``grad_y @ em.T(self.w)``, ``layers.py:55``)."""
    rows, m_out = _rows(grad_y)
    n_in, m_out2 = _rows(w)
    if m_out != m_out2:
        raise ValueError(f"Shape mismatch: {grad_y.shape} and {w.shape}")
    return Tensor._from_core(
        C._gemm(grad_y._core, w._core, 1, rows, n_in, m_out, False, True, None,
                None if residual is None else residual._core), (rows, n_in))


def col_sum(x: Tensor) -> Tensor:
    """Column sums of a 2-D Tensor (a Linear layer's bias gradient)."""
    n, m = _rows(x)
    return Tensor._from_core(C._col_sum(x._core, n, m), (m,))


def gated(x: Tensor, w: Tensor, b: Tensor | None = None, activation: str = "silu",
          training: bool = True) -> tuple[Tensor, Tensor | None]:
    """``act(x @ wg + bg) * (x @ wu + bu)`` in one GEMM with the gate in its
    epilogue, for w = [wg | wu] (in, 2 * hidden) and b = [bg | bu]; act is "silu",
    x / (1 + exp(-x)), or "gelu", Ember's.  Returns (h, pre), pre = x @ w + b being
    kept where ``training`` (``gated_grad`` needs it)."""
    n, d = _rows(x)
    d2, m = _rows(w)
    if d != d2 or m < 2 or m % 2:
        raise ValueError(f"Shape mismatch: {x.shape} takes a weight of ({d}, 2 * hidden), got {w.shape}")
    if b is not None and b.shape != (m,):
        raise ValueError(f"b must be ({m},), got {b.shape}")
    h, pre = C._gated_fwd(x._core, w._core, None if b is None else b._core, n, m // 2, d, activation_code(activation), training)
    return Tensor._from_core(h, (n, m // 2)), (Tensor._from_core(pre, (n, m)) if pre is not None else None)


def gated_grad(grad_y: Tensor, w_down: Tensor, pre: Tensor, activation: str = "silu") -> Tensor:
    """The gradient with respect to ``pre`` of y = gated(...) @ w_down, from y's:
    ``[dh * up * act'(gate) | dh * act(gate)]`` with dh = grad_y @ w_down^T, in one GEMM."""
    n, d = _rows(grad_y)
    hidden, d2 = _rows(w_down)
    if d != d2 or pre.shape != (n, 2 * hidden):
        raise ValueError(f"Shape mismatch: {grad_y.shape}, {w_down.shape} and {pre.shape}")
    return Tensor._from_core(C._gated_bwd(grad_y._core, w_down._core, pre._core, n, hidden, d, activation_code(activation)), pre.shape)


class Linear(Layer):
    """y = b + x @ w (``ember/nn/layers.py:9-56``), x of shape (rows, in).
    ``activation="gelu"`` fuses Ember's GELU into the GEMM epilogue.  Weights
    start U(+-1/sqrt(in)), biases 0, as the reference's ``reset``."""

    def __init__(self, in_features: int, out_features: int, activation: str | None = None):
        if activation not in (None, "gelu"):
            raise ValueError(f"unsupported activation {activation!r}")
        self.in_features = in_features
        self.out_features = out_features
        self.activation = activation
        self.reset()

    def reset(self) -> None:
        self.x = self.y = self.pre = None
        scale = 1.0 / math.sqrt(self.in_features)
        self.w = _random.uniform(-scale, scale, (self.in_features, self.out_features))
        self.b = _random.zeros((self.out_features,))
        self.grad_w = self.grad_b = None

    def parameters(self) -> list[Tensor]:
        return [self.w, self.b]

    def gradients(self) -> list[Tensor | None]:
        return [self.grad_w, self.grad_b]

    def forward(self, x: Tensor, training: bool = True, residual: Tensor | None = None) -> Tensor:
        self.x = x
        y, self.pre = linear(x, self.w, self.b, residual, self.activation == "gelu")
        return y

    def backward(self, grad_y: Tensor) -> Tensor:
        if self.x is None:
            raise RuntimeError("forward() must run before backward()")
        if self.activation == "gelu":
            # The GELU output is recomputed from the pre-activation in the
            # kernel (bit-identical to the forward's); the bias gradient is
            # summed in the same pass.
            n, m = _rows(grad_y)
            g_core, b_core = C._gelu_bwd_col_sum(grad_y._core, self.pre._core, n, m)
            grad_y = Tensor._from_core(g_core, grad_y.shape)
            self.grad_b = Tensor._from_core(b_core, (m,))
        else:
            self.grad_b = col_sum(grad_y)
        self.grad_w = weight_grad(self.x, grad_y)
        return input_grad(grad_y, self.w)


class Activation(Layer):
    """A parameter-free element-wise layer (``ember/nn/base.py:38-47``); its
    ``forward`` keeps x and y for ``backward``, so it may be called directly
    as well as through ``__call__``."""

    def __init__(self) -> None:
        self.reset()

    def reset(self) -> None:
        self.x = self.y = None

    def parameters(self) -> list[Tensor]:
        return []

    def gradients(self) -> list[Tensor | None]:
        return []

    def _need_forward(self) -> None:
        if self.y is None:
            raise RuntimeError("forward() must run before backward()")


class ReLU(Activation):
    """max(x, 0); backward grad * (y > 0) (``ember/nn/activations.py:7-19``)."""

    def forward(self, x: Tensor, training: bool = True) -> Tensor:
        from ember_amd.tensor import max as em_max
        self.x = x
        self.y = em_max(x, 0)
        return self.y

    def backward(self, grad_y: Tensor) -> Tensor:
        self._need_forward()
        return grad_y * (self.y > 0.0)


class Sigmoid(Activation):
    """1 / (1 + exp(-x)); backward grad * (y * (1 - y))
    (``ember/nn/activations.py:22-34``)."""

    def forward(self, x: Tensor, training: bool = True) -> Tensor:
        from ember_amd.tensor import exp
        self.x = x
        self.y = 1.0 / (1.0 + exp(-x))
        return self.y

    def backward(self, grad_y: Tensor) -> Tensor:
        self._need_forward()
        return grad_y * (self.y * (1.0 - self.y))


class Tanh(Activation):
    """tanh(x); backward grad * (1 - y*y) (``ember/nn/activations.py:37-49``)."""

    def forward(self, x: Tensor, training: bool = True) -> Tensor:
        from ember_amd.tensor import tanh
        self.x = x
        self.y = tanh(x)
        return self.y

    def backward(self, grad_y: Tensor) -> Tensor:
        self._need_forward()
        return grad_y * (1 - self.y * self.y)


class Dropout(Layer):
    """Inverted dropout (``ember/nn/layers.py:59-97``): in training, keep
    each element where a uniform(0, 1) draw exceeds p and scale the kept ones
    by 1/(1-p); identity otherwise.  The mask comes from the library's
    seeded generator (``ember_amd.random``)."""

    def __init__(self, p: float):
        if not 0 <= p < 1:
            raise ValueError("p must be between 0 and 1 (exclusive of 1)")
        self.p = p
        self.scale = 1.0 / (1.0 - p)
        self.reset()

    def reset(self) -> None:
        self.x = self.y = self.mask = None

    def parameters(self) -> list[Tensor]:
        return []

    def gradients(self) -> list[Tensor | None]:
        return []

    def forward(self, x: Tensor, training: bool = True) -> Tensor:
        self.x = x
        if training:
            self.mask = _random.uniform(0.0, 1.0, x.shape) > self.p
            self.y = x * self.mask * self.scale
        else:
            self.y = x
        return self.y

    def backward(self, grad_y: Tensor) -> Tensor:
        if self.mask is None:
            raise RuntimeError("forward(training=True) must run before backward()")
        return grad_y * self.mask * self.scale


class GELU(Activation):
    """Ember's GELU, 0.5*x*(1 + tanh(0.8x)) (``ember/nn/activations.py:51-66``):
    the forward composed from element-wise operators as the reference does,
    the backward one fused kernel."""

    def forward(self, x: Tensor, training: bool = True) -> Tensor:
        from ember_amd.tensor import tanh
        self.x = x
        self.y = 0.5 * x * (1 + tanh(0.8 * x))
        return self.y

    def backward(self, grad_y: Tensor) -> Tensor:
        if self.x is None or self.y is None:
            raise RuntimeError("forward() must run before backward()")
        return Tensor._from_core(C._gelu_bwd(grad_y._core, self.x._core, self.y._core), grad_y.shape)


class LayerNorm(Layer):
    """LayerNorm over the last dimension: (x - mean)/sqrt(var + eps)*gamma + beta
    (biased variance); gamma = 1, beta = 0 at reset."""

    def __init__(self, features: int, eps: float = 1e-5):
        self.features = features
        self.eps = eps
        self.reset()

    def reset(self) -> None:
        self.x = self.y = None
        self.gamma = _random.ones((self.features,))
        self.beta = _random.zeros((self.features,))
        self.grad_gamma = self.grad_beta = None
        self._stats = None

    def parameters(self) -> list[Tensor]:
        return [self.gamma, self.beta]

    def gradients(self) -> list[Tensor | None]:
        return [self.grad_gamma, self.grad_beta]

    def forward(self, x: Tensor, training: bool = True) -> Tensor:
        d = x.shape[-1]
        rows = x.size // d
        y, mean, rstd = C._layernorm_fwd(x._core, self.gamma._core, self.beta._core, rows, d, self.eps)
        self._stats = (mean, rstd)
        return Tensor._from_core(y, x.shape)

    def backward(self, grad_y: Tensor, residual: Tensor | None = None) -> Tensor:
        """Gradient with respect to x; ``residual`` (the gradient reaching x
        through a skip connection) is added in the same pass."""
        if self.x is None or self._stats is None:
            raise RuntimeError("forward() must run before backward()")
        d = self.x.shape[-1]
        dx, dg, db = C._layernorm_bwd(self.x._core, self.gamma._core, *self._stats, grad_y._core,
                                      self.x.size // d, d,
                                      None if residual is None else residual._core)
        self.grad_gamma = Tensor._from_core(dg, (d,))
        self.grad_beta = Tensor._from_core(db, (d,))
        return Tensor._from_core(dx, self.x.shape)


class RMSNorm(Layer):
    """RMS norm over the last dimension: s / sqrt(mean(s^2) + eps) * gamma with s = x,
    or x + residual where ``forward`` is given one (the sum is kept as ``sum``, and
    the gradient that ``backward`` returns is that of either); gamma = 1 at reset."""

    def __init__(self, features: int, eps: float = 1e-5):
        self.features = features
        self.eps = eps
        self.reset()

    def reset(self) -> None:
        self.x = self.y = self.sum = None
        self.gamma = _random.ones((self.features,))
        self.grad_gamma = None
        self._saved = None

    def parameters(self) -> list[Tensor]:
        return [self.gamma]

    def gradients(self) -> list[Tensor | None]:
        return [self.grad_gamma]

    def forward(self, x: Tensor, training: bool = True, residual: Tensor | None = None) -> Tensor:
        if residual is not None and residual.shape != x.shape:
            raise ValueError(f"residual must be {x.shape}, got {residual.shape}")
        d = x.shape[-1]
        y, s, rstd = C._rmsnorm_fwd(x._core, None if residual is None else residual._core, self.gamma._core, x.size // d, d, self.eps)
        self.sum = x if s is None else Tensor._from_core(s, x.shape)
        self._saved = (self.sum, rstd)
        return Tensor._from_core(y, x.shape)

    def backward(self, grad_y: Tensor, residual: Tensor | None = None) -> Tensor:
        """Gradient with respect to x; ``residual`` (the gradient reaching the
        sum through a skip connection) is added in the same pass."""
        if self._saved is None:
            raise RuntimeError("forward() must run before backward()")
        s, rstd = self._saved
        d = s.shape[-1]
        dx, dgamma = C._rmsnorm_bwd(s._core, self.gamma._core, rstd, grad_y._core, None if residual is None else residual._core,
                                    s.size // d, d)
        self.grad_gamma = Tensor._from_core(dgamma, (d,))
        return Tensor._from_core(dx, s.shape)


def _xavier(fan_in: int, fan_out: int) -> Tensor:
    a = math.sqrt(6.0 / (fan_in + fan_out))
    return _random.uniform(-a, a, (fan_in, fan_out))


def _gate_weights(d: int, hidden: int) -> Tensor:
    """Both projections of a gated layer side by side, each as ``_xavier``'s."""
    a = math.sqrt(6.0 / (d + hidden))
    return _random.uniform(-a, a, (d, 2 * hidden))


class GatedFeedForward(Layer):
    """(act(x wg + bg) * (x wu + bu)) w_out + b_out on (rows, features), with
    ``hidden`` columns between; ``activation`` is "silu" or "gelu" (Ember's).  w_in =
    [wg | wu] and b_in are one matrix and one vector; without ``bias`` there are only
    the weights.  Weights Xavier-uniform, biases 0."""

    def __init__(self, features: int, hidden: int, activation: str = "silu", bias: bool = True):
        activation_code(activation)
        if features < 1 or hidden < 1:
            raise ValueError(f"features and hidden must be positive, got {features} and {hidden}")
        self.features, self.hidden, self.activation, self.bias = features, hidden, activation, bias
        self.reset()

    def reset(self) -> None:
        d, hidden = self.features, self.hidden
        self.w_in, self.w_out = _gate_weights(d, hidden), _xavier(hidden, d)
        self.b_in = _random.zeros((2 * hidden,)) if self.bias else None
        self.b_out = _random.zeros((d,)) if self.bias else None
        self._grads: list[Tensor | None] = [None] * (4 if self.bias else 2)
        self.x = self.y = None
        self._saved = None

    def parameters(self) -> list[Tensor]:
        return [self.w_in, self.b_in, self.w_out, self.b_out] if self.bias else [self.w_in, self.w_out]

    def gradients(self) -> list[Tensor | None]:
        return list(self._grads)

    def forward(self, x: Tensor, training: bool = True, residual: Tensor | None = None) -> Tensor:
        h, pre = gated(x, self.w_in, self.b_in, self.activation, training)
        y, _ = linear(h, self.w_out, self.b_out, residual)
        self._saved = (x, h, pre) if training else None
        return y

    def backward(self, grad_y: Tensor) -> Tensor:
        if self._saved is None:
            raise RuntimeError("forward(training=True) must run before backward()")
        x, h, pre = self._saved
        dpre = gated_grad(grad_y, self.w_out, pre, self.activation)
        g_in, g_out = weight_grad(x, dpre), weight_grad(h, grad_y)
        self._grads = [g_in, col_sum(dpre), g_out, col_sum(grad_y)] if self.bias else [g_in, g_out]
        return input_grad(dpre, self.w_in)


class _Decoding:
    """What decoding takes beside the products, for a block of ``d`` features and ``h``
    heads whose norms are ``norm``."""

    d: int
    h: int
    causal: bool
    norm: str

    def make_cache(self, sequences: int, tokens: int, page_size: int = 64, pages: int | None = None) -> KVCache:
        """An empty cache for ``decode``: ``sequences`` of up to ``tokens`` tokens."""
        return KVCache(sequences, self.h, self.d // self.h, tokens, page_size, pages)

    def _new_tokens(self, x: Tensor, cache: KVCache) -> int:
        """T of ``decode``'s arguments, which it checks."""
        if not self.causal:
            raise ValueError("decode() needs a causal block")
        rows, d = _rows(x)
        if (cache.heads, cache.head_dim) != (self.h, self.d // self.h):
            raise ValueError(f"the cache has {cache.heads} heads of {cache.head_dim}, the block {self.h} of {self.d // self.h}")
        if d != self.d or rows % cache.sequences:
            raise ValueError(f"x must be ({cache.sequences} * T, {self.d}), got {x.shape}")
        return rows // cache.sequences

    def _normed(self, x: Tensor, norm: LayerNorm | RMSNorm) -> Tensor:
        rows, d = _rows(x)
        if self.norm == "rms":
            y = C._rmsnorm_fwd(x._core, None, norm.gamma._core, rows, d, norm.eps)[0]
        else:
            y = C._layernorm_fwd(x._core, norm.gamma._core, norm.beta._core, rows, d, norm.eps)[0]
        return Tensor._from_core(y, x.shape)

    def _attend(self, qkv: Tensor, cache: KVCache, T: int, count: Sequence[int] | None) -> Tensor:
        """Appends the keys and values of qkv (rows, 3 d) and attends to the cache."""
        d, D = self.d, cache.head_dim
        strides = (T * 3 * d, D, 3 * d)
        cache._append(qkv._core, d, qkv._core, 2 * d, T, strides, count)
        o, _ = cache._attend(qkv._core, 0, T, self.h, strides, True, float(1.0 / math.sqrt(D)))
        return Tensor._from_core(o, (qkv.shape[0], d))


class DecoderBlock(_Decoding, Layer):
    """One pre-norm transformer decoder block on (B*S, d) token rows:
        h = N1(x);  x2 = x + Attention(h Wqkv + bqkv) Wo + bo
        y = x2 + GELU(N2(x2) W1 + b1) W2 + b2
    with causal fused attention reading the packed QKV projection in place.  N1 and
    N2 are LayerNorm, or with ``norm="rms"`` RMSNorm.  ``gated`` "silu" or "gelu"
    makes the feed-forward layer (act(N2(x2) wg + bg) * (N2(x2) wu + bu)) W2 + b2 with
    W1 = [wg | wu].  Its width is ``hidden``, ``mlp_ratio * d_model`` without.
    Weights Xavier-uniform, biases 0, norms' gamma 1 / beta 0.  ``forward``
    takes (x, B, S); ``backward`` returns dx and fills ``gradients()``.
    ``decode`` runs new tokens against a 4-bit cache of the earlier ones, and
    ``quantize8`` gives a block that does so with its matrices in 8 bits."""

    def __init__(self, d_model: int, n_heads: int, mlp_ratio: int = 4, causal: bool = True, norm: str = "layer",
                 gated: str | None = None, hidden: int | None = None):
        if d_model % n_heads:
            raise ValueError("d_model must be a multiple of n_heads")
        if norm not in ("layer", "rms"):
            raise ValueError(f"norm must be 'layer' or 'rms', not {norm!r}")
        if gated is not None:
            activation_code(gated)
        if hidden is not None and hidden < 1:
            raise ValueError(f"hidden must be positive, not {hidden}")
        self.d, self.h, self.r, self.causal = d_model, n_heads, mlp_ratio, causal
        self.norm, self.gated = norm, gated
        self.hidden = mlp_ratio * d_model if hidden is None else hidden
        self.reset()

    def reset(self) -> None:
        d, hidden = self.d, self.hidden
        norm = RMSNorm if self.norm == "rms" else LayerNorm
        self.ln1 = norm(d)
        self.ln2 = norm(d)
        self.w_qkv, self.b_qkv = _xavier(d, 3 * d), _random.zeros((3 * d,))
        self.w_o, self.b_o = _xavier(d, d), _random.zeros((d,))
        self.w_1 = _gate_weights(d, hidden) if self.gated else _xavier(d, hidden)
        self.b_1 = _random.zeros((self.w_1.shape[1],))
        self.w_2, self.b_2 = _xavier(hidden, d), _random.zeros((d,))
        self._grads: list[Tensor | None] = [None] * len(self.parameters())
        self.x = self.y = None
        self._saved = None

    def parameters(self) -> list[Tensor]:
        return [*self.ln1.parameters(), self.w_qkv, self.b_qkv, self.w_o, self.b_o,
                *self.ln2.parameters(), self.w_1, self.b_1, self.w_2, self.b_2]

    def gradients(self) -> list[Tensor | None]:
        return list(self._grads)

    def __call__(self, x: Tensor, B: int, S: int, training: bool = True) -> Tensor:
        self.x = x
        self.y = self.forward((x, B, S), training)
        return self.y

    def forward(self, xbs, training: bool = True) -> Tensor:
        x, B, S = xbs
        D = self.d // self.h
        scale = float(1.0 / math.sqrt(D))
        self.ln1.x = x
        h1 = self.ln1.forward(x)
        qkv, _ = linear(h1, self.w_qkv, self.b_qkv)
        o_core, lse = C._attention_fwd_packed(qkv._core, B, S, self.h, D, scale, self.causal)
        o = Tensor._from_core(o_core, (B * S, self.d))
        x2, _ = linear(o, self.w_o, self.b_o, residual=x)
        self.ln2.x = x2
        h2 = self.ln2.forward(x2)
        if self.gated:
            a, u = gated(h2, self.w_1, self.b_1, self.gated)
        else:
            a, u = linear(h2, self.w_1, self.b_1, gelu=True)
        y, _ = linear(a, self.w_2, self.b_2, residual=x2)
        self._saved = (B, S, scale, h1, qkv, o, lse, x2, h2, a, u)
        return y

    def backward(self, grad_y: Tensor) -> Tensor:
        if self._saved is None:
            raise RuntimeError("forward() must run before backward()")
        B, S, scale, h1, qkv, o, lse, x2, h2, a, u = self._saved
        D = self.d // self.h
        # MLP: y = x2 + GELU(h2 W1 + b1) W2 + b2, or with the gate in GELU's place
        g_w2, g_b2 = weight_grad(a, grad_y), col_sum(grad_y)
        if self.gated:
            du = gated_grad(grad_y, self.w_2, u, self.gated)
            g_b1 = col_sum(du)
        else:
            da = input_grad(grad_y, self.w_2)
            n, m = _rows(da)
            du_core, g_b1_core = C._gelu_bwd_col_sum(da._core, u._core, n, m)  # a recomputed from u
            du, g_b1 = Tensor._from_core(du_core, da.shape), Tensor._from_core(g_b1_core, (m,))
        g_w1 = weight_grad(h2, du)
        dx2 = self.ln2.backward(input_grad(du, self.w_1), residual=grad_y)
        # attention: x2 = x + O Wo + bo
        g_wo, g_bo = weight_grad(o, dx2), col_sum(dx2)
        d_o = input_grad(dx2, self.w_o)
        dqkv = Tensor._from_core(
            C._attention_bwd_packed(qkv._core, o._core, lse, d_o._core, B, S, self.h, D, scale,
                                    self.causal), qkv.shape)
        g_wqkv, g_bqkv = weight_grad(h1, dqkv), col_sum(dqkv)
        dx = self.ln1.backward(input_grad(dqkv, self.w_qkv), residual=dx2)
        self._grads = [*self.ln1.gradients(), g_wqkv, g_bqkv, g_wo, g_bo, *self.ln2.gradients(), g_w1, g_b1, g_w2, g_b2]
        return dx

    def decode(self, x: Tensor, cache: KVCache, count: Sequence[int] | None = None) -> Tensor:
        """The block on rows that follow what ``cache`` holds: x is (sequences *
        T, d), T new tokens of each sequence (``count[b]`` of them where given,
        padded behind), which are appended to the cache and attend to it.  Causal
        blocks only; for inference: what ``backward`` needs stays as it was.
        In rows past ``count`` the attention gives 0."""
        T = self._new_tokens(x, cache)
        if T == 0:
            return _random.zeros(x.shape)
        qkv, _ = linear(self._normed(x, self.ln1), self.w_qkv, self.b_qkv)
        x2, _ = linear(self._attend(qkv, cache, T, count), self.w_o, self.b_o, residual=x)
        h2 = self._normed(x2, self.ln2)
        if self.gated:
            a, _ = gated(h2, self.w_1, self.b_1, self.gated, training=False)
        else:
            a, _ = linear(h2, self.w_1, self.b_1, gelu=True)
        y, _ = linear(a, self.w_2, self.b_2, residual=x2)
        return y

    def quantize8(self) -> DecoderBlock8:
        """This causal block for decoding with its four matrices in 8 bits, as they are now."""
        return DecoderBlock8(self)


def _copied(x: Tensor) -> Tensor:
    """A copy: the sum over its one row."""
    return Tensor._from_core(C._col_sum(x._core, 1, x.size), x.shape)


def _copied_norm(norm: LayerNorm | RMSNorm) -> LayerNorm | RMSNorm:
    new = type(norm)(norm.features, norm.eps)
    new.gamma = _copied(norm.gamma)
    if isinstance(norm, LayerNorm):
        new.beta = _copied(norm.beta)
    return new


class DecoderBlock8(_Decoding):
    """A ``DecoderBlock`` for inference whose matrices are held in 8 bits, 129/128 byte
    per element; what enters a product is rounded to 8 bits too, by the norm and the
    gate as they write it.  Norms, biases, attention and all sums stay float32.
    ``block.quantize8()`` makes one: a copy of the block's weights at that time, which
    needs the block no longer."""

    def __init__(self, block: DecoderBlock):
        if not block.causal:
            raise ValueError("decode() needs a causal block")
        self.d, self.h, self.causal, self.norm, self.gated = block.d, block.h, block.causal, block.norm, block.gated
        self.ln1, self.ln2 = _copied_norm(block.ln1), _copied_norm(block.ln2)
        self.w_qkv, self.w_o, self.w_1, self.w_2 = (quantize8(w, trans=True) for w in (block.w_qkv, block.w_o, block.w_1, block.w_2))
        self.b_qkv, self.b_o, self.b_1, self.b_2 = (_copied(b) for b in (block.b_qkv, block.b_o, block.b_1, block.b_2))

    @property
    def nbytes(self) -> int:
        """Device memory of the matrices."""
        return sum(w.nbytes for w in (self.w_qkv, self.w_o, self.w_1, self.w_2))

    def _normed8(self, x: Tensor, norm: LayerNorm | RMSNorm):
        if self.norm == "rms":
            return rms_norm8(x, norm.gamma, norm.eps)[0]
        return quantize8(self._normed(x, norm))

    def decode(self, x: Tensor, cache: KVCache, count: Sequence[int] | None = None) -> Tensor:
        """``DecoderBlock.decode`` with the matrices in 8 bits."""
        T = self._new_tokens(x, cache)
        if T == 0:
            return _random.zeros(x.shape)
        qkv = linear8(self._normed8(x, self.ln1), self.w_qkv, self.b_qkv)
        x2 = linear8(quantize8(self._attend(qkv, cache, T, count)), self.w_o, self.b_o, residual=x)
        h2 = self._normed8(x2, self.ln2)
        if self.gated:
            a = gated8(h2, self.w_1, self.b_1, self.gated)
        else:
            a = quantize8(linear8(h2, self.w_1, self.b_1, gelu=True))
        return linear8(a, self.w_2, self.b_2, residual=x2)
