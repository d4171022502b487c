"""Matrices in 8 bits and their products, for inference (no counterpart in the
reference, whose tensors are all float32).

``quantize8`` rounds a matrix to a ``Rows8``: 128 neighbours of a row share a
power of two and each has 4 bits of exponent and 3 of fraction
(``include/ember_amd.h`` describes the format), 129/128 byte per element.
``linear8`` multiplies two of them with the epilogue of ``nn.linear``,
``rms_norm8`` and ``gated8`` are layers whose output is one.  What they hold
enters products exactly, and sums are float32, so rounding to 8 bits is the only
difference to the float32 layers.  ``nn.DecoderBlock.quantize8`` puts them together.
"""

from __future__ import annotations

from ember_amd import _core as C
from ember_amd.tensor import Tensor, _need_tensor

ACTIVATIONS = {"gelu": 1, "silu": 2}


def activation_code(name: str) -> int:
    """The entry points' number of a gated layer's activation."""
    if name not in ACTIVATIONS:
        raise ValueError(f"unsupported activation {name!r}: {' or '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]


class Rows8:
    """A (rows, columns) matrix in 8 bits, as ``quantize8`` and the layers make them."""

    __slots__ = ("shape", "_codes", "_scales")

    def __init__(self, codes: C._Tensor, scales: C._Tensor, shape: tuple[int, int]):
        self._codes, self._scales, self.shape = codes, scales, tuple(shape)

    @property
    def nbytes(self) -> int:
        """Device memory of the codes and scales."""
        return 4 * (self._codes.size + self._scales.size)

    def to_tensor(self) -> Tensor:
        """The values held, in float32."""
        return Tensor._from_core(C._rows8_read(self._view()), self.shape)

    def _view(self) -> tuple:
        return (self._codes, self._scales, *self.shape)

    def __repr__(self) -> str:
        return f"Rows8(shape={self.shape})"


def _matrix(x: Tensor, what: str) -> tuple[int, int]:
    _need_tensor(x, what)
    if len(x.shape) != 2:
        raise ValueError(f"{what} must be 2-D (rows, features), got {x.shape}")
    return x.shape


def _need_rows8(*operands) -> None:
    for name, m in operands:
        if not isinstance(m, Rows8):
            raise TypeError(f"{name} must be a Rows8 (quantize8 makes one), got {type(m).__name__}")


def _optional(t: Tensor | None, shape: tuple[int, ...], what: str):
    if t is None:
        return None
    _need_tensor(t, what)
    if t.shape != shape:
        raise ValueError(f"{what} must be {shape}, got {t.shape}")
    return t._core


def quantize8(x: Tensor, trans: bool = False) -> Rows8:
    """x (rows, columns) rounded to 8 bits; with ``trans`` its transpose, which is
    how ``linear8`` and ``gated8`` take a weight stored (in, out)."""
    rows, cols = _matrix(x, "quantize8() x")
    if trans:
        rows, cols = cols, rows
    return Rows8(*C._rows8_write(x._core, rows, cols, bool(trans)), (rows, cols))


def linear8(x: Rows8, w: Rows8, b: Tensor | None = None, residual: Tensor | None = None, gelu: bool = False) -> Tensor:
    """``act(x @ w^T + b) + residual`` for x (rows, in) and w (out, in); b (out,),
    residual (rows, out), act Ember's GELU where ``gelu``."""
    _need_rows8(("linear8() x", x), ("linear8() w", w))
    (n, k), (m, k2) = x.shape, w.shape
    if k != k2:
        raise ValueError(f"Shape mismatch: {x.shape} and {w.shape} have different numbers of columns")
    bias, res = _optional(b, (m,), "linear8() b"), _optional(residual, (n, m), "linear8() residual")
    return Tensor._from_core(C._linear8(x._view(), w._view(), bias, res, 1 if gelu else 0), (n, m))


def gated8(x: Rows8, w: Rows8, b: Tensor | None = None, activation: str = "silu") -> Rows8:
    """``act(x @ wg^T + bg) * (x @ wu^T + bu)`` in 8 bits again, for x (rows, in) and
    w (2 * hidden, in): wg's rows, then wu's; b (2 * hidden,), act "silu" or "gelu"."""
    _need_rows8(("gated8() x", x), ("gated8() w", w))
    (n, k), (m, k2) = x.shape, w.shape
    if k != k2 or m < 2 or m % 2:
        raise ValueError(f"Shape mismatch: x {x.shape} takes w of (2 * hidden, {k}), got {w.shape}")
    act = activation_code(activation)
    return Rows8(*C._gated8(x._view(), w._view(), _optional(b, (m,), "gated8() b"), act), (n, m // 2))


def rms_norm8(x: Tensor, gamma: Tensor, eps: float = 1e-5, residual: Tensor | None = None) -> tuple[Rows8, Tensor]:
    """The RMS norm of the rows of s = x + residual, s / sqrt(mean(s^2) + eps) *
    gamma, in 8 bits, and s (x itself without ``residual``)."""
    n, d = _matrix(x, "rms_norm8() x")
    _need_tensor(gamma, "rms_norm8() gamma")
    if gamma.shape != (d,):
        raise ValueError(f"gamma must be ({d},), got {gamma.shape}")
    y, s = C._rmsnorm_fwd8(x._core, _optional(residual, (n, d), "rms_norm8() residual"), gamma._core, n, d, eps)
    return Rows8(*y, (n, d)), x if s is None else Tensor._from_core(s, x.shape)


__all__ = ["Rows8", "quantize8", "linear8", "gated8", "rms_norm8"]
