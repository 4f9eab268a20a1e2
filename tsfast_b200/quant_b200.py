"""Projections in 8-bit floating point on B200's tensor cores, for inference.

``proj_b200.linear`` is float32-faithful; here both operands are e4m3 with power-of-two scales and the products are
added in float32 (``tcgen05`` MMAs fed by TMA), at a quarter of the bytes per weight:

* ``quantize_weight(w)`` -> ``(q, scale)``, once per weight: a scale per 128 x 128 block;
* ``quant_linear(x, q, scale, bias=None)`` -> ``x q'^T + bias`` for bfloat16 or float16 ``x [..., K]``, which is quantised
  on the way in with a scale per row and 128 features; one token or many thousands.

A scale is the smallest power of two that brings its block's largest magnitude to 448 or below: scaling is exact, and the
rounding to e4m3 (half a step, 2^-4 of a value at most, subnormal steps of 2^-9 of a scale) is the only one.  There is no
gradient and no fallback.
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["quantize_weight", "quant_linear"]


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of a weight ``[N, K]`` (float32, bfloat16 or float16): ``q`` float8_e4m3fn ``[N, K]`` with a row pitch
    that is a multiple of 128, ``scale`` float32 ``[ceil(N / 128), ceil(K / 128)]``.  A value that is not finite becomes NaN and sets no scale:
    the others of its block are quantised as without it."""
    if not torch.compiler.is_compiling():
        out = _lib.host().quantize_weight(w)
        if out is not None:
            return out
    return _weight_op(w.detach())


@torch.library.custom_op("b200scan::quantize_weight", mutates_args=())
def _weight_op(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _lib.host().quant_weight(w)


@_weight_op.register_fake
def _(w):
    (N, K), blocks = w.shape, lambda n: (n + 127) // 128
    q = w.new_empty((N, 128 * blocks(K)), dtype=torch.uint8).view(torch.float8_e4m3fn).narrow(1, 0, K)
    return q, w.new_empty((blocks(N), blocks(K)), dtype=torch.float32)


@torch.library.custom_op("b200scan::quant_linear", mutates_args=())
def _linear_op(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor:
    return _lib.host().quant_product(x, q, scale, bias)


@_linear_op.register_fake
def _(x, q, scale, bias):
    return x.new_empty(*x.shape[:-1], q.shape[0])


def quant_linear(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x [..., K]`` (bfloat16 or float16) times the quantised weight ``q [N, K]``, plus ``bias [N]`` (x's type or float32).

    ``q`` and ``scale`` as ``quantize_weight`` returns them: the scales are powers of two, and another value gives NaN in the
    results that its block enters.  A ``q`` whose rows TMA cannot read (pitch or base not a multiple of 16 bytes) is copied first.  A row of x with a value that is not finite gives NaN
    throughout.  Sums are float32, the result is rounded once to x's type."""
    if not torch.compiler.is_compiling():
        out = _lib.host().quant_linear(x, q, scale, bias)
        if out is not None:
            return out
    return _linear_op(x, q, scale, bias)
