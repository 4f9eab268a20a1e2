"""The norms around a gated block on B200, each with what surrounds it fused into one pass over HBM, and their adjoints.

With ``n(v) = (v - mean) / sqrt(var + eps)`` over the last axis (``kind="layer"``) or without the mean (``kind="rms"``)
and ``act`` SiLU, the logistic function or one:

* ``gated_norm(x, gate, weight, bias=None)``: ``y = (n(x) weight + bias) act(gate)``, which closes a block's inner path;
* ``residual_norm(x, residual, weight, bias=None, gate=, scale=, post_weight=, post_bias=)``:
  ``r = residual + scale (n(x) post_weight + post_bias) act(gate)`` and ``y = n(r) weight + bias``, returned as
  ``(y, r)``: the seam between two blocks, with the norm after the one and the norm before the next.  Every part but the
  last norm is optional.

``glue_b200.layer_norm`` and ``gate_residual`` are the float32 operators of the LRU and S5 blocks up to 512 features; these
take float32, bfloat16 and float16 rows of up to 8192, sums and statistics in float32, every result rounded once.
Parameters are of the rows' type or float32.  Eager calls take the host path in ``csrc/host/block_host.cpp``; the custom
ops below are what ``torch.compile``, tracers, dispatch modes and fake tensors see (the host path returns None for those).  What
the kernels cannot take raises.
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["gated_norm", "residual_norm"]

_KINDS = {"rms": 0, "layer": 1}
_ACTS = {None: 0, "silu": 1, "sigmoid": 2}


def _like(t, wanted=True):
    return t.new_empty(t.shape if wanted else 0)


@torch.library.custom_op("b200scan::block_norm", mutates_args=())
def _norm_op(x: torch.Tensor, residual: torch.Tensor | None, gate: torch.Tensor | None, w1: torch.Tensor | None, b1: torch.Tensor | None,
             scale: torch.Tensor | None, w2: torch.Tensor | None, b2: torch.Tensor | None, kind: int, act: int,
             eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Rows ``[M, D]``: the result, the new residual (empty without one) and the statistics kept for the adjoint."""
    h, params = _lib.host(), [w1, b1, scale, w2, b2]
    h.check_norm("gated_norm" if residual is None else "residual_norm", x, residual, gate, params, kind, eps)
    y, r, stats = h.norm_forward(x, residual, gate, params, kind, act, eps)
    return y, x.new_empty(0) if r is None else r, stats


@_norm_op.register_fake
def _(x, residual, gate, w1, b1, scale, w2, b2, kind, act, eps):
    return _like(x), _like(x, residual is not None), x.new_empty(x.shape[0], 4, dtype=torch.float32)


@torch.library.custom_op("b200scan::block_norm_bwd", mutates_args=())
def _norm_bwd_op(gy: torch.Tensor | None, gr: torch.Tensor | None, x: torch.Tensor, residual: torch.Tensor | None,
                 gate: torch.Tensor | None, w1: torch.Tensor | None, b1: torch.Tensor | None, scale: torch.Tensor | None,
                 w2: torch.Tensor | None, b2: torch.Tensor | None, stats: torch.Tensor, kind: int, act: int, eps: float) -> list[torch.Tensor]:
    """Gradients of x, residual, gate and the five parameters, empty where there is no such operand; x's is empty too where it
    is the residual's (nothing stands between x and the sum)."""
    grads = _lib.host().norm_backward(gy, gr, x, residual, gate, [w1, b1, scale, w2, b2], stats, kind, act, eps)
    if _bare(residual, gate, w1, scale):
        grads[0] = None
    return [x.new_empty(0) if g is None else g for g in grads]


def _bare(residual, gate, w1, scale):
    return residual is not None and gate is None and w1 is None and scale is None


@_norm_bwd_op.register_fake
def _(gy, gr, x, residual, gate, w1, b1, scale, w2, b2, stats, kind, act, eps):
    return [_like(x, not _bare(residual, gate, w1, scale)), _like(x, residual is not None), _like(x, gate is not None),
            *(x.new_empty(0) if t is None else _like(t) for t in (w1, b1, scale, w2, b2))]


def _remember(ctx, inputs, output):
    *tensors, ctx.kind, ctx.act, ctx.eps = inputs
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*tensors, output[2])


def _adjoint(ctx, gy, gr, _gstats):
    *tensors, stats = ctx.saved_tensors
    x, residual, gate, w1, _b1, scale, *_ = tensors
    grads = _norm_bwd_op(gy, gr if residual is not None else None, *tensors, stats, ctx.kind, ctx.act, ctx.eps)
    if _bare(residual, gate, w1, scale):
        grads[0] = grads[1]
    return *(None if t is None else g for g, t in zip(grads, tensors)), None, None, None


_norm_op.register_autograd(_adjoint, setup_context=_remember)


def _codes(op, kind, activation):
    try:
        return _KINDS[kind], _ACTS[activation]
    except KeyError:
        raise RuntimeError(f"b200scan::{op}: kind={kind!r} and activation={activation!r}, expected 'rms' or 'layer' and 'silu', "
                           "'sigmoid' or None") from None


def _composed(op, x, residual, gate, params, kind, act, eps):
    for name, t in (("residual", residual), ("gate", gate)):
        _lib.check_shape(op, name, t, x.shape, " like x")
    flat = lambda t: None if t is None else t.reshape(-1, x.shape[-1])  # noqa: E731
    y, r, _ = _norm_op(flat(x), flat(residual), flat(gate), *params, kind, act, float(eps))
    return y.reshape(x.shape), r if residual is None else r.reshape(x.shape)


def gated_norm(x: torch.Tensor, gate: torch.Tensor | None, weight: torch.Tensor, bias: torch.Tensor | None = None, *, kind: str = "rms",
               eps: float = 1e-6, activation: str | None = "silu") -> torch.Tensor:
    """``(n(x) weight + bias) act(gate)`` over the last axis of ``x [..., D]``, ``D <= 8192``; ``gate`` None: no gate.
    ``bias`` goes with ``kind="layer"``.  Differentiable in all tensors; the result is dense."""
    kind, act = _codes("gated_norm", kind, activation)
    if not torch.compiler.is_compiling():
        out = _lib.host().gated_norm(x, gate, weight, bias, kind, act, eps)
        if out is not None:
            return out
    return _composed("gated_norm", x, None, gate, (weight, bias, None, None, None), kind, act, eps)[0]


def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                  gate: torch.Tensor | None = None, scale: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, kind: str = "rms", eps: float = 1e-6,
                  activation: str | None = "silu") -> tuple[torch.Tensor, torch.Tensor]:
    """``(n(r) weight + bias, r)`` with ``r = residual + scale (n(x) post_weight + post_bias) act(gate)``.

    ``x``, ``residual``, ``gate``: ``[..., D]`` of one type; ``weight``, ``bias``, ``scale``, ``post_weight``, ``post_bias``:
    ``[D]``.  Without ``post_weight`` x enters as it is, without ``gate`` or ``scale`` they are one; the norm reads the
    unrounded ``r``.  Differentiable in all tensors, with gradients through both results."""
    kind, act = _codes("residual_norm", kind, activation)
    if not torch.compiler.is_compiling():
        out = _lib.host().residual_norm(x, residual, weight, bias, gate, scale, post_weight, post_bias, kind, act, eps)
        if out is not None:
            return out
    if residual is None:  # (else it might pass for a gated norm)
        raise RuntimeError("b200scan::residual_norm: residual is required")
    return _composed("residual_norm", x, residual, gate, (post_weight, post_bias, scale, weight, bias), kind, act, eps)
