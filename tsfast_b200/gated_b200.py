"""The gated linear recurrence on B200: gates, scan and adjoint fused, for training, prompts and single tokens.

Per channel, with ``rho = sigmoid(r_t)``, ``iota = sigmoid(i_t)`` and ``a_t = exp(-c softplus(lam) rho)``,

    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) iota x_t

``selective_recurrence`` takes a ready ``a_t`` and float32 sequences; here the gates' pre-activations go in as the
projections leave them (float32, bfloat16 or float16, slices of one product's output are read in place), the state is
float32 whatever the sequences' type, and sequences may be packed end to end.  The first step of a sequence is like the others:
its input too has the factor ``sqrt(1 - a_t^2)`` (some released models of this recurrence use one there).

* ``gated_recurrence(x, r, i, lam, h0=None, cu_seqlens=None, c=8.0)`` -> ``(h, h_last)``, differentiable in ``x``,
  ``r``, ``i``, ``lam`` and ``h0``;
* ``gated_recurrence_step(x, r, i, lam, state, slots=None, c=8.0)`` -> ``h``: one token per row, against a cache of
  float32 states that is updated in place.

Eager calls take the host path in ``csrc/host/block_host.cpp``; the custom ops below are what ``torch.compile``, tracers,
dispatch modes and fake tensors see (the host path returns None for those).  Nothing falls back: what the kernels cannot take raises.
"""

from __future__ import annotations

import math

import torch

from . import _lib

__all__ = ["gated_recurrence", "gated_recurrence_step"]


def _extents(x, cu):
    """(sequences, steps of each, rows of the buffer, channels) as the library counts them."""
    return (x.shape[0], x.shape[1], 0, x.shape[2]) if cu is None else (cu.numel() - 1, 0, x.shape[0], x.shape[1])


def _dense_like(t):
    return t.new_empty(t.shape)


@torch.library.custom_op("b200scan::gated_recurrence", mutates_args=())
def _gated_op(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, lam: torch.Tensor, h0: torch.Tensor | None,
              cu: torch.Tensor | None, c: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _lib.host().gated_forward(x, r, i, lam, h0, cu, c, True)


@_gated_op.register_fake
def _(x, r, i, lam, h0, cu, c):
    S, L, T, D = _extents(x, cu)
    tile = 28  # steps between the states kept for the adjoint
    kept = S * ((L + tile - 1) // tile) if cu is None else T // tile + S + 1
    return _dense_like(x), lam.new_empty(S, D), lam.new_empty(kept, D)


@torch.library.custom_op("b200scan::gated_recurrence_bwd", mutates_args=())
def _gated_bwd_op(gh: torch.Tensor | None, glast: torch.Tensor | None, x: torch.Tensor, r: torch.Tensor, i: torch.Tensor,
                  lam: torch.Tensor, cu: torch.Tensor | None, chk: torch.Tensor, c: float,
                  want_h0: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _lib.host().gated_backward(gh, glast, x, r, i, lam, cu, chk, c, want_h0)


@_gated_bwd_op.register_fake
def _(gh, glast, x, r, i, lam, cu, chk, c, want_h0):
    S, _, _, D = _extents(x, cu)
    return _dense_like(x), _dense_like(x), _dense_like(x), _dense_like(lam), lam.new_empty(S if want_h0 else 0, D)


def _remember(ctx, inputs, output):
    x, r, i, lam, h0, cu, c = inputs
    ctx.c, ctx.want_h0 = c, h0 is not None
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, r, i, lam, cu, output[2])


def _adjoint(ctx, gh, glast, _gchk):
    x, r, i, lam, cu, chk = ctx.saved_tensors
    gx, gr, gi, glam, gh0 = _gated_bwd_op(gh, glast, x, r, i, lam, cu, chk, ctx.c, ctx.want_h0)
    return gx, gr, gi, glam, gh0 if ctx.want_h0 else None, None, None


_gated_op.register_autograd(_adjoint, setup_context=_remember)


def gated_recurrence(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, lam: torch.Tensor, h0: torch.Tensor | None = None, *,
                     cu_seqlens: torch.Tensor | None = None, c: float = 8.0) -> tuple[torch.Tensor, torch.Tensor]:
    """States of the gated recurrence and the final ones.

    ``x``, ``r``, ``i``: ``[..., L, D]`` of one type (float32, bfloat16, float16), any strides with unit channel stride
    (others are copied); ``lam``: float32 ``[D]``; ``h0``: float32 ``[..., D]`` or None for zeros.  Returns ``h`` of x's
    shape and type, dense, and ``h_last`` float32 ``[..., D]`` (``h0`` where L is 0).

    With ``cu_seqlens`` (int32 or int64 ``[S + 1]`` on the device, non-decreasing) ``x`` is ``[T, D]`` and sequence ``s``
    is rows ``cu_seqlens[s]`` to ``cu_seqlens[s + 1] - 1`` with its own ``h0[s]`` and ``h_last[s]``; sequences may be empty,
    and rows before the first and behind the last get zeros, in ``h`` and in the gradients.  First derivatives backward only: second
    ones, forward-mode ones and the transforms of ``torch.func`` raise.  ``h0`` is not kept for the backward pass.
    """
    if not torch.compiler.is_compiling():
        out = _lib.host().gated_recurrence(x, r, i, lam, h0, cu_seqlens, c)
        if out is not None:
            return out
    if cu_seqlens is not None or x.dim() == 3:
        return _gated_op(x, r, i, lam, h0, cu_seqlens, float(c))[:2]
    if x.dim() < 2:
        raise RuntimeError(f"b200scan::gated_recurrence: x is {list(x.shape)}, expected at least [L, D]")
    lead, tail = x.shape[:-2], x.shape[-2:]
    n = math.prod(lead)
    for name, t in (("r", r), ("i", i)):
        _lib.check_shape("gated_recurrence", name, t, x.shape, " like x")
    _lib.check_shape("gated_recurrence", "h0", h0, (*lead, tail[1]))
    h, last, _ = _gated_op(*(t.reshape(n, *tail) for t in (x, r, i)), lam, None if h0 is None else h0.reshape(n, tail[1]), None, float(c))
    return h.reshape(x.shape), last.reshape(*lead, tail[1])


@torch.library.custom_op("b200scan::gated_recurrence_step", mutates_args=("state",))
def _step_op(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, lam: torch.Tensor, state: torch.Tensor, slots: torch.Tensor | None,
             c: float) -> torch.Tensor:
    return _lib.host().gated_step(x, r, i, lam, state, slots, c)


@_step_op.register_fake
def _(x, r, i, lam, state, slots, c):
    return _dense_like(x)


def gated_recurrence_step(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, lam: torch.Tensor, state: torch.Tensor,
                          slots: torch.Tensor | None = None, *, c: float = 8.0) -> torch.Tensor:
    """One token per row: ``h`` of ``x [B, D]``, with ``state`` (float32 ``[n, D]``) updated in place.

    ``slots`` (int32 or int64 ``[B]`` on the device) names each row's state; without it row b has state b.  A slot
    outside the cache (-1 for an empty row of a padded batch) leaves the cache alone and its row of ``h`` is zeros; rows
    that name the same slot are applied in row order.  Up to 65535 rows.  There is no gradient: train with ``gated_recurrence``.
    """
    if not torch.compiler.is_compiling():
        out = _lib.host().gated_recurrence_step(x, r, i, lam, state, slots, c)
        if out is not None:
            return out
    return _step_op(x, r, i, lam, state, slots, float(c))
