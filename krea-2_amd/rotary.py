"""Rotary positions of queries and keys, between the quantized projections and the attention (reference ``mmdit.py:13-30``
for the DiT; the text encoder's layers use the half layout).

:class:`RotaryEmbedding` holds the frequencies; calling it turns every head of ``q`` and ``k`` by its token's position in
one gfx950 launch (``k2q_rotary``), and its backward is the same launch with the angles reversed.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn

from . import _lib

LAYOUTS = ("interleaved", "half")
SCALINGS = ("linear", "ntk", "yarn")


@dataclass(frozen=True)
class RotaryScaling:
    """How frequencies ``f_i = theta ** (-2 i / d)`` are scaled for contexts ``factor`` times the length trained on.

    * ``linear``: ``f_i / factor`` (positions interpolated).
    * ``ntk``: ``theta * factor ** (d / (d - 2))`` in place of theta (the slowest pair is interpolated, the fastest kept).
    * ``yarn``: pairs that turn more than ``beta_fast`` times within ``original_length`` positions are kept, those that
      turn less than ``beta_slow`` times interpolated, a linear ramp over the pairs between; the rotated part is multiplied
      by ``attention_factor`` (default ``0.1 ln(factor) + 1``)."""

    kind: str
    factor: float
    original_length: int | None = None
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self):
        if self.kind not in SCALINGS:
            raise ValueError(f"kind must be one of {SCALINGS}, got {self.kind!r}")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError(f"factor must be at least 1, got {self.factor}")
        if self.kind == "yarn":
            if self.original_length is None or self.original_length < 1:
                raise ValueError("yarn needs the original_length that the frequencies were trained on")
            if not self.beta_fast > self.beta_slow > 0:
                raise ValueError(f"yarn needs beta_fast > beta_slow > 0, got {self.beta_fast} and {self.beta_slow}")

    def magnitude(self) -> float:
        if self.kind != "yarn":
            return 1.0
        if self.attention_factor is not None:
            return float(self.attention_factor)
        return 0.1 * math.log(self.factor) + 1.0

    def frequencies(self, d: int, theta: float) -> list[float]:
        if self.kind == "ntk":
            if d < 4:
                raise ValueError(f"ntk scaling needs at least 4 rotated values, got {d}")
            return _frequencies(d, theta * self.factor ** (d / (d - 2)))
        f = _frequencies(d, theta)
        if self.kind == "linear":
            return [v / self.factor for v in f]

        def pair(turns):        # the pair that turns so often within the original length
            return d * math.log(self.original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = max(math.floor(pair(self.beta_fast)), 0), min(math.ceil(pair(self.beta_slow)), d - 1)
        width = max(high - low, 0.001)
        ramp = [min(max((i - low) / width, 0.0), 1.0) for i in range(len(f))]
        return [v * (1 - r) + v / self.factor * r for v, r in zip(f, ramp)]


def _frequencies(d: int, theta: float) -> list[float]:
    return [theta ** (-2.0 * i / d) for i in range(d // 2)]


class _RotaryFn(torch.autograd.Function):
    """Forward: every pair turned by its angle.  Backward: the transpose, by the reversed angle."""

    @staticmethod
    def forward(ctx, q, k, positions, table, half, factor, heads_first):
        ctx.save_for_backward(positions)
        ctx.rest = (table, half, factor, heads_first)
        ctx.set_materialize_grads(False)
        return _lib.rotary(q, k, positions, *table, half, factor, False, heads_first)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        positions, = ctx.saved_tensors
        table, half, factor, heads_first = ctx.rest
        grads = [_heads(g) if need and g is not None else None for g, need in zip((dq, dk), ctx.needs_input_grad)]
        given = [g for g in grads if g is not None]
        if given:
            out = iter(_lib.rotary(given[0], given[1] if len(given) > 1 else None, positions, *table, half, factor, True,
                                   heads_first))
            grads = [None if g is None else next(out) for g in grads]
        return (*grads, None, None, None, None, None)


def _heads(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


class RotaryEmbedding(nn.Module):
    """Rotary positions over the first ``dim`` values of every head: the pair of values ``i`` turns by ``position * f_i``
    radians, ``f_i = theta ** (-2 i / dim)``, scaled for long contexts by ``scaling``; values past ``dim`` pass unchanged.

    ``layout``: pair ``i`` is the values ``(2 i, 2 i + 1)`` (``interleaved``) or ``(i, i + dim / 2)`` (``half``).
    ``axes``: the sizes (even, summing to ``dim``) of the sections that follow separate position axes, each with its own
    frequencies (the DiT's text / row / column); without it there is one axis.

    Angles are products in float64 and the rotation is float32, rounded once to the tensors' type (bf16, float16 or
    float32).  An angle of ``position * f_i`` radians is off by at most ``3 * 2^-53`` of itself (the rounded revolutions
    per position and one product) and 2^-26 turns (the rest behind the whole turns, in float32): the first is the smaller
    up to 2^28 radians, 1e-4 turns at 2^41, and a whole turn, so that nothing is left, near 2^54.

    It holds no parameters and no state: the frequencies of a device are built at its first call there (before a graph
    captures one), or for ``device`` at once."""

    def __init__(self, dim: int, theta: float = 10000.0, layout: str = "interleaved", axes=None,
                 scaling: RotaryScaling | None = None, device=None):
        super().__init__()
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
        if dim < 2 or dim % 2 or dim > _lib.MAX_ROTARY:
            raise ValueError(f"dim={dim} must be even, from 2 to {_lib.MAX_ROTARY}")
        sections = (dim,) if axes is None else tuple(int(d) for d in axes)
        if sum(sections) != dim or any(d < 2 or d % 2 for d in sections):
            raise ValueError(f"axes {sections} must be even sizes that sum to {dim}")
        if not (math.isfinite(theta) and theta > 1.0):
            raise ValueError(f"theta must be above 1, got {theta}")
        self.dim, self.theta, self.layout, self.scaling = dim, float(theta), layout, scaling
        self.axes = None if axes is None else sections
        self.factor = 1.0 if scaling is None else scaling.magnitude()
        self.frequencies = [f for d in sections for f in (scaling.frequencies(d, self.theta) if scaling is not None
                                                          else _frequencies(d, self.theta))]
        self._tables = {}
        if device is not None:
            self._table(torch.empty(0, device=device).device)

    def _table(self, dev: torch.device):
        """``(turns, axis, axes)`` on ``dev``: revolutions per position of every pair, f64, and its axis."""
        t = self._tables.get(dev)
        if t is None:
            if dev.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"the frequencies are not on {dev} yet and a capture cannot copy them there: call the "
                                   "module once before it, or make it with device=")
            tracing = torch._C._get_tracing_state()
            torch._C._set_tracing_state(None)       # the module's own, not values of a trace that ends before it
            try:
                turns = torch.tensor([f / (2 * math.pi) for f in self.frequencies], dtype=torch.float64, device=dev)
                axis = None
                if self.axes is not None:
                    axis = torch.tensor([a for a, d in enumerate(self.axes) for _ in range(d // 2)], dtype=torch.int32,
                                        device=dev)
            finally:
                torch._C._set_tracing_state(tracing)
            t = self._tables[dev] = (turns, axis, len(self.axes or ()))
        return t

    def extra_repr(self) -> str:
        return f"dim={self.dim}, theta={self.theta}, layout={self.layout}, axes={self.axes}, scaling={self.scaling}"

    def forward(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, heads_first: bool = False):
        """``(q', k')``, with the strides of ``q`` and ``k``.  ``q`` (B, L, H, D), or with ``heads_first`` (B, H, L, D), or
        either without the batch; ``k`` the same with its own number of heads, or None.  ``positions``: int64, int32,
        float32 or float64, (L,) or (B, L), with ``axes`` a last dimension of one value per axis; they get no gradient."""
        if positions.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("positions get no gradient: detach them")
        grad = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) or _lib.observed()
        table = self._tables.get(q.device)
        if table is not None and not grad:      # the call as it is, where the kernel takes it
            out = _lib.rotary_native(q, k, positions, *table, self.layout == "half", self.factor, False, heads_first)
            if out is not None:
                return out
        if q.dim() not in (3, 4) or (k is not None and k.dim() != q.dim()):
            raise ValueError(f"q {tuple(q.shape)} and k must have 4 dimensions, or 3 without a batch")
        if self.dim > q.shape[-1]:
            raise ValueError(f"{self.dim} rotated values in heads of {q.shape[-1]}")
        if q.shape[-1] > _lib.MAX_HEAD:
            raise ValueError(f"heads of {q.shape[-1]} values exceed the kernel's {_lib.MAX_HEAD}")
        if q.dim() == 3:
            # forward itself: the module's hooks have run
            q2, k2 = self.forward(q.unsqueeze(0), None if k is None else k.unsqueeze(0), positions, heads_first)
            return q2.squeeze(0), None if k2 is None else k2.squeeze(0)
        if q.numel() == 0 or (k is not None and k.numel() == 0):
            if q.numel() or (k is not None and k.numel()):
                raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)}: one of them is empty")
            return q.clone(), None if k is None else k.clone()
        _lib._device_check(q.device)
        q, k = _heads(q), None if k is None else _heads(k)
        table, half = self._table(q.device), self.layout == "half"
        if grad:
            return _RotaryFn.apply(q, k, positions, table, half, self.factor, heads_first)
        return _lib.rotary(q, k, positions, *table, half, self.factor, False, heads_first)
