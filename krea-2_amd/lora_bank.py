"""Adapters of many requests over one base: a bank of LoRA factors beside a projection, a row of the batch using the adapter
that its request names, or none.

:class:`LoRALinear` holds one adapter, whose arithmetic is ``lora.py:43-48`` of the reference.  :class:`LoRABank` holds
``count`` of them over the same frozen base, so that requests with different adapters run in one batch, and several adapters
train at once: each gets the gradients of its own rows.  :func:`add_adapters` is the operator behind it.
"""
from __future__ import annotations

import contextlib
import contextvars
import math
import sys
import threading
import weakref

import torch
import torch.nn as nn

from . import _lib
from . import lora as _lora
from .lora import DEFAULT_TARGETS


class _AddAdaptersFn(torch.autograd.Function):
    """Backward: ``g = s dy B_a``, ``dx = g A_a``, ``dA_a = sum g^T x`` and ``dB_a = sum dy^T u`` over the adapter's rows.
    Fixed order of sums, no atomics."""

    @staticmethod
    def forward(ctx, y, x, A, B, ids, scales, ranks, scale):
        out, u = _lib.bank_fwd(y, x, A, B, ids, scales, ranks, scale, ctx.needs_input_grad[3])
        need_A = ctx.needs_input_grad[2]
        ctx.save_for_backward(x if need_A else None, u, A, B, ids, scales, ranks)
        ctx.scale = scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, u, A, B, ids, scales, ranks = ctx.saved_tensors
        need = ctx.needs_input_grad
        d = _rows(dy)
        grads = _lib.bank_bwd(d, x, u, A, B, ids, scales, ranks, ctx.scale, None, *need[1:4]) if any(need[1:4]) else (None,) * 3
        return (dy if need[0] else None, *grads, None, None, None, None)


class _NoRowsFn(torch.autograd.Function):
    """A batch without rows: products of no rows, whose gradients are zeros."""

    @staticmethod
    def forward(ctx, y, x, A, B):
        ctx.save_for_backward(x, A, B)
        return y.clone()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        return (dy if need[0] else None, *(torch.zeros_like(t) if n else None for t, n in zip(ctx.saved_tensors, need[1:])))


class _BankLinearFn(torch.autograd.Function):
    """``add_adapters`` over the output of a frozen quantized base, as one node: the base's input gradient is what the adapters'
    is added to, in place (autograd would make both tensors, and a third)."""

    @staticmethod
    def forward(ctx, x, A, B, ids, scales, ranks, scale, base):
        out, u = _lib.bank_fwd(_rows(base(x)), x, A, B, ids, scales, ranks, scale, ctx.needs_input_grad[2])
        # the base's too: autograd refuses one that changed in place
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, u, A, B, ids, scales, ranks,
                              *base.input_grad_reads())
        ctx.scale, ctx.base = scale, base
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, u, A, B, ids, scales, ranks = ctx.saved_tensors[:7]
        need = ctx.needs_input_grad[:3]
        d, dx = _rows(dy), None
        if need[0]:
            dx = ctx.base.input_grad(d.view(-1, d.shape[-1])).view(*d.shape[:-1], -1)
        return (*_lib.bank_bwd(d, x, u, A, B, ids, scales, ranks, ctx.scale, dx, *need), None, None, None, None, None)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous, 16-byte aligned and in bf16 (itself when it is that)."""
    if t.dtype != torch.bfloat16:
        t = t.to(torch.bfloat16)
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def add_adapters(y: torch.Tensor, x: torch.Tensor, lora_A: torch.Tensor, lora_B: torch.Tensor, adapters: torch.Tensor,
                 scales: torch.Tensor | None = None, ranks: torch.Tensor | None = None, scale: float = 1.0) -> torch.Tensor:
    """``y + s_a (x A_a^T) B_a^T``, the adapter ``a`` of every row from ``adapters``; rows without one (a number outside
    ``0 .. count - 1``, such as -1) keep ``y``.

    ``x`` (.., in) and ``y`` (.., out) bf16 with the same leading dimensions; ``lora_A`` (count, rank, in) and ``lora_B``
    (count, out, rank), float32 or bfloat16, the rank a multiple of 16; ``adapters`` int32 or int64, one number for each of
    ``x``'s first dimension, or first dimensions (a request's rows, or every row), on the device, where nothing waits for it.
    ``s_a = scale * scales[a]`` (``scales`` float32, default 1).  ``ranks`` (int32): the ranks of each adapter that count; what
    the storage holds behind them enters nothing, and gets zero gradients.

    Sums are float32 and ``out`` is rounded once.  Float32 factors (and the sums between the products) enter the matrix
    units as two bf16 parts, 2^-17 of a value off at most, or on the way to a float32 gradient as three, which hold it.  Rows
    may have any order; rows of one adapter that lie together are faster.  Differentiable in ``y``, ``x`` and both factors.  A
    value that is infinite or NaN spoils its own row, and the gradients of its row's adapter."""
    grad = torch.is_grad_enabled() and (y.requires_grad or x.requires_grad or lora_A.requires_grad or lora_B.requires_grad)
    if not grad and not _lib.observed() and not (scales is not None and scales.requires_grad):
        out = _lib.bank_native(y, x, lora_A, lora_B, adapters, scales, ranks, scale, False)
        if out is not None:
            return out[0]
    if x.dim() < 2 or y.shape[:-1] != x.shape[:-1]:
        raise ValueError(f"y {tuple(y.shape)} and x {tuple(x.shape)} differ in their rows")
    if scales is not None and scales.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("scales get no gradient: detach them")
    if x.numel() == 0 and x.shape[-1] == lora_A.shape[-1] and y.shape[-1] == lora_B.shape[1]:
        return _NoRowsFn.apply(y, x, lora_A, lora_B) if grad else y.clone()
    if x.dtype == y.dtype == torch.bfloat16:
        x, y = _rows(x), _rows(y)
    A, B, ids = lora_A.contiguous(), lora_B.contiguous(), adapters.contiguous()
    if _lib.observed() or grad:
        return _AddAdaptersFn.apply(y, x, A, B, ids, scales, ranks, float(scale))
    return _lib.bank_fwd(y, x, A, B, ids, scales, ranks, float(scale), False)[0]


class _Body:
    """A ``with`` body of :func:`lora_requests`: the requests of some banks, ahead of those of the bodies around it."""

    def __init__(self, banks, ids, outer):
        self.banks, self.ids, self.outer, self.open = weakref.WeakSet(banks), ids, outer, True
        self.named = ids is not None
        self._count(1)

    def close(self) -> None:
        self.open, self.ids = False, None
        self._count(-1)

    def _count(self, by: int) -> None:
        if self.named:
            with _counting:
                for bank in self.banks:
                    bank.__dict__["_named"] = bank._named + by

    def of(self, bank) -> "_Body | None":
        """The innermost body of ``bank``, from this one outwards."""
        body = self
        while body is not None and bank not in body.banks:
            body = body.outer
        return body


_counting = threading.Lock()

# The body that the caller is in: a thread's, or an asyncio task's (what it starts with a copy of its context included)
_body: contextvars.ContextVar = contextvars.ContextVar("lora_requests", default=None)
# The body of a thread's last entry or forward pass, for passes that autograd recomputes: those run on threads of its own,
# which have none here
_last: dict = {}


def _entered() -> _Body | None:
    body = _body.get()
    while body is not None and not body.open:       # a task that outlived the body it was started in
        body = body.outer
    return body


def _ids_in(body: _Body | None, bank) -> torch.Tensor | None:
    found = None if body is None else body.of(bank)
    return bank._own if found is None or not found.open else found.ids


def _backward_callers() -> list:
    """The threads that are inside a backward pass: this one if it called one, and those that wait for theirs."""
    me, name, out = threading.get_ident(), "_engine_run_backward", []
    for ident, frame in sys._current_frames().items():
        if ident == me:
            while frame is not None and frame.f_code.co_name != name:
                frame = frame.f_back
        if frame is not None and frame.f_code.co_name == name:
            out.append(ident)
    return out


def _requests(bank) -> torch.Tensor | None:
    """The requests that ``bank`` runs with now where its call names none."""
    if torch.compiler.is_compiling() and not bank._named and bank._own is None:
        return None         # no body names any: what follows cannot be traced into a graph
    body, me = _entered(), threading.get_ident()
    if torch._C._current_graph_task_id() < 0:
        last = _last.get(me)
        if body is not None or last is None or last.of(bank) is not None:
            _last[me] = body
        return _ids_in(body, bank)
    if body is None or body.of(bank) is None:       # on a thread of autograd's own, or with no body left
        callers = [_last[t] for t in _backward_callers() if t in _last]
        callers = callers or [b for b in list(_last.values()) if b is None or b.open]
        bodies = [None if b is None else b.of(bank) for b in callers]
        if any(b is not None and not b.open and b.named for b in bodies):
            raise RuntimeError("a bank's forward is recomputed outside the lora_requests body that it ran in, where it would run "
                               "without its adapters: keep the backward pass inside the body")
        ids = [_ids_in(b, bank) for b in callers]
        if any(i is not ids[0] for i in ids):
            raise RuntimeError("backward passes of several threads recompute a bank's forward at once: nothing tells whose "
                               "requests it wants; open lora_requests in the recomputed function")
        return ids[0] if ids else bank._own
    return _ids_in(body, bank)


class LoRABank(nn.Module):
    """``base(x) + s_a (x A_a^T) B_a^T`` over a bank of ``count`` adapters of up to ``rank`` ranks: ``lora_A`` (count, rank, in),
    ``lora_B`` (count, out, rank), with the rank rounded up to a multiple of 16 (zero ranks, which training leaves zero).
    Initialised as ``LoRALinear`` (``lora.py:30-41``): ``A`` kaiming-uniform, ``B`` zeros, ``scale = alpha / rank``.

    Which rows use which adapter comes with the call, or from :func:`lora_requests` around the model's, or from ``adapters``
    (one setting for all threads); without any the output is ``base(x)``.  ``scale_mul`` and ``lora_scaled`` act on all adapters.

    The adapters are one parameter to an optimizer.  One that no row of a step had gets gradients of zeros, and a step moves
    it all the same: by its weight decay, and by the momentum that earlier steps left (its count of steps goes on too).
    Without decay, one that never had a row stays bit for bit.  Adapters that are to stay as they are while others train
    belong in a bank that is not stepped, or are put back (:meth:`set_adapter`) from their files."""

    _own = None     # the requests of all calls that are in no body
    _named = 0      # bodies that are open now, in any thread, and name requests

    def __init__(self, base: nn.Module, count: int, rank: int, alpha: float | None = None, dtype: torch.dtype = torch.float32):
        super().__init__()
        if not 1 <= count <= _lib.MAX_ADAPTERS:
            raise ValueError(f"{count} adapters: a bank holds 1 to {_lib.MAX_ADAPTERS}")
        if not 1 <= rank <= _lib.MAX_RANK:
            raise ValueError(f"LoRA rank must be 1 to {_lib.MAX_RANK}, got {rank}")
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"the factors must be float32 or bfloat16, got {dtype}")
        K, N = base.in_features, base.out_features
        if K % _lib.BANK_ALIGN or N % _lib.BANK_ALIGN:
            raise ValueError(f"a bank needs in/out features that are multiples of {_lib.BANK_ALIGN}, got {K} -> {N}")
        self.base = base
        base.requires_grad_(False)
        self.count, self.rank, self.scale_mul = count, rank, 1.0
        home = base.weight.device
        held = rank + -rank % _lib.RANK_ALIGN
        self.lora_A = nn.Parameter(torch.zeros(count, held, K, device=home, dtype=dtype))
        self.lora_B = nn.Parameter(torch.zeros(count, N, held, device=home, dtype=dtype))
        with torch.no_grad():
            for A in self.lora_A:
                nn.init.kaiming_uniform_(A[:rank], a=math.sqrt(5))
        # the scales as f32 bits: Module.to(dtype) casts floating buffers and leaves integer ones alone
        scale = torch.full((count,), (rank if alpha is None else alpha) / rank, dtype=torch.float32, device=home)
        self.register_buffer("scale_bits", scale.view(torch.int32))
        self.register_buffer("ranks", torch.full((count,), rank, dtype=torch.int32, device=home))

    @property
    def adapters(self) -> torch.Tensor | None:
        """The requests of the caller's body of :func:`lora_requests`, else those set here."""
        return _ids_in(_entered(), self)

    @adapters.setter
    def adapters(self, ids: torch.Tensor | None) -> None:
        self._own = ids

    @property
    def scales(self) -> torch.Tensor:
        """Every adapter's ``alpha / rank`` (a view)."""
        return self.scale_bits.view(torch.float32)

    @torch.no_grad()
    def set_adapter(self, index: int, A: torch.Tensor, B: torch.Tensor, alpha: float | None = None) -> None:
        """Put an adapter's factors (rank, in) and (out, rank) in place ``index``; ``alpha`` defaults to their rank."""
        r = self._fits(index, A, B)
        for held, t in ((self.lora_A[index], A), (self.lora_B[index].t(), B.t())):
            held[:r].copy_(t)
            held[r:].zero_()
        self.scales[index] = (r if alpha is None else alpha) / r
        self.ranks[index] = r

    @torch.no_grad()
    def _remove(self, index: int) -> None:
        """No adapter in place ``index``: rank 0, whose rows keep the base's output."""
        self._place(index)
        self.lora_A[index].zero_()
        self.lora_B[index].zero_()
        self.scales[index] = 1.0
        self.ranks[index] = 0

    def _place(self, index: int) -> None:
        if not 0 <= index < self.count:
            raise ValueError(f"adapter {index} of {self.count}")

    def _fits(self, index: int, A: torch.Tensor, B: torch.Tensor) -> int:
        """The rank of factors that have a place here."""
        self._place(index)
        (held, K), N, r = self.lora_A.shape[1:], self.lora_B.shape[1], A.shape[0] if A.dim() else 0
        if A.shape != (r, K) or B.shape != (N, r) or not 1 <= r <= held:
            raise ValueError(f"factors {tuple(A.shape)} and {tuple(B.shape)} do not fit a bank of rank {held}, {K} -> {N}")
        return r

    def adapter(self, index: int):
        """``(A, B, alpha)`` of an adapter, without the zero ranks (views; waits for the device)."""
        self._place(index)
        r = int(self.ranks[index])
        return self.lora_A[index, :r], self.lora_B[index, :, :r], float(self.scales[index]) * r

    def extra_repr(self) -> str:
        return f"count={self.count}, rank={self.rank}"

    def forward(self, x: torch.Tensor, adapters: torch.Tensor | None = None) -> torch.Tensor:
        ids, base = _requests(self) if adapters is None else adapters, self.base
        if ids is None or self.scale_mul == 0.0:
            return base(x)
        A, B = self.lora_A, self.lora_B
        grad = torch.is_grad_enabled() and (x.requires_grad or A.requires_grad or B.requires_grad)
        if (grad and isinstance(base, _lora._HIP_BASES) and "_k2q_group" not in base.__dict__ and not _lib.observed()
                and x.dtype == torch.bfloat16 and x.dim() > 1 and x.numel()):
            return _BankLinearFn.apply(_rows(x), A.contiguous(), B.contiguous(), ids.contiguous(), self.scales, self.ranks,
                                       float(self.scale_mul), base)
        return add_adapters(base(x), x, A, B, ids, self.scales, self.ranks, self.scale_mul)


_lora._SCALED += (LoRABank,)


@contextlib.contextmanager
def lora_requests(model: nn.Module, adapters: torch.Tensor | None):
    """Within the ``with`` body the rows of every bank's input in ``model`` use the adapters of ``adapters``: one number for
    each entry of the input's first dimension (the requests of a batch), or of its first dimensions; None: the base alone.

    A body is its thread's, or its asyncio task's, alone (``asyncio.to_thread`` and tasks take it with them while it is open;
    a plain thread opens its own), so threads may run requests of their own through one model.  A checkpointed forward runs
    again in its backward pass, with the requests of the thread that called that: keep it inside the body too (a bank whose last
    body the thread has left is refused there)."""
    body = _Body([m for m in model.modules() if isinstance(m, LoRABank)], adapters, _entered())
    token, me, outside = _body.set(body), threading.get_ident(), torch._C._current_graph_task_id() < 0
    if outside:
        _last[me] = body
    try:
        yield
    finally:
        body.close()
        with contextlib.suppress(ValueError):       # left in another context than entered: its holders see that it is closed
            _body.reset(token)
        if outside:
            _last[me] = _entered() or body      # closed: a backward pass that comes yet finds that it came too late


def inject_lora_bank(dit, count: int, rank: int, alpha: float | None = None, *, targets=DEFAULT_TARGETS,
                     include_txtfusion: bool = False, include_txtmlp: bool = False, dtype: torch.dtype = torch.float32) -> dict:
    """Freeze ``dit`` and put a :class:`LoRABank` around every linear that :func:`inject_lora` would wrap with these
    arguments.  The stages outside the blocks are left out by default: their inputs need the batch as their first dimension.
    Returns ``{module path: bank}``; raises ``RuntimeError`` when nothing matched."""
    return _lora._inject(dit, lambda base: LoRABank(base, count, rank, alpha, dtype), targets, include_txtfusion,
                         include_txtmlp, "inject_lora_bank")


def load_lora_into(banks: dict, index: int, path: str, *, key_prefix: str = "diffusion_model") -> int:
    """Load a saved adapter (:func:`save_lora`) into place ``index`` of ``banks``, its scale ``alpha / rank`` from the file's
    metadata (1 without).  A bank that the file does not name gets no adapter there (rank 0).  Returns how many of the file's
    adapters have no bank (0: everything loaded).  A file that does not fit one of the banks changes none."""
    from safetensors import safe_open

    with safe_open(path, framework="pt") as f:
        meta = f.metadata() or {}
        saved = {k: f.get_tensor(k) for k in f.keys()}
    names = {k[len(key_prefix) + 1:].rsplit(".lora_", 1)[0] for k in saved if k.startswith(key_prefix + ".")}
    if not names:
        raise ValueError(f"{path} holds no adapters under {key_prefix!r}")
    ratio = float(meta["alpha"]) / float(meta["rank"]) if "alpha" in meta and "rank" in meta else 1.0
    pairs = {name: [saved.get(_lora._key(key_prefix, name, w)) for w in ("A", "B")] for name in banks}
    for name, bank in banks.items():
        if any(t is None for t in pairs[name]):
            bank._place(index)
        else:
            bank._fits(index, *pairs[name])
    for name, bank in banks.items():
        A, B = pairs[name]
        if A is None or B is None:
            bank._remove(index)
        else:
            bank.set_adapter(index, A, B, ratio * A.shape[0])
    return len(names - set(banks))


def save_lora_from(banks: dict, index: int, path: str, *, metadata: dict | None = None,
                   key_prefix: str = "diffusion_model") -> None:
    """Write adapter ``index`` of ``banks`` as a file of its own, as :func:`save_lora` writes one.  All banks that hold one there
    must hold one rank and one alpha; those of rank 0 are left out."""
    parts = {name: bank.adapter(index) for name, bank in banks.items()}
    parts = {name: part for name, part in parts.items() if part[0].shape[0]}
    if not parts:
        raise ValueError(f"no adapter is held in place {index}")
    kinds = {(A.shape[0], alpha) for A, _, alpha in parts.values()}
    if len(kinds) != 1:
        raise ValueError(f"the banks' ranks and alphas differ at {index}: {sorted(kinds)}")
    (rank, alpha), = kinds
    held = {name: _lora._Factors(A, B) for name, (A, B, _) in parts.items()}
    _lora.save_lora(held, path, rank=rank, alpha=alpha, metadata=metadata, key_prefix=key_prefix)
