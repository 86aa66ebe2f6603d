"""GPU tests of a bank of adapters at its edges: ranks that are no multiple of 16 in storage that holds something behind them,
gradients in the precision of their type, batches and adapters without rows, bases that change between the passes, and
requests of several threads."""
import contextlib
import copy
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from test_gpu_lora_bank import DTYPES, _check, _formula, _ids, _linear, _make

pytestmark = pytest.mark.gpu


# -- ranks ------------------------------------------------------------------------------------------------------------
RANKS = [5, 0, 64, 33, 17, 16, 1, 50]


@pytest.mark.parametrize("behind", [3.0, float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lead, of, R, K, N", [
    ((40,), (40,), 64, 128, 192),           # single rows in one launch
    ((40,), (40,), 128, 1600, 192),         # and in two
    ((500,), (500,), 64, 128, 320),         # tiles that meet several adapters
    ((4, 300), (4,), 144, 1088, 2112),      # tiles of one, ranks past a workgroup's, slices
    ((2, 20000), (2,), 64, 64, 128)])       # a "down" in one slice, pieces
def test_ranks_are_counted_one_by_one(k2, dev, lead, of, R, K, N, dtype, behind):
    """An adapter's rank counts as it is, whatever the storage holds behind it: the formula's values with zeros there, and
    gradients of exactly zero."""
    ids = _ids(of, len(RANKS), "mixed")
    x, y, A, B, ids, scales, rk, dy = _make(dev, lead, ids, len(RANKS), R, K, N, DTYPES[dtype], RANKS)
    want, size = _formula(x, y, A, B, ids, scales, dy)
    for a, r in enumerate(RANKS):
        A[a, r:], B[a, :, r:] = behind, behind
    with torch.no_grad():
        served = k2.add_adapters(y, x, A, B, ids, scales, rk)
    leaves = [t.clone().requires_grad_() for t in (x, A, B)]
    out = k2.add_adapters(y, *leaves, ids, scales, rk)
    grads = torch.autograd.grad(out, leaves, dy)
    rows = out.shape[:-1].numel()
    assert torch.equal(out, served)
    for got, w, s, terms in zip((out.detach(), *grads), want, size, (K + R, N + R, N + rows, K + rows)):
        _check(got, w, s, terms, dtype)
    for a, r in enumerate(RANKS):
        assert not int(grads[1][a, r:].count_nonzero()) and not int(grads[2][a, :, r:].count_nonzero()), a


@pytest.mark.parametrize("rows", [30, 300])
def test_ranks_behind_an_adapters_own_keep_zero_gradients(k2, dev, rows):
    """Also where a row of its own is not finite."""
    ids = torch.arange(rows) % 2
    x, y, A, B, ids, scales, rk, dy = _make(dev, (rows,), ids, 2, 64, 128, 64, torch.float32, [5, 20])
    x[0, 3], dy[0, 5] = float("nan"), float("inf")
    leaves = [t.clone().requires_grad_() for t in (A, B)]
    dA, dB = torch.autograd.grad(k2.add_adapters(y, x, *leaves, ids, scales, rk), leaves, dy)
    for a, r in enumerate((5, 20)):
        assert not int(dA[a, r:].count_nonzero()) and not int(dB[a, :, r:].count_nonzero())
    assert torch.isfinite(dA[1]).all() and torch.isfinite(dB[1]).all() and not torch.isfinite(dA[0]).all()


# -- precision --------------------------------------------------------------------------------------------------------
def _two_parts(t):
    """float32 as two bf16 parts, in float64."""
    hi = t.bfloat16()
    return hi.double() + (t - hi.float()).bfloat16().double()


@pytest.mark.parametrize("how", ["sorted", "mixed"])
@pytest.mark.parametrize("lead, of, count, R, K, N", [
    ((65,), (65,), 3, 32, 320, 64), ((3, 50), (3,), 5, 48, 128, 256), ((2, 120), (2,), 1, 16, 256, 320),
    ((70,), (70,), 2, 144, 64, 128), ((2, 33, 3), (2, 33), 4, 64, 64, 192)])
def test_gradients_of_f32_factors_hold_its_bits(k2, dev, lead, of, count, R, K, N, how):
    """dA and dB in f32 are off by the sums' roundings alone.  Their operands enter in three bf16 parts, which hold them
    whole.  A sum of n products (n at most 320 here) takes 3 n / 32 matrix instructions, of which each rounds a running sum a
    few times (4, say): 120 roundings of up to 2^-24 of a sum that grows as the root of its terms come to 2^-24 sqrt(120 / 2)
    of the result, as a norm over many, 4.6e-7 for the first product and as much for the second: 6.5e-7 together.  With two
    parts an operand is off by 2^-17 of itself at most, and that is above the bar for these inputs (shown in float64)."""
    bar = 1e-6
    ids = _ids(of, count, how)
    x, y, A, B, ids, scales, _, dy = _make(dev, lead, ids, count, R, K, N, torch.float32)
    want, _ = _formula(x, y, A, B, ids, scales, dy)
    leaves = [t.clone().requires_grad_() for t in (A, B)]
    got = torch.autograd.grad(k2.add_adapters(y, x, *leaves, ids, scales), leaves, dy)
    for g, w in zip(got, want[2:]):
        assert float((g.double() - w).norm()) <= bar * float(w.norm())
    rows = x.shape[:-1].numel()
    each = ids.reshape(-1).repeat_interleave(rows // ids.numel())
    off = torch.zeros(2, dtype=torch.float64)
    for a in range(count):
        at = (each == a).nonzero()[:, 0]
        xa, da, s = x.reshape(rows, K)[at].double(), dy.reshape(rows, N)[at].double(), float(scales[a])
        g, u = s * da @ _two_parts(B[a]), s * xa @ _two_parts(A[a]).t()
        off[0] += float((_two_parts(g.float()).t() @ xa - want[2][a]).square().sum())
        off[1] += float((da.t() @ _two_parts(u.float()) - want[3][a]).square().sum())
    assert all(float(o) ** 0.5 > bar * float(w.norm()) for o, w in zip(off, want[2:]))


# -- batches without rows ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["w8a8", "linear"])
def test_a_batch_without_rows_trains_nothing(k2, dev, kind):
    """Its pass back gives zeros, as products of no rows do."""
    bank = k2.LoRABank(_linear(k2, dev, 256, 256, kind), 2, 16)
    x = torch.zeros(0, 5, 256, device=dev, dtype=torch.bfloat16, requires_grad=True)
    out = bank(x, torch.zeros(0, dtype=torch.int64, device=dev))
    assert out.shape == (0, 5, 256)
    out.float().sum().backward()
    assert x.grad.shape == x.shape
    for p in (bank.lora_A, bank.lora_B):
        assert p.grad.shape == p.shape and p.grad.dtype == p.dtype and not int(p.grad.count_nonzero())


# -- adapters without rows --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_adapters_without_rows_are_stepped_as_zero_gradients(k2, dev, bits):
    """A bank's adapters are one parameter: the step decays one that no row had, and moves one that had rows before on, as
    torch's step does with a gradient of zeros.  Without decay, one that never had rows stays bit for bit."""
    banks = []
    for decay in (0.0, 0.1):
        torch.manual_seed(0)
        bank = k2.LoRABank(_linear(k2, dev, 128, 192, "linear"), 3, 16)
        with torch.no_grad():
            bank.lora_B.normal_()
        banks.append((bank, k2.AdamW([bank.lora_A, bank.lora_B], lr=1e-2, weight_decay=decay, state_bits=bits)))
    alike = copy.deepcopy(banks[1][0])
    other = torch.optim.AdamW([alike.lora_A, alike.lora_B], lr=1e-2, weight_decay=0.1)
    x = torch.randn(2, 9, 128, generator=torch.Generator().manual_seed(1)).to(dev).bfloat16()
    start = [p.detach().clone() for p in (banks[0][0].lora_A, banks[0][0].lora_B)]
    before = None
    for ids in ([0, 1], [1, 1]):        # adapter 0 in the first step alone, adapter 2 in none
        ids = torch.tensor(ids, device=dev)
        for bank, opt in banks:
            opt.zero_grad()
            bank(x, ids).float().square().sum().backward()
        for p, q in zip((alike.lora_A, alike.lora_B), (banks[1][0].lora_A, banks[1][0].lora_B)):
            p.grad = q.grad.clone()
        before = [p.detach().clone() for p in (banks[1][0].lora_A, banks[1][0].lora_B)]
        for _, opt in banks:
            opt.step()
        other.step()
    for p, s in zip((banks[0][0].lora_A, banks[0][0].lora_B), start):
        assert torch.equal(p[2], s[2])                      # no decay and never a row
    for p, q, b, s in zip((banks[1][0].lora_A, banks[1][0].lora_B), (alike.lora_A, alike.lora_B), before, start):
        if bits == 32:
            # two updates of 1e-2, each off by 8 roundings of its terms
            assert bool(((p - q).abs() <= 2.0 ** -22 * q.abs() + 2 * 1e-2 * 2.0 ** -20).all())
        # two steps of 1 - 1e-2 * 0.1, each rounded once, and the factor itself
        assert bool(((p[2].double() - s[2].double() * (1 - 1e-3) ** 2).abs() <= 4 * 2.0 ** -24 * s[2].abs()).all())
        assert not torch.equal(p[0], b[0])                  # on its momentum


# -- a base that changes ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["w8a8", "w4a8", "fp8"])
def test_a_base_changed_in_place_between_the_passes_is_refused(k2, dev, kind):
    """As autograd refuses it where LoRALinear's node saves the weights."""
    base = _linear(k2, dev, 256, 256, kind)
    bank = k2.LoRABank(base, 1, 16)
    x = torch.randn(4, 256, device=dev).bfloat16().requires_grad_()
    ids = torch.zeros(4, dtype=torch.int64, device=dev)
    out = bank(x, ids)
    with torch.no_grad():
        weight = base.weight_fp8 if kind == "fp8" else base.qweight
        weight.view(torch.uint8).add_(1) if kind == "fp8" else weight.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()
    bank(x, ids).float().sum().backward()


# -- requests of threads ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reentrant", [True, False])
def test_recomputed_passes_use_the_requests_of_the_thread_that_called_them(k2, dev, reentrant):
    """Two threads with requests of their own and one without, their bodies open all at once, one backward pass after another:
    each gets the gradients that it gets alone."""
    bank = k2.LoRABank(_linear(k2, dev, 256, 256, "w8a8"), 2, 16)
    with torch.no_grad():
        bank.lora_B.normal_(0.0, 0.1)
    x = torch.randn(2, 8, 256, device=dev).bfloat16()
    wanted = [torch.tensor([0, 1], device=dev), None, torch.tensor([1, -1], device=dev)]

    def forward(leaf):
        return checkpoint(lambda t: bank(bank(t)), leaf, use_reentrant=reentrant)

    def grads(y, leaf):
        bank.zero_grad()
        y.float().square().sum().backward()
        out = [t.grad for t in (leaf, bank.lora_A, bank.lora_B)]
        return [None if t is None else t.clone() for t in out]

    alone = []
    for ids in wanted:
        leaf = x.clone().requires_grad_()
        with k2.lora_requests(bank, ids) if ids is not None else contextlib.nullcontext():
            alone.append(grads(forward(leaf), leaf))
    got, errors, gate = [None] * 3, [], threading.Barrier(3, timeout=60)

    def work(i):
        try:
            leaf = x.clone().requires_grad_()
            with k2.lora_requests(bank, wanted[i]) if wanted[i] is not None else contextlib.nullcontext():
                y = forward(leaf)
                for turn in (2, 0, 1):
                    gate.wait()
                    if turn == i:
                        got[i] = grads(y, leaf)
                    gate.wait()
        except Exception as e:          # noqa: BLE001 - shown below
            errors.append(e)
            gate.abort()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for a, b in zip(got, alone):
        assert all((p is None) == (q is None) and (p is None or torch.equal(p, q)) for p, q in zip(a, b))
    assert alone[1][1] is None and not torch.equal(alone[0][0], alone[2][0])


# -- recomputed passes ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reentrant", [True, False])
def test_a_pass_recomputed_outside_its_body_is_refused(k2, dev, reentrant):
    """On autograd's own thread: it would run without the adapters, whose factors would get no gradients."""
    bank = k2.LoRABank(_linear(k2, dev, 256, 256, "w8a8"), 2, 16)
    x = torch.randn(2, 8, 256, device=dev).bfloat16().requires_grad_()
    ids = torch.tensor([0, 1], device=dev)
    with k2.lora_requests(bank, ids):
        y = checkpoint(lambda t: bank(bank(t)), x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="outside the lora_requests body"):
        y.float().sum().backward()
    with k2.lora_requests(bank, ids):
        checkpoint(lambda t: bank(bank(t)), x, use_reentrant=reentrant).float().sum().backward()
    assert bank.lora_B.grad is not None
    bank.zero_grad()
    checkpoint(lambda t: bank(bank(t)), x, use_reentrant=reentrant).float().sum().backward()      # the base alone
    assert bank.lora_B.grad is None
