"""GPU tests of adapters that share a base, as they are used: several trained at once through quantized blocks (banks, the
gradients' norm, AdamW), saved one by one, and served by request, each against adapters that run alone."""
import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from restated_block import Dit, FEAT

pytestmark = pytest.mark.gpu


def _dit(k2, dev, seed=0, mode="w8a8", fused=True):
    torch.manual_seed(seed)
    dit = Dit().to(dev, torch.bfloat16)
    for b in dit.blocks:
        b.mod.lin.data.normal_(0, 0.1)
    k2.quantize_dit_convrot(dit, mode)
    return dit


def _run(dit, x, vec):
    for b in dit.blocks:
        x = b(x, vec, None)
    return x


def _inputs(dev, requests, tokens, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(requests, tokens, FEAT, generator=g).to(dev).bfloat16()
    vec = (torch.randn(requests, 1, 6 * FEAT, generator=g) * 0.1).to(dev).bfloat16()
    return x, vec, torch.randn(requests, tokens, FEAT, generator=g).to(dev).bfloat16() * 1e-2


def _fill(banks, seed=2):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for b in banks.values():
            r = b.rank
            b.lora_B[..., :r] = (torch.randn(*b.lora_B.shape[:2], r, generator=g) * 0.05).to(b.lora_B.device)


@pytest.mark.parametrize("mode", ["w8a8", "w4a8"])
@pytest.mark.parametrize("grouped", [False, True])
def test_each_request_as_alone(k2, dev, tmp_path, mode, grouped):
    """A batch of requests with adapters of their own, and one without, against models that hold one of them, loaded from a
    bank's files (which hold bf16: the bank's factors are rounded to it first): outputs, and the gradients of each adapter
    and of the input.  Both sides round per linear, and a changed bit of an activation flips codes: the blocks' bars."""
    x, vec, dy = _inputs(dev, 4, 40)
    ids = torch.tensor([1, -1, 0, 1], device=dev)
    dit = _dit(k2, dev, mode=mode)
    if grouped:
        assert k2.group_siblings(dit) == (4 if mode == "w8a8" else 0)
    banks = k2.inject_lora_bank(dit, 3, 12, 24.0)
    _fill(banks)
    with torch.no_grad():
        for b in banks.values():
            for t in (b.lora_A, b.lora_B):
                t.copy_(t.bfloat16())
    k2.fuse_producers(dit)
    params = [t for b in banks.values() for t in (b.lora_A, b.lora_B)]
    leaf = x.clone().requires_grad_()
    with k2.lora_requests(dit, ids):
        out = _run(dit, leaf, vec)
        grads = torch.autograd.grad(out, [leaf, *params], dy)
        with torch.no_grad():
            served = _run(dit, x, vec)
    assert (out.detach() - served).double().norm() <= 1e-2 * served.double().norm()
    for a, path in ((0, "a"), (1, "b")):
        k2.save_lora_from(banks, a, str(tmp_path / path))
    for a, rows in ((0, [2]), (1, [0, 3]), (-1, [1])):
        one = _dit(k2, dev, mode=mode)
        adapters = {}
        if a >= 0:
            adapters = k2.load_lora(one, str(tmp_path / "ab"[a]))
            for m in adapters.values():
                m.scale = 2.0
        k2.fuse_producers(one)
        t = x[rows].clone().requires_grad_()
        alone = _run(one, t, vec[rows])
        assert (out.detach()[rows] - alone.detach()).double().norm() <= 1e-2 * alone.double().norm()
        want = torch.autograd.grad(alone, [t, *k2.lora_parameters(adapters)], dy[rows])
        assert (grads[0][rows] - want[0]).double().norm() <= 2e-2 * want[0].double().norm()
        for i, (name, m) in enumerate(adapters.items()):
            dA, dB = grads[1 + 2 * i][a, :12], grads[2 + 2 * i][a, :, :12]
            for got, e in ((dA, want[1 + 2 * i]), (dB, want[2 + 2 * i])):
                assert (got.double() - e.double()).norm() <= 2e-2 * e.double().norm(), name
    for i, b in enumerate(banks.values()):          # no request has adapter 2, and ranks 12 to 15 are padding
        assert not int(grads[1 + 2 * i][2].count_nonzero()) and not int(grads[2 + 2 * i][2].count_nonzero())
        assert not int(grads[1 + 2 * i][:, 12:].count_nonzero()) and not int(grads[2 + 2 * i][..., 12:].count_nonzero())


def test_codes_are_shared_and_recomputed_passes_are_equal(k2, dev):
    """The linears of a block that read one tensor make its codes once, with banks between them; a checkpointed step is the
    plain one bit for bit."""
    from krea2_amd.quantize import shared_input_quant
    x, vec, dy = _inputs(dev, 3, 24)
    dit = _dit(k2, dev)
    banks = k2.inject_lora_bank(dit, 2, 16)
    _fill(banks)
    ids = torch.tensor([1, 0, -1], device=dev)
    params = [t for b in banks.values() for t in (b.lora_A, b.lora_B)]

    def step(run):
        t = x.clone().requires_grad_()
        with k2.lora_requests(dit, ids):
            y = run(t)
            return [y.detach(), *torch.autograd.grad(y, [t, *params], dy)]

    before = shared_input_quant.misses
    plain = step(lambda t: _run(dit, t, vec))
    assert shared_input_quant.misses - before == 2 * 4      # a block: attention's input, wo's, the MLP's, down's
    again = step(lambda t: checkpoint(lambda u: _run(dit, u, vec), t, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(plain, again))


@pytest.mark.parametrize("bits", [32, 8])
def test_joint_training_and_serving(k2, dev, tmp_path, bits):
    """Two of three adapters trained at once: the third stays bit for bit, as do padded ranks; the weights follow AdamW's formula
    (float64, 32-bit moments); the state goes on after a save; a file of one adapter serves alone what the bank serves."""
    x, vec, dy = _inputs(dev, 4, 24)
    dit = _dit(k2, dev)
    banks = k2.inject_lora_bank(dit, 3, 8)
    _fill(banks)
    ids = torch.tensor([1, 0, -1, 1], device=dev)
    params = [t for b in banks.values() for t in (b.lora_A, b.lora_B)]
    opt = k2.AdamW(params, lr=1e-3, weight_decay=0.0, max_norm=0.5, state_bits=bits, seed=3)
    start = [p.detach().clone() for p in params]
    ref = [p.detach().double() for p in params]
    m, v = [torch.zeros_like(r) for r in ref], [torch.zeros_like(r) for r in ref]
    for t in range(1, 4):
        opt.zero_grad()
        with k2.lora_requests(dit, ids):
            _run(dit, x, vec).backward(dy)
        grads = [p.grad.double() for p in params]
        norm = math.sqrt(sum(float(g.square().sum()) for g in grads))
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -22 * norm
        by = min(1.0, 0.5 / (norm + 1e-6))
        for i, g in enumerate(grads):
            m[i] = 0.9 * m[i] + 0.1 * by * g
            v[i] = 0.999 * v[i] + 0.001 * (by * g) ** 2
            u = m[i] / (1 - 0.9 ** t) / ((v[i] / (1 - 0.999 ** t)).sqrt() + 1e-8)
            if bits == 32:
                # an update is m's rounding against sqrt(v) off: 8 roundings of its terms, which cancel at most 8 times here
                off = (params[i].detach().double() - (ref[i] - 1e-3 * u)).abs()
                assert bool((off <= 2.0 ** -22 * ref[i].abs() + 1e-3 * 2.0 ** -16).all())
            ref[i] = params[i].detach().double()
    for p, s in zip(params, start):
        assert torch.equal(p[2], s[2])
        assert not torch.equal(p[0], s[0]) and not torch.equal(p[1], s[1])
    for b in banks.values():
        assert not int(b.lora_A[:, 8:].count_nonzero()) and not int(b.lora_B[..., 8:].count_nonzero())
    k2.save_lora_from(banks, 1, str(tmp_path / "one"))
    bank2 = k2.inject_lora_bank(_dit(k2, dev), 5, 8, dtype=torch.bfloat16)
    assert k2.load_lora_into(bank2, 4, str(tmp_path / "one")) == 0
    name = "blocks.1.mlp.down"
    h = torch.randn(2, 3, banks[name].base.in_features, device=dev).bfloat16()
    with torch.no_grad():
        a = banks[name](h, torch.tensor([1, -1], device=dev))
        b = bank2[name](h, torch.tensor([4, 7], device=dev))
        assert torch.equal(a[1], b[1])
        # the file holds bf16 factors: 2^-8 of each in every product of two
        one = banks[name]
        size = (h[0].double().abs() @ one.lora_A[1].double().abs().t()) @ one.lora_B[1].double().abs().t()
        assert bool(((a[0] - b[0]).double().abs() <= size * 2.0 ** -7 * 1.02 + 2.0 ** -7 * a[0].double().abs()).all())


def test_captured_training_step(k2, dev):
    """Forward, backward, norm and step in one graph: every replay gives the eager step's weights, as the inputs and the
    requests change."""
    models = []
    for _ in range(2):
        dit = _dit(k2, dev)
        banks = k2.inject_lora_bank(dit, 2, 16)
        _fill(banks)
        params = [t for b in banks.values() for t in (b.lora_A, b.lora_B)]
        with torch.no_grad():
            for i, p in enumerate(params[0::2]):
                p.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(i)) * 0.05)
        models.append((dit, params, k2.AdamW(params, lr=1e-3, max_norm=1.0)))
    x, vec, dy = _inputs(dev, 3, 24)
    ids = torch.tensor([0, 1, -1], device=dev)

    def step(model, x, ids):
        dit, params, opt = model
        with k2.lora_requests(dit, ids):
            y = _run(dit, x, vec)
            for p, g in zip(params, torch.autograd.grad(y, params, dy)):
                p.grad = g
        opt.step()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(models[0], x, ids)
    torch.cuda.current_stream().wait_stream(side)
    step(models[1], x, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(models[0], x, ids)
    for s in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(20 + s)))
        ids.copy_(torch.randint(-1, 2, (3,), generator=torch.Generator().manual_seed(s)))
        graph.replay()
        torch.cuda.synchronize()
        step(models[1], x.clone(), ids.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(models[0][1], models[1][1]))
