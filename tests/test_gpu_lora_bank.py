"""GPU tests of the adapters of many requests beside one projection: values and gradients against the formulas in float64,
rows without adapter, every order of rows, and the bank's module."""
import copy

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _make(dev, lead, ids, count, R, K, N, dtype, ranks=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*lead, K, generator=g).bfloat16()
    x[..., 1] *= 20
    y = torch.randn(*lead, N, generator=g).bfloat16()
    A = torch.randn(count, R, K, generator=g) * K ** -0.5
    B = torch.randn(count, N, R, generator=g) * 0.2
    if ranks is not None:
        for a, r in enumerate(ranks):
            A[a, r:], B[a, :, r:] = 0, 0
    scales = torch.rand(count, generator=g) + 0.5
    dy = torch.randn(*lead, N, generator=g).bfloat16()
    rk = None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device=dev)
    return x.to(dev), y.to(dev), A.to(dev, dtype), B.to(dev, dtype), ids.to(dev), scales.to(dev), rk, dy.to(dev)


def _formula(x, y, A, B, ids, scales, dy=None):
    """(out, dx, dA, dB) in float64, and the sums of magnitudes behind each: what roundings are counted against."""
    rows = x.shape[:-1].numel()
    K, N, count = x.shape[-1], y.shape[-1], A.shape[0]
    ids = ids.reshape(-1).repeat_interleave(rows // ids.numel())
    x2, y2 = x.reshape(rows, K).double(), y.reshape(rows, N).double()
    d2 = None if dy is None else dy.reshape(rows, N).double()
    out, size = y2.clone(), torch.zeros_like(y2)
    res = [torch.zeros(rows, K, dtype=torch.float64, device=x.device), torch.zeros(A.shape, dtype=torch.float64, device=x.device),
           torch.zeros(B.shape, dtype=torch.float64, device=x.device)]
    sizes = [torch.zeros_like(r) for r in res]
    for a in range(count):
        at = (ids == a).nonzero()[:, 0]
        Aa, Ba, s = A[a].double(), B[a].double(), float(scales[a])
        u, su = s * x2[at] @ Aa.t(), s * x2[at].abs() @ Aa.abs().t()
        out[at] += u @ Ba.t()
        size[at] = su @ Ba.abs().t()
        if d2 is not None:
            g, sg = s * d2[at] @ Ba, s * d2[at].abs() @ Ba.abs()
            res[0][at], sizes[0][at] = g @ Aa, sg @ Aa.abs()
            res[1][a], sizes[1][a] = g.t() @ x2[at], sg.t() @ x2[at].abs()
            res[2][a], sizes[2][a] = d2[at].t() @ u, d2[at].abs().t() @ su
    res[0], sizes[0] = res[0].view(x.shape), sizes[0].view(x.shape)
    return [out.view(y.shape), *res], [size.view(y.shape), *sizes]


def _check(got, want, size, terms, dtype):
    """Roundings, of the sums' magnitudes: each operand in f32 enters a product as two bf16 parts (off by 2^-16 of it; two of
    them, and the product of both rests that is left out, in each of two products: 6 at most), each f32 sum of n terms n of
    2^-24; and the result's own."""
    half = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[got.dtype]
    d = (got.double() - want).abs()
    bound = half * want.abs() + size * (6 * 2.0 ** -16 + terms * 2.0 ** -24) * (1 + half)
    assert bool((d <= bound).all()), float((d - bound).max())


CASES = {
    # name: (leading dimensions, the ids' dimensions, adapters, rank, in, out)
    "token": ((1,), (1,), 1, 16, 64, 64),
    "tokens": ((9, 1), (9,), 4, 16, 192, 320),
    "flat": ((65,), (65,), 3, 32, 320, 64),
    "batch": ((3, 50), (3,), 5, 48, 128, 256),
    "grid": ((2, 33, 3), (2, 33), 40, 64, 64, 192),
    "one": ((2, 300), (2,), 1, 16, 256, 576),
    "deep": ((70,), (70,), 2, 144, 64, 128),
    "deeper": ((5, 13), (5,), 3, 272, 128, 64),
    "wide": ((130,), (130,), 6, 16, 1088, 1344),
    "many": ((40, 2), (40,), 300, 16, 64, 64),
}


def _ids(shape, count, how, seed=1):
    g = torch.Generator().manual_seed(seed)
    n = torch.Size(shape).numel()
    if how == "sorted":
        t = torch.randint(0, count, shape, generator=g).reshape(-1).sort().values.view(shape)
    elif how == "mixed":        # any order, some without an adapter, numbers that are none's
        t = torch.randint(-1, count, shape, generator=g)
        t.view(-1)[n // 2] = count
        if n > 3:
            t.view(-1)[1], t.view(-1)[2] = -(1 << 40), (1 << 40) + 1
    else:
        t = torch.full(shape, -1)
    return t


@pytest.mark.parametrize("how", ["sorted", "mixed", "none"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", list(CASES))
def test_values_and_gradients(k2, dev, case, dtype, how):
    _values_and_gradients(k2, dev, *CASES[case], dtype, how)


def _values_and_gradients(k2, dev, lead, of, count, R, K, N, dtype, how):
    ids = _ids(of, count, how)
    x, y, A, B, ids, scales, _, dy = _make(dev, lead, ids, count, R, K, N, DTYPES[dtype])
    want, size = _formula(x, y, A, B, ids, scales, dy)
    with torch.no_grad():
        served = k2.add_adapters(y, x, A, B, ids, scales)
    leaves = [t.clone().requires_grad_() for t in (y, x, A, B)]
    out = k2.add_adapters(*leaves, ids, scales)
    grads = torch.autograd.grad(out, leaves, dy)
    rows = out.shape[:-1].numel()
    assert torch.equal(out, served)
    assert torch.equal(grads[0], dy)
    for got, w, s, terms in zip((out.detach(), *grads[1:]), want, size, (K + R, N + R, N + rows, K + rows)):
        assert got.shape == w.shape
        _check(got, w, s, terms, dtype)
    again = torch.autograd.grad(k2.add_adapters(*leaves, ids, scales), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    if how == "none":
        assert torch.equal(out, y) and not any(int(g.count_nonzero()) for g in grads[1:])


@pytest.mark.parametrize("how", ["sorted", "mixed"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lead, of, count, R, K, N", [
    ((80,), (80,), 1, 32, 192, 320), ((81,), (81,), 1, 32, 192, 320),           # single rows and tiles, either side of the
    ((176,), (176,), 7, 48, 320, 64), ((177,), (177,), 7, 48, 320, 64),         # rule between them
    ((768,), (768,), 64, 16, 64, 192), ((769,), (769,), 64, 16, 64, 192),
    ((5, 20), (5,), 5, 64, 128, 64), ((3, 50), (3,), 5, 64, 128, 64),
    ((2, 30), (2,), 3, 32, 1536, 320), ((2, 30), (2,), 3, 32, 1600, 320),       # single rows in one launch, or in two
    ((3,), (3,), 2, 16, 3008, 256), ((1,), (1,), 1, 16, 6144, 64), ((700,), (700,), 50, 16, 64, 8192),
    ((300,), (300,), 6, 144, 1088, 192), ((4, 500), (4,), 3, 64, 1088, 5120),   # slices that "up" adds up, and the join
    ((1000,), (1000,), 40, 64, 1088, 576), ((300,), (300,), 6, 144, 64, 128), ((11, 40), (11,), 9, 272, 128, 1344)])
def test_single_rows_and_tiles(k2, dev, lead, of, count, R, K, N, dtype, how):
    _values_and_gradients(k2, dev, lead, of, count, R, K, N, dtype, how)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 64, 65, 127, 255, 256, 257, 300, 513])
def test_every_length(k2, dev, rows):
    """One request after another, rows of a batch entry for each, lengths around the tiles' and the pieces'."""
    for lead, of in (((rows,), (rows,)), ((3, rows), (3,))):
        ids = _ids(of, 2, "mixed", seed=rows)
        x, y, A, B, ids, scales, _, dy = _make(dev, lead, ids, 2, 16, 64, 128, torch.float32, seed=rows)
        want, size = _formula(x, y, A, B, ids, scales, dy)
        leaves = [t.clone().requires_grad_() for t in (x, A, B)]
        out = k2.add_adapters(y, *leaves, ids, scales)
        grads = torch.autograd.grad(out, leaves, dy)
        n = out.shape[:-1].numel()
        for got, w, s, terms in zip((out.detach(), *grads), want, size, (80, 144, 128 + n, 64 + n)):
            _check(got, w, s, terms, "f32")


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_ranks_of_their_own(k2, dev, dtype):
    """Adapters of several ranks in one bank: past an adapter's rank (rounded up to 16) nothing is read, and the gradients are
    zeros."""
    ranks = [16, 0, 64, 33, 128]
    ids = _ids((90,), 5, "mixed")
    x, y, A, B, ids, scales, rk, dy = _make(dev, (90,), ids, 5, 128, 128, 192, DTYPES[dtype], ranks)
    want, size = _formula(x, y, A, B, ids, scales, dy)
    for a, r in enumerate(ranks):
        A[a, -(-r // 16) * 16:], B[a, :, -(-r // 16) * 16:] = float("nan"), float("nan")
    leaves = [t.clone().requires_grad_() for t in (x, A, B)]
    out = k2.add_adapters(y, *leaves, ids, scales, rk)
    grads = torch.autograd.grad(out, leaves, dy)
    for got, w, s, terms in zip((out.detach(), *grads), want, size, (256, 320, 290, 220)):
        for a, r in enumerate(ranks):       # between a rank and its 16 the factors are zeros: their gradients are too
            if w is want[2]:
                assert not int(got[a, -(-r // 16) * 16:].count_nonzero())
            if w is want[3]:
                assert not int(got[a, :, -(-r // 16) * 16:].count_nonzero())
        _check(got, w, s, terms, dtype)


def test_gradients_against_differences(k2, dev):
    """The output is linear in x, in A and in B, so the gradient along a direction is a difference of two outputs, each off by
    its own rounding of 2^-8."""
    ids = _ids((50,), 3, "mixed")
    x, y, A, B, ids, scales, _, dy = _make(dev, (50,), ids, 3, 16, 128, 64, torch.float32)
    leaves = [t.clone().requires_grad_() for t in (x, A, B)]
    grads = torch.autograd.grad(k2.add_adapters(y, *leaves, ids, scales), leaves, dy)
    g = torch.Generator().manual_seed(7)
    for i, t in enumerate(leaves):
        step = torch.randn(t.shape, generator=g).to(dev).bfloat16().to(t.dtype)
        moved = [v.detach().clone() for v in leaves]
        moved[i] = (moved[i] + step).to(t.dtype)
        step = moved[i].double() - t.detach().double()
        outs = [k2.add_adapters(torch.zeros_like(y), *v, ids, scales).double() for v in (moved, [v.detach() for v in leaves])]
        want = float((dy.double() * (outs[0] - outs[1])).sum())
        off = float((dy.double().abs() * (outs[0].abs() + outs[1].abs())).sum()) * (2.0 ** -8 + 2.0 ** -13)
        # a gradient in bf16 (x's) is off by 2^-8 of each of its values
        off += float((grads[i].double().abs() * step.abs()).sum()) * (2.0 ** -8 if i == 0 else 2.0 ** -13)
        assert abs(float((grads[i].double() * step).sum()) - want) <= off


def test_some_gradients_alone(k2, dev):
    ids = _ids((70,), 3, "mixed")
    x, y, A, B, ids, scales, _, dy = _make(dev, (70,), ids, 3, 32, 128, 64, torch.float32)
    leaves = [t.clone().requires_grad_() for t in (y, x, A, B)]
    every = torch.autograd.grad(k2.add_adapters(*leaves, ids, scales), leaves, dy)
    for which in range(1, 16):
        some = [t.detach().requires_grad_(bool(which >> i & 1)) for i, t in enumerate((y, x, A, B))]
        asked = [t for t in some if t.requires_grad]
        got = torch.autograd.grad(k2.add_adapters(*some, ids, scales), asked, dy)
        want = [e for i, e in enumerate(every) if which >> i & 1]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), which


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite_stay_in_their_rows(k2, dev, bad):
    ids = torch.tensor([0, 1, -1, 0, 1] * 8)
    x, y, A, B, ids, scales, _, dy = _make(dev, (40,), ids, 2, 16, 64, 64, torch.float32)
    want, size = _formula(x, y, A, B, ids, scales, dy)
    x[0, 3] = x[2, 5] = bad           # a row of adapter 0, and one without
    dy[0, 3] = bad
    leaves = [t.clone().requires_grad_() for t in (x, A, B)]
    out = k2.add_adapters(y, *leaves, ids, scales)
    grads = torch.autograd.grad(out, leaves, dy)
    assert not torch.isfinite(out[0]).all() and torch.isfinite(out[1:]).all()
    assert torch.equal(out[2], y[2])
    _check(out.detach()[1:], want[0][1:], size[0][1:], 80, "f32")
    _check(grads[0][1:], want[1][1:], size[1][1:], 80, "f32")
    for got, w, s in zip(grads[1:], want[2:], size[2:]):
        _check(got[1], w[1], s[1], 104, "f32")
        assert not torch.isfinite(got[0]).all()
    B[0, 3, 2] = bad                  # a factor of adapter 0 alone
    out = k2.add_adapters(y, x, A, B, ids, scales)
    others = (ids != 0).nonzero()[:, 0]
    _check(out[others], want[0][others], size[0][others], 80, "f32")


def test_forms_of_arguments(k2, dev):
    """Ids in 32 bits, no scales, one scale for all, operands that are not contiguous or aligned, no rows."""
    ids = _ids((3,), 4, "mixed")
    x, y, A, B, ids, scales, _, dy = _make(dev, (3, 20), ids, 4, 16, 128, 192, torch.float32)
    ids = torch.tensor([3, -1, 1], device=dev)
    want = k2.add_adapters(y, x, A, B, ids, scales)
    assert torch.equal(k2.add_adapters(y, x, A, B, ids.int(), scales), want)
    assert torch.equal(k2.add_adapters(y, x, A, B, ids.view(3, 1).expand(3, 20), scales), want)
    assert torch.equal(k2.add_adapters(y, x, A, B, ids, scales * 4, scale=0.25), want)
    ones = k2.add_adapters(y, x, A, B, ids, torch.ones_like(scales))
    assert torch.equal(k2.add_adapters(y, x, A, B, ids), ones)
    apart = torch.empty(3, 20, 129, device=dev, dtype=torch.bfloat16)[..., 1:]
    apart.copy_(x)
    turned = y.transpose(0, 1).contiguous().transpose(0, 1)
    strided = torch.stack([A, A], -1)[..., 0]
    leaves = [t.requires_grad_() for t in (turned, apart, strided)]
    out = k2.add_adapters(*leaves, B, ids, scales)
    assert torch.equal(out, want)
    plain = [t.clone().requires_grad_() for t in (y, x, A)]
    far = torch.empty(3, 20, 193, device=dev, dtype=torch.bfloat16)[..., :-1]
    far.copy_(dy)
    near = torch.autograd.grad(k2.add_adapters(*plain, B, ids, scales), plain, dy)
    for a, b in zip(torch.autograd.grad(out, leaves, far), near):
        assert torch.equal(a, b)
    none = k2.add_adapters(y[:0], x[:0], A, B, ids[:0], scales)
    assert none.shape == (0, 20, 192)
    with pytest.raises(NotImplementedError):
        k2.add_adapters(y, x, A, B, ids, scales.clone().requires_grad_())
    for bad in (lambda: k2.add_adapters(y, x, A, B, ids[:2], scales), lambda: k2.add_adapters(y, x, A, B, ids.float(), scales),
                lambda: k2.add_adapters(y, x, A, B.bfloat16(), ids, scales), lambda: k2.add_adapters(y[:2], x, A, B, ids, scales),
                lambda: k2.add_adapters(y, x, A[:, :8].contiguous(), B[..., :8].contiguous(), ids, scales),
                lambda: k2.add_adapters(y, x, A, B, ids, scales[:3]), lambda: k2.add_adapters(y, x, A, B, ids.cpu(), scales),
                lambda: k2.add_adapters(y, x, A[:3], B, ids, scales)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        k2.add_adapters(y.float(), x.float(), A, B, ids, scales)


def test_offsets_past_32_bits(k2, dev):
    """More than 2^32 elements of the output: the last rows' values and gradients."""
    T, K, N = 66000, 64, 65536
    ids = torch.full((T,), -1)
    ids[-70:] = torch.arange(70) % 2
    y = torch.zeros(T, N, device=dev, dtype=torch.bfloat16)
    x, tail, A, B, ids, scales, _, dy = _make(dev, (70,), ids, 2, 16, K, N, torch.float32)
    every = torch.zeros(T, K, device=dev, dtype=torch.bfloat16)
    every[-70:] = x
    y[-70:] = tail
    want, size = _formula(x, tail, A, B, ids[-70:], scales, dy)
    leaves = [t.requires_grad_() for t in (every, A, B)]
    out = k2.add_adapters(y, *leaves, ids, scales)
    _check(out.detach()[-70:], want[0], size[0], K + 16, "f32")
    assert not int(out[:70].count_nonzero()) and not int(out[32000:32100].count_nonzero())
    grad = torch.zeros(T, N, device=dev, dtype=torch.bfloat16)
    grad[-70:] = dy
    del y
    grads = torch.autograd.grad(out, leaves, grad)
    _check(grads[0][-70:], want[1], size[1], N + 16, "f32")
    assert not int(grads[0][:-70].count_nonzero())
    for got, w, s, terms in zip(grads[1:], want[2:], size[2:], (N + 70, K + 70)):
        _check(got, w, s, terms, "f32")


def test_streams_and_captures(k2, dev):
    """A captured pass follows its static ids, inputs and factors; two graphs and another stream do not meet."""
    ids = _ids((6,), 3, "mixed")
    x, y, A, B, ids, scales, _, dy = _make(dev, (6, 40), ids, 3, 16, 128, 192, torch.float32)
    ids = ids.clamp(-1, 3)
    static = [t.clone() for t in (y, x, A, B)]
    leaves = [static[0], *(t.requires_grad_() for t in static[1:])]
    number = ids.clone()

    def call(y, x, A, B, ids):
        out = k2.add_adapters(y, x, A, B, ids, scales)
        return [out.detach(), *torch.autograd.grad(out, [x, A, B], dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = call(*leaves, number)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(warm, call(*leaves, number)))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call(*leaves, number))
    for s in range(4):
        new = [torch.randn(t.shape, generator=torch.Generator().manual_seed(s)).to(dev, t.dtype) for t in leaves]
        with torch.no_grad():
            for t, v in zip(leaves, new):
                t.copy_(v)
        number.copy_(torch.randint(-1, 3, (6,), generator=torch.Generator().manual_seed(s)))
        graphs[s % 2].replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs[s % 2]]
        graphs[1 - s % 2].replay()
        torch.cuda.synchronize()
        want = call(*[v.requires_grad_(i > 0) for i, v in enumerate(new)], number.clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(outs[1 - s % 2], want))


def test_refuses_tangents_and_second_gradients(k2, dev):
    ids = torch.zeros(4, dtype=torch.int64)
    x, y, A, B, ids, scales, _, dy = _make(dev, (4,), ids, 1, 16, 64, 64, torch.float32)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
        k2.add_adapters(y, fwad.make_dual(x, torch.ones_like(x)), A, B, ids, scales)
    x.requires_grad_()
    first, = torch.autograd.grad(k2.add_adapters(y, x, A, B, ids, scales), x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.float().sum(), x)


# -- the module -------------------------------------------------------------------------------------------------------
def _linear(k2, dev, K, N, kind, seed=0):
    lin = nn.Linear(K, N, bias=False, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=torch.Generator().manual_seed(seed)) * 0.05)
    return {"w8a8": lambda: k2.ConvRotLinear(lin, "w8a8"), "w4a8": lambda: k2.ConvRotLinear(lin, "w4a8"),
            "fp8": lambda: k2.Fp8Linear(lin), "linear": lambda: lin}[kind]()


@pytest.mark.parametrize("kind", ["w8a8", "w4a8", "fp8", "linear"])
def test_bank_beside_every_base(k2, dev, kind):
    """Each request's rows are base(x) plus its adapter (the formula's, from the base's own output), and what LoRALinear gives
    with that adapter, up to roundings: 2^-8 of the base's output and of both sums, and 2^-8 of u and of B in every product of
    LoRALinear's second one, whose operands are bf16 (over a plain linear: 2^-8 of the product), which is 2^-7 of the sum of
    their magnitudes."""
    base = _linear(k2, dev, 256, 384, kind)
    bank = k2.LoRABank(base, 3, 20, 40.0)
    assert bank.lora_A.shape == (3, 32, 256) and bank.lora_B.shape == (3, 384, 32)
    g = torch.Generator().manual_seed(2)
    single = []
    for a, r in enumerate((20, 8, 32)):
        A, B = (torch.randn(r, 256, generator=g) * 0.05).to(dev), (torch.randn(384, r, generator=g) * 0.05).to(dev)
        bank.set_adapter(a, A, B, alpha=2.0 * r + a)
        one = k2.LoRALinear(base, r, 2.0 * r + a)
        with torch.no_grad():
            one.lora_A.copy_(A)
            one.lora_B.copy_(B)
        single.append(one)
        back = bank.adapter(a)
        assert torch.equal(back[0], A) and torch.equal(back[1], B) and abs(back[2] - (2.0 * r + a)) < 1e-4
    x = torch.randn(5, 30, 256, generator=g).to(dev).bfloat16()
    ids = torch.tensor([2, 0, -1, 1, 2], device=dev)
    with torch.no_grad():
        y = base(x)
        assert torch.equal(bank(x), y)
        out = bank(x, ids)
        want, size = _formula(x, y, bank.lora_A, bank.lora_B, ids, bank.scales)
        _check(out, want[0], size[0], 256 + 32, "f32")
        for i, a in enumerate(ids.tolist()):
            if a < 0:
                assert torch.equal(out[i], y[i])
                continue
            one = single[a](x[i]).double()
            u = single[a].scale * x[i].double() @ single[a].lora_A.double().t()
            terms = u.abs() @ single[a].lora_B.double().abs().t()
            bound = 2.0 ** -8 * (y[i].double().abs() + out[i].double().abs() + one.abs()) + 2.0 ** -7 * terms
            assert bool(((out[i].double() - one).abs() <= bound * (1 + 2.0 ** -6) + 2.0 ** -12 * size[0][i]).all())
        with k2.lora_requests(bank, ids):
            assert torch.equal(bank(x), out)
            with k2.lora_requests(bank, None):
                assert torch.equal(bank(x), y)
            with k2.lora_scaled(bank, 0.5):
                half = bank(x)
            assert torch.equal(half, k2.add_adapters(y, x, bank.lora_A, bank.lora_B, ids, bank.scales * 0.5, bank.ranks))
            with k2.lora_disabled(bank):
                assert torch.equal(bank(x), y)
        assert torch.equal(bank(x), y)
        cast = copy.deepcopy(bank).to(torch.float16).to(torch.float32)
        assert torch.equal(cast.scales, bank.scales) and torch.equal(cast.ranks, bank.ranks)


@pytest.mark.parametrize("kind", ["w8a8", "w4a8", "fp8", "linear"])
def test_bank_gradients_beside_every_base(k2, dev, kind):
    """x's gradient is the base's plus the adapters': each rounded once, and their sum."""
    base = _linear(k2, dev, 256, 384, kind)
    bank = k2.LoRABank(base, 3, 16)
    with torch.no_grad():
        bank.lora_B.normal_(0.0, 0.05)
    x = torch.randn(4, 30, 256, generator=torch.Generator().manual_seed(0)).to(dev).bfloat16()
    dy = torch.randn(4, 30, 384, generator=torch.Generator().manual_seed(1)).to(dev).bfloat16()
    ids = torch.tensor([1, -1, 0, 1], device=dev)
    xa, xb = x.clone().requires_grad_(), x.clone().requires_grad_()
    out = bank(xa, ids)
    dx, dA, dB = torch.autograd.grad(out, [xa, bank.lora_A, bank.lora_B], dy)
    own, = torch.autograd.grad(base(xb), xb, dy)
    want, size = _formula(x, torch.zeros_like(dy), bank.lora_A.detach(), bank.lora_B.detach(), ids, bank.scales, dy)
    near = (dx.double() - (own.double() + want[1])).abs()
    parts = own.double().abs() + want[1].abs()
    assert bool((near <= parts * (3 * 2.0 ** -8) + size[1] * 2.0 ** -13).all())
    _check(dA, want[2], size[2], 384 + 120, "f32")
    _check(dB, want[3], size[3], 256 + 120, "f32")
    assert not int(dA[2].count_nonzero()) and not int(dB[2].count_nonzero())


def test_two_streams_at_once(k2, dev):
    """Calls on two streams share no workspace: each gives what it gives alone."""
    a = _make(dev, (300,), _ids((300,), 5, "mixed"), 5, 32, 256, 320, torch.float32)
    b = _make(dev, (70,), _ids((70,), 5, "mixed", seed=2), 5, 32, 256, 320, torch.float32, seed=7)

    def call(x, y, A, B, ids, scales, _, dy):
        leaves = [t.detach().requires_grad_() for t in (x, A, B)]
        out = k2.add_adapters(y, *leaves, ids, scales)
        return (out.detach(), *torch.autograd.grad(out, leaves, dy))

    want = [call(*a), call(*b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        for s, args in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(call(*args))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g, want[i % 2])), i
