"""GPU tests of the optimizer's step: AdamW over many tensors, its moments in 32 and in 8 bits, and the gradients' norm,
against the formulas in float64."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # a rounding, of the value
BLOCK = 256


def _params(dev, sizes, dtype, seed=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for s in sizes:
        n = math.prod(s)
        buf = torch.empty(n + offset, dtype=dtype, device=dev)
        p = torch.nn.Parameter(buf[offset:].view(s))
        with torch.no_grad():
            p.copy_(torch.randn(s, generator=g) * 0.1)
        p.grad = torch.empty(n + offset, dtype=dtype, device=dev)[offset:].view(s)
        p.grad.copy_(torch.randn(s, generator=g) * 0.01)
        out.append(p)
    return out


class _Formula:
    """AdamW in float64; parameters rounded to their type to nearest after every step."""

    def __init__(self, params, lr, betas, eps, decay, max_norm=None):
        self.p = [p.detach().double() for p in params]
        self.m = [torch.zeros_like(p) for p in self.p]
        self.v = [torch.zeros_like(p) for p in self.p]
        self.t = [0] * len(self.p)
        self.rest = lr, betas, eps, decay, max_norm

    def step(self, grads):
        lr, (b1, b2), eps, decay, most = self.rest
        gs = [None if g is None else g.double() for g in grads]
        if most is not None:
            norm = math.sqrt(sum(float(g.square().sum()) for g in gs if g is not None))
            gs = [None if g is None else g * min(1.0, most / (norm + 1e-6)) for g in gs]
        for i, g in enumerate(gs):
            if g is None:
                continue
            self.t[i] += 1
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
            u = self.m[i] / (1 - b1 ** self.t[i]) / ((self.v[i] / (1 - b2 ** self.t[i])).sqrt() + eps)
            self.p[i] = (1 - lr * decay) * self.p[i] - lr * u


def _near(got, want, rel, floor=0.0):
    d = (got.double() - want).abs()
    assert bool((d <= rel * want.abs() + floor).all()), float((d - rel * want.abs() - floor).max())


def _same(a, b):
    return torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


SIZES = {
    "one": [(1,)],
    "layer": [(16, 640), (384, 16)],
    "odd": [(3, 5), (257,), (8191, 3), (1, 1), (255,), (8192,), (8193,), (7, 1031)],
    "many": [(16, 8 + i % 3) for i in range(150)],
}


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("sizes", list(SIZES))
def test_steps_in_32_bits(k2, dev, sizes, dtype, offset):
    """Four steps.  A moment is two products and a sum a step (3 roundings of 2^-24, and 3 more in the squared gradient's
    share), over 4 steps under 24 of them; its constants beta and 1 - beta are off by 2^-24 and 2^-24 / (1 - beta2 = 0.001,
    held to 2^-24 of itself).  The update takes sqrt, quotient, sum and products: under 32 roundings; a parameter is its
    own rounding and lr times that."""
    dt = DTYPES[dtype]
    lr, betas, eps, decay = 1e-2, (0.9, 0.999), 1e-8, 0.05
    params = _params(dev, SIZES[sizes], dt, offset=offset)
    ref = _Formula(params, lr, betas, eps, decay)
    opt = k2.AdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=decay)
    for s in range(4):
        for i, p in enumerate(params):
            p.grad.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * s + i)) * 0.01)
        versions = [p._version for p in params]
        ref.step([p.grad for p in params])
        opt.step()
        assert all(p._version > v for p, v in zip(params, versions))
        for i, p in enumerate(params):
            st = opt.state[p]
            assert float(st["step"]) == s + 1
            m_scale = 0.04 * torch.ones_like(ref.m[i])      # terms of m may cancel: roundings count against their size
            _near(st["exp_avg"], ref.m[i], 24 * 2.0 ** -24, 24 * 2.0 ** -24 * 0.1 * m_scale)
            _near(st["exp_avg_sq"], ref.v[i], 32 * 2.0 ** -24)
            # |update| <= 1 / sqrt(1 - b2)-ish bounded by 4 here; m's error against its terms is carried into it
            m_err = 24 * 2.0 ** -24 * 0.004 / (ref.v[i] / (1 - betas[1] ** (s + 1))).sqrt().clamp(min=1e-12)
            _near(p.detach(), ref.p[i], HALF[dt] + 2.0 ** -23, lr * (64 * 2.0 ** -24 * 4 + m_err * 4))
            ref.p[i] = p.detach().double()


def test_equals_torch_on_one_more_step(k2, dev):
    """The moments of a torch optimizer that has run are taken over; the next step of both agrees to their roundings."""
    ours = _params(dev, [(64, 96), (33, 7)], torch.float32)
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    a = torch.optim.AdamW(theirs, lr=1e-3, weight_decay=0.1)
    b = k2.AdamW(ours, lr=5.0)
    for s in range(3):
        for p in theirs:
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(s)).to(dev)
        if s == 2:
            for p, q in zip(ours, theirs):
                p.data.copy_(q.data)
                p.grad = q.grad.clone()
            b.load_state_dict(a.state_dict())
            b.step()
        a.step()
    assert b.param_groups[0]["lr"] == 1e-3 and b.param_groups[0]["weight_decay"] == 0.1
    for p, q in zip(ours, theirs):
        assert float(b.state[p]["step"]) == 3
        _near(p.detach(), q.detach().double(), 2.0 ** -22, 1e-3 * 2.0 ** -18)


def test_parameters_without_a_gradient_stay(k2, dev):
    params = _params(dev, [(16, 24), (40,), (8, 8), (5, 5)], torch.float32)
    opt = k2.AdamW([{"params": params[:3], "lr": 1e-2}, {"params": params[3:], "lr": 1e-3, "betas": (0.8, 0.99)}])
    before = [p.detach().clone() for p in params]
    params[1].grad = None
    opt.step()
    assert torch.equal(params[1], before[1])
    assert [float(opt.state[p]["step"]) for p in params] == [1, 0, 1, 1]
    params[1].grad = torch.ones_like(params[1])
    params[0].grad = params[3].grad = None
    opt.step()
    assert [float(opt.state[p]["step"]) for p in params] == [1, 1, 2, 1]
    _near(params[1].detach(), before[1].double() * (1 - 1e-4) - 1e-2, 4 * 2.0 ** -24, 1e-2 * 2.0 ** -20)
    empty = torch.nn.Parameter(torch.empty(0, 4, device=dev))
    empty.grad = torch.empty_like(empty)
    opt = k2.AdamW([empty, params[0]], max_norm=1.0)
    opt.step()                                       # nothing to do
    assert opt.grad_norm is None


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("sizes", list(SIZES))
def test_norm_and_scaling(k2, dev, sizes, dtype):
    """The norm is a float64 sum rounded once; a scaled gradient has the factor's rounding, the product's and its type's."""
    params = _params(dev, SIZES[sizes], DTYPES[dtype])
    want = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
    for most in (2 * want, want / 3, 0.0):
        for p in params:
            p.grad.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(3)) * 0.01)
        grads = [p.grad.clone() for p in params]
        want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        versions = [p.grad._version for p in params]
        norm = k2.clip_grad_norm_(params, most)
        assert norm.dtype == torch.float32 and norm.shape == ()
        assert abs(float(norm) - want) <= 2.0 ** -23 * want
        by = min(1.0, most / (want + 1e-6))
        for p, g, version in zip(params, grads, versions):
            assert p.grad._version > version
            # float16's smallest step below its normal numbers: half of 2^-24
            _near(p.grad, g.double() * by, HALF[p.dtype] + 2.0 ** -22, 2.0 ** -25 if dtype == "f16" else 0.0)
    assert float(k2.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3, device=dev))], 1.0)) == 0
    one = params[0]
    assert torch.equal(k2.clip_grad_norm_(one, 1e9), k2.clip_grad_norm_([one], 1e9))


def test_norm_of_large_small_and_mixed_gradients(k2, dev):
    """Squares that leave float32's range, gradients that are transposed, and types side by side."""
    big = torch.nn.Parameter(torch.zeros(1000, device=dev))
    big.grad = torch.full_like(big, 1e25)
    assert abs(float(k2.clip_grad_norm_(big, 1.0)) / (1e25 * math.sqrt(1000)) - 1) < 2.0 ** -22
    assert abs(float(big.grad.double().square().sum()) - 1) < 1e-5
    small = torch.nn.Parameter(torch.zeros(1000, device=dev))
    small.grad = torch.full_like(small, 1e-30)
    assert abs(float(k2.clip_grad_norm_(small, 1.0)) / (1e-30 * math.sqrt(1000)) - 1) < 2.0 ** -22
    mixed = [p for name in DTYPES for p in _params(dev, [(33, 20)], DTYPES[name], seed=len(name))]
    turned = torch.nn.Parameter(torch.zeros(12, 20, device=dev))
    turned.grad = torch.randn(20, 12, generator=torch.Generator().manual_seed(1)).to(dev).t()
    mixed.append(turned)
    grads = [p.grad.double() for p in mixed]
    want = math.sqrt(sum(float(g.square().sum()) for g in grads))
    assert abs(float(k2.clip_grad_norm_(mixed, want / 2)) - want) <= 2.0 ** -23 * want
    for p, g in zip(mixed, grads):
        _near(p.grad, g * (want / 2 / (want + 1e-6)), HALF[p.dtype] + 2.0 ** -22, 2.0 ** -25)
    a, b = (torch.nn.Parameter(torch.zeros(5, device=dev)) for _ in range(2))
    for value in (float("inf"), float("nan")):
        for f, p in ((k2.clip_grad_norm_, a), (torch.nn.utils.clip_grad_norm_, b)):
            p.grad = torch.tensor([1.0, value, 0.0, -2.0, 3.0], device=dev)
            norm = f([p], 1.0)
            assert not math.isfinite(float(norm))
        assert torch.equal(a.grad.isnan(), b.grad.isnan()) and torch.equal(a.grad.nan_to_num(), b.grad.nan_to_num())


@pytest.mark.parametrize("bits", [32, 8])
def test_step_with_a_largest_norm(k2, dev, bits):
    """max_norm inside the step is clip_grad_norm_ before it, and leaves the gradients as they are."""
    sizes = SIZES["odd"]
    a, b = (_params(dev, sizes, torch.float32) for _ in range(2))
    oa, ob = k2.AdamW(a, max_norm=0.5, state_bits=bits), k2.AdamW(b, state_bits=bits)
    for s in range(3):
        grads = [torch.randn(p.shape, generator=torch.Generator().manual_seed(s)).to(dev) for p in a]
        for p, q, g in zip(a, b, grads):
            p.grad, q.grad = g.clone(), g.clone()
        oa.step()
        norm = k2.clip_grad_norm_(b, 0.5)
        ob.step()
        assert torch.equal(oa.grad_norm, norm)
        assert all(torch.equal(p.grad, g) for p, g in zip(a, grads))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        assert all(_same(x, y) for p, q in zip(a, b)
                   for x, y in zip(oa.state[p].values(), ob.state[q].values()))


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(k2, dev, bits, value):
    params = _params(dev, [(16, 40), (300,)], torch.float32)
    opt = k2.AdamW(params, max_norm=1.0, state_bits=bits)
    opt.step()
    params[1].grad[7] = value
    kept = [p.detach().clone() for p in params]
    state = copy.deepcopy(opt.state_dict()["state"])
    opt.step()                                       # skipped
    assert not math.isfinite(float(opt.grad_norm))
    assert all(torch.equal(p, k) for p, k in zip(params, kept))
    for i, p in enumerate(params):
        assert all(_same(opt.state[p][n], state[i][n]) for n in state[i])
    opt.max_norm = None
    opt.step()                                       # the element alone is spoilt
    assert torch.isfinite(params[0]).all()
    assert torch.nonzero(~torch.isfinite(params[1])).flatten().tolist() == [7]
    params[1].grad[7] = 0.0
    opt.step()
    assert torch.nonzero(~torch.isfinite(params[1])).flatten().tolist() == [7]
    m = opt.moments()[0]
    assert int((~torch.isfinite(m)).sum()) == 1


# -- moments in 8 bits ------------------------------------------------------------------------------------------------
def _mix(h):
    h = ((h ^ h >> 16) * 0x7FEB352D) & 0xFFFFFFFF
    h = ((h ^ h >> 15) * 0x846CA68B) & 0xFFFFFFFF
    return h ^ h >> 16


def _bits(seed, step, places):
    return _mix((places & 0xFFFFFFFF) ^ _mix(_mix(seed) ^ step) ^ ((places >> 32) * 0x9E3779B9 & 0xFFFFFFFF))


def _neighbours(a, places, low):
    """The number of ``places`` binary places at or below every value, and the step to the next one."""
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -140))).clamp(min=low) - places)
    return torch.floor(a / step) * step, step


def _held(a, places, low, top, random, least):
    """Blocks' values as codes hold them, from float64, and the size of a code's step at each."""
    n = a.numel()
    a = torch.nn.functional.pad(a, (0, -n % BLOCK)).view(-1, BLOCK)
    unit = (a.amax(1, keepdim=True) / top).expand_as(a).reshape(-1)[:n]
    a = a.reshape(-1)[:n]
    t = a / unit.clamp(min=2.0 ** -140)
    low_value, step = _neighbours(t, places, low)
    up = t / step - low_value / step + random >= 1
    out = low_value + up * step
    return torch.where((a > 0) & (out < least), least, out) * unit, step * unit


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1, 31, 255, 256, 257, 3000, 8192 + 77])
def test_moments_in_8_bits_follow_the_formula(k2, dev, size, dtype):
    """From the same state one step in float64 with the same random bits.  A value within 2^-18 of its border between two codes
    may fall to either side (the operands of the comparison are off by under 32 roundings of 2^-24, the random number's place
    by 2^-16 at most of a step); everywhere else the code has to be the formula's."""
    dt = DTYPES[dtype]
    params = _params(dev, [(40,), (size,)], dt, seed=size)
    p = params[1]
    opt = k2.AdamW(params, lr=1e-3, state_bits=8, stochastic=dtype == "bf16", seed=77)
    b1, b2 = 0.9, 0.999
    for s in range(4):
        for q in params:
            scale = torch.exp2(torch.randint(-12, 4, q.shape, generator=torch.Generator().manual_seed(s)).float())
            q.grad.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(50 + s)) * scale * 1e-2)
        m, v = (t[BLOCK:BLOCK + size].double() for t in opt.moments()) if s else (torch.zeros(size, device=dev).double(),) * 2
        old = p.detach().double()
        opt.step()
        g = p.grad.double()
        h = _bits(77, s + 1, torch.arange(BLOCK, BLOCK + size, device=dev))
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        new = old * (1 - 1e-3 * 1e-2) - 1e-3 * (m / (1 - b1 ** (s + 1))) / ((v / (1 - b2 ** (s + 1))).sqrt() + 1e-8)
        got = [t[BLOCK:BLOCK + size].double() for t in opt.moments()]
        for a, have, places, low, top, random, least in (
                (m.abs(), got[0].abs(), 3, -6, 448.0, (h & 0xFFFF).double() / 65536, 0.0),
                (v.sqrt(), got[1].sqrt(), 4, 0, 31744.0, (h >> 16).double() / 65536, 1 / 16)):
            want, step = _held(a, places, low, top, random, least)
            off = (have - want).abs()
            exact = off <= 64 * 2.0 ** -24 * want
            assert bool((off <= step * (1 + 2.0 ** -18) + 64 * 2.0 ** -24 * want).all())
            assert int((~exact).sum()) <= 1 + size * 2.0 ** -10       # borders: 2 * 2^-18 + 32 * 2^-24 * 2^5 each, far fewer
        assert torch.equal(torch.sign(got[0]), torch.sign(m) * (got[0] != 0))
        if dtype == "f32":
            _near(p.detach(), new, 2.0 ** -22, 1e-3 * 2.0 ** -17)
        else:
            low_value, step = _neighbours(new.abs(), 7, -126)
            up = new.abs() / step - low_value / step + (_mix(h ^ 0x9E3779B9) & 0xFFFF).double() / 65536 >= 1
            off = (p.detach().double() - torch.sign(new) * (low_value + up * step)).abs()
            assert bool((off <= step * (1 + 2.0 ** -18)).all())
            assert int((off > 0).sum()) <= 1 + size * 2.0 ** -7       # update errors of 1e-3 * 2^-17 against steps of 2^-10


def test_moments_in_8_bits_do_not_stand_still(k2, dev):
    """A second moment that moves by a thousandth a step, far under half a code, still reaches its mean: the roots of 65536
    elements are on the average within 1 % (a random choice between neighbours adds a variance of a step squared, 2^-8 of v at
    most, and the mean over the elements scatters by 2^-4 / 256)."""
    n = 65536
    p = torch.nn.Parameter(torch.zeros(n, device=dev))
    size = torch.exp2(torch.rand(n, generator=torch.Generator().manual_seed(0)) * 8 - 12).to(dev)
    opt = k2.AdamW([p], lr=0.0, state_bits=8)
    for s in range(1500):
        p.grad = size * (1.0 if s < 300 else 0.5)
        opt.step()
    v = 0.0
    for s in range(1500):
        v = 0.999 * v + 0.001 * (1.0 if s < 300 else 0.25)
    m, got = opt.moments()
    assert abs(float((got.double().sqrt() / size.double() / math.sqrt(v)).mean()) - 1) < 0.01
    assert abs(float((m.double() / size.double() / 0.5).mean()) - 1) < 0.01


def test_rounding_at_random_keeps_small_updates(k2, dev):
    """Updates of a hundredth of a bf16 step: to the nearest nothing moves, at random the mean does."""
    n = 65536
    out = []
    for stochastic in (False, True):
        p = torch.nn.Parameter(torch.ones(n, device=dev, dtype=torch.bfloat16))
        opt = k2.AdamW([p], lr=2.0 ** -8 / 100, betas=(0.0, 0.0), weight_decay=0.0, stochastic=stochastic)
        for _ in range(50):
            p.grad = torch.ones_like(p)
            opt.step()
        out.append(float(p.detach().double().mean()))
    assert out[0] == 1.0
    # 50 updates of 2^-8 / 100; 65536 elements whose steps of 2^-8 (2^-7 above 1) scatter by their root
    assert abs(out[1] - (1 - 50 * 2.0 ** -8 / 100)) < 5 * 2.0 ** -8 / 256


# -- states, streams, captures ----------------------------------------------------------------------------------------
def _three(opt, params, first=0):
    for s in range(first, first + 3):
        for i, p in enumerate(params):
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(31 * s + i)).to(p.device, p.dtype)
        opt.step()


@pytest.mark.parametrize("how", ["load", "deepcopy"])
@pytest.mark.parametrize("bits,dtype", [(32, "f32"), (32, "bf16"), (8, "f32"), (8, "bf16")])
def test_states_go_on_where_they_were(k2, dev, tmp_path, bits, dtype, how):
    sizes = [(16, 40), (300,), (3, 3)]
    dt = DTYPES[dtype]
    a = _params(dev, sizes, dt)
    kw = {"lr": 1e-2, "state_bits": bits, "stochastic": dtype == "bf16", "seed": 5, "max_norm": 1.0}
    oa = k2.AdamW(a, **kw)
    _three(oa, a)
    if how == "load":
        torch.save(oa.state_dict(), tmp_path / "o.pt")
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        ob = k2.AdamW(b, lr=1.0, state_bits=bits, max_norm=1.0)
        ob.load_state_dict(torch.load(tmp_path / "o.pt", map_location="cpu", weights_only=True))
    else:
        ob = copy.deepcopy(oa)
        b = ob.param_groups[0]["params"]
        assert ob.max_norm == 1.0
    _three(oa, a, 3)
    _three(ob, b, 3)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert all(torch.equal(x, y) for x, y in zip(oa.moments(), ob.moments()))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(k2, dev, bits):
    sizes = [(16, 640), (257,), (100, 16)]
    a, b = (_params(dev, sizes, torch.float32) for _ in range(2))
    lr = torch.full((), 1e-3, device=dev)
    oa = k2.AdamW(a, lr=lr, state_bits=bits, max_norm=0.3)
    ob = k2.AdamW(b, lr=1e-3, state_bits=bits, max_norm=0.3)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            oa.step()
    torch.cuda.synchronize()
    oa.step()
    ob.step()
    with torch.cuda.graph(graph):
        oa.step()
    for s in range(5):
        for p, q in zip(a, b):
            g = torch.randn(p.shape, generator=torch.Generator().manual_seed(s)).to(dev)
            p.grad.copy_(g)
            q.grad = g
        if s == 3:
            lr.fill_(5e-3)
            ob.param_groups[0]["lr"] = 5e-3
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        assert all(float(oa.state[p]["step"]) == s + 2 for p in a)
        assert torch.equal(oa.grad_norm, ob.grad_norm)
        for p, q in zip(a, b):      # the learning rate as a float32 number and as a float64 one
            _near(p.detach(), q.detach().double(), 2.0 ** -23, 5e-3 * 2.0 ** -22 * 4 * (s + 1))
            if bits == 32:
                assert torch.equal(oa.state[p]["exp_avg"], ob.state[q]["exp_avg"])


def test_on_another_stream(k2, dev):
    a, b = (_params(dev, [(64, 2048), (33,)], torch.float32) for _ in range(2))
    oa, ob = k2.AdamW(a, max_norm=1.0, state_bits=8), k2.AdamW(b, max_norm=1.0, state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _three(oa, a)
    torch.cuda.current_stream().wait_stream(side)
    _three(ob, b)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_grads_of_other_strides(k2, dev):
    a = _params(dev, [(48, 20)], torch.float32)[0]
    b = torch.nn.Parameter(a.detach().clone())
    b.grad = a.grad.t().contiguous().t()
    k2.AdamW([a]).step()
    k2.AdamW([b], max_norm=1e9).step()
    assert torch.equal(a, b)


def test_places_past_32_bits(k2, dev):
    """A tensor of more than 2^32 elements: its last ones move as a short tensor's at their place do."""
    n, tail = (1 << 32) + 3 * 8192 + 77, 2048
    p = torch.nn.Parameter(torch.zeros(n, device=dev, dtype=torch.bfloat16))
    p.grad = torch.zeros(n, device=dev, dtype=torch.bfloat16)
    values = torch.randn(tail, generator=torch.Generator().manual_seed(0)).to(dev).bfloat16()
    p.grad[-tail:] = values
    opt = k2.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8, stochastic=True, seed=9, max_norm=1.0)
    opt.step()
    norm = math.sqrt(float(values.double().square().sum()))
    assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
    assert int(torch.count_nonzero(p.detach()[:1 << 20])) == 0 and int(torch.count_nonzero(p.detach()[-tail:])) == tail
    update = 0.5 * torch.sign(values.double())      # a first step's m / sqrt(v), of magnitude 1
    got = p.detach()[-tail:].double()
    assert bool(((got + update).abs() <= 0.5 * 2.0 ** -7).all())
    codes = opt.state[p]["exp_avg"].view(torch.uint8)
    assert int(torch.count_nonzero(codes[:-tail].view(torch.int8)[:1 << 20])) == 0
    at = torch.arange(n - tail, n, device=dev)
    first = (n - tail) // BLOCK * BLOCK
    g = torch.zeros(n - first, device=dev, dtype=torch.float64)
    g[-tail:] = values.double() / (norm + 1e-6)
    want, step = _held((0.1 * g).abs(), 3, -6, 448.0,
                       (_bits(9, 1, torch.arange(first, n, device=dev)) & 0xFFFF).double() / 65536, 0.0)
    scale = opt.state[p]["exp_avg_scale"][first // BLOCK:].double().repeat_interleave(BLOCK)[:n - first]
    have = opt.state[p]["exp_avg"][first:].double().abs() * scale
    off = (have - want).abs() > 64 * 2.0 ** -24 * want
    assert int(off.sum()) <= 2 and at.numel() == tail


def test_groups_that_move(k2, dev):
    """A group taken out or put elsewhere keeps its parameters' moments with the others; an empty one is passed over; one
    that grows is refused."""
    a, b = (_params(dev, [(16, 24), (40,), (300,)], torch.float32) for _ in range(2))
    oa = k2.AdamW([{"params": [a[0]]}, {"params": []}, {"params": [a[1]], "lr": 1e-2}, {"params": [a[2]]}], max_norm=1e9)
    ob = k2.AdamW([{"params": [b[0]]}, {"params": [b[1]], "lr": 1e-2}, {"params": [b[2]]}], max_norm=1e9)
    _three(oa, a)
    _three(ob, b)
    oa.param_groups.reverse()
    ob.param_groups[0]["params"][0].grad = None
    oa.param_groups.pop()
    for p, q in zip(a[1:], b[1:]):
        p.grad = q.grad = torch.ones_like(p)
    b[0].grad = None
    oa.step()
    ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    oa.param_groups[0]["params"].append(_params(dev, [(4,)], torch.float32)[0])
    with pytest.raises(ValueError, match="the group has 2 parameters"):
        oa.step()


def test_a_state_that_does_not_fit_changes_nothing(k2, dev):
    a = _params(dev, [(16, 24)], torch.float32)
    opt = k2.AdamW([{"params": a, "state_bits": 8, "lr": 3e-3}])
    _three(opt, a)
    before = copy.deepcopy(opt.state_dict())
    torch_opt = torch.optim.AdamW(a, lr=1.0)
    torch_opt.step()
    with pytest.raises(ValueError, match="8 bits"):         # the group's own bits, which the state does not name
        opt.load_state_dict(torch_opt.state_dict())
    after = opt.state_dict()
    assert after["param_groups"] == before["param_groups"] and opt.param_groups[0]["lr"] == 3e-3
    assert all(_same(after["state"][0][n], before["state"][0][n]) for n in before["state"][0])
    _three(opt, a)


@pytest.mark.parametrize("bits", [0x7FFFFFFF, -1, 0x7FC00000, 0x7F800000])
def test_values_that_are_not_finite_are_rounded_at_random_to_what_they_are(k2, dev, bits):
    """A NaN stays one whatever its bits (16 random ones must not carry past its sign), an infinity stays infinite."""
    p = torch.nn.Parameter(torch.zeros(512, device=dev, dtype=torch.bfloat16))
    value = torch.tensor([bits >> 16 & 0xFFFF], dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    with torch.no_grad():
        p[100:200] = value.to(dev)
    opt = k2.AdamW([p], lr=1e-3, stochastic=True)
    p.grad = torch.ones_like(p)
    opt.step()
    assert torch.isfinite(p[:100]).all() and torch.isfinite(p[200:]).all()
    want = torch.isnan if math.isnan(float(value)) else torch.isinf
    assert want(p[100:200]).all()


def test_memory_written_twice_is_refused(k2, dev):
    """Parameters or gradients that share memory, and a parameter that outgrew its moments: refused, nothing changes."""
    flat = torch.zeros(600, device=dev)
    a, b, c = (torch.nn.Parameter(t) for t in (flat[:300], flat[299:400], flat[400:]))
    for p in (a, b, c):
        p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="parameters 0 and 1 share memory"):
        k2.AdamW([a, b, c]).step()
    assert not int(flat.count_nonzero())
    k2.AdamW([a, c]).step()             # neighbours
    assert bool((flat[:300] != 0).all()) and bool((flat[400:] != 0).all()) and not int(flat[300:400].count_nonzero())
    with pytest.warns(UserWarning, match="duplicate"):
        opt = k2.AdamW([c, c])
    with pytest.raises(ValueError, match="parameters 0 and 1 share memory"):
        opt.step()
    grads = torch.ones(600, device=dev)
    a.grad, b.grad = grads[:300], grads[200:301]
    with pytest.raises(ValueError, match="parameters 0 and 1 share memory"):
        k2.clip_grad_norm_([a, b, c], 1e-3)
    assert bool((grads == 1).all())
    opt = k2.AdamW([a, c])
    opt.step()                          # gradients that share memory are only read
    kept = [t.clone() for t in opt.moments()]
    a.data = torch.zeros(513, device=dev)
    a.grad = torch.ones(513, device=dev)
    with pytest.raises(ValueError, match="grown to 513"):
        opt.step()
    assert all(torch.equal(x, y) for x, y in zip(opt.moments(), kept)) and not int(a.count_nonzero())


def test_empty_parameters(k2, dev):
    p = torch.nn.Parameter(torch.zeros(0, 4, device=dev))
    p.grad = torch.zeros(0, 4, device=dev)
    for bits in (32, 8):
        opt = k2.AdamW([p], state_bits=bits, max_norm=1.0)
        opt.step()
        assert opt.grad_norm is None and all(t.numel() == 0 for t in opt.moments(dtype=torch.bfloat16))
    assert float(k2.clip_grad_norm_([p], 1.0)) == 0.0


@pytest.mark.parametrize("gap", [2, 7])
def test_many_parameters_without_gradients_between(k2, dev, gap):
    """Counts and values of the others stay; those with a gradient move as in a list of their own, beyond 512 of them too."""
    n = 560 * gap
    a = _params(dev, [(5,)] * n, torch.float32)
    for p in a:
        p.grad = None
    few = [torch.nn.Parameter(p.detach().clone()) for p in a[::gap]]
    oa, ob = k2.AdamW(a, max_norm=1.0), k2.AdamW(few, max_norm=1.0)
    for k in range(3):
        for i, p in enumerate(few):
            p.grad = torch.full_like(p, (i % 13 - 6) * 0.25 + k)
            a[i * gap].grad = p.grad.clone()
        before = [p.detach().clone() for p in a]
        oa.step()
        ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a[::gap], few))
    assert all(torch.equal(p, q) for i, (p, q) in enumerate(zip(a, before)) if i % gap)
    counts = torch.stack([oa.state[p]["step"] for p in a]).view(-1, gap)
    assert bool((counts[:, 0] == 3).all()) and not int(counts[:, 1:].count_nonzero())
