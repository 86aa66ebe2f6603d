"""GPU tests of the RMSNorm with the residual's addition (``residual_rmsnorm``) and its backward."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

EPS = 1e-5


class Norm(nn.Module):          # mmdit.py:146-161: weight scale + 1
    def __init__(self, scale):
        super().__init__()
        self.eps, self.scale = EPS, nn.Parameter(scale, requires_grad=False)


def _inputs(shape, dev, entries=0, seed=0, spread=1.0):
    """x, y and, for entries > 0, gate / scale / shift as chunks of one tensor."""
    g = torch.Generator().manual_seed(sum(shape) + seed)
    K = shape[-1]
    x, y = (torch.randn(shape, generator=g) * spread).bfloat16().to(dev), torch.randn(shape, generator=g).bfloat16().to(dev)
    x[..., : max(1, K // 100)] *= 20
    mods = [None] * 3
    if entries:
        lead = (entries, 1) if len(shape) == 3 else (entries,)
        mods = list((torch.randn(*lead, 3 * K, generator=g) * 0.3).bfloat16().to(dev).chunk(3, -1))
    norm = Norm((torch.randn(K, generator=g) * 0.1).to(dev))
    return norm, x, y, mods


SHAPES = [((1, 128), 0), ((1, 1, 6144), 1), ((3, 640), 3), ((2, 77, 2560), 2), ((1, 333, 4096), 1), ((2, 5, 4224), 1),
          ((3, 3, 8192), 3), ((2, 9, 8320), 2), ((1, 7, 16384), 1), ((4, 1, 12288), 4), ((1025, 256), 0)]


@pytest.mark.parametrize("modulated", [False, True])
@pytest.mark.parametrize("shape,entries", SHAPES)
def test_equals_the_separate_operations(k2, dev, shape, entries, modulated):
    """r is the eager bf16 residual, h the norm kernel's on r, the codes those of h: bit for bit, one or more entries."""
    from krea2_amd.quantize import shared_input_quant
    norm, x, y, (gate, p, b) = _inputs(shape, dev, entries)
    K = shape[-1]
    if not modulated:
        p = b = None
    r, h = k2.residual_rmsnorm(norm, x, y, gate, p, b)
    misses = shared_input_quant.misses
    q, s = k2.input_codes(h)
    assert shared_input_quant.misses == misses                  # the pass left them
    assert torch.equal(r, x + (y if gate is None else gate * y))
    zero = torch.zeros(1, K, device=dev, dtype=torch.bfloat16)
    if p is None:                                               # (1 + 0) n + 0 = n
        ref = k2.modulated_rmsnorm(norm, r, zero, zero)
    else:
        ref = k2.modulated_rmsnorm(norm, r, p, b)
    assert torch.equal(h, ref)
    q0, s0, _ = k2._lib.rotquant(h.reshape(-1, K))
    assert torch.equal(q, q0) and torch.equal(s, s0)


def test_plain_weight(k2, dev):
    """A norm with a ``weight`` weighs by it: the value in float64, within the rounding of n to bf16 and the float32
    statistics (K = 1024 squares summed: under 2^-18 of the mean)."""
    g = torch.Generator().manual_seed(3)
    for dt in (torch.float32, torch.bfloat16):
        norm = nn.RMSNorm(1024, eps=1e-6, device=dev, dtype=dt)
        with torch.no_grad():
            norm.weight.copy_(torch.randn(1024, generator=g))
        norm.requires_grad_(False)
        x, y = torch.randn(2, 33, 1024, generator=g).bfloat16().to(dev), torch.randn(2, 33, 1024, generator=g).bfloat16().to(dev)
        r, h = k2.residual_rmsnorm(norm, x, y)
        r64 = (x + y).double()
        ref = r64 / (r64.square().mean(-1, keepdim=True) + 1e-6).sqrt() * norm.weight.double()
        assert torch.equal(r, x + y)
        assert ((h.double() - ref).abs() <= (2 ** -8 + 2 ** -17) * ref.abs()).all()


def test_rows_zero_strided_offset_and_nonfinite(k2, dev):
    """A row of zeros has the norm 0 (eps keeps it finite); strided and unaligned rows give what contiguous ones do; a
    row with an infinity or NaN touches no other row."""
    norm, x, y, (gate, p, b) = _inputs((6, 512), dev, 6)
    x[2] = 0
    y[2] = 0
    r, h = k2.residual_rmsnorm(norm, x, y, gate, p, b)
    assert (r[2] == 0).all() and torch.equal(h[2], b[2])
    wide = torch.empty(6, 1024, device=dev, dtype=torch.bfloat16)
    wide[:, 512:] = x
    odd = torch.empty(6 * 512 + 3, device=dev, dtype=torch.bfloat16)[3:].view(6, 512)
    odd.copy_(y)
    r2, h2 = k2.residual_rmsnorm(norm, wide[:, 512:], odd, gate.contiguous(), p, b.clone())
    assert torch.equal(r2, r) and torch.equal(h2, h)
    tr = torch.empty(512, 6, device=dev, dtype=torch.bfloat16).t()
    tr.copy_(x)
    assert torch.equal(k2.residual_rmsnorm(norm, tr, y, gate, p, b)[1], h)
    same, both = x[:1].expand(6, 512), x[:1].repeat(6, 1)
    assert torch.equal(k2.residual_rmsnorm(norm, same, y, gate, p, b)[1], k2.residual_rmsnorm(norm, both, y, gate, p, b)[1])
    x[1, 3], y[4, 7] = float("inf"), float("nan")
    r3, h3 = k2.residual_rmsnorm(norm, x, y, gate, p, b)
    keep = [0, 2, 3, 5]
    assert torch.equal(r3[keep], r[keep]) and torch.equal(h3[keep], h[keep])
    assert r3[4].isnan().sum() == 1 and h3[4].isnan().all() and h3[1].isnan().any()


def test_no_rows(k2, dev):
    norm, x, y, _ = _inputs((2, 4, 256), dev)
    gate = torch.ones(2, 1, 256, device=dev, dtype=torch.bfloat16, requires_grad=True)
    r, h = k2.residual_rmsnorm(norm, x[:, :0], y[:, :0], gate)
    assert r.shape == h.shape == (2, 0, 256)
    (r.sum() + h.sum()).backward()
    assert (gate.grad == 0).all()


def test_gradients_of_other_layouts(k2, dev, monkeypatch):
    """Transposed, expanded and unaligned inputs, vectors of one entry in any shape, and a device that the wrappers have not
    seen: the gradients of contiguous tensors, in the inputs' shapes."""
    B, L, K = 2, 6, 256
    norm, x, y, (gate, p, b) = _inputs((B, L, K), dev, B)
    dr, dh = torch.randn_like(x), torch.randn_like(x)

    def run(x, y, gate, p, b):
        leaves = [x, y, gate, p, b]
        return _grads(k2.residual_rmsnorm(norm, *leaves), leaves, dr, dh)

    plain = run(*(t.detach().clone().requires_grad_() for t in (x, y, gate, p, b)))
    xt = x.transpose(0, 1).contiguous().requires_grad_()
    odd = torch.empty(y.numel() + 3, device=dev, dtype=torch.bfloat16)[3:].view(y.shape).copy_(y).requires_grad_()
    spread = torch.empty(B, 1, 2 * K, device=dev, dtype=torch.bfloat16)[..., ::2].copy_(gate).requires_grad_()
    leaves = [xt, odd, spread, *(t.detach().clone().view(B, K).requires_grad_() for t in (p, b))]
    got = _grads(k2.residual_rmsnorm(norm, xt.transpose(0, 1), *leaves[1:]), leaves, dr.transpose(0, 1).contiguous().transpose(0, 1), dh)
    assert torch.equal(got[0].transpose(0, 1), plain[0])
    for a, e in zip(got[1:], plain[1:]):
        assert torch.equal(a.reshape(e.shape), e)
    real = k2._lib._fast().resnorm
    calls = []

    class Native:                       # refuses the first call, as before the device's check
        def __getattr__(self, name):
            return getattr(k2._lib._native_saved, name)

        def resnorm(self, *a):
            calls.append(a)
            return None if len(calls) == 1 else real(*a)

    k2._lib._native_saved = k2._lib._native
    monkeypatch.setattr(k2._lib, "_native", Native())
    again = run(*(t.detach().clone().requires_grad_() for t in (x, y, gate, p, b)))
    assert len(calls) == 2 and all(torch.equal(a, e) and a.shape == e.shape for a, e in zip(again, plain))
    with torch.no_grad():
        calls.clear()
        r, h = k2.residual_rmsnorm(norm, x, y, gate, p, b)
    assert len(calls) == 2 and r.shape == h.shape == x.shape
    del k2._lib._native_saved


def _separate(norm, x, y, gate, p, b):
    """The operation in float64, each tensor that the model holds in bf16 rounded, the gradient passed through."""
    def bf(t):
        return t + (t.float().bfloat16().double() - t).detach()

    r = bf(x + (y if gate is None else bf(gate * y)))
    h = bf(r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * (norm + 1))
    if p is not None:
        h = bf(bf(bf(1 + p) * h) + b)
    return r, h


def _grads(out, leaves, dr, dh):
    return torch.autograd.grad(out, leaves, (dr, dh), allow_unused=True)


# enough rows that one pass makes the row's gradients and the column sums (last strips short, one row an entry more or less)
LONG = [((1, 1101, 2176), 1), ((2, 601, 6144), 2), ((3, 259, 8192), 3), ((250, 5, 2560), 250), ((1, 768, 4096), 1),
        ((1, 4609, 6144), 1), ((1030, 6016), 0), ((64, 33, 2304), 64)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape,entries", SHAPES + LONG)
def test_gradients_against_float64(k2, dev, shape, entries, gated):
    """Every gradient against the formula's in float64: float32 inside and one rounding to bf16, at most 2^-8 of the value;
    a quarter of that for the float32 sums of a row or a column (16384 terms: 2^-10 at the very most)."""
    if gated and not entries:
        pytest.skip("no entries to gate")
    norm, x, y, (gate, p, b) = _inputs(shape, dev, entries, seed=1)
    if not gated:
        gate = p = b = None
    g = torch.Generator().manual_seed(7)
    dr, dh = (torch.randn(shape, generator=g).bfloat16().to(dev) for _ in range(2))
    leaves = [t.detach().clone().requires_grad_() for t in (x, y, gate, p, b) if t is not None]
    full = leaves + [None] * (5 - len(leaves))
    norm.scale.requires_grad_()
    out = k2.residual_rmsnorm(norm, *full)
    got = _grads(out, [*leaves, norm.scale], dr, dh)
    l64 = [t.detach().double().requires_grad_() for t in leaves]
    w64 = norm.scale.detach().double().requires_grad_()
    ref = _grads(_separate(w64, *(l64 + [None] * (5 - len(l64)))), [*l64, w64], dr.double(), dh.double())
    for a, e, t in zip(got, ref, [*leaves, norm.scale]):
        assert a.shape == t.shape and a.dtype == t.dtype
        assert (a.double() - e).norm() <= 1.25 * 2 ** -8 * e.norm()
    # the norm's gradient is float32 throughout: K or M products summed, n rounded nowhere
    assert (got[-1].double() - ref[-1]).norm() <= 1e-5 * ref[-1].norm()
    # the same with the parameters frozen, and again: the same bits
    norm.scale.requires_grad_(False)
    out = k2.residual_rmsnorm(norm, *full)
    two = _grads(out, leaves[:2], dr, dh)
    assert torch.equal(two[0], got[0]) and torch.equal(two[1], got[1])
    norm.scale.requires_grad_()
    again = _grads(k2.residual_rmsnorm(norm, *full), [*leaves, norm.scale], dr, dh)
    assert all(torch.equal(a, e) for a, e in zip(again, got))


@pytest.mark.parametrize("read", ["both", "h"])
@pytest.mark.parametrize("shape", [(2, 9, 640), (2, 450, 2304)])
def test_some_of_the_gradients(k2, dev, shape, read):
    """Each input alone, and h alone read: the same bits as when every gradient is asked for."""
    norm, x, y, mods = _inputs(shape, dev, 2, seed=3)
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    base = [t.detach() for t in (x, y, *mods)]

    def run(asked):
        leaves = [t.clone().requires_grad_(i in asked) for i, t in enumerate(base)]
        norm.scale.requires_grad_(5 in asked)
        r, h = k2.residual_rmsnorm(norm, *leaves)
        of = [t for i, t in enumerate((*leaves, norm.scale)) if i in asked]
        g = torch.autograd.grad([r, h], of, [dr, dh]) if read == "both" else torch.autograd.grad(h, of, dh)
        norm.scale.requires_grad_(False)
        return g

    full = run(range(6))
    for i in range(6):
        assert torch.equal(run([i])[0], full[i]), i
    none = torch.zeros_like(dr)
    if read == "h":             # r unread is r read with a gradient of zeros
        leaves = [t.clone().requires_grad_() for t in base]
        got = torch.autograd.grad(k2.residual_rmsnorm(norm, *leaves), leaves, [none, dh])
        assert all(torch.equal(a, e) for a, e in zip(got, full))


@pytest.mark.parametrize("K", [640, 6144, 8320])
def test_eager_gradients_equal_the_separate_operations(k2, dev, K):
    """The block's form (gate, modulation and norm frozen): the gradients of the eager residual and the norm kernel; the
    form that rounds once is within their three and four roundings of them."""
    from krea2_amd.fused import _residual_rmsnorm
    norm, x, y, (gate, p, b) = _inputs((2, 40, K), dev, 2)
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    a = [t.detach().clone().requires_grad_() for t in (x, y)]
    ga = _grads(_residual_rmsnorm(norm, *a, gate, p, b, True), a, dr, dh)
    e = [t.detach().clone().requires_grad_() for t in (x, y)]
    r = e[0] + gate * e[1]
    ge = _grads((r, k2.modulated_rmsnorm(norm, r, p, b)), e, dr, dh)
    assert torch.equal(ga[0], ge[0]) and torch.equal(ga[1], ge[1])
    once = _grads(k2.residual_rmsnorm(norm, *a, gate, p, b), a, dr, dh)
    assert not torch.equal(once[1], ge[1])
    for u, v in zip(once, ge):
        assert (u.double() - v.double()).norm() <= 4 * 2 ** -8 * v.double().norm()


def test_gradient_against_differences(k2, dev):
    """The directional derivative of a smooth function of h against central differences in float64 of the formula."""
    norm, x, y, (gate, p, b) = _inputs((1, 3, 128), dev, 1, seed=5)
    v = torch.randn_like(x)
    leaves = [t.detach().clone().requires_grad_() for t in (x, y, gate, p, b)]
    r, h = k2.residual_rmsnorm(norm, *leaves)
    got = torch.autograd.grad((h * v).sum() + r.sum(), leaves)

    def value(ts):
        rr = ts[0] + ts[2] * ts[1]
        hh = rr * torch.rsqrt(rr.square().mean(-1, keepdim=True) + EPS) * (norm.scale.double() + 1) * (1 + ts[3]) + ts[4]
        return ((hh * v.double()).sum() + rr.sum()).item()

    base = [t.detach().double() for t in leaves]
    for i, gi in enumerate(got):
        d = torch.randn_like(base[i])
        hi = [t + 1e-4 * d if j == i else t for j, t in enumerate(base)]
        lo = [t - 1e-4 * d if j == i else t for j, t in enumerate(base)]
        num = (value(hi) - value(lo)) / 2e-4
        # the kernel differentiates at the rounded r, n and 1 + p: a few 2^-8 of the products' magnitudes
        assert abs(num - (gi.double() * d).sum().item()) <= 8 * 2 ** -8 * (gi.double().abs() * d.abs()).sum().item(), i


def test_an_entry_per_row(k2, dev):
    """Rows with a gate and a modulation of their own, more of them than a launch has workgroups in its second extent."""
    M, K = 66000, 128
    norm, x, y, (gate, p, b) = _inputs((M, K), dev, M)
    leaves = [t.detach().clone().requires_grad_() for t in (x, y, gate, p, b)]
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    got = _grads(k2.residual_rmsnorm(norm, *leaves), leaves, dr, dh)
    l64 = [t.detach().double().requires_grad_() for t in leaves]
    ref = _grads(_separate(norm.scale.detach().double(), *l64), l64, dr.double(), dh.double())
    for a, e in zip(got, ref):
        assert a.shape == e.shape and (a.double() - e).norm() <= 1.25 * 2 ** -8 * e.norm()
    one = torch.randn(K, device=dev).as_strided((1, K), (1, 1)).bfloat16().as_strided((1, K), (1, 1))
    assert torch.equal(k2.residual_rmsnorm(norm, one, one)[0], one + one)


@pytest.mark.parametrize("shape", [(3, 77, 640), (3, 280, 2176)])
@pytest.mark.parametrize("one", [(0,), (1,), (2,), (0, 1, 2)])
def test_vectors_that_every_entry_shares(k2, dev, one, shape):
    """One gate, scale or shift beside others with an entry per batch row: the sum over every row, rounded once (2^-8 of
    it; float32 sums of K terms in a row and B L in a column, 2^-24 of the products' magnitudes a term, twice that for the
    products' own roundings), and the same bits from a captured backward, also of r alone."""
    norm, x, y, mods = _inputs(shape, dev, 3, seed=2)
    terms = shape[2] + shape[0] * shape[1]
    leaves = [t.detach().clone()[:1 if i in one else 3].requires_grad_() for i, t in enumerate(mods)]
    leaves = [x.detach().clone().requires_grad_(), y.detach().clone().requires_grad_(), *leaves]
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    got = _grads(k2.residual_rmsnorm(norm, *leaves), leaves, dr, dh)
    l64 = [t.detach().double().requires_grad_() for t in leaves]
    r64 = l64[0] + l64[2] * l64[1]
    r64 = r64 + ((x + leaves[2].detach() * y).double() - r64).detach()              # the bf16 r, the gradient passed through
    n64 = r64 * torch.rsqrt(r64.square().mean(-1, keepdim=True) + EPS) * (norm.scale.double() + 1)
    nb = n64.float().bfloat16().double()
    p64 = (1 + leaves[3].detach()).double() + (l64[3] - l64[3].detach())
    h64 = n64 * p64 + l64[4] + (nb - n64).detach() * (l64[3] - l64[3].detach())
    ref = _grads((r64, h64), l64, dr.double(), dh.double())
    r = r64.detach()
    inv = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
    g = (dh.double() * p64.detach() * (norm.scale.double() + 1)).abs()
    dR = dr.double().abs() + g * inv + r.abs() * inv ** 3 * (g * r.abs()).mean(-1, keepdim=True)
    mags = dR * y.double().abs(), dh.double().abs() * nb.detach().abs(), dh.double().abs()
    for i in range(3):
        a, e, over = got[2 + i], ref[2 + i], (0, 1) if i in one else 1
        bound = 2 ** -8 * e.abs() + 2 * terms * 2 ** -24 * mags[i].sum(over, keepdim=True)
        if i == 1:      # an n at a tie rounds to either side: two products of a column a step (2^-7) off
            bound += 2 * 2 ** -7 * mags[i].amax(over, keepdim=True)
        assert a.shape == e.shape and ((a.double() - e).abs() <= bound).all(), i
    static = [t.detach().clone().requires_grad_() for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _grads(k2.residual_rmsnorm(norm, *static), static, dr, dh)
    torch.cuda.current_stream().wait_stream(side)
    graph, alone = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = _grads(k2.residual_rmsnorm(norm, *static), static, dr, dh)
    with torch.cuda.graph(alone):                                                   # the stream's gradient without h's
        stream = torch.autograd.grad(k2.residual_rmsnorm(norm, *static)[0], static[:3], dr)
    ref = (dr.double() * y.double()).sum((0, 1) if 0 in one else 1, keepdim=True)
    mag = (dr.double() * y.double()).abs().sum((0, 1) if 0 in one else 1, keepdim=True)
    for _ in range(3):
        for t in (*cap, *stream[1:]):       # stream[0] is dr itself
            t.zero_()
        graph.replay()
        alone.replay()
        again = _grads(k2.residual_rmsnorm(norm, *leaves), leaves, dr, dh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) and torch.equal(c, e) for a, c, e in zip(again, cap, got))
        assert torch.equal(stream[0], dr) and stream[2].shape == static[2].shape
        assert ((stream[2].double() - ref).abs() <= 2 ** -8 * ref.abs() + terms * 2 ** -24 * mag).all()


def test_unused_and_broadcast_outputs(k2, dev):
    """Only r, only h, or neither used; a gate of one entry beside a modulation per batch row; a bf16 norm scale."""
    norm, x, y, (gate, p, b) = _inputs((3, 4, 256), dev, 3)
    one = gate[:1].detach().clone().requires_grad_()
    xs = x.detach().clone().requires_grad_()
    r, h = k2.residual_rmsnorm(norm, xs, y, one, p, b)
    dr = torch.randn_like(x)
    gx, gg = torch.autograd.grad(r, (xs, one), dr, retain_graph=True)
    assert torch.equal(gx, dr)
    ref = (dr.double() * y.double()).sum((0, 1), keepdim=True)
    mag = (dr.double() * y.double()).abs().sum((0, 1), keepdim=True)
    assert gg.shape == one.shape and ((gg.double() - ref).abs() <= 2 ** -7 * mag).all()
    full = [t.detach().clone().requires_grad_() for t in (x, y, gate, p, b)]
    norm.scale.requires_grad_()
    bad = x.detach().clone()
    bad[1, 2, 5] = float("inf")                     # a row that the norm cannot take, whose norm nothing reads
    full[0] = bad.requires_grad_()
    gs = torch.autograd.grad(k2.residual_rmsnorm(norm, *full)[0], [*full, norm.scale], dr)
    norm.scale.requires_grad_(False)
    assert torch.equal(gs[0], dr) and torch.equal(gs[1], gate * dr)
    assert ((gs[2].double() - (dr.double() * y.double()).sum(1, keepdim=True)).abs() <= 2 ** -8 * mag).all()
    assert all((t == 0).all() and t.shape == u.shape for t, u in zip(gs[3:], [*full[3:], norm.scale]))
    gx2, = torch.autograd.grad(h, xs, dr)
    e = x.detach().clone().requires_grad_()
    ge, = torch.autograd.grad(k2.modulated_rmsnorm(norm, e + one.detach() * y, p, b), e, dr)
    assert (gx2.double() - ge.double()).norm() <= 3 * 2 ** -8 * ge.double().norm()      # dn rounded, the result twice
    half = Norm(norm.scale.detach().bfloat16())
    half.scale.requires_grad_()
    gs, = torch.autograd.grad(k2.residual_rmsnorm(half, x, y)[1], half.scale, dr)
    assert gs.dtype == torch.bfloat16 and gs.shape == half.scale.shape
    with pytest.raises(RuntimeError):                           # differentiable once
        q = x.detach().clone().requires_grad_()
        g1, = torch.autograd.grad(k2.residual_rmsnorm(norm, q, y)[1].float().square().sum(), q, create_graph=True)
        g1.float().sum().backward()


def test_captured_and_other_stream(k2, dev):
    """Replays of a captured pass and a pass on another stream equal the eager one."""
    norm, x, y, (gate, p, b) = _inputs((2, 50, 1024), dev, 2)
    k2.residual_rmsnorm(norm, x, y, gate, p, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rs, hs = k2.residual_rmsnorm(norm, x, y, gate, p, b)
    torch.cuda.current_stream().wait_stream(side)
    xs, ys = x.clone(), y.clone()
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    graph = torch.cuda.CUDAGraph()
    w = norm.scale
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        r, h = k2.residual_rmsnorm(norm, xs, ys, gate, p, b)
        flat = [t.reshape(-1, 1024) for t in (dh, dr, r, ys)]
        ent = [t.reshape(2, 1024) for t in (p, gate)]
        grads = k2._lib.resnorm_bwd(flat[0], flat[1], flat[2], w, 1.0, EPS, ent[0], ent[1], 50, flat[3], True, True, True)
    for i in range(3):
        xs.copy_(x * (i + 1))
        graph.replay()
        er, eh = k2.residual_rmsnorm(norm, x * (i + 1), y, gate, p, b)
        ref = k2._lib.resnorm_bwd(flat[0], flat[1], er.reshape(-1, 1024), w, 1.0, EPS, ent[0], ent[1], 50, flat[3], True,
                                  True, True)
        torch.cuda.synchronize()
        assert torch.equal(r, er) and torch.equal(h, eh), i
        assert all(torch.equal(a, e) for a, e in zip(grads, ref)), i
        if i == 0:
            assert torch.equal(rs, r) and torch.equal(hs, h)


def test_fused_block_keeps_its_bits(k2, dev):
    """A patched block, forward and gradients, against the composition it replaces."""
    from tests import restated_block as rb
    torch.manual_seed(0)
    dit = rb.Dit(1).to(dev).to(torch.bfloat16)
    for blk in dit.blocks:
        blk.prenorm.float(), blk.postnorm.float()
        blk.postnorm.scale.data.normal_(0, 0.1)
    k2.quantize_dit_convrot(dit)
    ad = k2.inject_lora(dit, 16)
    for m in ad.values():
        m.lora_B.data.normal_(0, 0.02)
    assert k2.fuse_producers(dit) == 2
    blk = dit.blocks[0]
    x = torch.randn(2, 33, rb.FEAT, device=dev, dtype=torch.bfloat16)
    vec = (torch.randn(2, 1, 6 * rb.FEAT, device=dev) * 0.3).bfloat16()
    dy = torch.randn_like(x)

    def before(x):
        ps, pb, pg, qs, qb, qg = blk.mod(vec)
        x = x + pg * blk.attn(k2.modulated_rmsnorm(blk.prenorm, x, ps, pb), None, None)
        return x + qg * blk.mlp(k2.modulated_rmsnorm(blk.postnorm, x, qs, qb))

    params = k2.lora_parameters(ad)
    outs = []
    for f in (lambda t: blk(t, vec, None), before):
        t = x.detach().clone().requires_grad_()
        out = f(t)
        outs.append((out, *torch.autograd.grad(out, [t, *params], dy)))
    for a, e in zip(*outs):
        assert torch.equal(a, e)


def test_refusals(k2, dev):
    norm, x, y, (gate, p, b) = _inputs((2, 4, 256), dev, 2)
    for bad in (lambda: k2.residual_rmsnorm(norm, x, y[:1]), lambda: k2.residual_rmsnorm(norm, x, y, gate, p),
                lambda: k2.residual_rmsnorm(norm, x, y, gate[..., :128]), lambda: k2.residual_rmsnorm(norm, x, y, p, b[:0], p),
                lambda: k2.residual_rmsnorm(norm, x[..., :192], y[..., :192]), lambda: k2.residual_rmsnorm(nn.Module(), x, y),
                lambda: k2.residual_rmsnorm(Norm(norm.scale[:128]), x, y),
                lambda: k2.residual_rmsnorm(nn.LayerNorm(256, device=dev), x, y),
                lambda: k2.residual_rmsnorm(nn.RMSNorm(256, device=dev), x, y),
                lambda: k2._lib.resnorm_rotquant(x[0], y[0], None, norm.scale, 1.0, EPS, None, None, 3),
                lambda: k2._lib.resnorm_bwd(x[0], None, x[0], norm.scale, 1.0, EPS, None, None, 4, y[0]),
                lambda: k2._lib.resnorm_bwd(x[0], None, x[0], norm.scale, 1.0, EPS, p[0], None, 1, None, False, True, True, 3)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        k2.residual_rmsnorm(norm, x.float(), y)
    with pytest.raises(ValueError):
        k2.residual_rmsnorm(norm, x, y.cpu())


def test_offsets_past_32_bits(k2, dev):
    """2^31 elements and more: the last rows are those of the same rows alone, forward and backward."""
    M, K, n = 350208, 6144, 8
    g = torch.Generator(device=dev).manual_seed(0)
    x, y, dr, dh = (torch.empty(M, K, device=dev, dtype=torch.bfloat16).normal_(generator=g) for _ in range(4))
    norm = Norm((torch.randn(K, generator=g, device=dev) * 0.1))
    gate = torch.randn(1, K, generator=g, device=dev).bfloat16()

    def run(rows):
        leaves = [t[rows].requires_grad_() for t in (x, y)]
        r, h = k2.residual_rmsnorm(norm, *leaves, gate)
        q, s = k2.input_codes(h)
        out = [r.detach(), h.detach(), q, s, *torch.autograd.grad([r, h], leaves, [dr[rows], dh[rows]])]
        return [t[-n:].clone() for t in out]

    for a, e in zip(run(slice(None)), run(slice(M - n, M))):
        assert torch.equal(a, e)
