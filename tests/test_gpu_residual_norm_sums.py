"""GPU tests of the residual norm's gradients that are sums over rows: many entries, entries of a few rows, sums over every
row, and rows past 32 bits of offset."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

EPS = 1e-5


class Norm(nn.Module):
    def __init__(self, scale):
        super().__init__()
        self.eps, self.scale = EPS, nn.Parameter(scale)


def _inputs(M, K, entries, dev, seed=0):
    """x, y (entries, rows, K), gate / scale / shift (entries, 1, K), dr, dh."""
    g = torch.Generator(device=dev).manual_seed(M + K + seed)

    def bf(*shape):
        return torch.randn(shape, generator=g, device=dev).bfloat16()

    shape = (entries, M // entries, K)
    vectors = [(bf(entries, 1, K).float() * 0.3).bfloat16() for _ in range(3)]
    return Norm(torch.randn(K, generator=g, device=dev) * 0.1), bf(*shape), bf(*shape), vectors, bf(*shape), bf(*shape)


def _grads(k2, norm, x, y, vectors, dr, dh, asked=range(6)):
    leaves = [t.detach().clone().requires_grad_(i in asked) for i, t in enumerate((x, y, *vectors))]
    norm.scale.requires_grad_(5 in asked)
    out = k2.residual_rmsnorm(norm, *leaves)
    return torch.autograd.grad(out, [t for i, t in enumerate((*leaves, norm.scale)) if i in asked], (dr, dh))


def _sums64(norm, x, y, vectors, dr, dh):
    """The three vectors' and the norm weight's gradients per entry in float64, the sums of the terms' magnitudes and the
    largest of them.  The tensors that the model holds in bf16 (r, n, 1 + scale) are rounded as there."""
    gate, scale, _ = vectors
    r = (x + gate * y).double()
    w, p1 = norm.scale.detach().double() + 1, (1 + scale).double()
    inv = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
    n = (r * inv * w).float().bfloat16().double()
    dn = dh.double() * p1
    g = dn * w
    dR = dr.double() + g * inv - r * inv ** 3 * (g * r).mean(-1, keepdim=True)
    mR = dr.double().abs() + g.abs() * inv + r.abs() * inv ** 3 * (g * r).abs().mean(-1, keepdim=True)
    terms = [(dR * y.double(), mR * y.double().abs()), (dh.double() * n,) * 2, (dh.double(),) * 2, (dn * r * inv,) * 2]
    return ([t.sum(1, keepdim=True) for t, _ in terms], [m.abs().sum(1, keepdim=True) for _, m in terms],
            [m.abs().amax(1, keepdim=True) for _, m in terms])


# (rows of an entry, entries, K): a wave's own entries (fewer than 16 rows; a last wave and workgroup that are short), one
# strip an entry (their partials folded above 1024), strips of an entry
MANY = [(1, 5, 128), (1, 4099, 640), (3, 1003, 384), (15, 77, 1152), (7, 4, 8320), (1, 66000, 128), (13, 2500, 256),
        (17, 1100, 128), (16, 4200, 256), (33, 129, 2304), (40, 3, 640), (2, 2, 512)]


@pytest.mark.parametrize("shared", [(), (0,), (1, 2), (0, 1, 2)])
@pytest.mark.parametrize("rows,entries,K", MANY)
def test_sums_of_many_entries(k2, dev, rows, entries, K, shared):
    """Each sum within 2^-8 of its value (one rounding to bf16; none for the norm weight's) and 2^-24 of its terms' magnitudes
    for every addition that a term passes: an entry's rows at most 64 in a wave and four waves, or 16 rows' strip and its
    joins (under 200 together), the products' own roundings and the row sums of K terms beside them (K / 64 + 16).  An n that
    lies at a tie may round to either side, a step of 2^-7: one in 1e4 of a sum's terms at most, and two of a short sum's."""
    norm, x, y, vectors, dr, dh = _inputs(rows * entries, K, entries, dev)
    vectors = [t[:1].contiguous() if i in shared else t for i, t in enumerate(vectors)]
    got = _grads(k2, norm, x, y, vectors, dr, dh)
    ref, mag, top = _sums64(norm, x, y, [t.expand(entries, 1, K) for t in vectors], dr, dh)
    eps = (200 + K / 64 + 16) * 2 ** -24
    for i in range(4):
        e, m, t, terms = ref[i], mag[i], top[i], rows
        if i == 3 or i in shared:
            e, m, t, terms = e.sum(0, keepdim=True), m.sum(0, keepdim=True), t.amax(0, keepdim=True), rows * entries
        bound = eps * m + (0 if i == 3 else 2 ** -8) * e.abs()
        if i == 1:
            bound = bound + (2 + 1e-4 * terms) * 2 ** -7 * t
        a = got[2 + i].double().reshape(e.shape)
        assert ((a - e).abs() <= bound).all(), i
    for asked in ((0, 1), (2,), (3,), (4,), (5,), (4, 5)):      # some of them, and again: the same bits
        for a, i in zip(_grads(k2, norm, x, y, vectors, dr, dh, asked), asked):
            assert torch.equal(a, got[i]), (asked, i)


def test_equal_terms_of_every_row(k2, dev):
    """66000 rows with a vector each and the same terms: a sum of equal values in one accumulator would be off by a part of
    each addition's last digit, the same way every time (3e-4 of the sum).  Here no term passes 100 additions."""
    M, K = 66000, 128
    x = torch.ones(M, K, device=dev, dtype=torch.bfloat16)
    x[:, ::2] = 2
    vectors = [torch.zeros(M, K, device=dev, dtype=torch.bfloat16) for _ in range(3)]
    norm = Norm(torch.zeros(K, device=dev))
    dw, = _grads(k2, norm, x, torch.zeros_like(x), vectors, torch.zeros_like(x), torch.ones_like(x), (5,))
    want = M * x[0].double() / (2.5 + EPS) ** 0.5
    assert ((dw.double() - want).abs() <= 108 * 2 ** -24 * want).all()


@pytest.mark.parametrize("M,K", [(350208, 6144), (1050624, 2048)])
@pytest.mark.parametrize("entries", [1, None])
def test_sums_past_32_bits(k2, dev, M, K, entries):
    """2^31 elements and more with every gradient asked for, one vector for all rows (one pass makes rows and columns, or two)
    and one every 16 rows.  The gradients of r and h are zeros but in the last rows: the sums are those rows' own."""
    entries = entries or M // 16
    n = 2 * M // entries if entries > 1 else 64
    g = torch.Generator(device=dev).manual_seed(1)
    x, y = (torch.empty(entries, M // entries, K, device=dev, dtype=torch.bfloat16).normal_(generator=g) for _ in range(2))
    norm = Norm(torch.randn(K, generator=g, device=dev) * 0.1)
    vectors = [(torch.randn(entries, 1, K, generator=g, device=dev) * 0.3).bfloat16() for _ in range(3)]
    dr, dh = torch.zeros_like(x), torch.zeros_like(x)
    for t in (dr, dh):
        t.view(M, K)[-n:].normal_(generator=g)
    got = _grads(k2, norm, x, y, vectors, dr, dh)
    few = 2 if entries > 1 else 1

    def last(t):
        return t.view(M, K)[-n:].view(few, -1, K)

    part = [t if entries == 1 else t[-2:] for t in vectors]
    one = _grads(k2, norm, *(last(t) for t in (x, y)), part, *(last(t) for t in (dr, dh)))
    for a, e in zip(got[:2], one[:2]):
        assert torch.equal(last(a), e) and not a.view(M, K)[:-n].any()
    ref, mag, _ = _sums64(norm, *(last(t) for t in (x, y)), part, *(last(t) for t in (dr, dh)))
    for i, a in enumerate(got[2:5]):
        # the same terms in another order: float32 sums of at most 64 (their magnitudes), then one rounding either way
        assert ((a[-few:].double() - one[2 + i].double()).abs() <= 2 * 2 ** -8 * ref[i].abs() + 128 * 2 ** -24 * mag[i]).all()
        assert not a[:-few].any()
    assert ((got[5] - one[5]).double().abs() <= 200 * 2 ** -24 * mag[3].sum((0, 1))).all()


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("rows,entries,K", [*MANY, (4608, 1, 6144), (300, 2, 2560)])
def test_stream_alone(k2, dev, rows, entries, K, shared):
    """Nothing reads h: dx is r's gradient, dy its product with the gate rounded once, the gate's gradient the rows' sum of
    dr y, exact products added in float32 (16 rows of a strip or 64 of a wave, and the joins: under 200) and rounded once."""
    norm, x, y, vectors, dr, _ = _inputs(rows * entries, K, entries, dev, seed=5)
    if shared:
        vectors[0] = vectors[0][:1].contiguous()
    leaves = [t.detach().clone().requires_grad_() for t in (x, y, *vectors)]
    norm.scale.requires_grad_()
    r, _ = k2.residual_rmsnorm(norm, *leaves)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    gx, gy, gg, gs, gb, gw = torch.autograd.grad(r, [*leaves, norm.scale], dr)
    used = torch.cuda.max_memory_allocated() - before
    # dy, the vectors' gradients and the sums' partials, in the allocator's blocks (each up to 2 MB larger): no copy of the
    # stream in float32
    ws = k2._lib.load().k2q_resnorm_bwd_ws_bytes(rows * entries, K, rows)
    assert used <= 2 * x.numel() + 6 * gs.numel() + 4 * K + ws + 6 * (2 << 20)
    assert torch.equal(gx, dr) and torch.equal(gy, vectors[0] * dr)
    assert not (gs.any() or gb.any() or gw.any())
    over = (0, 1) if shared else 1
    e, m = (f(dr.double() * y.double()).sum(over, keepdim=True) for f in (lambda t: t, torch.abs))
    assert gg.shape == vectors[0].shape and ((gg.double() - e).abs() <= 2 ** -8 * e.abs() + 200 * 2 ** -24 * m).all()
    assert torch.equal(torch.autograd.grad(k2.residual_rmsnorm(norm, *leaves)[0], leaves[1], dr)[0], gy)
    assert torch.equal(torch.autograd.grad(k2.residual_rmsnorm(norm, *leaves)[0], leaves[2], dr)[0], gg)


def test_stream_refusals(k2, dev):
    x, g = torch.zeros(2, 4, 256, device=dev, dtype=torch.bfloat16), torch.zeros(2, 1, 256, device=dev, dtype=torch.bfloat16)
    f = k2._lib.resnorm_stream_bwd
    for bad in (lambda: f(x.float(), g, 4), lambda: f(x, g, 3), lambda: f(x, g[..., :128], 4), lambda: f(x, g, 4, x[:1]),
                lambda: f(x, g, 4, None, False), lambda: f(x, g.float(), 4), lambda: f(x, torch.cat([g, g]), 4)):
        with pytest.raises(ValueError):
            bad()
