"""GPU tests of the rotary positions against the rotation in float64.

A rotated value is two products and a sum in float32, with cos and sin of the float64 angle in float32: fewer than six
roundings of 2^-24 of the pair's length (times the factor), and one to the tensor's type (half its epsilon)."""
import math
from decimal import Decimal, localcontext

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11, torch.float32: 2 ** -24}


def _reference(rope, t, positions, heads_first=False, sign=1.0):
    """(value, pair length) in float64."""
    pos = positions.double()
    if rope.axes is not None:
        which = torch.tensor([a for a, d in enumerate(rope.axes) for _ in range(d // 2)], device=t.device)
        pos = pos[..., which]
    else:
        pos = pos.unsqueeze(-1)
    angle = pos * torch.tensor(rope.frequencies, dtype=torch.float64, device=t.device)
    if angle.dim() == 2:
        angle = angle.unsqueeze(0)
    angle = angle.unsqueeze(1 if heads_first else 2)
    c, s = angle.cos() * rope.factor, angle.sin() * rope.factor * sign
    d = t.double()
    n = rope.dim
    a, b = (d[..., 0:n:2], d[..., 1:n:2]) if rope.layout == "interleaved" else (d[..., :n // 2], d[..., n // 2:n])
    u, v, size = a * c - b * s, a * s + b * c, (a * a + b * b).sqrt() * rope.factor

    def join(p, q):
        return torch.stack([p, q], -1).flatten(-2) if rope.layout == "interleaved" else torch.cat([p, q], -1)

    rest = torch.zeros_like(d[..., n:])
    return torch.cat([join(u, v), d[..., n:]], -1), torch.cat([join(size, size), rest], -1)


def _check(rope, got, t, positions, heads_first=False, sign=1.0):
    ref, size = _reference(rope, t, positions, heads_first, sign)
    assert got.shape == t.shape and got.dtype == t.dtype
    # subnormal halves round by half of 2^-24
    assert ((got.double() - ref).abs() <= HALF_STEP[t.dtype] * ref.abs() + 6 * 2 ** -24 * size + 2.0 ** -25).all()


CASES = [  # (B, L, H, KV, D, dim, axes, heads first)
    (1, 1, 1, 1, 2, 2, None, False), (8, 1, 32, 8, 128, 128, None, False), (1, 333, 16, 4, 80, 32, None, False),
    (2, 77, 48, 12, 128, 128, (32, 48, 48), False), (2, 65, 6, 6, 96, 24, None, True), (1, 19, 5, 3, 80, 20, None, False),
    (3, 7, 2, 1, 13, 6, None, True), (1, 4097, 3, 1, 64, 64, (16, 24, 24), True), (1, 5, 2, 2, 1024, 1024, None, False),
    (1, 3, 1, 1, 4096, 512, None, False), (1, 1000, 1, 1, 16, 16, None, False), (2, 300, 60, 60, 128, 64, None, False),
    (1, 2, 700, 700, 32, 32, None, False)]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,H,KV,D,dim,axes,first", CASES)
def test_forward_and_gradient(k2, dev, B, L, H, KV, D, dim, axes, first, dtype, layout):
    rope = k2.RotaryEmbedding(dim, layout=layout, axes=axes)
    g = torch.Generator().manual_seed(B + L + H + D)

    def heads(n):
        return torch.randn(*((B, n, L, D) if first else (B, L, n, D)), generator=g).to(dtype).to(dev)

    q, k = heads(H).requires_grad_(), heads(KV).requires_grad_()
    pos = torch.randint(0, 1 << 18, (B, L) if axes is None else (B, L, len(axes)), generator=g).to(dev)
    q2, k2_ = rope(q, k, pos, heads_first=first)
    _check(rope, q2, q.detach(), pos, first)
    _check(rope, k2_, k.detach(), pos, first)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    gq, gk = torch.autograd.grad((q2, k2_), (q, k), (dq, dk))
    _check(rope, gq, dq, pos, first, -1.0)
    _check(rope, gk, dk, pos, first, -1.0)
    with torch.no_grad():                                       # the call without a node, and k alone behind None
        again = rope(q, None, pos, heads_first=first)
    assert again[1] is None and torch.equal(again[0], q2)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.float32, torch.float64])
def test_position_types_and_far_positions(k2, dev, dtype):
    """Angles keep their digits past 2^24 positions; negative and fractional positions turn the other way and in part."""
    rope = k2.RotaryEmbedding(64, layout="half")
    pos = torch.tensor([0, 1, -1, 4095, (1 << 24) + 1, (1 << 31) - 1, -(1 << 30) - 7], dtype=torch.float64)
    if dtype.is_floating_point:
        pos[3] = 4095.625
    if dtype == torch.float64:
        pos[5] = float(1 << 44) + 3
    pos = pos.to(dtype).to(dev)
    t = torch.randn(1, 7, 3, 64, device=dev)
    got, _ = rope(t, None, pos)
    # the reference's own angle is one float64 product: half a unit of 2^44 radians' last digit is 2^-9
    near = slice(0, 5) if dtype == torch.float64 else slice(0, 7)
    _check(rope, got[:, near], t[:, near], pos[near])
    if dtype == torch.float64:
        length = lambda v: (v[..., :32].double() ** 2 + v[..., 32:].double() ** 2).sqrt()       # noqa: E731
        assert (length(got) - length(t)).abs().max() < 1e-5
    assert torch.equal(got[:, 0], t[:, 0])


def _rest(position, frequency):
    """``position * frequency`` radians less the whole turns, from exact integers and 60 digits of pi."""
    with localcontext() as c:
        c.prec = 90
        turn = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
        a = Decimal(position) * Decimal(frequency)          # both binary fractions: exact
        return float(a - turn * (a / turn).to_integral_value())


@pytest.mark.parametrize("dtype", [torch.int64, torch.float64])
def test_angles_of_far_positions(k2, dev, dtype):
    """Every angle within the documented bound of the exact one, to a position of 2^44: 3 * 2^-53 of the angle and 2^-26
    turns; cos and sin in float32 are two units of 2^-24 more, their product with ones and zeros exact."""
    rope = k2.RotaryEmbedding(64, layout="half")
    far = [1, 4095, (1 << 20) + 1, (1 << 24) + 1, (1 << 28) - 3, -(1 << 31) + 5, (1 << 37) + 11, (1 << 44) + 3]
    t = torch.zeros(1, len(far), 1, 64, device=dev)
    t[..., :32] = 1
    got = rope(t, None, torch.tensor(far, dtype=dtype, device=dev))[0][0, :, 0].double().cpu()
    for i, p in enumerate(far):
        for j, f in enumerate(rope.frequencies):
            a = _rest(p, f)
            bound = abs(p * f) * 3 * 2.0 ** -53 + 2 * math.pi * 2.0 ** -26 + 2 * 2.0 ** -24
            assert abs(got[i, j] - math.cos(a)) <= bound and abs(got[i, j + 32] - math.sin(a)) <= bound, (p, j)


@pytest.mark.parametrize("scaling", [("linear", 4.0, None), ("ntk", 8.0, None), ("yarn", 4.0, 2048), ("yarn", 16.0, 32768)])
def test_scaled_frequencies(k2, dev, scaling):
    s = k2.RotaryScaling(*scaling)
    rope, plain = k2.RotaryEmbedding(128, layout="half", scaling=s), k2.RotaryEmbedding(128, layout="half")
    f, p = rope.frequencies, plain.frequencies
    assert f[0] == p[0] / (scaling[1] if s.kind == "linear" else 1.0)
    assert math.isclose(f[-1], p[-1] / scaling[1], rel_tol=1e-12)       # the slowest pair is interpolated
    assert all(a <= b for a, b in zip(f[1:], f[:-1]))
    assert rope.factor == (1.0 if s.kind != "yarn" else 0.1 * math.log(scaling[1]) + 1.0)
    t = torch.randn(2, 31, 4, 128, device=dev)
    pos = torch.randint(0, 1 << 17, (2, 31), device=dev)
    _check(rope, rope(t, None, pos)[0], t, pos)


def test_strides_views_and_positions_broadcast(k2, dev):
    """Heads sliced out of a fused projection, transposed, offset by odd elements, expanded; positions shared by the
    batch: the results of contiguous copies, in the layout of the input where that is dense."""
    rope = k2.RotaryEmbedding(32, layout="half")
    L, H, D = 21, 4, 64
    fused = torch.randn(2, L, 3 * H * D, device=dev).bfloat16()
    q = fused[..., :H * D].view(2, L, H, D)
    pos = torch.arange(L, device=dev) * 7
    ref, _ = rope(q.contiguous(), None, pos)
    assert torch.equal(rope(q, None, pos)[0], ref)
    t = q.contiguous().transpose(1, 2)
    got, _ = rope(t, None, pos, heads_first=True)
    assert got.stride() == t.stride() and torch.equal(got.transpose(1, 2), ref)
    odd = torch.empty(q.numel() + 5, device=dev, dtype=torch.bfloat16)[5:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(rope(odd, None, pos.expand(2, L))[0], ref)
    one = q[:, :, :1].expand(2, L, H, D)
    assert torch.equal(rope(one, None, pos[None])[0], rope(one.contiguous(), None, pos)[0])
    spread = torch.empty(2, L, H, 2 * D, device=dev, dtype=torch.bfloat16)[..., ::2]
    spread.copy_(q)
    assert torch.equal(rope(spread, q, pos)[0], ref)
    back = torch.arange(L - 1, -1, -1, device=dev) * 7
    assert torch.equal(rope(q.flip(1), None, back)[0].flip(1), ref)
    assert torch.equal(rope(q[0], q[0], pos)[1], ref[0])
    strided = torch.stack([pos, -pos], -1)[:, 0]
    assert strided.stride(0) == 2 and torch.equal(rope(q, None, strided)[0], ref)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,D", [(64, 64), (24, 96), (20, 80), (12, 30), (6, 7)])
@pytest.mark.parametrize("start", [0, 1, 2, 4, 8])
def test_every_vector_width(k2, dev, dim, D, start, dtype, layout):
    """Heads that start anywhere in their storage, and sizes that cut into vectors of eight, four, two or one: the bits of
    aligned copies, values between the rows untouched."""
    rope = k2.RotaryEmbedding(dim, layout=layout)
    wide = torch.randn(2, 9, 3, D + start, device=dev).to(dtype)
    q = wide[..., start:]
    pos = torch.arange(9, device=dev) * 11
    aligned = torch.zeros(2, 9, 3, (D + 15) // 16 * 16, device=dev, dtype=dtype)[..., :D]
    aligned.copy_(q)
    a, b = rope(q, None, pos)[0], rope(aligned, None, pos)[0]
    assert torch.equal(a, b)
    _check(rope, a, q, pos)


def test_gradients_of_one_of_both_and_expanded(k2, dev):
    rope = k2.RotaryEmbedding(64)
    q, k = torch.randn(1, 9, 4, 64, device=dev), torch.randn(1, 9, 2, 64, device=dev, requires_grad=True)
    pos = torch.arange(9, device=dev)
    q2, k2_ = rope(q, k, pos)
    gk, = torch.autograd.grad(k2_.sum(), k, retain_graph=True)      # an expanded gradient
    _check(rope, gk, torch.ones_like(k), pos, sign=-1.0)
    assert not q2.requires_grad or torch.autograd.grad(q2.sum(), k, allow_unused=True)[0] is None
    shared = torch.randn(1, 9, 1, 64, device=dev, requires_grad=True)   # one head read by four
    gs, = torch.autograd.grad(rope(shared.expand(1, 9, 4, 64), None, pos)[0], shared, torch.ones(1, 9, 4, 64, device=dev))
    ref, size = _reference(rope, torch.ones(1, 9, 1, 64, device=dev), pos, sign=-1.0)
    assert ((gs.double() - 4 * ref).abs() <= 4 * 8 * 2 ** -24 * size).all()
    x = torch.randn(1, 3, 2, 64, device=dev, dtype=torch.float32, requires_grad=True)
    v = torch.randn_like(x)
    g, = torch.autograd.grad((rope(x, None, pos[:3])[0] * v).sum(), x)
    d, e = torch.randn_like(x), 2.0 ** -6                            # linear in x: differences are exact but for rounding
    num = ((rope(x + e * d, None, pos[:3])[0] - rope(x - e * d, None, pos[:3])[0]).double() * v.double()).sum() / (2 * e)
    assert abs(num - (g.double() * d.double()).sum()) <= 2 ** -16 * (g.double().abs() * d.double().abs()).sum() + 1e-3
    with pytest.raises(RuntimeError):
        g1, = torch.autograd.grad(rope(x, None, pos[:3])[0].square().sum(), x, create_graph=True)
        g1.sum().backward()


def test_captured_and_other_stream(k2, dev):
    rope = k2.RotaryEmbedding(128, axes=(32, 48, 48), device=dev)
    q, k = torch.randn(2, 40, 6, 128, device=dev).bfloat16(), torch.randn(2, 40, 3, 128, device=dev).bfloat16()
    pos = torch.randint(0, 64, (2, 40, 3), device=dev)
    ref = rope(q, k, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rope(q, k, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, other))
    qs, ps = q.clone(), pos.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope(qs, k, ps)
    for i in range(3):
        ps.copy_(pos + i)
        qs.copy_(q * (i + 1))
        graph.replay()
        want = rope(q * (i + 1), k, pos + i)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_rest_and_neighbours_untouched(k2, dev):
    """Values past the rotated part are copied bit for bit (NaN payloads too), a NaN position spoils its token alone, and
    nothing is written outside a strided output's rows."""
    rope = k2.RotaryEmbedding(16)
    t = torch.randn(1, 5, 2, 40, device=dev)
    t[0, 2, 1, 30] = float("nan")
    pos = torch.tensor([0.0, 1.0, float("nan"), 3.0, float("inf")], device=dev)
    got, _ = rope(t, None, pos)
    assert torch.equal(got[..., 16:].contiguous().view(torch.int32), t[..., 16:].contiguous().view(torch.int32))
    assert got[0, [2, 4], :, :16].isnan().all() and not got[0, [0, 1, 3], :, :16].isnan().any()


def test_refusals(k2, dev):
    q, pos = torch.randn(2, 6, 4, 64, device=dev), torch.arange(6, device=dev)
    rope, three = k2.RotaryEmbedding(64), k2.RotaryEmbedding(64, axes=(16, 24, 24))
    for bad in (lambda: rope(q, None, pos[:5]), lambda: rope(q, None, pos.expand(3, 6)), lambda: rope(q, q[:1], pos),
                lambda: rope(q, q.bfloat16(), pos), lambda: rope(q.double(), None, pos), lambda: rope(q, None, pos.short()),
                lambda: rope(q, None, pos.cpu()), lambda: rope(q[..., :32], None, pos), lambda: rope(q[0, 0], None, pos),
                lambda: three(q, None, pos), lambda: three(q, None, torch.zeros(6, 2, device=dev)),
                lambda: rope(q, None, torch.zeros(6, 3, device=dev)), lambda: rope(q, q[:, :, :0], pos)):
        with pytest.raises(ValueError):
            bad()
    assert rope(q[:, :0], q[:, :0], pos[:0])[0].shape == (2, 0, 4, 64)


def test_offsets_past_32_bits(k2, dev):
    """2^31 elements and more in q: the last tokens are those of the same tokens alone, either way round."""
    L, H, D, n = 350000, 48, 128, 4
    q = torch.empty(1, L, H, D, device=dev, dtype=torch.bfloat16).normal_()
    k = torch.empty(1, L, 2, D, device=dev, dtype=torch.bfloat16).normal_()
    pos = torch.arange(L, device=dev)
    rope = k2.RotaryEmbedding(D, layout="half")
    a, e = rope(q, k, pos), rope(q[:, -n:], k[:, -n:], pos[-n:])
    assert all(torch.equal(u[:, -n:], v) for u, v in zip(a, e))
    t = q.requires_grad_()
    got, = torch.autograd.grad(rope(t, None, pos)[0], t, a[0])
    one = q[:, -n:].detach().requires_grad_()
    ref, = torch.autograd.grad(rope(one, None, pos[-n:])[0], one, e[0])
    assert torch.equal(got[:, -n:], ref)
