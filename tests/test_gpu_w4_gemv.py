"""GPU tests of the W4A8 forward for 1 to 8 rows (the matrix-vector paths) against the product in float64.

Every float32 sum starts from exact int32 dots of half groups or groups.  A lane adds at most K / 512 products with a
scale (the matrix cores' 32 groups of K = 16384; two half groups on the vector path), then at most ten more sums join lanes
and waves; with the epilogue's product and sums that is fewer than K / 512 + 16 float32 roundings (and one a rank), each at
most 2^-24 of the sum of the terms' magnitudes, and one rounding to bf16 (2^-8 of the value)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EDGES = [(1, 4, 128), (1, 1536, 6144), (2, 132, 2048), (3, 36, 2176), (4, 260, 4096), (5, 512, 640), (6, 1028, 8192),
         (7, 6144, 16384), (8, 18432, 1024), (8, 64, 16384), (2, 36864, 6144), (1, 2000, 256), (1, 4100, 2048),
         (2, 4108, 16384), (3, 4100, 128), (8, 4124, 8320), (5, 6148, 1152), (3, 4096, 8192), (1, 8196, 10240),
         (3, 4100, 9344), (8, 8192, 16384), (5, 6148, 12288), (6, 8196, 10240), (4, 4104, 9216)]


def _codes(q4):
    """(N, K/2) packed -> (N, K) int codes: byte j of a 16-wide chunk holds codes j and j + 8."""
    b = q4.view(q4.shape[0], -1, 8).int()
    c = torch.cat([b & 15, b >> 4], -1).reshape(q4.shape[0], -1)
    return torch.where(c > 7, c - 16, c)


def _inputs(M, N, K, dev, exact):
    g = torch.Generator(device=dev).manual_seed(M + N + K)
    qx = torch.randint(-128, 128, (M, K), device=dev, dtype=torch.int8, generator=g)
    q4 = torch.randint(0, 256, (N, K // 2), device=dev, dtype=torch.uint8, generator=g)
    if exact:
        s4 = torch.exp2(torch.randint(-1, 1, (K // 64, N), device=dev, generator=g).float()).bfloat16()
        sx = torch.exp2(torch.randint(-3, 3, (M,), device=dev, generator=g).float())
    else:
        s4 = (torch.rand(K // 64, N, device=dev, generator=g) * 1e-2 - 2e-3).bfloat16()
        s4[0] = 0
        sx = torch.rand(M, device=dev, generator=g) * 0.05 + 0.01
    w = (_codes(q4).double().view(N, -1, 64) * s4.t().double().unsqueeze(-1)).view(N, K)
    return g, qx, sx, q4, s4, w


@pytest.mark.parametrize("M,N,K", EDGES)
def test_exact_sums(k2, dev, M, N, K):
    """Power-of-two scales: every float32 sum is exact in any order, so the output is the product rounded once."""
    L = k2._lib
    g, qx, sx, q4, s4, w = _inputs(M, N, K, dev, True)
    acc = qx.double() @ w.t()
    assert acc.abs().max() * 2 < 2 ** 24
    y = L.gemm_w4a8(qx, sx, q4, s4)
    assert torch.equal(y, (acc * (sx.double() / 128).unsqueeze(1)).bfloat16())


@pytest.mark.parametrize("r", [0, 16, 48])
@pytest.mark.parametrize("M,N,K", EDGES)
def test_against_float64(k2, dev, M, N, K, r):
    L = k2._lib
    g, qx, sx, q4, s4, w = _inputs(M, N, K, dev, False)
    bias = torch.randn(N, device=dev, generator=g) if r else None
    u = torch.randn(M, r, device=dev, generator=g) if r else None
    B = torch.randn(N, r, device=dev, generator=g) * 0.01 if r else None
    y = L.gemm_w4a8(qx, sx, q4, s4, bias, u, B, 0.75)
    s = (sx.double() / 128).unsqueeze(1)
    ref, mag = (qx.double() @ w.t()) * s, (qx.double().abs() @ w.abs().t()) * s
    if r:
        ub, Bb = (u * 0.75).bfloat16().double(), B.bfloat16().double()     # the factors' bf16 rounding is the operator's
        ref, mag = ref + bias.double() + ub @ Bb.t(), mag + bias.double().abs() + ub.abs() @ Bb.abs().t()
    off = (y.double() - ref).abs()
    assert (off <= 2 ** -8 * ref.abs() + (K / 512 + 16 + r) * 2 ** -24 * mag).all()
    # the same bits again, and for a row in another's place
    assert torch.equal(L.gemm_w4a8(qx, sx, q4, s4, bias, u, B, 0.75), y)
    p = torch.arange(M - 1, -1, -1, device=dev)
    assert torch.equal(L.gemm_w4a8(qx[p], sx[p], q4, s4, bias, u[p] if r else None, B, 0.75), y[p])


@pytest.mark.parametrize("N,K", [(64, 128), (512, 512), (1536, 2048), (1536, 6144), (4092, 8192), (4100, 6272), (8188, 1024),
                                 (8192, 1024), (1536, 8320)])
def test_codes_made_on_the_way(k2, dev, N, K):
    """One token whose codes are not given: the codes, scale and output of the separate launches, bit for bit; a row of
    zeros, and the row's neighbours in a longer buffer untouched."""
    L = k2._lib
    g, _, _, q4, s4, _ = _inputs(1, N, K, dev, False)
    bias = torch.randn(N, device=dev, generator=g)
    x = torch.randn(2, K, device=dev, generator=g)
    x[:, ::37] *= 20
    x[1] = 0
    for row in x.bfloat16().split(1):
        qx, sx = torch.full((2, K), 99, dtype=torch.int8, device=dev), torch.full((2,), 7.0, device=dev)
        y, _ = L.linear_fwd(row, qx[:1], sx[:1], False, None, None, 0.0, q4, s4, bias, True, need_u=False)
        q0, s0, _ = L.rotquant(row)
        assert torch.equal(qx[:1], q0) and torch.equal(sx[:1], s0) and (qx[1] == 99).all() and sx[1] == 7
        assert torch.equal(y, L.gemm_w4a8(q0, s0, q4, s4, bias))


def test_rows_behind_the_output_stay(k2, dev):
    """The last rows of a partly filled workgroup: nothing is written past y."""
    L = k2._lib
    lib = L.load()
    M, N, K = 3, 20, 384
    _, qx, sx, q4, s4, _ = _inputs(M, N, K, dev, False)
    buf = torch.full((M * N + 64,), 7.0, device=dev, dtype=torch.bfloat16)
    P = L._ptr
    assert lib.k2q_gemm_w4a8(P(qx), P(sx), P(q4), P(s4), None, None, None, 0, 1.0, M, N, K, P(buf), L._stream(dev)) == 0
    assert torch.equal(buf[:M * N].view(M, N), L.gemm_w4a8(qx, sx, q4, s4)) and (buf[M * N:] == 7).all()


@pytest.mark.parametrize("rows", [1, 2, 8])
@pytest.mark.parametrize("rank", [0, 16, 24])
def test_layer_serves_tokens(k2, dev, rows, rank):
    """The module's call for a few tokens: the same rows inside a longer call go through the tiles and agree with it to
    the two schedules' float32 sums and the output's rounding; a captured graph replays it on new inputs."""
    K, N = 1024, 768
    g = torch.Generator().manual_seed(rows + rank)
    lin = torch.nn.Linear(K, N, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=g) * 0.02)
        lin.bias.copy_(torch.randn(N, generator=g))
    layer = k2.ConvRotLinear(lin, "w4a8")
    if rank:
        layer = k2.LoRALinear(layer, rank, 2.0 * rank)
        with torch.no_grad():
            layer.lora_B.copy_(torch.randn(N, rank, generator=g) * 0.02)
    x = torch.randn(40, K, generator=g).bfloat16().to(dev)
    with torch.no_grad():
        few, many = layer(x[:rows].clone()).double(), layer(x)[:rows].double()
        # two roundings of values that differ by float32 sums, and of u's sums before their bf16 rounding
        assert (few - many).norm() <= 2 ** -7 * many.norm()
        static = x[:rows].clone()
        layer(static.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(static.clone())
        for i in range(3):
            new = x[8 * i:8 * i + rows].clone()
            static.copy_(new)
            graph.replay()
            eager = layer(new.clone())
            torch.cuda.synchronize()
            assert torch.equal(out, eager), i


def test_refusals(k2, dev):
    """Widths that the path does not take are refused, few rows or many."""
    L = k2._lib
    _, qx, sx, q4, s4, _ = _inputs(2, 64, 256, dev, False)
    with pytest.raises((ValueError, RuntimeError)):
        L.gemm_w4a8(qx[:, :192].contiguous(), sx, q4, s4)
    with pytest.raises((ValueError, RuntimeError)):
        L.gemm_w4a8(qx, sx, q4[:63].contiguous(), s4)
    with pytest.raises((ValueError, RuntimeError)):
        L.gemm_w4a8(qx, sx[:1].clone(), q4, s4)


@pytest.mark.parametrize("M", [1, 2, 8])
def test_offsets_past_32_bits(k2, dev, M):
    """More than 2^31 bytes of packed weights: the last rows are those of the same rows alone (exact sums)."""
    L, N, K, n = k2._lib, 263168, 16384, 64
    g, qx, sx, q4, s4, _ = _inputs(M, n, K, dev, True)
    big = torch.empty(N, K // 2, device=dev, dtype=torch.uint8)
    big.random_(0, 256, generator=g)
    scales = torch.ones(K // 64, N, device=dev, dtype=torch.bfloat16)
    big[-n:], scales[:, -n:] = q4, s4
    assert torch.equal(L.gemm_w4a8(qx, sx, big, scales)[:, -n:], L.gemm_w4a8(qx, sx, q4, s4))
