"""GPU tests of 8-bit moments, code by code: every operation that leads to one rounds on its own and correctly, so the codes
are those of the formula's 32-bit operations, restated here with elementary ones on the CPU, bit for bit."""
import pytest
import torch

from test_gpu_adamw import BLOCK, _bits

pytestmark = pytest.mark.gpu

N = 1 << 22
B1, B2 = 0.9, 0.999


def _value_m(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _value_v(codes):
    c = codes.int()
    e = (c >> 4).clamp(min=1)
    return (c - 16 * (e - 1)).float() * torch.exp2((e - 5).float())


def _codes(t, random, places, low, top):
    """The number of so many places below a value, or, with the chance that its distance gives, the one above; as integers
    from the evenly spaced ones near zero on."""
    blocks = t.abs().view(-1, BLOCK)
    most = blocks.amax(1)
    by = torch.where(most < 2.0 ** -100, 0.0, most.reciprocal() * top)
    a = (blocks * by.view(-1, 1)).clamp(max=top).view(-1)
    x = torch.maximum(a, (a + 2.0 ** low) * 0.5)        # below 2^low in the binary order under it: its steps are a's
    code = (x.view(torch.int32) + random.int() * (1 << 23 - places - 16) - ((126 + low) << 23)) >> (23 - places)
    return code, a, torch.where(most < 2.0 ** -100, 0.0, most) * torch.tensor(1 / top, dtype=torch.float32)


def _inputs(seed, kind):
    g = torch.Generator().manual_seed(seed)
    grad = torch.randn(N, generator=g) * 1e-3
    if kind == "wide":          # 60 binary orders, zeros among them
        grad *= torch.exp2(torch.randint(-50, 10, (N,), generator=g).float())
        grad[torch.rand(N, generator=g) < 0.01] = 0.0
        grad[5 * BLOCK:9 * BLOCK] = 0.0
    return grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["even", "wide"])
def test_codes_are_the_formulas_in_32_bits(k2, dev, kind, dtype):
    p = torch.nn.Parameter(torch.zeros(N, device=dev, dtype=dtype))
    opt = k2.AdamW([p], lr=1e-3, betas=(B1, B2), state_bits=8, seed=11)
    cm, cv = torch.zeros(N, dtype=torch.uint8), torch.zeros(N, dtype=torch.uint8)
    sm, sv = torch.zeros(N // BLOCK), torch.zeros(N // BLOCK)
    for step in range(1, 5):
        grad = _inputs(step, kind).to(dtype)
        p.grad = grad.to(dev)
        opt.step()
        g = grad.float()
        m = (_value_m(cm).view(-1, BLOCK) * sm.view(-1, 1)).view(-1) * B1 + g * (1 - B1)
        root = (_value_v(cv).view(-1, BLOCK) * sv.view(-1, 1)).view(-1)
        v = root * root * B2 + g * g * (1 - B2)
        random = _bits(11, step, torch.arange(N))
        cm, _, sm = _codes(m, random & 0xFFFF, 3, -6, 448.0)
        cm = (cm | m.signbit().int() << 7).to(torch.uint8)
        r = torch.sqrt(v.double()).float()      # of 53 bits, which rounds as a root of 24 does
        cv, a, sv = _codes(r, random >> 16, 4, 0, 31744.0)
        cv = cv.maximum((a > 0).int()).to(torch.uint8)
        st = opt.state[p]
        for name, want in (("exp_avg", cm), ("exp_avg_sq", cv)):
            have = st[name].view(torch.uint8).cpu()
            assert torch.equal(have, want), (step, name, int((have != want).sum()))
        assert torch.equal(st["exp_avg_scale"].cpu(), sm) and torch.equal(st["exp_avg_sq_scale"].cpu(), sv)
