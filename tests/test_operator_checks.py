"""CPU tests of the arguments that the residual norm, the rotary positions and the W4A8 matrix-vector product refuse, and
of the rotary frequencies."""
import ctypes
import math

import pytest
import torch
import torch.nn as nn


class _Norm(nn.Module):
    def __init__(self, k):
        super().__init__()
        self.eps, self.scale = 1e-5, nn.Parameter(torch.zeros(k), requires_grad=False)


def test_residual_norm_refuses_before_any_launch(k2):
    x = torch.zeros(2, 3, 256, dtype=torch.bfloat16)
    v = torch.zeros(2, 1, 256, dtype=torch.bfloat16)
    f = k2.residual_rmsnorm
    for bad in (lambda: f(_Norm(256), x, x[:, :2]), lambda: f(_Norm(256), x, x, v, v), lambda: f(_Norm(128), x, x),
                lambda: f(_Norm(256), x, x, v[..., :128]), lambda: f(_Norm(256), x, x, v.expand(2, 3, 256)),
                lambda: f(_Norm(256), x, x, torch.cat([v, v[:1]])), lambda: f(nn.Module(), x, x),
                lambda: f(_Norm(64), x[..., :64], x[..., :64])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        f(_Norm(256), x, x.float())
    with pytest.raises(NotImplementedError):
        k2.input_codes(x.float())
    with pytest.raises(RuntimeError):
        f(_Norm(256), x, x, v)
    with pytest.raises(RuntimeError):
        f(_Norm(256), x[:, :0], x[:, :0])


def test_residual_norm_refuses_a_module_without_eps(k2):
    """A norm that names its eps otherwise is no argument of this function: the refusal says what is missing."""
    class Other(nn.Module):
        def __init__(self):
            super().__init__()
            self.weight, self.variance_epsilon = nn.Parameter(torch.ones(256)), 1e-6

    x = torch.zeros(2, 3, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="Other has no eps"):
        k2.residual_rmsnorm(Other(), x, x)


def test_entry_points_refuse_bad_arguments(k2):
    """The C entries' own checks (addresses that are never read)."""
    lib = k2._lib.load()
    p, odd = 4096, 4100

    def norm(x=p, ldx=256, y=p, gate=p, ldg=0, M=4, K=256, w=p, eps=1e-5, ms=p, ls=0, mb=p, lb=0, rows=4, r=p, h=p, q=p,
             s=p):
        return lib.k2q_resnorm_rotquant(x, ldx, y, 256, gate, ldg, M, K, w, 1.0, eps, ms, ls, mb, lb, rows, r, h, q, s, None)

    for bad in ({"x": None}, {"x": odd}, {"ldx": 255}, {"ldx": 128}, {"y": None}, {"gate": odd}, {"ldg": 4}, {"M": 0},
                {"K": 192}, {"w": None}, {"eps": float("nan")}, {"ms": None}, {"mb": None}, {"lb": -8}, {"rows": 0},
                {"r": None}, {"h": odd}, {"q": None}, {"s": None}):
        assert norm(**bad) == -1, bad
    assert norm(K=16512, ldx=16512) == -4 and norm(M=1 << 31) == -4

    def bwd(dh=p, r=p, M=4, K=256, ms=p, gate=p, rows=2, dx=p, dy=p, y=p, dw=p, ds=p, dg=p, ws=p, nws=1 << 30,
            shared=0):
        return lib.k2q_resnorm_bwd(dh, None, r, M, K, p, 1.0, 1e-5, ms, 0, gate, 0, rows, 0, dx, dy, y, 256, dw, ds, None, dg,
                                   shared, ws, nws, None)

    for bad in ({"dh": None}, {"r": odd}, {"M": 0}, {"K": 100}, {"ms": None}, {"gate": None}, {"dy": None}, {"rows": 3},
                {"rows": 0}, {"dx": None}, {"y": None}, {"ws": None}, {"nws": 16}, {"shared": 8}, {"shared": -1}):
        assert bwd(**bad) == -1, bad
    assert bwd(M=1 << 31) == -4 and bwd(M=1 << 30, rows=1, nws=1 << 62) == -4

    def stream(dr=p, M=4, K=256, gate=p, ld=0, rows=2, dy=p, y=p, ldy=256, dg=p, shared=0, ws=p, nws=1 << 30):
        return lib.k2q_resnorm_stream_bwd(dr, M, K, gate, ld, rows, dy, y, ldy, dg, shared, ws, nws, None)

    for bad in ({"dr": None}, {"dr": odd}, {"M": 0}, {"K": 100}, {"gate": None}, {"gate": odd}, {"ld": 4}, {"rows": 3},
                {"rows": 0}, {"dy": None, "dg": None}, {"dy": odd}, {"y": None}, {"y": odd}, {"ldy": 255}, {"dg": odd},
                {"ws": None}, {"ws": odd}, {"nws": 16}, {"shared": 8}, {"shared": -1}):
        assert stream(**bad) == -1, bad
    assert stream(M=1 << 31) == -4 and stream(K=16512) == -4

    heads = k2._lib.RotaryHeads(p, p, 4, 64 * 4 * 6, 256, 64, 64 * 4 * 6, 256, 64)

    def rot(t=heads, n=1, dtype=0, B=1, L=6, D=64, dim=64, layout=0, pos=p, pt=0, turns=p):
        return lib.k2q_rotary(ctypes.byref(t) if t is not None else None, n, dtype, B, L, D, dim, layout, pos, pt, 0, 1, 0,
                              turns, None, 1.0, 0, None)

    for bad in ({"t": None}, {"n": 0}, {"n": 3}, {"dtype": 3}, {"dtype": -1}, {"B": 0}, {"L": 0}, {"dim": 66}, {"dim": 63},
                {"dim": 0}, {"layout": 2}, {"pos": None}, {"pos": odd}, {"pt": 4}, {"turns": None},
                {"t": k2._lib.RotaryHeads(p, None, 4, 0, 0, 0, 0, 0, 0)}, {"t": k2._lib.RotaryHeads(p, p, 0, 0, 0, 0, 0, 0, 0)}):
        assert rot(**bad) == -1, bad
    assert rot(D=8192) == -4 and rot(D=4096, dim=2048) == -4 and rot(B=1 << 20, L=1 << 20) == -4


def test_residual_norm_workspace_is_small(k2):
    """The partial sums never exceed the tensors that they are sums of (an entry per row: 16 bytes of four sums an element
    once), however the rows are cut."""
    lib = k2._lib.load()
    for K in (128, 640, 2304, 6144, 16384):
        for rpb in (1, 2, 3, 7, 15, 16, 17, 40, 333):
            for entries in (1, 3, 64, 999, 9216):
                M = rpb * entries
                if M < 4096:
                    continue
                ws = lib.k2q_resnorm_bwd_ws_bytes(M, K, rpb)
                assert ws <= 2 * M * K + 16 * M, (M, K, rpb, ws)


def test_w4_gemv_needs_no_workspace(k2):
    lib = k2._lib.load()
    for M in range(1, 9):
        assert lib.k2q_linear_fwd_ws_bytes(1, M, 1536, 16384, 0) == 0


def test_rotary_module_refuses(k2):
    R, S = k2.RotaryEmbedding, k2.RotaryScaling
    for bad in (lambda: R(0), lambda: R(63), lambda: R(2048), lambda: R(64, layout="both"), lambda: R(64, axes=(32, 16)),
                lambda: R(64, axes=(33, 31)), lambda: R(64, theta=1.0), lambda: S("other", 2.0), lambda: S("linear", 0.5),
                lambda: S("linear", float("nan")), lambda: S("yarn", 4.0), lambda: S("yarn", 4.0, 2048, 1.0, 32.0),
                lambda: R(2, scaling=S("ntk", 2.0))):
        with pytest.raises(ValueError):
            bad()
    rope = R(64)
    q = torch.zeros(1, 5, 2, 64)
    with pytest.raises(RuntimeError):
        rope(q, None, torch.arange(5))
    with pytest.raises(ValueError):
        rope(q[..., :32], None, torch.arange(5))
    with pytest.raises(NotImplementedError):                    # a gradient that it would not give
        rope(q, None, torch.zeros(5, requires_grad=True))
    assert rope(q[:, :0], None, torch.arange(0))[0].shape == (1, 0, 2, 64)
    assert not list(rope.parameters()) and not rope.state_dict()


@pytest.mark.parametrize("shape", [(5, 2, 64), (1, 5, 2, 64)])
def test_rotary_hooks_run_once(k2, monkeypatch, shape):
    """Also where the call has no batch: a hook of the module sees the caller's tensors, once."""
    rope = k2.RotaryEmbedding(64)
    monkeypatch.setattr(k2._lib, "_device_check", lambda dev: None)
    monkeypatch.setattr(k2._lib, "rotary", lambda q, k, *rest: (q.clone(), None if k is None else k.clone()))
    seen = []
    rope.register_forward_pre_hook(lambda m, args: seen.append(args[0].shape))
    rope.register_forward_hook(lambda m, args, out: seen.append(out[0].shape))
    q = torch.zeros(shape)
    rope(q, q, torch.arange(5))
    assert seen == [q.shape, q.shape]


def test_rotary_frequencies(k2):
    R, S = k2.RotaryEmbedding, k2.RotaryScaling
    f = R(8, theta=10000.0).frequencies
    assert all(math.isclose(a, b) for a, b in zip(f, (1.0, 0.1, 0.01, 0.001)))
    assert R(8, axes=(4, 4)).frequencies == R(4).frequencies * 2
    g = R(128, scaling=S("yarn", 4.0, 4096)).frequencies
    p = R(128).frequencies
    kept = [2 * math.pi / v * 32 <= 4096 for v in p]             # over 32 turns within the original length
    slow = [2 * math.pi / v >= 4096 for v in p]                  # under one
    assert any(kept) and any(slow)
    for i, v in enumerate(p):
        if kept[i] and i + 1 < len(p) and kept[i + 1]:
            assert math.isclose(g[i], v)
        elif slow[i] and slow[i - 1]:
            assert math.isclose(g[i], v / 4)
        else:
            assert v / 4 <= g[i] * (1 + 1e-12) and g[i] <= v * (1 + 1e-12)
    assert R(64, scaling=S("yarn", 4.0, 4096, attention_factor=1.5)).factor == 1.5


def test_scaled_frequencies_of_every_pair(k2):
    """Each scaling's frequencies from its formula, every pair.  yarn at 128 values, theta 1e4 and 4096 positions: a pair i
    turns 4096 f_i / 2 pi times, 32 times at i = 64 ln(4096 / 64 pi) / ln 1e4 = 20.94 and once at 64 ln(4096 / 2 pi) / ln 1e4
    = 45.03, so the ramp runs from pair 20 to pair 46, a 26th a pair; at 8 positions no pair turns 32 times (from pair 0)
    and one at i = 1.68 once."""
    R, S = k2.RotaryEmbedding, k2.RotaryScaling
    p = R(128).frequencies
    for i, (lin, ntk, yarn, short) in enumerate(zip(*(R(128, scaling=s).frequencies for s in (
            S("linear", 4.0), S("ntk", 8.0), S("yarn", 4.0, 4096), S("yarn", 16.0, 8))))):
        base = math.exp(-2 * i / 128 * math.log(10000))
        assert math.isclose(p[i], base, rel_tol=1e-12) and math.isclose(lin, base / 4, rel_tol=1e-12)
        assert math.isclose(ntk, (10000 * 8 ** (128 / 126)) ** (-i / 64), rel_tol=1e-12)
        r = min(max((i - 20) / 26, 0), 1)
        assert math.isclose(yarn, base * (1 - 0.75 * r), rel_tol=1e-12)
        assert math.isclose(short, base * (1 - 15 / 16 * min(i / 2, 1)), rel_tol=1e-12)


def test_no_codes_kept_in_inference_mode(k2):
    """A tensor without a version counter is never known again, so an in-place write cannot leave stale codes."""
    from krea2_amd.quantize import _SharedInputQuant
    cache = _SharedInputQuant()
    with torch.inference_mode():
        h = torch.zeros(2, 128, dtype=torch.bfloat16)
        cache.seed(h, None, None)
        key, codes = cache.find(h)
        cache.keep(h, key, None, None)
    assert key is None and codes is None and cache.ref is None and cache.misses == 1


def test_calls_run_on_their_tensors_device(k2, monkeypatch):
    """The device of a call's tensors is the current one while it runs, and the caller's again afterwards."""
    class There:
        device = torch.device("cuda", 3)

    now = [0]

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            now.append(self.dev.index)

        def __exit__(self, *a):
            now.pop()

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[-1])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(k2._lib, "load", lambda: 1 / 0)
    call = k2._lib._on_its_device(lambda first, more=None: (now[-1], more))
    assert call(There(), more=5) == (3, 5) and call([None, There()]) == (3, None) and call([(There(), 1)]) == (3, None)
    assert call(torch.zeros(1)) == (0, None) and call(None) == (0, None) and call([]) == (0, None) and now == [0]
    now[0] = 3
    assert call(There()) == (3, None)
    for name in ("rotquant", "rmsmod_rotquant", "swiglu_rotquant", "rmsmod_bwd", "swiglu_bwd", "gemm_w4a8",
                 "gemm_dx_grouped"):
        assert hasattr(getattr(k2._lib, name), "__wrapped__"), name
