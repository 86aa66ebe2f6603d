"""CPU tests: the block's operators under a tracer and a forward-mode level.  The trace has to hold the call as a node of its
graph, and a tangent has to be refused, not dropped."""
import pytest
import torch
from torch.autograd import forward_ad


def _unseen(t):
    """The values of ``t`` in a tensor that no tracer and no forward-mode level has seen."""
    return torch.tensor(t.detach().float().tolist())


def _codes(h):
    """Codes without the rotation, on the tensor's values, as a kernel makes them."""
    v = _unseen(h).reshape(-1, h.shape[-1])
    s = v.abs().amax(1) / 127
    return (v / s[:, None]).round().to(torch.int8), s


@pytest.fixture
def codes(k2, monkeypatch):
    lib = k2._lib
    monkeypatch.setattr(lib, "rotquant", lambda x, want_xrot=False: (*_codes(x), None))
    monkeypatch.setattr(lib, "_stream", lambda dev: 0)
    k2.quantize.shared_input_quant.clear()
    yield k2.input_codes
    k2.quantize.shared_input_quant.clear()


def test_codes_in_a_trace_follow_their_input(codes):
    x, other = torch.randn(2, 4, 128).to(torch.bfloat16)
    traced = torch.jit.trace(lambda h: codes(h), x, check_trace=False)
    for a, e in zip(traced(other), _codes(other)):
        assert torch.equal(a, e)


def test_codes_refuse_a_tangent(codes):
    x = torch.randn(4, 128).to(torch.bfloat16)
    want = _codes(x)
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            codes(forward_ad.make_dual(x, torch.ones_like(x)))
        assert all(torch.equal(a, e) for a, e in zip(codes(x.clone()), want))    # no tangent: taken


def test_codes_kept_before_a_trace_are_no_part_of_it(codes):
    x, other = torch.randn(2, 4, 128).to(torch.bfloat16)
    codes(x)
    traced = torch.jit.trace(lambda h: codes(h), x, check_trace=False)
    again = torch.jit.trace(lambda h: codes(h), x, check_trace=False)
    for t in (traced, again):
        for a, e in zip(t(other), _codes(other)):
            assert torch.equal(a, e)


def test_a_norm_scale_kept_in_float32_is_no_part_of_a_recording(k2, monkeypatch):
    """On the CPU: the copy is a stream's own, and a capture neither keeps one nor takes a kept one."""
    from krea2_amd.fused import _norm_scale_f32
    at, now = 0, 0

    class Scale(torch.nn.Parameter):        # a parameter that says it is on the device
        is_cuda = True

    norm = torch.nn.Module()
    norm.scale = Scale(torch.ones(8, dtype=torch.bfloat16), requires_grad=False)
    monkeypatch.setattr(k2._lib, "_stream", lambda dev: at)
    monkeypatch.setattr(k2._lib, "_native", type("Native", (), {"capture_id": staticmethod(lambda stream: now)}))
    plain = _norm_scale_f32(norm)
    assert _norm_scale_f32(norm) is plain
    at = 16
    other = _norm_scale_f32(norm)
    assert other is not plain and _norm_scale_f32(norm) is other
    now = 5
    assert _norm_scale_f32(norm) is not other and _norm_scale_f32(norm) is not _norm_scale_f32(norm)
    now = 0
    assert _norm_scale_f32(norm) is other


def test_stacked_factors_are_no_part_of_a_recording(k2, monkeypatch):
    """On the CPU: a captured training step stacks the factors that its optimizer changes, and does not keep what only its
    replays fill."""
    from krea2_amd.fused import _SiblingGroup
    at, now = 0, 0

    class Factor(torch.nn.Parameter):
        is_cuda = True

    group, pair = _SiblingGroup([]), [Factor(torch.ones(16, 8)), Factor(torch.ones(16, 8))]
    monkeypatch.setattr(k2._lib, "_stream", lambda dev: at)
    monkeypatch.setattr(k2._lib, "_native", type("Native", (), {"capture_id": staticmethod(lambda stream: now)}))
    kept = group._a_stack(pair)
    assert group._a_stack(pair) is kept
    at = 16
    other = group._a_stack(pair)
    assert other is not kept and group._a_stack(pair) is other
    now = 5
    assert group._a_stack(pair) is not other
    now = 0
    assert group._a_stack(pair) is other


def test_an_effective_weight_built_in_a_capture_is_not_kept(k2, monkeypatch):
    now = 5
    q = torch.zeros(64, 128, dtype=torch.int8)
    layer = k2.ConvRotLinear.from_quantized(q, torch.zeros(64, dtype=torch.int32), None)
    monkeypatch.setattr(k2._lib, "dx_weight", lambda q, s, w4=False: torch.zeros(128, 64))
    monkeypatch.setattr(k2._lib, "recording", lambda stream: now)
    k2.set_dx_weight_cache(layer, True)
    layer.dx_weight()
    assert layer.dx_weight_kept is None
    now = 0
    kept = layer.dx_weight()
    now = 5
    assert layer.dx_weight() is kept


def test_codes_kept_by_another_thread_in_between(k2, monkeypatch):
    """Between a call's look at the kept tensor and its taking the codes another thread may keep others: the call takes the
    codes of its own tensor."""
    cache, x, y = k2.quantize._SharedInputQuant(), torch.zeros(2, 128), torch.ones(2, 128)

    class Key:
        def __eq__(self, other):            # what runs between the two
            cache.keep(y, other, "qy", "sy")
            return True

    monkeypatch.setattr(cache, "_key", lambda t: Key())
    cache.seed(x, "qx", "sx")
    assert cache.find(x)[1] == ("qx", "sx")
    cache.seed(x, "qx", "sx")
    assert cache.lookup(x, x) == ("qx", "sx")


def test_codes_of_one_recording_are_no_part_of_another(k2, monkeypatch):
    """On the CPU: a hit needs the stream's capture, or none, that the codes were kept in."""
    cache, now = k2.quantize._SharedInputQuant(), 0
    monkeypatch.setattr(k2._lib, "_stream", lambda dev: 16)
    monkeypatch.setattr(k2._lib, "_native", type("Native", (), {"capture_id": staticmethod(lambda stream: now)}))
    x = torch.zeros(2, 128)
    for now in (0, 7, 8, 0, -3, -3):
        assert cache.find(x)[1] is None
        cache.seed(x, now, now)
        assert cache.find(x)[1] == ((now, now) if now >= 0 else None)       # -3: the stream could not be asked


class _Norm(torch.nn.Module):
    def __init__(self, k):
        super().__init__()
        self.eps, self.scale = 1e-5, torch.nn.Parameter(torch.zeros(k), requires_grad=False)


@pytest.fixture
def residual(k2, monkeypatch):
    def native(x, y, gate, w, add, eps, scale, shift):
        r = (_unseen(x) + (1 if gate is None else _unseen(gate)) * _unseen(y)).to(torch.bfloat16)
        h = (r.float() * torch.rsqrt(r.float().square().mean(-1, keepdim=True) + eps) * (_unseen(w) + add)).to(torch.bfloat16)
        return _unseen(r).to(r.dtype), _unseen(h).to(h.dtype), *_codes(h)

    monkeypatch.setattr(k2._lib, "resnorm_native", native)
    monkeypatch.setattr(k2._lib, "_stream", lambda dev: 0)
    norm = _Norm(128)
    yield lambda x, y: k2.residual_rmsnorm(norm, x, y)
    k2.quantize.shared_input_quant.clear()


@pytest.fixture
def rotary(k2, monkeypatch):
    def turned(q, k, positions, turns, axis, axes, half, factor, inverse, heads_first):
        a = _unseen(positions)[:, None, None] * _unseen(turns) * 6.283185307179586
        u, v = _unseen(q).chunk(2, -1)
        return torch.tensor(torch.cat([u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()], -1).tolist()), None

    monkeypatch.setattr(k2._lib, "rotary", turned)
    monkeypatch.setattr(k2._lib, "_device_check", lambda dev: None)
    rope = k2.RotaryEmbedding(16, layout="half")
    return lambda q, pos: rope(q, None, pos)[0]


def test_residual_norm_and_rotary_in_a_trace_follow_their_inputs(residual, rotary):
    a, b, c, d = torch.randn(4, 2, 3, 128).to(torch.bfloat16)
    with torch.no_grad():
        traced = torch.jit.trace(residual, (a, b), check_trace=False)
        for got, want in zip(traced(c, d), residual(c, d)):
            assert torch.equal(got, want)
        q, pos = torch.randn(1, 5, 2, 16), torch.arange(5.0)
        traced = torch.jit.trace(rotary, (q, pos), check_trace=False)
        assert torch.equal(traced(2 * q, pos + 3), rotary(2 * q, pos + 3))


def test_residual_norm_and_rotary_refuse_a_tangent(residual, rotary):
    x, q, pos = torch.randn(2, 3, 128).to(torch.bfloat16), torch.randn(1, 5, 2, 16), torch.arange(5.0)
    with torch.no_grad():
        want = residual(x, x)[1], rotary(q, pos)
        with forward_ad.dual_level():
            for call in (lambda: residual(forward_ad.make_dual(x, torch.ones_like(x)), x),
                         lambda: rotary(forward_ad.make_dual(q, torch.ones_like(q)), pos)):
                with pytest.raises((RuntimeError, NotImplementedError)):
                    call()
            assert torch.equal(residual(x, x)[1], want[0]) and torch.equal(rotary(q, pos), want[1])
