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
