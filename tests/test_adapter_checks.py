"""CPU tests of what the optimizer's step refuses, and of its options and states."""
import ctypes

import pytest
import torch


def _p(*shape, dtype=torch.float32, grad=True):
    p = torch.nn.Parameter(torch.zeros(shape, dtype=dtype))
    if grad:
        p.grad = torch.zeros(shape, dtype=dtype)
    return p


@pytest.mark.parametrize("bad", [{"lr": -1.0}, {"lr": float("nan")}, {"lr": torch.zeros(2)}, {"betas": (1.0, 0.9)},
                                 {"betas": (0.9, -0.1)}, {"eps": -1.0}, {"weight_decay": -1.0}, {"max_norm": -1.0},
                                 {"max_norm": float("nan")}, {"state_bits": 16}, {"seed": -1}, {"seed": 1 << 32},
                                 {"seed": 0.5}])
def test_adamw_refuses_options(k2, bad):
    with pytest.raises(ValueError):
        k2.AdamW([_p(4)], **bad)
    with pytest.raises(ValueError):
        k2.AdamW([{"params": [_p(4)], **bad}]) if "max_norm" not in bad else k2.AdamW([_p(4)], **bad)


def test_steps_run_on_the_gpu_alone(k2):
    opt = k2.AdamW([_p(4)])
    with pytest.raises(RuntimeError):
        opt.step()
    with pytest.raises(RuntimeError):
        k2.AdamW([_p(4)], max_norm=1.0).step()
    with pytest.raises(RuntimeError):
        k2.clip_grad_norm_([_p(4)], 1.0)


def test_gradients_that_are_refused(k2):
    with pytest.raises(ValueError, match="float64"):
        k2.clip_grad_norm_([_p(4, dtype=torch.float64)], 1.0)
    with pytest.raises(ValueError):
        k2.clip_grad_norm_([_p(4)], -1.0)
    with pytest.raises(ValueError):
        k2.clip_grad_norm_([_p(4)], float("nan"))
    with pytest.raises(ValueError, match="tensor"):
        k2.clip_grad_norm_(["p"], 1.0)
    p = _p(4)
    with pytest.raises(ValueError, match="twice"):
        k2.clip_grad_norm_([p, p], 1.0)
    q = _p(4, 3)
    q.grad = torch.zeros(1, 3).expand(4, 3)
    with pytest.raises(ValueError, match="gaps"):
        k2.clip_grad_norm_(q, 1.0)
    s = _p(4, 3)
    s.grad = torch.zeros(4, 3).to_sparse()
    with pytest.raises(ValueError, match="sparse"):
        k2.clip_grad_norm_(s, 1.0)
    assert float(k2.clip_grad_norm_([_p(4, grad=False)], 1.0)) == 0


def test_states_that_are_refused(k2):
    p = _p(3, 5)
    opt8 = k2.AdamW([p], state_bits=8)
    torch_opt = torch.optim.AdamW([_p(3, 5)])
    torch_opt.step()
    with pytest.raises(ValueError, match="8 bits"):
        opt8.load_state_dict(torch_opt.state_dict())
    assert not opt8.state
    other = torch.optim.AdamW([_p(3, 4)])
    other.step()
    with pytest.raises(ValueError, match="exp_avg must be"):
        k2.AdamW([p]).load_state_dict(other.state_dict())
    ams = torch.optim.AdamW([_p(3, 5)], amsgrad=True)
    with pytest.raises(ValueError, match="amsgrad"):
        k2.AdamW([p]).load_state_dict(ams.state_dict())
    with pytest.raises(ValueError):
        k2.AdamW([p]).load_state_dict(torch.optim.AdamW([_p(3, 5), _p(1)]).state_dict())


def test_step_entries_refuse_bad_arguments(k2):
    """The C entries' own checks (addresses that are never read)."""
    lib = k2._lib.load()
    a = 4096

    def one(**kw):
        return k2._lib.StepTensor(**{"p": a, "g": a, "n": 4, "at": 0, "index": 0, "dtype": 1, **kw})

    def call(t=None, count=None, bits=32, m=a, v=a, ms=None, vs=None, steps=a, lr=1e-3, b1=0.9, b2=0.9, eps=0.0, wd=0.0, norm=None,
             stochastic=0, ws=a, nws=1 << 20):
        t = [one()] if t is None else t
        arr = (k2._lib.StepTensor * max(len(t), 1))(*t)
        return lib.k2q_adamw(ctypes.addressof(arr), len(t) if count is None else count, bits, m, v, ms, vs, steps, lr, None, b1,
                             b2, eps, wd, norm, stochastic, 0, ws, nws, None)

    for bad in ({"count": 0}, {"t": [one(p=None)]}, {"t": [one(g=None)]}, {"t": [one(n=0)]}, {"t": [one(at=8)]},
                {"t": [one(at=-256)]}, {"t": [one(index=-1)]}, {"t": [one(dtype=3)]}, {"t": [one(p=a + 2)]},
                {"t": [one(), one()]}, {"bits": 4}, {"m": None}, {"v": a + 4}, {"bits": 8}, {"steps": None},
                {"lr": float("nan")}, {"b1": 1.0}, {"b2": -0.5}, {"eps": -1.0}, {"wd": float("nan")}, {"norm": a + 4},
                {"ws": None}, {"nws": 8}, {"stochastic": 1, "t": [one(dtype=2)]}):
        assert call(**bad) == -1, bad
    assert call(t=[one(n=1 << 43)]) == -4
    arr = (k2._lib.StepTensor * 2)(one(), one(n=100000))
    addr = ctypes.addressof(arr)
    need = lib.k2q_grad_norm_ws_bytes(addr, 2)
    assert need == 8 * (1 + 13) and lib.k2q_grad_norm_ws_bytes(addr, 0) == 0
    for args in ((addr, 2, -1.0, a, need, a), (addr, 2, 1.0, None, need, a), (addr, 2, 1.0, a, need - 1, a),
                 (addr, 2, 1.0, a, need, None), (addr, 0, 1.0, a, need, a), (None, 2, 1.0, a, need, a)):
        assert lib.k2q_grad_norm(*args, None) == -1
    assert lib.k2q_scale_grads(addr, 2, None, None) == -1
    for args in ((None, a, a, a, 256, 0, a, a), (a, a, a, a, 255, 0, a, a), (a, a, a, a, 256, 2, a, a), (a, a, a, a, 0, 0, a, a)):
        assert lib.k2q_moments(*args, None) == -1
