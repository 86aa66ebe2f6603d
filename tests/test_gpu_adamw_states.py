"""GPU tests of the optimizer's moments as its ``state`` says they are: cleared, replaced, and of parameters that change places,
against torch's own AdamW under the same edits."""
from collections import defaultdict

import pytest
import torch

from test_gpu_adamw import _near, _params

pytestmark = pytest.mark.gpu

SIZES = [(16, 40), (300,), (3, 3)]


def _grads(params, seed):
    for i, p in enumerate(params):
        p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(31 * seed + i)).to(p.device)


def _pair(k2, dev, **kw):
    a, b = (_params(dev, SIZES, torch.float32) for _ in range(2))
    return a, b, k2.AdamW(a, **kw), torch.optim.AdamW(b, **kw)


def _steps(oa, ob, a, b, first, n=2):
    for s in range(first, first + n):
        _grads(a, s)
        _grads(b, s)
        oa.step()
        ob.step()


def _equal(a, b, oa, ob, steps):
    """``steps`` updates of 1e-2, each off by 16 roundings of terms that are 4 times the update at most."""
    for p, q in zip(a, b):
        _near(p.detach(), q.detach().double(), 2.0 ** -22 * steps, steps * 1e-2 * 2.0 ** -18)
        assert float(oa.state[p]["step"]) == float(ob.state[q]["step"])


def _clear(opt, params):
    opt.state.clear()


def _new_dict(opt, params):
    opt.state = defaultdict(dict)


def _pop_one(opt, params):
    del opt.state[params[1]]


def _empty_one(opt, params):
    opt.state[params[0]] = {}


def _zero_moment(opt, params):
    st = opt.state[params[0]]
    st["exp_avg"] = torch.zeros_like(st["exp_avg"])


def _new_entries(opt, params):
    st = opt.state[params[2]]
    opt.state[params[2]] = {"step": torch.tensor(7.0), "exp_avg": st["exp_avg"] * 2, "exp_avg_sq": st["exp_avg_sq"] * 4}


@pytest.mark.parametrize("edit", [_clear, _new_dict, _pop_one, _empty_one, _zero_moment, _new_entries])
def test_the_state_is_what_the_next_step_uses(k2, dev, edit):
    a, b, oa, ob = _pair(k2, dev, lr=1e-2)
    _steps(oa, ob, a, b, 0)
    edit(oa, a)
    edit(ob, b)
    _steps(oa, ob, a, b, 2)
    _equal(a, b, oa, ob, 4)
    assert set(oa.state) == set(a)
    again = oa.state_dict()["state"]
    assert all(torch.equal(again[i][n], oa.state[p][n]) for i, p in enumerate(a) for n in ("step", "exp_avg", "exp_avg_sq"))
    m, v = oa.moments()
    at = 0
    for p in a:
        assert torch.equal(m[at:at + p.numel()].view(p.shape), oa.state[p]["exp_avg"])
        assert torch.equal(v[at:at + p.numel()].view(p.shape), oa.state[p]["exp_avg_sq"])
        at += -(-p.numel() // 256) * 256


def test_a_cleared_state_is_saved_as_cleared_and_read_as_zeros(k2, dev):
    a, b, oa, ob = _pair(k2, dev, lr=1e-2)
    _steps(oa, ob, a, b, 0)
    oa.state.clear()
    assert not oa.state_dict()["state"]
    assert not any(int(t.count_nonzero()) for t in oa.moments())


@pytest.mark.parametrize("size", [(300,), (512,), (40,)])
def test_a_parameter_in_anothers_place_starts_anew(k2, dev, size):
    """Of the same size, of more blocks, and of fewer."""
    a, b, oa, ob = _pair(k2, dev, lr=1e-2)
    _steps(oa, ob, a, b, 0)
    for params, opt in ((a, oa), (b, ob)):
        old, params[1] = params[1], torch.nn.Parameter(torch.ones(size, device=dev))
        opt.param_groups[0]["params"][1] = params[1]
        del opt.state[old]
    _steps(oa, ob, a, b, 2)
    assert float(oa.state[a[1]]["step"]) == 2 and float(oa.state[a[0]]["step"]) == 4
    _equal(a, b, oa, ob, 4)
    assert len(oa.state_dict()["state"]) == 3


def test_edits_of_one_group_leave_the_others(k2, dev):
    a, b = (_params(dev, SIZES, torch.float32) for _ in range(2))
    oa, ob = (cls([{"params": [p[0], p[2]]}, {"params": [p[1]]}], lr=1e-2)
              for cls, p in ((k2.AdamW, a), (torch.optim.AdamW, b)))
    _steps(oa, ob, a, b, 0)
    untouched = oa.state[a[1]]["exp_avg"].data_ptr()
    for opt, p in ((oa, a), (ob, b)):
        opt.state[p[2]] = {}
    _steps(oa, ob, a, b, 2)
    _equal(a, b, oa, ob, 4)
    assert oa.state[a[1]]["exp_avg"].data_ptr() == untouched
    oa.param_groups.pop()
    ob.param_groups.pop()
    _steps(oa, ob, a, b, 4)
    _equal(a, b, oa, ob, 6)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_fits_no_more_is_refused(k2, dev, bits):
    p = torch.nn.Parameter(torch.zeros(300, device=dev))
    p.grad = torch.ones_like(p)
    opt = k2.AdamW([p], state_bits=bits)
    opt.step()
    before = p.detach().clone()
    opt.state[p]["exp_avg"] = torch.zeros(299, device=dev)
    with pytest.raises(ValueError, match="exp_avg must be"):
        opt.step()
    assert torch.equal(p, before)
    opt.state.clear()
    opt.step()
    assert float(opt.state[p]["step"]) == 1


def test_edits_in_place_are_seen_and_copies_go_on(k2, dev):
    a, b, oa, ob = _pair(k2, dev, lr=1e-2)
    _steps(oa, ob, a, b, 0)
    for opt, p in ((oa, a), (ob, b)):
        opt.state[p[0]]["exp_avg"].zero_()
        opt.state[p[0]]["step"].fill_(0.0)
    held = oa.state[a[1]]["exp_avg"].data_ptr()
    _steps(oa, ob, a, b, 2)
    _equal(a, b, oa, ob, 4)
    assert oa.state[a[1]]["exp_avg"].data_ptr() == held


def test_other_bits_than_the_moments_have_are_refused(k2, dev):
    p = torch.nn.Parameter(torch.zeros(300, device=dev))
    p.grad = torch.ones_like(p)
    opt = k2.AdamW([p])
    opt.step()
    opt.param_groups[0]["state_bits"] = 8
    with pytest.raises(ValueError, match="a state in 8 bits"):
        opt.step()
    opt.state.clear()
    opt.step()
    assert opt.state[p]["exp_avg"].dtype == torch.float8_e4m3fn and float(opt.state[p]["step"]) == 1


def test_entries_of_the_users_own_stay(k2, dev):
    """What a program keeps in the state beside the parameters', and a parameter's that no group has any more."""
    a, b, oa, ob = _pair(k2, dev, lr=1e-2)
    oa.state["note"] = 3
    oa.state["more"]["x"] = a[0]
    _steps(oa, ob, a, b, 0)
    held = oa.state[a[1]]["exp_avg"].data_ptr()
    oa.state["note"] = 4
    _steps(oa, ob, a, b, 2)
    _equal(a, b, oa, ob, 4)
    assert oa.state["note"] == 4 and oa.state["more"]["x"] is a[0] and oa.state[a[1]]["exp_avg"].data_ptr() == held
