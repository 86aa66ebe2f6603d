"""CPU tests of what the optimizer's hooks are given and may return: what torch's own AdamW gives them."""
import pytest
import torch


def _optimizers(k2):
    out = []
    for cls in (torch.optim.AdamW, k2.AdamW):
        p = torch.nn.Parameter(torch.zeros(4))
        opt = cls([p])
        if cls is k2.AdamW:
            opt._step = lambda: None            # the kernels run on the GPU alone
        out.append(opt)
    return out


def _calls():
    f = lambda: 3.0     # noqa: E731
    return {"plain": ((), {}), "positional": ((f,), {}), "keyword": ((), {"closure": f}), "none": ((None,), {})}


@pytest.mark.parametrize("call", list(_calls()))
def test_hooks_get_torchs_arguments(k2, call):
    args, kwargs = _calls()[call]
    got = []
    for opt in _optimizers(k2):
        seen = []
        opt.register_step_pre_hook(lambda o, a, k: seen.append(("pre", o is opt, a[0] is opt, a[1:], dict(k))))
        opt.register_step_post_hook(lambda o, a, k: seen.append(("post", o is opt, a[0] is opt, a[1:], dict(k))))
        seen.append(opt.step(*args, **kwargs))
        got.append(seen)
    assert got[0] == got[1]


def test_a_hook_replaces_the_arguments(k2):
    for opt in _optimizers(k2):
        behind = []
        opt.register_step_post_hook(lambda o, a, k: behind.append((a[1:], k)))
        f = lambda: 7.0     # noqa: E731
        first = opt.register_step_pre_hook(lambda o, a, k: ((o, f), {}))
        assert opt.step() == 7.0 and opt.step(lambda: 1.0) == 7.0
        first.remove()
        opt.register_step_pre_hook(lambda o, a, k: ((o,), {"closure": f}))
        assert opt.step(lambda: 1.0) == 7.0
        assert behind == [((f,), {}), ((f,), {}), ((), {"closure": f})]


@pytest.mark.parametrize("result", [3, (1,), (1, 2, 3), [(), {}]])
def test_a_hook_that_returns_no_pair_is_refused(k2, result):
    for opt in _optimizers(k2):
        ran = []
        opt.register_step_pre_hook(lambda o, a, k: result)
        with pytest.raises(RuntimeError, match="must return None or a tuple"):
            opt.step(lambda: ran.append(1))
        assert not ran


def test_calls_that_fit_no_step_are_refused(k2):
    for opt in _optimizers(k2):
        with pytest.raises(TypeError):
            opt.step(None, None)
        with pytest.raises(TypeError):
            opt.step(other=1)
