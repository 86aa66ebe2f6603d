"""CPU tests of what the optimizer's step and the banks of adapters refuse, of their options and states, and of what walks a
model to place banks, files and requests."""
import ctypes

import pytest
import torch
import torch.nn as nn


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


def test_hooks_closures_and_schedulers(k2):
    """What torch runs around a step: hooks of all optimizers and of one, the closure with gradients on, a scheduler's count,
    and its label under the profiler."""
    import importlib
    every = importlib.import_module("torch.optim.optimizer")
    opt, seen = k2.AdamW([_p(4, grad=False)]), []
    opt._step = lambda: seen.append("step")
    handles = [every.register_optimizer_step_pre_hook(lambda o, a, k: seen.append("all before")),
               every.register_optimizer_step_post_hook(lambda o, a, k: seen.append("all behind")),
               opt.register_step_pre_hook(lambda o, a, k: seen.append("before")),
               opt.register_step_post_hook(lambda o, a, k: seen.append("behind"))]

    def closure():
        seen.append(torch.is_grad_enabled())
        return 3.0

    with torch.no_grad():
        assert opt.step(closure) == 3.0
    assert seen == ["all before", "before", True, "step", "behind", "all behind"]
    for h in handles:
        h.remove()
    scheduler = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    del seen[:]
    assert opt.step() is None and seen == ["step"]
    scheduler.step()
    assert opt.param_groups[0]["lr"] == 5e-4
    with torch.profiler.profile() as p:
        opt.step()
    assert any(e.key == "Optimizer.step#AdamW.step" for e in p.key_averages())


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

    def call(t=None, count=None, bits=32, m=a, v=a, ms=None, vs=None, steps=a, lr=1e-3, b1=0.9, b2=0.9, eps=0.0, wd=0.0, sq=None,
             nsq=1, most=1.0, norm=a, stochastic=0, ws=a, nws=1 << 20):
        t = [one()] if t is None else t
        arr = (k2._lib.StepTensor * max(len(t), 1))(*t)
        return lib.k2q_adamw(ctypes.addressof(arr), len(t) if count is None else count, bits, m, v, ms, vs, steps, lr, None, b1,
                             b2, eps, wd, sq, nsq, most, norm, stochastic, 0, ws, nws, None)

    for bad in ({"count": 0}, {"t": [one(p=None)]}, {"t": [one(g=None)]}, {"t": [one(n=0)]}, {"t": [one(at=8)]},
                {"t": [one(at=-256)]}, {"t": [one(index=-1)]}, {"t": [one(dtype=3)]}, {"t": [one(p=a + 2)]},
                {"t": [one(), one()]}, {"bits": 4}, {"m": None}, {"v": a + 4}, {"bits": 8}, {"steps": None},
                {"lr": float("nan")}, {"b1": 1.0}, {"b2": -0.5}, {"eps": -1.0}, {"wd": float("nan")}, {"sq": a, "norm": a + 4},
                {"sq": a + 4}, {"sq": a, "nsq": 0}, {"sq": a, "most": -1.0}, {"sq": a, "norm": None},
                {"ws": None}, {"nws": 8}, {"stochastic": 1, "t": [one(dtype=2)]}):
        assert call(**bad) == -1, bad
    assert call(t=[one(n=1 << 43)]) == -4
    assert call(t=[one(n=(1 << 34) + 1)]) == -4 and call(t=[one(at=(1 << 46) + 256)]) == -4     # a launch's threads
    assert lib.k2q_moments(a, a, a, a, (1 << 34) + 256, 1, a, a, None) == -4
    arr = (k2._lib.StepTensor * 2)(one(), one(n=100000))
    addr = ctypes.addressof(arr)
    need = lib.k2q_grad_norm_ws_bytes(addr, 2)
    assert need == 8 * (1 + 98) and lib.k2q_grad_norm_ws_bytes(addr, 0) == 0
    for args in ((addr, 2, -1.0, a, need, a), (addr, 2, 1.0, None, need, a), (addr, 2, 1.0, a, need - 1, a),
                 (addr, 2, 1.0, a, need, a + 4), (addr, 0, 1.0, a, need, a), (None, 2, 1.0, a, need, a)):
        assert lib.k2q_grad_norm(*args, 0, None) == -1
    assert lib.k2q_grad_norm(addr, 2, 1.0, a, need, None, 1, None) == -1
    for args in ((None, a, a, a, 256, 0, a, a), (a, a, a, a, 255, 0, a, a), (a, a, a, a, 256, 2, a, a), (a, a, a, a, 0, 0, a, a)):
        assert lib.k2q_moments(*args, None) == -1


def test_bank_entries_refuse_bad_arguments(k2):
    """The C entries' own checks (addresses that are never read)."""
    lib, a = k2._lib.load(), 4096

    def bank(**kw):
        return k2._lib.Bank(**{"A": a, "B": a, "ids": a, "scale": 1.0, "ids64": 1, "dtype": 1, "count": 3, "R": 16, "K": 64,
                               "N": 128, **kw})

    def fwd(b, T=12, per=4, x=a, y=a, out=a, u=a, ws=a, nws=1 << 30):
        return lib.k2q_bank_fwd(ctypes.addressof(b), T, per, x, y, out, u, ws, nws, None)

    def bwd(b, T=12, per=4, dy=a, x=a, u=a, base=None, dx=a, dA=a, dB=a, ws=a, nws=1 << 30):
        return lib.k2q_bank_bwd(ctypes.addressof(b), T, per, dy, x, u, base, dx, dA, dB, ws, nws, None)

    for bad in ({"A": None}, {"B": a + 4}, {"ids": None}, {"ids": a + 4}, {"dtype": 2}, {"count": 0}, {"R": 8}, {"R": 24},
                {"K": 32}, {"K": 96}, {"N": 0}, {"N": 100}, {"ranks": a + 2}, {"scales": a + 2}):
        b = bank(**bad)
        assert fwd(b) == -1 and bwd(b) == -1, bad
        assert lib.k2q_bank_fwd_ws_bytes(ctypes.addressof(b), 12, 4) == 0
        assert lib.k2q_bank_bwd_ws_bytes(ctypes.addressof(b), 12, 4, 1) == 0
    for bad in ({"count": 1025}, {"R": 4112}, {"K": (1 << 24) + 64}):
        assert fwd(bank(**bad)) == -4 and bwd(bank(**bad)) == -4, bad
    assert fwd(bank(), T=0x7fffff04, per=4) == -4
    for T, bad in (((1 << 30) + 4, {"K": 64, "N": 64}), (1 << 30, {"K": 192, "N": 64}), (1 << 30, {"R": 16, "K": 64, "N": 192}),
                   (1 << 26, {"R": 144, "K": 64, "N": 64}), (12, {"R": 4096, "K": (1 << 19) + 64}),
                   (12, {"R": 4096, "N": 1 << 20})):      # the grids' threads, a piece's row numbers
        b = bank(**bad)
        assert fwd(b, T=T, per=4, nws=1 << 62) == -4 and bwd(b, T=T, per=4, nws=1 << 62) == -4, (T, bad)
        assert lib.k2q_bank_fwd_ws_bytes(ctypes.addressof(b), T, 4) == 0
    b = bank(R=16, K=64, N=64)
    assert lib.k2q_bank_fwd_ws_bytes(ctypes.addressof(b), 1 << 29, 4) >= (1 << 29) * 16 * 4     # at the limits
    for bad in ({"T": 0}, {"per": 0}, {"T": 13}, {"ws": None}, {"ws": a + 8}, {"nws": 0}):
        assert fwd(bank(), **bad) == -1 and bwd(bank(), **bad) == -1, bad
    for bad in ({"x": None}, {"x": a + 2}, {"y": a + 2}, {"out": None}, {"u": a + 4}):
        assert fwd(bank(), **bad) == -1, bad
    for bad in ({"dy": None}, {"dy": a + 2}, {"x": None}, {"u": None}, {"base": a + 2}, {"dA": a + 4},
                {"dx": None, "dA": None, "dB": None}):
        assert bwd(bank(), **bad) == -1, bad
    b = bank()
    need = lib.k2q_bank_bwd_ws_bytes(ctypes.addressof(b), 12, 4, 1)
    assert need > lib.k2q_bank_bwd_ws_bytes(ctypes.addressof(b), 12, 4, 0) > 0
    assert bwd(b, nws=need - 1) == -1


def test_add_adapters_refuses(k2):
    x, y = torch.zeros(2, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 3, 128, dtype=torch.bfloat16)
    A, B, ids = torch.zeros(4, 16, 64), torch.zeros(4, 128, 16), torch.zeros(2, dtype=torch.int64)
    f = k2.add_adapters
    for bad in (lambda: f(y[:1], x, A, B, ids), lambda: f(y, x, A[:3], B, ids), lambda: f(y, x, A, B[..., :8], ids),
                lambda: f(y, x, A[:, :8], B[..., :8], ids), lambda: f(y, x, A.half(), B.half(), ids),
                lambda: f(y, x, A, B.bfloat16(), ids), lambda: f(y, x, A, B, ids.float()), lambda: f(y, x, A, B, ids[:1]),
                lambda: f(y, x, A, B, torch.zeros(2, 3, 64, dtype=torch.int64)), lambda: f(y, x, A, B, ids.sum()),
                lambda: f(y, x, A, B, ids, torch.zeros(3)), lambda: f(y, x, A, B, ids, ranks=torch.zeros(4)),
                lambda: f(y, x, A[..., :32], B, ids), lambda: f(y[0, 0], x[0, 0], A, B, ids),
                lambda: f(y, x[..., :32], A[..., :32], B, ids), lambda: f(y, x, A[0], B[0], ids)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        f(y.float(), x.float(), A, B, ids)
    with pytest.raises(NotImplementedError):
        f(y, x, A, B, ids, torch.zeros(4, requires_grad=True))
    with pytest.raises(RuntimeError):
        f(y, x, A, B, ids)                  # arguments that fit, on a device that does not
    assert torch.equal(f(y[:0], x[:0], A, B, ids[:0]), y[:0])


@pytest.mark.parametrize("bad", [{"count": 0}, {"count": 1025}, {"rank": 0}, {"rank": 4097}, {"dtype": torch.float16},
                                 {"base": (96, 128)}, {"base": (128, 96)}])
def test_bank_refuses(k2, bad):
    args = {"base": (128, 192), "count": 2, "rank": 16, **bad}
    base = nn.Linear(*args.pop("base"))
    with pytest.raises(ValueError):
        k2.LoRABank(base, **args)


class _Block(nn.Module):
    def __init__(self):
        super().__init__()
        self.attn, self.mlp = nn.Module(), nn.Module()
        for n in ("wq", "wo"):
            setattr(self.attn, n, nn.Linear(64, 128 if n == "wq" else 64, bias=False))
        self.mlp.up = nn.Linear(64, 64, bias=False)


class _Dit(nn.Module):
    def __init__(self):
        super().__init__()
        self.blocks = nn.ModuleList(_Block() for _ in range(2))
        self.txtmlp = nn.Sequential(nn.Linear(64, 64))


def test_banks_hold_adapters_of_files(k2, tmp_path):
    """Adapters saved one by one fill a bank, in their own ranks and scales, and a bank's adapter is a file like any."""
    files = []
    for i, (rank, alpha) in enumerate(((4, 8.0), (16, 16.0), (20, 5.0))):
        dit = _Dit()
        adapters = k2.inject_lora(dit, rank, alpha, include_txtmlp=i == 1)
        with torch.no_grad():
            for m in adapters.values():
                m.lora_A.copy_(m.lora_A.bfloat16())
                m.lora_B.copy_(torch.randn(m.lora_B.shape).bfloat16())
        files.append((str(tmp_path / f"{i}.safetensors"), adapters, rank, alpha))
        k2.save_lora(adapters, files[-1][0], rank=rank, alpha=alpha)
    dit = _Dit()
    banks = k2.inject_lora_bank(dit, 3, 20)
    assert len(banks) == 6 and all(b.lora_A.shape[:2] == (3, 32) for b in banks.values())
    assert not any(p.requires_grad for n, p in dit.named_parameters() if "lora_" not in n)
    for i, (path, adapters, rank, alpha) in enumerate(files):
        assert k2.load_lora_into(banks, i, path) == (1 if i == 1 else 0)
        for name, bank in banks.items():
            A, B, a = bank.adapter(i)
            assert torch.equal(A, adapters[name].lora_A) and torch.equal(B, adapters[name].lora_B) and abs(a - alpha) < 1e-5
            assert float(bank.scales[i]) == torch.tensor(alpha / rank)
            assert not int(bank.lora_A[i, rank:].count_nonzero()) and not int(bank.lora_B[i, :, rank:].count_nonzero())
    out = str(tmp_path / "out.safetensors")
    k2.save_lora_from(banks, 2, out, metadata={"step": 3})
    again = k2.load_lora(_Dit(), out)
    assert all(torch.equal(again[n].lora_A, files[2][1][n].lora_A) for n in banks)
    # a file without some of the banks: those have no adapter there
    part = str(tmp_path / "part.safetensors")
    k2.save_lora({n: m for n, m in files[0][1].items() if "attn" in n}, part, rank=4, alpha=8.0)
    assert k2.load_lora_into(banks, 1, part) == 0
    assert not int(banks["blocks.0.mlp.up"].lora_B[1].count_nonzero())
    with pytest.raises(ValueError, match="no adapters"):
        k2.load_lora_into(banks, 0, part, key_prefix="text_encoder")
    with pytest.raises(ValueError, match="fit a bank"):
        next(iter(banks.values())).set_adapter(0, torch.zeros(33, 64), torch.zeros(128, 33))
    for bad in (3, -1):
        with pytest.raises(ValueError):
            next(iter(banks.values())).adapter(bad)
        with pytest.raises(ValueError):
            k2.load_lora_into(banks, bad, part)
    with pytest.raises(RuntimeError, match="inject_lora_bank"):
        k2.inject_lora_bank(_Dit(), 1, 4, targets=("attn.none",))


def test_requests_and_scales_reach_every_bank(k2):
    dit = _Dit()
    banks = k2.inject_lora_bank(dit, 2, 4)
    x = torch.randn(3, 5, 64)
    bank = banks["blocks.1.mlp.up"]
    assert torch.equal(bank(x), bank.base(x))
    ids = torch.tensor([0, 1, -1])
    with pytest.raises(RuntimeError):
        with k2.lora_requests(dit, ids):
            assert all(b.adapters is ids for b in banks.values())
            with k2.lora_disabled(dit):
                assert torch.equal(bank(x), bank.base(x))
            bank.base.bfloat16()
            bank(x.bfloat16())              # there is no kernel off the GPU
    assert all(b.adapters is None and b.scale_mul == 1.0 for b in banks.values())


def test_gradients_that_overlap_are_not_scaled(k2):
    flat = torch.ones(100)
    p, q = _p(60), _p(40)
    p.grad, q.grad = flat[:60], flat[59:99]
    with pytest.raises(ValueError, match="parameters 0 and 1 share memory"):
        k2.clip_grad_norm_([p, q], 1.0)
    assert bool((flat == 1).all())
