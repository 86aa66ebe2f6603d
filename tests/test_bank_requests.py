"""CPU tests of what a bank of adapters is asked for, and of its files."""
import asyncio
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from test_adapter_checks import _Dit


@pytest.fixture
def seen(k2, monkeypatch):
    """A model of banks, and the requests that each of their calls used, in place of the kernel (there is none on the CPU)."""
    import krea2_amd.lora_bank as lb
    calls = []

    def add(y, x, A, B, ids, scales, ranks, scale):
        calls.append(ids)
        return y + (x @ A[0].t()) @ B[0].t()

    monkeypatch.setattr(lb, "add_adapters", add)
    dit = _Dit()
    banks = k2.inject_lora_bank(dit, 2, 16)
    return dit, banks, calls


def _ids(*v):
    return torch.tensor(v)


def test_threads_keep_their_requests(k2, seen):
    """Two threads whose bodies overlap, the first one out first: each sees its own, and nothing stays behind."""
    dit, banks, calls = seen
    bank = banks["blocks.0.mlp.up"]
    mine, its = _ids(0), _ids(1)
    turns = [threading.Event() for _ in range(4)]
    out, x = {}, torch.zeros(1, 64)

    def other():
        assert turns[0].wait(20)
        out["before"] = bank.adapters
        with k2.lora_requests(dit, its):
            turns[1].set()
            assert turns[2].wait(20)            # the first body has ended
            out["inside"] = bank.adapters
            bank(x)
            out["used"] = calls[-1]
        out["behind"] = bank.adapters
        turns[3].set()

    t = threading.Thread(target=other)
    t.start()
    with k2.lora_requests(dit, mine):
        turns[0].set()
        assert turns[1].wait(20)
        assert bank.adapters is mine
        bank(x)
        assert calls[-1] is mine
    turns[2].set()
    assert turns[3].wait(20)
    t.join()
    assert out["before"] is None and out["inside"] is its and out["used"] is its and out["behind"] is None
    assert all(b.adapters is None for b in banks.values())
    n = len(calls)
    bank(x)
    assert len(calls) == n                      # the base alone


def test_tasks_keep_their_requests(k2, seen):
    """Two tasks of one thread that wait inside their bodies, and a function that one sends to another thread."""
    dit, banks, calls = seen
    bank = banks["blocks.0.mlp.up"]
    found = []

    async def one(ids, n):
        with k2.lora_requests(dit, ids):
            for _ in range(n):
                await asyncio.sleep(0.01)
                found.append(bank.adapters is ids)
            found.append(await asyncio.to_thread(lambda: bank.adapters is ids))
        found.append(bank.adapters is None)

    async def both():
        await asyncio.gather(one(_ids(0), 2), one(_ids(1), 4))

    asyncio.run(both())
    assert found and all(found) and bank.adapters is None


def test_bodies_nest(k2, seen):
    dit, banks, calls = seen
    bank, a, b = banks["blocks.1.attn.wo"], _ids(0), _ids(1)
    with k2.lora_requests(dit, a):
        with k2.lora_requests(dit.blocks[0], b):        # other banks
            assert bank.adapters is a and banks["blocks.0.attn.wo"].adapters is b
        with pytest.raises(KeyError):
            with k2.lora_requests(dit, None):
                assert bank.adapters is None
                raise KeyError
        assert bank.adapters is a
    assert bank.adapters is None
    bank.adapters = b                                   # requests of the bank's own, where no body is open
    assert bank.adapters is b
    with k2.lora_requests(dit, a):
        assert bank.adapters is a
    assert bank.adapters is b
    bank.adapters = None


def _train(dit, x, reentrant):
    def run(t):
        for b in dit.blocks:
            t = b.mlp.up(t)
        return t

    return checkpoint(run, x, use_reentrant=reentrant)


def test_passes_of_two_threads_are_recomputed_with_their_own(k2, seen):
    """Also where one has no requests and the other's body is open meanwhile."""
    dit, banks, calls = seen
    ids, used, errors = _ids(0), {}, []
    gate = threading.Barrier(2, timeout=20)

    def work(name, wanted):
        try:
            x = torch.randn(1, 64, requires_grad=True)
            if wanted is None:
                gate.wait()
                y = _train(dit, x, False)
                n = len(calls)
                y.sum().backward()
                used[name] = len(calls) - n
                gate.wait()
            else:
                with k2.lora_requests(dit, wanted):
                    y = _train(dit, x, False)
                    gate.wait()
                    gate.wait()
                    n = len(calls)
                    y.sum().backward()
                    used[name] = calls[n:]
        except Exception as e:          # noqa: BLE001 - shown below
            errors.append(e)
            gate.abort()

    threads = [threading.Thread(target=work, args=a) for a in (("with", ids), ("without", None))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and used["without"] == 0 and [u is ids for u in used["with"]] == [True, True]


@pytest.mark.parametrize("other", ["same", "another", "none", "own"])
def test_a_recomputed_pass_that_two_threads_may_want_is_refused(k2, seen, monkeypatch, other):
    """A thread of autograd's own, while two threads wait for their backward passes: it runs where both have the same requests
    or it opened a body, and with one of them alone as that one."""
    import krea2_amd.lora_bank as lb
    dit, banks, calls = seen
    bank, x, ids = banks["blocks.0.mlp.up"], torch.zeros(1, 64), _ids(0)
    bodies = [lb._Body(banks.values(), i, None) for i in (ids, _ids(0) if other == "another" else ids)]
    monkeypatch.setattr(lb, "_last", {-5: bodies[0], -6: None if other == "none" else bodies[1]})
    monkeypatch.setattr(lb, "_backward_callers", lambda: [-7, -5, -6])
    monkeypatch.setattr(torch._C, "_current_graph_task_id", lambda: 1)
    if other == "same":
        bank(x)
        assert calls[-1] is ids
    elif other == "own":
        mine = _ids(1)
        with k2.lora_requests(dit, mine):
            bank(x)
        assert calls[-1] is mine and set(lb._last) == {-5, -6}
    else:
        with pytest.raises(RuntimeError, match="several threads"):
            bank(x)
    monkeypatch.setattr(lb, "_backward_callers", lambda: [-5])
    bank(x)
    assert calls[-1] is ids


def test_a_compiled_bank_without_requests_is_one_graph(k2):
    bank = k2.LoRABank(torch.nn.Linear(64, 128), 2, 16)
    x = torch.randn(2, 64)
    run = torch.compile(bank, backend="eager", fullgraph=True)
    assert torch.equal(run(x), bank.base(x))
    with k2.lora_requests(bank, None):
        assert torch.equal(run(x), bank.base(x))
    with k2.lora_requests(bank, _ids(0)):
        assert bank._named == 1
    assert bank._named == 0 and torch.equal(run(x), bank.base(x))


# -- recomputed passes ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reentrant", [True, False])
def test_a_pass_recomputed_outside_its_body_is_refused(k2, seen, reentrant):
    """It would run without the adapters.  Inside the body, in one of its own, and without requests it runs."""
    dit, banks, calls = seen
    ids = _ids(0)
    x = torch.randn(1, 64, requires_grad=True)
    with k2.lora_requests(dit, ids):
        y = _train(dit, x, reentrant)
        y.sum().backward()
    assert len(calls) == 4 and all(c is ids for c in calls)
    with k2.lora_requests(dit, ids):
        y = _train(dit, x, reentrant)
    with pytest.raises(RuntimeError, match="lora_requests"):
        y.sum().backward()
    with k2.lora_requests(dit, ids):
        y = _train(dit, x, reentrant)
    with k2.lora_requests(dit, ids):
        y.sum().backward()
    for body in (False, True):                          # a forward pass without requests, and with those of no adapter
        del calls[:]
        if body:
            with k2.lora_requests(dit, None):
                y = _train(dit, x, reentrant)
        else:
            y = _train(dit, x, reentrant)
        y.sum().backward()
        assert not calls


# -- batches without rows ---------------------------------------------------------------------------------------------
def test_a_batch_without_rows_has_a_pass_back(k2):
    """Zeros for both factors, as products of no rows give."""
    x = torch.zeros(0, 3, 64, dtype=torch.bfloat16, requires_grad=True)
    y = torch.zeros(0, 3, 128, dtype=torch.bfloat16, requires_grad=True)
    A, B, ids = torch.ones(4, 16, 64, requires_grad=True), torch.ones(4, 128, 16, requires_grad=True), torch.zeros(0, dtype=torch.int64)
    for leaves in ((y, x, A, B), (A,), (B,), (x,)):
        args = [t if any(t is v for v in leaves) else t.detach() for t in (y, x, A, B)]
        out = k2.add_adapters(*args, ids)
        assert out.shape == y.shape and out.requires_grad
        for g, t in zip(torch.autograd.grad(out, leaves, torch.zeros_like(out)), leaves):
            assert g.shape == t.shape and g.dtype == t.dtype and not int(g.count_nonzero())
    with torch.no_grad():
        assert not k2.add_adapters(y, x, A, B, ids).requires_grad


# -- files ------------------------------------------------------------------------------------------------------------
def _file(k2, path, rank, only="", seed=0):
    adapters = k2.inject_lora(_Dit(), rank, float(rank))
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for m in adapters.values():
            m.lora_A.copy_(m.lora_A.bfloat16())
            m.lora_B.copy_(torch.randn(m.lora_B.shape, generator=g).bfloat16())
    kept = {n: m for n, m in adapters.items() if only in n}
    k2.save_lora(kept, str(path), rank=rank, alpha=float(rank))
    return str(path), kept


def test_a_file_that_does_not_fit_every_bank_changes_none(k2, tmp_path):
    banks = k2.inject_lora_bank(_Dit(), 2, 32)
    small = k2.inject_lora_bank(_Dit(), 2, 16)
    last = list(banks)[-1]
    banks[last] = small[last]
    path, _ = _file(k2, tmp_path / "a", 20)
    before = [t.clone() for b in banks.values() for t in (b.lora_A, b.lora_B, b.scales, b.ranks)]
    with pytest.raises(ValueError, match="fit a bank"):
        k2.load_lora_into(banks, 1, path)
    with pytest.raises(ValueError, match="adapter 2 of 2"):
        k2.load_lora_into(banks, 2, path)
    after = [t for b in banks.values() for t in (b.lora_A, b.lora_B, b.scales, b.ranks)]
    assert all(torch.equal(a, b) for a, b in zip(before, after))


def test_banks_that_a_file_does_not_name_hold_no_adapter_there(k2, tmp_path):
    """Rank 0, which the file written back leaves out again."""
    banks = k2.inject_lora_bank(_Dit(), 2, 16)
    path, kept = _file(k2, tmp_path / "a", 16, only="attn")
    assert k2.load_lora_into(banks, 1, path) == 0
    for name, b in banks.items():
        assert b.ranks.tolist() == [16, 16 if "attn" in name else 0]
        A, B, alpha = b.adapter(1)
        assert A.shape[0] == B.shape[1] == int(b.ranks[1]) and alpha == float(b.ranks[1])
        if "attn" not in name:
            assert not int(b.lora_A[1].count_nonzero()) and not int(b.lora_B[1].count_nonzero())
    out = str(tmp_path / "b")
    k2.save_lora_from(banks, 1, out)
    from safetensors.torch import load_file
    a, b = load_file(path), load_file(out)
    assert set(a) == set(b) and all(torch.equal(a[k], b[k]) for k in a)
    assert k2.load_lora_into(banks, 0, out) == 0
    for b in banks.values():                # an adapter that none of the banks holds
        b.ranks[0] = 0
    with pytest.raises(ValueError, match="no adapter"):
        k2.save_lora_from(banks, 0, out)
