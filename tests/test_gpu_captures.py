"""GPU tests: what is kept between calls (an input's codes, siblings' outputs, float32 copies) and graph captures.  A graph
follows its static input at every replay, whatever ran before its capture on the same stream, and eager calls after a capture
take nothing that only a replay computes."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


def make_x(M, K, seed):
    return torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _layer(k2, dev, mode="w8a8", K=512, N=256, seed=0):
    lin = nn.Linear(K, N, bias=False, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        lin.weight.copy_(make_x(N, K, seed=seed).to(dev) * 0.05)
    return k2.ConvRotLinear(lin, mode)


def _replays(graph, static, outs, call, values):
    """Every replay against the eager result on the same values, with eager work between."""
    for v in values:
        static.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = call(v.clone())
        assert all(torch.equal(a, e) for a, e in zip(got, want))


@pytest.mark.parametrize("rows", [3, 64])
@pytest.mark.parametrize("mode", ["w8a8", "w4a8"])
def test_captured_after_a_call_on_the_same_stream(k2, dev, mode, rows):
    layer = _layer(k2, dev, mode)
    values = [make_x(rows, 512, seed=s).to(dev) for s in range(3)]

    def call(x):
        with torch.no_grad():
            return (*k2.input_codes(x), layer(x))

    for first in (layer, k2.input_codes):
        static = values[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        outs = []
        with torch.cuda.stream(side), torch.no_grad():
            first(static)                                       # its codes are kept for this tensor
        torch.cuda.synchronize()
        for g in graphs:                                        # the second capture finds the first one's codes
            with torch.cuda.graph(g, stream=side):
                outs.append(call(static))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            eager = call(static)                                # before any replay
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(eager, call(values[0].clone())))
        for g, o in zip(reversed(graphs), reversed(outs)):
            _replays(g, static, o, call, values)


def test_siblings_kept_before_a_capture(k2, dev):
    from krea2_amd.fused import _SiblingGroup
    layers = [_layer(k2, dev, N=256, seed=s) for s in range(2)]
    group = _SiblingGroup(layers)
    values = [make_x(64, 512, seed=s).to(dev) for s in range(3)]
    static = values[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            group.call(0, static)                               # keeps the other member's output
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = group.call(1, static)
        _replays(graph, static, [out], lambda x: [layers[1](x)], values)


def test_rotary_first_called_in_a_capture_says_what_it_needs(k2, dev):
    """A refusal, before anything is launched: the capture goes on, and takes the module once it has its frequencies."""
    rope, q, pos = k2.RotaryEmbedding(64), torch.randn(1, 5, 2, 64, device=dev), torch.arange(5, device=dev)
    k2.RotaryEmbedding(64, device=dev)(q, None, pos)
    ready = k2.RotaryEmbedding(64, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before it"):
            rope(q, None, pos)
        out, _ = ready(q, None, pos)
    for i in range(3):
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rope(q, None, pos)[0])


class Norm(nn.Module):
    def __init__(self, dev, K=512):
        super().__init__()
        self.eps, self.scale = 1e-5, nn.Parameter(torch.randn(K, device=dev).bfloat16(), requires_grad=False)


@pytest.mark.parametrize("entry", ["residual", "modulated"])
def test_a_norm_scale_first_seen_or_changed_around_a_capture(k2, dev, entry):
    """A bf16 norm scale is held in float32 between calls.  The copy that a capture makes belongs to its graph, and a graph
    follows the scale as it follows every input, also where a later eager call has replaced the kept copy."""
    norm, x = Norm(dev), make_x(33, 512, seed=4).to(dev)
    zero = torch.zeros(1, 512, device=dev, dtype=torch.bfloat16)

    def call(n):
        with torch.no_grad():
            return k2.residual_rmsnorm(n, x, x)[1] if entry == "residual" else k2.modulated_rmsnorm(n, x, zero, zero)

    def fresh():                                                # nothing kept
        n = Norm(dev)
        n.scale.copy_(norm.scale)
        return call(n)

    call(Norm(dev))                                             # the device is known to the wrappers
    torch.cuda.synchronize()
    first = torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        out = call(norm)
    assert torch.equal(call(norm), fresh())                     # eager, before any replay
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        out2 = call(norm)
    for i in range(3):
        norm.scale.normal_()
        want = fresh()
        assert torch.equal(call(norm), want)
        junk = torch.full((1 << 16,), float("nan"), device=dev)     # takes the memory of what was let go
        for g, o in ((first, out), (second, out2)):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want), i
        del junk


def test_a_captured_grouped_step_follows_its_factors(k2, dev):
    """Siblings with adapters: the stacked LoRA factors that eager calls keep are no part of a graph, whose replays follow
    an update of the factors in place."""
    from krea2_amd.fused import _SiblingGroup

    def members():
        return [k2.LoRALinear(_layer(k2, dev, N=256, seed=s), 16, 16.0) for s in range(2)]

    layers = members()
    group, x = _SiblingGroup(layers), make_x(64, 512, seed=7).to(dev)
    for m in layers:
        m.lora_B.data.normal_()
    with torch.no_grad():
        group.call(0, x.clone())                                # the stack is kept
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [group.call(0, x), group.call(1, x)]
        for _ in range(3):
            for m in layers:
                m.lora_A.normal_()
            graph.replay()
            torch.cuda.synchronize()
            fresh = _SiblingGroup(layers)
            y = x.clone()
            assert all(torch.equal(a, fresh.call(i, y)) for i, a in enumerate(out))


def test_siblings_kept_without_gradients_are_not_taken_with_them(k2, dev):
    """An output kept under no_grad, for an input or an adapter that did not ask for a gradient, has none to give: a call
    that asks runs its own forward."""
    from krea2_amd.fused import _SiblingGroup
    layers = [k2.LoRALinear(_layer(k2, dev, N=256, seed=s), 16, 16.0) for s in range(2)]
    for m in layers:
        m.lora_B.data.normal_()
    x = make_x(64, 512, seed=8).to(dev)
    group = _SiblingGroup(layers)
    with torch.no_grad():
        group.call(0, x)
    y = group.call(1, x)
    gA, = torch.autograd.grad(y.float().sum(), layers[1].lora_A)
    assert gA.any()
    group.call(0, x)
    x.requires_grad_()
    gx, = torch.autograd.grad(group.call(1, x).float().sum(), x)
    assert gx.any()
    x.requires_grad_(False)
    layers[1].lora_A.requires_grad_(False)
    group.call(0, x)
    layers[1].lora_A.requires_grad_()
    gA2, = torch.autograd.grad(group.call(1, x).float().sum(), layers[1].lora_A)
    assert torch.equal(gA2, gA)
