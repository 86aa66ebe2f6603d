"""The operators between the quantized linears of a transformer block, and the linear's form for single tokens: the
RMSNorm with the residual's addition and 8-bit codes, rotary positions of queries and keys, and the matrix-vector product
with 4-bit weights and group scales.

Every case is one call as a program makes it.  ``run`` computes it in plain torch operations, or, where ``own`` is true,
through the package.  Every tensor that an operator's formula names is a bf16 tensor in the model, so both round there.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------
def _norm(name, batch, tokens, width, gated, grads="none"):
    c = {"kind": "norm", "batch": batch, "tokens": tokens, "width": width, "gated": gated, "grads": grads}
    return {"name": name, **c} if name else c


def _rotary(name, batch, tokens, heads, kv, dim, rotary, layout, axes="", scaling="none", factor=1.0, original=0,
            far=0, dtype="bf16", heads_first=False, train=False):
    c = {"kind": "rotary", "batch": batch, "tokens": tokens, "heads": heads, "kv": kv, "dim": dim, "rotary": rotary,
         "layout": layout, "axes": axes, "scaling": scaling, "factor": factor, "original": original, "far": far,
         "dtype": dtype, "heads_first": heads_first, "train": train}
    return {"name": name, **c} if name else c


def _w4(name, rows, k, n, rank, bias):
    c = {"kind": "w4", "rows": rows, "in": k, "out": n, "rank": rank, "bias": bias}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one new token: the residual's addition before a plain norm, as in a decoder that answers token by token
        _norm("norm_token", 1, 1, 6144, False),
        # a prompt in the text encoder's width, its length whatever the prompt gives
        _norm("norm_prompt", 1, 333, 2560, False),
        # the gated residual and modulated norm of a block at 1024 x 1024 (4096 image + 512 text tokens), guidance batch 2
        _norm("norm_image", 2, 4608, 6144, True),
        # LoRA training at 1024 x 1024: gradients of the stream and of the attention's output
        _norm("norm_train", 1, 4608, 6144, True, "inputs"),
        # full fine-tuning at 256 x 256, batch 2: gradients of the gate, the modulation and the norm's scale too
        _norm("norm_finetune", 2, 768, 6144, True, "all"),
        # eight requests far into a long context, one new token each
        _rotary("rotary_token", 8, 1, 32, 8, 128, 128, "half", scaling="yarn", factor=4.0, original=32768, far=131072),
        # a prompt whose heads carry positions in part (odd length, fp16)
        _rotary("rotary_prompt", 1, 333, 16, 4, 80, 32, "half", scaling="linear", factor=2.0, far=4096, dtype="f16"),
        # the DiT's queries and keys at 1024 x 1024: 48 heads over 12, positions along three axes
        _rotary("rotary_image", 1, 4608, 48, 12, 128, 128, "interleaved", axes="32,48,48"),
        # training at 2048 x 2048 (16384 image + 512 text tokens), forward and backward
        _rotary("rotary_train", 1, 16896, 48, 12, 128, 128, "interleaved", axes="32,48,48", train=True),
        # one token through the key projection over an int4 base
        _w4("w4_token", 1, 6144, 1536, 0, False),
        # the modulation linear at batch 2: the whole weight is streamed for two rows
        _w4("w4_modulation", 2, 6144, 36864, 16, False),
        # a few tokens through the MLP down-projection
        _w4("w4_tokens", 7, 16384, 6144, 16, True),
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, min(hi, step * round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    """One more call of the same ranges: one token to the longest sequence, widths from the small blocks' to the widest
    linear's, every layout, scaling and type."""
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("norm", "rotary", "w4"))
        if kind == "norm":
            c = _norm(None, rng.choice((1, 1, 2, 3)), _log_int(rng, 1, 9000), _log_int(rng, 256, 16384, 128),
                      rng.random() < 0.6, rng.choice(("none", "none", "inputs", "all")))
        elif kind == "rotary":
            dim = rng.choice((64, 80, 96, 128, 128, 256))
            layout = rng.choice(("interleaved", "half"))
            axes = rng.choice(("", "", "three"))
            rotary = dim if axes else rng.choice((dim, dim, dim // 2, dim // 4 - dim // 4 % 2))
            if axes:
                first = rotary // 4 // 2 * 2
                rest = (rotary - first) // 2 // 2 * 2
                axes = "%d,%d,%d" % (rotary - 2 * rest, rest, rest)
            scaling = "none" if axes else rng.choice(("none", "linear", "ntk", "yarn"))
            heads = rng.choice((4, 16, 32, 48))
            c = _rotary(None, rng.choice((1, 1, 2, 5)), _log_int(rng, 1, 16896), heads, rng.choice((heads, heads // 4)),
                        dim, rotary, layout, axes, scaling, 1.0 if scaling == "none" else rng.choice((2.0, 4.0, 7.5)),
                        rng.choice((2048, 32768)) if scaling == "yarn" else 0, 0 if axes else _log_int(rng, 1, 1 << 20),
                        rng.choice(("bf16", "bf16", "f16", "f32")), rng.random() < 0.3, rng.random() < 0.4)
        else:
            c = _w4(None, rng.randint(1, 8), _log_int(rng, 128, 16384, 128), _log_int(rng, 128, 36864, 128),
                    rng.choice((0, 16, 16, 32, 64)), rng.random() < 0.4)
        if _cost(c) <= most:
            return c


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------
def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(shape, device=DEV, dtype=torch.float32).normal_(0.0, std, generator=g).to(dtype)


def _stream(g, *shape):
    """A residual stream: N(0, 1), 1 % of the channels 20 times as large."""
    x = torch.empty(shape, device=DEV, dtype=torch.float32).normal_(generator=g)
    x[..., torch.randperm(shape[-1], device=DEV, generator=g)[:max(1, shape[-1] // 100)]] *= 20.0
    return x.to(torch.bfloat16)


class _NormModule(torch.nn.Module):
    """The block's norm: weight ``scale + 1``."""

    def __init__(self, scale):
        super().__init__()
        self.eps = EPS
        self.scale = torch.nn.Parameter(scale, requires_grad=False)


def _norm_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    b, t, k = case["batch"], case["tokens"], case["width"]
    s = {"x": _stream(g, b, t, k), "y": _normal(g, b, t, k), "scale": _normal(g, k, std=0.1, dtype=torch.float32)}
    if case["gated"]:
        # the chunks of one modulation tensor, as the block's modulation gives them
        s["gate"], s["p"], s["b"] = _normal(g, b, 1, 3 * k, std=0.3).chunk(3, -1)
    if case["grads"] != "none":
        s["dr"], s["dh"] = _normal(g, b, t, k, std=1e-3), _normal(g, b, t, k, std=1e-3)
    return s


def _axes(case):
    return [int(v) for v in case["axes"].split(",")] if case["axes"] else [case["rotary"]]


def _positions(case, g):
    """Token indices up to ``far``; or, along three axes, 512 text tokens at the origin and a square grid of image
    tokens (fewer where the sequence is shorter)."""
    b, t = case["batch"], case["tokens"]
    if not case["axes"]:
        start = torch.randint(0, max(1, case["far"] - t + 1), (b, 1), device=DEV, generator=g)
        return start + torch.arange(t, device=DEV)
    text = min(512, t // 2)
    side = max(1, math.isqrt(t - text))
    i = torch.arange(t - text, device=DEV)
    grid = torch.stack([torch.zeros_like(i), i // side, i % side], -1)
    return torch.cat([torch.zeros(text, 3, dtype=torch.int64, device=DEV), grid]).expand(b, t, 3).contiguous()


def _rotary_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def heads(n, std):
        shape = (case["batch"], n, case["tokens"]) if case["heads_first"] else (case["batch"], case["tokens"], n)
        return _normal(g, *shape, case["dim"], std=std, dtype=dt)

    s = {"q": heads(case["heads"], 1.0), "k": heads(case["kv"], 1.0), "positions": _positions(case, g)}
    if case["train"]:
        s["dq"], s["dk"] = heads(case["heads"], 1e-3), heads(case["kv"], 1e-3)
    return s


def _w4_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    m, k, n, r = case["rows"], case["in"], case["out"], case["rank"]
    codes = torch.empty(n, k, device=DEV, dtype=torch.float32).normal_(0.0, 2.7, generator=g).round_().clamp_(-7, 7)
    codes = codes.to(torch.int8).view(n, k // 16, 2, 8) & 15
    s = {"x": _stream(g, m, k), "codes": (codes[:, :, 0] | codes[:, :, 1] << 4).view(torch.uint8).reshape(n, k // 2),
         "scales": (torch.rand(k // 64, n, device=DEV, generator=g) * 0.06 + 0.05).to(torch.bfloat16)}
    s["bias"] = _normal(g, n, std=0.1, dtype=torch.float32) if case["bias"] else None
    s["A"] = _normal(g, r, k, std=0.01, dtype=torch.float32) if r else None
    s["B"] = _normal(g, n, r, std=0.01, dtype=torch.float32) if r else None
    return s


def _frequencies(case):
    """Radians per position of every pair, in 64 bits, and the factor on the rotated values."""
    base, s, out = 10000.0, case["factor"], []
    for d in _axes(case):
        i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
        if case["scaling"] == "ntk":
            base = 10000.0 * s ** (d / (d - 2))
        f = base ** (-2.0 * i / d)
        if case["scaling"] == "linear":
            f = f / s
        if case["scaling"] == "yarn":
            edge = [d * math.log(case["original"] / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
            low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), d - 1)
            ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
            f = f * (1 - ramp) + f / s * ramp
        out.append(f)
    return torch.cat(out), 0.1 * math.log(s) + 1.0 if case["scaling"] == "yarn" else 1.0


def prepare(case, seed):
    if case["kind"] == "norm":
        s = _norm_inputs(case, seed)
        s["norm"] = _NormModule(s.pop("scale"))
    elif case["kind"] == "rotary":
        s = _rotary_inputs(case, seed)
        s["f"], s["m"] = _frequencies(case)
        s["axis"] = torch.repeat_interleave(torch.arange(len(_axes(case)), device=DEV),
                                            torch.tensor([d // 2 for d in _axes(case)], device=DEV))
    else:
        s = _w4_inputs(case, seed)
    if case["kind"] != "rotary":
        s["hadamard"] = _hadamard()
    s["case"] = case
    if own:
        _keep(s)
    return s


def _keep(s):
    """What a program that uses the package holds: the rotary module, the quantized layer with its adapter."""
    import __graft_entry__
    k2 = s["k2"] = __graft_entry__.load_package()
    case = s["case"]
    if case["kind"] == "rotary":
        scaling = None
        if case["scaling"] != "none":
            scaling = k2.RotaryScaling(case["scaling"], case["factor"], case["original"] or None)
        s["rotary"] = k2.RotaryEmbedding(case["rotary"], layout=case["layout"], scaling=scaling,
                                         axes=_axes(case) if case["axes"] else None)
    elif case["kind"] == "w4":
        base = k2.ConvRotLinear.from_quantized(s["codes"], s["scales"].view(torch.int16), s["bias"], "w4a8")
        s["layer"] = base
        if case["rank"]:
            s["layer"] = k2.LoRALinear(base, case["rank"], float(case["rank"]))
            with torch.no_grad():
                s["layer"].lora_A.copy_(s["A"])
                s["layer"].lora_B.copy_(s["B"])


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    return {"norm": _run_norm, "rotary": _run_rotary, "w4": _run_w4}[s["case"]["kind"]](s)


def _grad_leaves(s):
    """The tensors that get gradients, as new leaves: (x, y, gate, p, b, the norm's scale)."""
    grads, gated = s["case"]["grads"], s["case"]["gated"]
    x, y = s["x"].detach(), s["y"].detach()
    mods = [s[n].detach() for n in ("gate", "p", "b")] if gated else [None] * 3
    leaves = []
    if grads != "none":
        leaves = [x.requires_grad_(), y.requires_grad_()]
    if grads == "all":
        leaves += [m.requires_grad_() for m in mods if m is not None]
        leaves.append(s["norm"].scale.requires_grad_())
    return x, y, mods, leaves


def _run_norm(s):
    x, y, mods, leaves = _grad_leaves(s)
    if own:
        k2 = s["k2"]
        r, h = k2.residual_rmsnorm(s["norm"], x, y, *mods)
        q, scale = k2.input_codes(h)
        codes = torch.mul(q, scale.unsqueeze(-1), out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))
    else:
        r, h = _plain_norm(x, y, *mods, s["norm"].scale)
        codes = _plain_codes(h.detach(), s["hadamard"])
    out = [r.detach(), h.detach(), codes]
    if leaves:
        out += torch.autograd.grad([r, h], leaves, [s["dr"], s["dh"]])
    return out


def _bf16(t):
    """To the nearest bf16 value, kept in 32 bits; its gradient passes as it is."""
    return t + (t.to(torch.bfloat16).float() - t).detach()


def _plain_norm(x, y, gate, p, b, scale):
    t = y.float() if gate is None else _bf16(gate.float() * y.float())
    r = _bf16(x.float() + t)
    h = _bf16(r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * (scale + 1.0))
    if p is not None:
        h = _bf16(_bf16(1.0 + p.float()) * h) + b.float()
    return r.to(torch.bfloat16), h.to(torch.bfloat16)


def _hadamard():
    h = torch.ones(1, 1, device=DEV)
    while h.shape[0] < 128:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h


def _rotate(t, hadamard):
    """Block-diagonal unnormalised Walsh-Hadamard transform of the rows of a (rows, K) tensor."""
    return (t.reshape(-1, 128) @ hadamard).reshape(t.shape)


def _quantize(v):
    """Per-row 8-bit codes, as whole numbers, and the rows' scales."""
    amax = v.abs().amax(-1, keepdim=True).clamp_min(1e-8)
    return torch.round(v * (127.0 / amax)), amax / 127.0


def _plain_codes(h, hadamard):
    q, scale = _quantize(_rotate(h.reshape(-1, h.shape[-1]).float(), hadamard))
    return (q * scale).to(torch.bfloat16)


def _run_rotary(s):
    case = s["case"]
    q, k = s["q"].detach(), s["k"].detach()
    if case["train"]:
        q.requires_grad_()
        k.requires_grad_()
    if own:
        out = s["rotary"](q, k, s["positions"], heads_first=case["heads_first"])
    else:
        pos = s["positions"] if case["axes"] else s["positions"].unsqueeze(-1)
        angle = pos[..., s["axis"]].double() * s["f"]
        angle = angle.unsqueeze(1 if case["heads_first"] else 2)
        cos, sin = (angle.cos() * s["m"]).float(), (angle.sin() * s["m"]).float()
        out = [_plain_rotate(t, cos, sin, case) for t in (q, k)]
    if not case["train"]:
        return list(out)
    return [t.detach() for t in out] + list(torch.autograd.grad(out, [q, k], [s["dq"], s["dk"]]))


def _plain_rotate(t, cos, sin, case):
    rd = case["rotary"]
    f = t[..., :rd].float()
    if case["layout"] == "half":
        a, b = f[..., :rd // 2], f[..., rd // 2:]
        f = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = f[..., 0::2], f[..., 1::2]
        f = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([f.to(t.dtype), t[..., rd:]], -1)


def _run_w4(s):
    x = s["x"].detach()
    if own:
        with torch.no_grad():
            return s["layer"](x)
    q, scale = _quantize(_rotate(x.float(), s["hadamard"]))
    y = (q @ _plain_weight(s["codes"], s["scales"].float()).t()) * (scale / 128.0)
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["A"] is not None:
        y = y + (x.float() @ s["A"].t()) @ s["B"].t()
    return y.to(torch.bfloat16)


def _plain_weight(codes, scales):
    """The (out, in) weight that packed codes stand for: byte j of 8 holds value j and, in its upper half, value j + 8."""
    n, half = codes.shape
    c = codes.view(n, half // 8, 1, 8)
    c = torch.cat([c & 15, c >> 4], 2).to(torch.int8)
    w = torch.where(c > 7, c - 16, c).to(scales.dtype).view(n, half // 32, 64)
    return (w * scales.t().unsqueeze(-1)).view(n, 2 * half)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "norm":
        rows, k = case["batch"] * case["tokens"], case["width"]
        size, mods = rows * k, case["batch"] * k * 2 if case["gated"] else 0
        nbytes = size * (4 + 5) + 4 * rows + 4 * k + 3 * mods
        flops = 30.0 * size
        if case["grads"] != "none":         # both gradients in, those of x and y out (one tensor without a gate)
            nbytes += size * (4 + (4 if case["gated"] else 2))
            flops += 20.0 * size
        if case["grads"] == "all":
            nbytes += 4 * k + 3 * mods
            flops += 10.0 * size
        return {"bytes": float(nbytes), "flops": flops}
    if case["kind"] == "rotary":
        tokens = case["batch"] * case["tokens"]
        size = tokens * (case["heads"] + case["kv"]) * case["dim"]
        passes = 2 if case["train"] else 1
        width = 4 if case["dtype"] == "f32" else 2
        turned = tokens * (case["heads"] + case["kv"]) * case["rotary"]
        return {"bytes": float(passes * 2 * width * size + 8 * tokens * len(_axes(case))), "flops": passes * 3.0 * turned}
    m, k, n, r = case["rows"], case["in"], case["out"], case["rank"]
    return {"bytes": float(n * k // 2 + n * k // 32 + 2 * m * (k + n) + 4 * r * (k + n) + (4 * n if case["bias"] else 0)),
            "flops": 2.0 * m * n * k + 2.0 * m * r * (n + k)}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ---------------------------------------------------------------------------------------------------------------
# The same from the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    return {"norm": _exact_norm, "rotary": _exact_rotary, "w4": _exact_w4}[case["kind"]](case, seed)


class _Stored(torch.autograd.Function):
    """A tensor of the formula that the model holds in bf16: the value rounded, the gradient as it is."""

    @staticmethod
    def forward(ctx, t):
        return t.to(torch.bfloat16).double()

    @staticmethod
    def backward(ctx, g):
        return g


def _exact_values(v):
    """What the 8-bit codes of the rows of v (rotated) stand for."""
    v = v.reshape(-1, v.shape[-1])
    blocks = v.view(v.shape[0], -1, 128)
    for stage in range(7):                       # butterflies of stride 2 ** stage
        w = blocks.reshape(*blocks.shape[:2], 128 >> stage + 1, 2, 1 << stage)
        blocks = torch.stack([w[..., 0, :] + w[..., 1, :], w[..., 0, :] - w[..., 1, :]], -2).reshape(blocks.shape)
    v = blocks.reshape(v.shape)
    step = v.abs().amax(-1, keepdim=True).clamp_min(1e-8) / 127
    return torch.round(v / step) * step


def _exact_norm(case, seed):
    t = {n: v.double() for n, v in _norm_inputs(case, seed).items()}
    grads, stored = case["grads"], _Stored.apply
    names = ["x", "y"] + (["gate", "p", "b"] if case["gated"] else [])
    leaves = [t[n] for n in (names + ["scale"] if grads == "all" else names[:2] if grads == "inputs" else [])]
    for v in leaves:
        v.requires_grad_()
    r = stored(t["x"] + (stored(t["gate"] * t["y"]) if case["gated"] else t["y"]))
    h = stored((1 + t["scale"]) * r / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + EPS))
    if case["gated"]:
        h = stored(stored(stored(1 + t["p"]) * h) + t["b"])
    out = [r.detach(), h.detach(), _exact_values(h.detach())]
    if leaves:
        out += torch.autograd.grad([r, h], leaves, [t["dr"], t["dh"]])
    return out


def _exact_rotary(case, seed):
    s = _rotary_inputs(case, seed)
    freqs, which, factor = [], [], case["factor"]
    for axis, d in enumerate(_axes(case)):
        for i in range(d // 2):
            theta = 10000.0 * (factor ** (d / (d - 2.0)) if case["scaling"] == "ntk" else 1.0)
            f = math.exp(-math.log(theta) * 2 * i / d)
            if case["scaling"] == "linear":
                f /= factor
            elif case["scaling"] == "yarn":
                # pairs that turn over 32 times within the original length stay, those below once are interpolated
                at = [d / 2 * math.log(case["original"] / (2 * math.pi * n)) / math.log(theta) for n in (32, 1)]
                lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
                keep = 1 - min(max((i - lo) / (hi - lo if hi > lo else 0.001), 0), 1)
                f = keep * f + (1 - keep) * f / factor
            freqs.append(f)
            which.append(axis)
    m = 1 + math.log(factor) / 10 if case["scaling"] == "yarn" else 1.0
    pos = s["positions"].double()
    pos = pos[..., torch.tensor(which, device=DEV)] if case["axes"] else pos[..., None]
    angle = pos * torch.from_numpy(np.array(freqs)).to(DEV)
    turn = torch.polar(torch.full_like(angle, m), angle).unsqueeze(1 if case["heads_first"] else 2)

    def rotate(t, by):
        t, rd = t.double(), case["rotary"]
        if case["layout"] == "half":
            z = torch.complex(t[..., :rd // 2], t[..., rd // 2:rd]) * by
            head = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(t[..., :rd].reshape(*t.shape[:-1], rd // 2, 2).contiguous()) * by
            head = torch.view_as_real(z).flatten(-2)
        return torch.cat([head, t[..., rd:]], -1)

    out = [rotate(s["q"], turn), rotate(s["k"], turn)]
    if case["train"]:
        out += [rotate(s["dq"], turn.conj()), rotate(s["dk"], turn.conj())]
    return out


def _exact_w4(case, seed):
    s = _w4_inputs(case, seed)
    n, k = case["out"], case["in"]
    byte = s["codes"].to(torch.int64).view(n, k // 16, 8)
    code = torch.cat([byte % 16, byte // 16], -1).view(n, k // 64, 64)
    del byte
    w = (code - 16 * (code >= 8)).double() * s["scales"].double().t()[..., None]
    del code
    y = _exact_values(s["x"].double()) @ w.view(n, k).t() / 128
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if s["A"] is not None:
        y = y + s["x"].double() @ s["A"].double().t() @ s["B"].double().t()
    return y
