"""Operators of adapters that share one base: the low-rank adapters of many requests added beside a projection, in
serving and in training, and the step behind it over many tensors at once: AdamW with moments in 32 bits or in 8, and the
scaling of gradients to a largest norm.

Every case is one call as a program makes it.  ``run`` computes it in plain torch operations, or, where ``own`` is true,
through the package.  Parameters, gradients and moments of an optimizer lie one behind another in flat buffers, each
tensor at a multiple of 256 elements.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 256                      # elements that share a scale, where moments are held in 8 bits
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 1e-4, 0.9, 0.999, 1e-8, 0.01, 1.0
STEPS = 100                      # steps that the optimizer has behind it
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# (in, out) of the linears that adapters go beside in a block of width 6144, and the tensors of a whole block
SITES = ((6144, 6144), (6144, 1536), (6144, 1536), (6144, 6144), (6144, 6144), (6144, 16384), (6144, 16384), (16384, 6144))


# ---------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------
def _adapters(name, batch, tokens, k, n, count, rank, dtype, ragged=False, mixed=False, train=False):
    c = {"kind": "adapters", "batch": batch, "tokens": tokens, "in": k, "out": n, "count": count, "rank": rank,
         "dtype": dtype, "ragged": ragged, "mixed": mixed, "train": train}
    return {"name": name, **c} if name else c


def _adamw(name, tensors, rank, bits, dtype="f32", clip=True, odd=False):
    c = {"kind": "adamw", "tensors": tensors, "rank": rank, "bits": bits, "dtype": dtype, "clip": clip, "odd": odd}
    return {"name": name, **c} if name else c


def _clip(name, tensors, rank, dtype="f32", odd=False):
    c = {"kind": "clip", "tensors": tensors, "rank": rank, "dtype": dtype, "odd": odd}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one request, one new token, through the key projection
        _adapters("adapters_token", 1, 1, 6144, 1536, 4, 16, "bf16"),
        # 64 requests, one new token each, adapters of several ranks, some requests without one
        _adapters("adapters_requests", 64, 1, 6144, 16384, 32, 64, "bf16", mixed=True),
        # prompts of uneven lengths in one batch, through the text MLP
        _adapters("adapters_prompts", 7, 1000, 2560, 6144, 8, 16, "f32", ragged=True),
        # four pictures at 1024 x 1024 (4096 image + 512 text tokens), a style of its own for each
        _adapters("adapters_images", 4, 4608, 6144, 6144, 6, 32, "bf16"),
        # several adapters trained at once at 256 x 256 (256 image + 512 text tokens) through the MLP's up-projection
        _adapters("adapters_train", 4, 768, 6144, 16384, 4, 64, "f32", train=True),
        # samples of uneven lengths in one batch of 16384 image + 512 text tokens, through the MLP's down-projection
        _adapters("adapters_train_long", 5, 16896, 16384, 6144, 3, 16, "f32", ragged=True, train=True),
        # the two factors of one adapter: a step's latency
        _adamw("adamw_layer", 2, 16, 32),
        # every factor of rank 64 beside the linears of 28 blocks, moments in 32 bits
        _adamw("adamw_lora", 448, 64, 32),
        # the same with moments in 8 bits
        _adamw("adamw_lora8", 448, 64, 8),
        # one block's own weights in bf16 with random rounding, moments in 8 bits
        _adamw("adamw_block8", 8, 0, 8, "bf16", clip=False),
        # the gradients of one adapter scaled to a largest norm
        _clip("clip_layer", 2, 16),
        # those of every factor of rank 64
        _clip("clip_lora", 448, 64),
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, min(hi, step * round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    """One more call of the same ranges: one token to the longest batch, widths from a small block's to the widest linear's,
    one adapter or many, one tensor or a whole model's, odd sizes among them."""
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("adapters", "adamw", "clip")}
    while True:
        kind = rng.choice(("adapters", "adapters", "adapters", "adamw", "adamw", "clip"))
        if kind == "adapters":
            ragged = rng.random() < 0.4
            batch = _log_int(rng, 1, 64)
            tokens = _log_int(rng, batch, 16896) if ragged else rng.choice((1, _log_int(rng, 1, 4608)))
            c = _adapters(None, batch, tokens, _log_int(rng, 256, 16384, 64), _log_int(rng, 256, 16384, 64),
                          _log_int(rng, 1, 32), rng.choice((16, 16, 32, 48, 64, 128)), rng.choice(("bf16", "f32")), ragged,
                          rng.random() < 0.3, rng.random() < 0.4)
        else:
            tensors, rank, odd = _log_int(rng, 1, 448), rng.choice((4, 8, 16, 32, 64)), rng.random() < 0.4
            if kind == "adamw":
                c = _adamw(None, tensors, rank, rng.choice((32, 8)), rng.choice(("f32", "f32", "bf16")), rng.random() < 0.6,
                           odd)
            else:
                c = _clip(None, tensors, rank, rng.choice(("f32", "f32", "bf16")), odd)
        if _cost(c) <= most[c["kind"]]:
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


def _ranks(case):
    """Every adapter's rank: the bank's, or that and half and a quarter of it in turn, in steps of 16."""
    r = case["rank"]
    return [max(16, (r >> i % 3) // 16 * 16) if case["mixed"] else r for i in range(case["count"])]


def _adapter_inputs(case, seed):
    """Requests one behind another: all of ``tokens`` rows, or, ragged, ``tokens`` rows cut at random places.  The last of
    several requests has no adapter."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    b, t, k, n, count, r = (case[v] for v in ("batch", "tokens", "in", "out", "count", "rank"))
    lead = (t,) if case["ragged"] else (b, t)
    ids = torch.randint(0, count, (b,), device=DEV, generator=g)
    if b > 2:
        ids[-1] = -1
    if case["ragged"]:
        cuts = torch.randint(0, t, (b - 1,), device=DEV, generator=g).sort().values
        ids = ids[torch.searchsorted(cuts, torch.arange(t, device=DEV), right=True)]
    rank = torch.tensor(_ranks(case), device=DEV)
    live = (torch.arange(r, device=DEV) < rank[:, None]).float()
    dt = DTYPES[case["dtype"]]
    s = {"y": _normal(g, *lead, n), "x": _stream(g, *lead, k), "ids": ids,
         "A": _normal(g, count, r, k, std=1.0 / math.sqrt(k), dtype=torch.float32).mul_(live[:, :, None]).to(dt),
         "B": _normal(g, count, n, r, std=0.05, dtype=torch.float32).mul_(live[:, None, :]).to(dt),
         "scales": torch.rand(count, device=DEV, generator=g) + 0.5}
    if case["train"]:
        s["dy"] = _normal(g, *lead, n, std=1e-3)
    return s


def _shapes(case):
    """The tensors' shapes: an adapter's two factors beside each of a block's linears in turn, or the linears' own weights.
    Odd: a few elements more in a tensor's width."""
    out = []
    for i in range(case["tensors"]):
        k, n = SITES[i // 2 % len(SITES)] if case["rank"] else SITES[i % len(SITES)]
        more = i % 5 if case["odd"] else 0
        r = case["rank"]
        out.append((n, k) if not r else (r, k + more) if i % 2 == 0 else (n + more, r))
    return out


def _starts(case):
    """Where each tensor starts in a flat buffer, and the buffer's elements."""
    at, starts = 0, []
    for a, b in _shapes(case):
        starts.append(at)
        at += -(-a * b // BLOCK) * BLOCK
    return starts, at


def _inside(case):
    """True where an element of the flat buffers belongs to a tensor."""
    starts, total = _starts(case)
    inside = torch.ones(total, dtype=torch.bool, device=DEV)
    if case["odd"]:
        for start, (a, b), end in zip(starts, _shapes(case), starts[1:] + [total]):
            inside[start + a * b:end] = False
    return inside


def _flat_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    total, dt = _starts(case)[1], DTYPES[case["dtype"]]
    live = _inside(case) if case["odd"] else 1

    def flat(std, dtype=torch.float32):
        return torch.empty(total, device=DEV).normal_(0.0, std, generator=g).mul_(live).to(dtype)

    s = {"g": flat(1e-3, dt)}
    if case["kind"] == "adamw":
        s["p"] = flat(0.02, dt)
        s["m"], s["v"] = flat(3e-4), flat(1e-3).square_()
        if case["bits"] == 8:
            s["m"], s["m_scale"] = _codes8(s["m"], None, _M_STEPS)
            s["v"], s["v_scale"] = _codes8(s["v"].sqrt(), None, _V_STEPS)
        s["step"], s["seed"] = STEPS, int(seed) & 0xFFFFFFFF
    return s


def _cut(case, flat):
    return [flat[start:start + a * b].view(a, b) for start, (a, b) in zip(_starts(case)[0], _shapes(case))]


def prepare(case, seed):
    if case["kind"] == "adapters":
        s = _adapter_inputs(case, seed)
        s["ranks"] = torch.tensor(_ranks(case), dtype=torch.int32, device=DEV)
    else:
        s = _flat_inputs(case, seed)
    s["case"] = case
    if own:
        _keep(s)
    return s


def _keep(s):
    """What a program that uses the package holds: parameters with their gradients, and an optimizer that has run."""
    import __graft_entry__
    k2 = s["k2"] = __graft_entry__.load_package()
    case = s["case"]
    if case["kind"] == "adapters":
        return
    grads = _cut(case, s["g"])
    s["params"] = [torch.nn.Parameter(p) for p in _cut(case, s["p"] if case["kind"] == "adamw" else torch.zeros_like(s["g"]))]
    for p, g in zip(s["params"], grads):
        p.grad = g
    if case["kind"] == "clip":
        return
    opt = s["opt"] = k2.AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                              max_norm=MAX_NORM if case["clip"] else None, state_bits=case["bits"],
                              stochastic=case["dtype"] == "bf16", seed=s["seed"])
    names = {"exp_avg": "m", "exp_avg_sq": "v"}
    if case["bits"] == 8:
        names.update(exp_avg_scale="m_scale", exp_avg_sq_scale="v_scale")
    state = {i: {"step": torch.tensor(float(s["step"]))} for i in range(len(s["params"]))}
    for name, key in names.items():
        if key.endswith("scale"):
            ends = [-(-a * b // BLOCK) for a, b in _shapes(case)]
            parts = s[key].split(ends)
        else:
            parts = _cut(case, s[key])
        for i, part in enumerate(parts):
            state[i][name] = part.view(torch.float8_e4m3fn) if name == "exp_avg" and case["bits"] == 8 else part
    opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
    for key in ("m", "v", "m_scale", "v_scale"):
        s.pop(key, None)


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    return {"adapters": _run_adapters, "adamw": _run_adamw, "clip": _run_clip}[s["case"]["kind"]](s)


def _run_adapters(s):
    train = s["case"]["train"]
    x, A, B = (s[n].detach().requires_grad_(train) for n in ("x", "A", "B"))
    if own:
        out = s["k2"].add_adapters(s["y"], x, A, B, s["ids"], s["scales"], s["ranks"])
    else:
        out = _plain_adapters(s["y"], x, A, B, s["ids"], s["scales"])
    if not train:
        return out
    return [out.detach(), *torch.autograd.grad(out, [x, A, B], s["dy"])]


def _plain_adapters(y, x, A, B, ids, scales):
    """All adapters' factors as one product each, rows masked to the adapter that they have."""
    count, r, k = A.shape
    ids = ids.view(*ids.shape, *[1] * (x.dim() - 1 - ids.dim()), 1)
    weight = (ids == torch.arange(count, device=ids.device)).float() * scales
    u = (x.float() @ A.float().view(count * r, k).t()).unflatten(-1, (count, r)) * weight.unsqueeze(-1)
    return (y.float() + u.flatten(-2) @ B.float().transpose(1, 2).reshape(count * r, -1)).to(y.dtype)


def _run_clip(s):
    if own:
        norm = s["k2"].clip_grad_norm_(s["params"], MAX_NORM)
    else:
        norm, by = _plain_norm(s["g"])
        s["g"].copy_((s["g"].float() * by).to(s["g"].dtype))
    return [s["g"], norm]


def _plain_norm(g):
    """The norm and the factor that brings it to the largest one."""
    norm = g.double().square().sum().sqrt()
    return norm.float(), (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()


def _run_adamw(s):
    case = s["case"]
    if own:
        s["opt"].step()
        m, v = s["opt"].moments(dtype=torch.bfloat16 if case["bits"] == 8 else torch.float32)
        return [s["p"], m, v] + ([s["opt"].grad_norm] if case["clip"] else [])
    g, out = s["g"].float(), []
    if case["clip"]:
        norm, by = _plain_norm(s["g"])
        g, out = g * by, [norm]
    s["step"] += 1
    m, v = s["m"], s["v"]
    if case["bits"] == 8:
        m = _values8(m, s["m_scale"], _M_STEPS)
        v = _values8(v, s["v_scale"], _V_STEPS).square()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    root = v.sqrt()
    update = m / (root * (1 / math.sqrt(1 - BETA2 ** s["step"])) + EPS)
    p = s["p"].float() * (1 - LR * DECAY) - update * (LR / (1 - BETA1 ** s["step"]))
    if case["bits"] == 8 or case["dtype"] == "bf16":
        dither = _dither(p.numel(), s["seed"], s["step"])
    if case["dtype"] == "bf16":     # a 16-bit random number below the kept bits, then the rest cut off
        p = ((p.view(torch.int32) + (_mix(dither ^ 0x9E3779B9) & 0xFFFF).int()) & -65536).view(torch.float32)
    s["p"].copy_(p.to(s["p"].dtype))
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
        return [s["p"], m, v] + out
    s["m"], s["m_scale"] = _codes8(m, (dither & 0xFFFF) << 4, _M_STEPS)
    s["v"], s["v_scale"] = _codes8(root, (dither >> 16) << 3, _V_STEPS)
    return [s["p"], _values8(s["m"], s["m_scale"], _M_STEPS).to(torch.bfloat16),
            _values8(s["v"], s["v_scale"], _V_STEPS).square().to(torch.bfloat16)] + out


# Numbers in 8 bits: (kept bits of the fraction, exponent of the smallest full-precision value, largest value, sign).  Below
# that value they are evenly spaced, down to zero.
_M_STEPS = (3, -6, 448.0, True)
_V_STEPS = (4, 0, 31744.0, False)


def _codes8(t, dither, steps):
    """Codes and scales of blocks of values.  ``dither`` (integers below the step of one code) is added under the kept bits
    before the rest is cut off; without it half a step is.  No value above zero has the unsigned code 0."""
    keep, low, top, signed = steps
    t = t.view(-1, BLOCK)
    most = t.abs().amax(1, keepdim=True)
    a = (t.abs() * torch.where(most < 2.0 ** -100, 0.0, top / most)).clamp(max=top).view(-1)
    small = a < 2.0 ** low
    bits = (a + 2.0 ** low * small).view(torch.int32).long()
    cut = 23 - keep
    code = (bits + (dither if dither is not None else (1 << cut - 1) - 1 + (bits >> cut & 1)) >> cut)
    code = code - ((127 + low - 1 << keep) + (small.long() << keep))
    if dither is None:
        code = code.clamp(max=126 if signed else 255)
    code = code + (t.view(-1).signbit().long() << 7) if signed else code.maximum((a > 0).long())
    return code.to(torch.uint8), (torch.where(most < 2.0 ** -100, 0.0, most) / top).view(-1)


def _table8(steps):
    keep, low, top, signed = steps
    c = torch.arange(256 >> signed, device=DEV)
    e = (c >> keep).clamp(min=1) - 1
    v = ((c & (1 << keep) - 1) + ((c >> keep) > 0).long() * (1 << keep)).float() * torch.exp2((e + low - keep).float())
    return torch.cat([v, -v]) if signed else v


def _values8(codes, scale, steps):
    return (_table8(steps)[codes.int()].view(-1, BLOCK) * scale.view(-1, 1)).view(-1)


def _mix(h):
    """A 32-bit mixer: shifts and products modulo 2^32."""
    h = ((h ^ h >> 16) * 0x7FEB352D) & 0xFFFFFFFF
    h = ((h ^ h >> 15) * 0x846CA68B) & 0xFFFFFFFF
    return h ^ h >> 16


def _dither(n, seed, step):
    """32 random bits for every element: of the seed, the step and the element's place."""
    key = _mix(_mix(seed & 0xFFFFFFFF) ^ step)
    return _mix(torch.arange(n, device=DEV) ^ key)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "adapters":
        k, n, b = case["in"], case["out"], case["batch"]
        rows = case["tokens"] * (1 if case["ragged"] else b)
        used = sorted(_ranks(case), reverse=True)[:max(1, min(case["count"], b - (b > 2)))]
        width = 4 if case["dtype"] == "f32" else 2
        r = sum(used) / len(used)
        nbytes = rows * 2 * (k + 2 * n) + width * sum(used) * (k + n)
        flops = 2.0 * rows * r * (k + n)
        if case["train"]:       # the gradient in, x's and the factors' out
            nbytes += rows * 2 * (k + n) + width * case["count"] * case["rank"] * (k + n)
            flops *= 3
        return {"bytes": float(nbytes), "flops": flops}
    size = sum(a * b for a, b in _shapes(case))
    width = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "clip":
        return {"bytes": float(2 * width * size), "flops": 3.0 * size}
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": float(size * (3 * width + state)), "flops": 20.0 * size}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ---------------------------------------------------------------------------------------------------------------
# The same from the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    return {"adapters": _exact_adapters, "adamw": _exact_adamw, "clip": _exact_clip}[case["kind"]](case, seed)


def _exact_adapters(case, seed):
    s = _adapter_inputs(case, seed)
    rows = s["x"].shape[:-1].numel()
    ids = s["ids"].repeat_interleave(rows // s["ids"].numel())
    x, out = s["x"].view(rows, -1), s["y"].view(rows, -1).double()
    dy = s["dy"].view(rows, -1) if case["train"] else None
    dx, dA, dB = (torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (x, s["A"], s["B"]))
    for a in range(case["count"]):
        at = (ids == a).nonzero()[:, 0]
        A, B, c = s["A"][a].double(), s["B"][a].double(), s["scales"][a].double()
        xa = x[at].double()
        u = c * (xa @ A.t())
        out[at] += u @ B.t()
        if dy is not None:
            da = dy[at].double()
            g = c * (da @ B)
            dx[at], dA[a], dB[a] = g @ A, g.t() @ xa, da.t() @ u
    out = out.view(s["y"].shape)
    return out if dy is None else [out, dx.view(s["x"].shape), dA, dB]


def _exact_norm(g):
    norm = torch.linalg.vector_norm(g.double())
    return norm, min(1.0, MAX_NORM / (float(norm) + 1e-6))


def _exact_clip(case, seed):
    g = _flat_inputs(case, seed)["g"]
    norm, by = _exact_norm(g)
    return [g.double() * by, norm]


def _exact_round(a, places, low, random):
    """Values above zero to the number of so many binary places of the fraction below them, or, with the chance that
    ``random`` (0 to 1) gives, above them."""
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -140))).clamp(min=low) - places)
    return torch.floor(a / step + random) * step


def _exact_adamw(case, seed):
    s = _flat_inputs(case, seed)
    t, out = s["step"] + 1, []
    g = s["g"].double()
    if case["clip"]:
        norm, by = _exact_norm(s["g"])
        g, out = g.mul_(by), [norm]
    m, v = s["m"], s["v"]
    if case["bits"] == 8:
        m = m.view(torch.float8_e4m3fn).double() * s["m_scale"].double().repeat_interleave(BLOCK)
        c = s["v"].double()
        e = torch.floor(c / 16).clamp(min=1)
        v = ((c - 16 * (e - 1)) * torch.exp2(e - 5) * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
        del c, e
    m = m.double() * BETA1 + (1 - BETA1) * g
    v = v.double() * BETA2 + (1 - BETA2) * g ** 2
    del g
    p = s["p"].double() * (1 - LR * DECAY) - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    if case["bits"] == 32 and case["dtype"] == "f32":
        return [p, m, v] + out
    h = _dither(p.numel(), s["seed"], t)
    if case["dtype"] == "bf16":
        p = torch.sign(p) * _exact_round(p.abs(), 7, -126, (_mix(h ^ 0x9E3779B9) & 0xFFFF).double() / 65536)
    if case["bits"] == 32:
        return [p, m, v] + out

    def held(a, places, low, top, random):
        unit = a.view(-1, BLOCK).amax(1).div_(top).repeat_interleave(BLOCK)
        return _exact_round(a / unit.clamp(min=2.0 ** -140), places, low, random) * unit

    m = torch.sign(m) * held(m.abs(), 3, -6, 448.0, (h & 0xFFFF).double() / 65536)
    unit = torch.sqrt(v).view(-1, BLOCK).amax(1).div_(31744.0).repeat_interleave(BLOCK)
    v = torch.where(v > 0, held(torch.sqrt(v), 4, 0, 31744.0, (h >> 16).double() / 65536).maximum(unit / 16), 0.0) ** 2
    return [p, m, v] + out
