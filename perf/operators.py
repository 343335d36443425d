"""Cases and plain forms of the gradient-norm operators: the global norm of many gradients,
clipping by it in place, and the AdamW-SR step that clips the gradients as it reads them.

A case describes the gradients of a decoder-shaped model (``layers``, ``width``, ``kv``,
``ff``, ``vocab``); ``pad`` is the alignment, in elements, of each tensor's slot in the packed
buffer that holds them (64: as a sharded step packs them; 1: back to back, so that tensors
after an odd-sized one start at odd addresses).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BETAS, EPS, LR, DECAY = (0.9, 0.95), 1e-8, 3e-4, 0.01


def _case(name, op, layers, width, kv, ff, vocab, dtype="bf16", pad=64, norm="2", max_norm=1.0, grad_scale=1.0):
    c = dict(op=op, layers=layers, width=width, kv=kv, ff=ff, vocab=vocab, dtype=dtype, pad=pad, norm=norm,
             max_norm=max_norm, grad_scale=grad_scale)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one block of a toy model with float32 gradients: launch latency is all there is
        _case("norm small fp32", "norm", 1, 64, 16, 171, 96, dtype="fp32"),
        # the unclipped odd-sized case: sizes that no vector width divides, slots back to back
        _case("norm odd inf fp16", "norm", 5, 1001, 143, 2731, 10007, dtype="fp16", pad=1, norm="inf"),
        # matrices in bfloat16 beside float32 vectors, the sum of magnitudes
        _case("norm mixed one", "norm", 8, 1536, 384, 4096, 32000, dtype="mixed", norm="1"),
        # every gradient of the benchmark's own training step (8.03 G elements, 16 GB)
        _case("norm 8B model", "norm", 32, 4096, 1024, 14336, 128256),
        # fine-tuning a few small tensors: latency again, with the write
        _case("clip small fp32", "clip", 1, 80, 20, 213, 100, dtype="fp32", max_norm=0.5, grad_scale=4.0),
        # a small model whose tensors start at odd addresses
        _case("clip odd bf16", "clip", 7, 1003, 251, 2677, 7919, pad=1, max_norm=1.0, grad_scale=4.0),
        # a model of about 1.8 G parameters: larger than any cache, clipping active
        _case("clip 1.8B bf16", "clip", 24, 2304, 576, 8192, 50257, max_norm=1.0, grad_scale=4.0),
        # late in training: the norm is below the bound and the gradients stay
        _case("clip idle fp16", "clip", 12, 1024, 256, 4096, 32000, dtype="fp16", max_norm=1e4),
        # vectors and one small table
        _case("step small", "step", 1, 72, 18, 191, 90, max_norm=0.5),
        # an embedding table with the norm vectors of a small model, odd sizes
        _case("step odd", "step", 3, 511, 73, 1365, 20011, pad=64, max_norm=1.0),
        # a model of 118 M parameters, averaging over 8 micro-batches as it clips
        _case("step ordinary", "step", 8, 896, 224, 2400, 32000, max_norm=1.0, grad_scale=0.125),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "norm", "clip", "clip", "step"])
    most = {"norm": 2.0e9, "clip": 1.2e9, "step": 8.0e7}[op]
    while True:
        width = log(33, 4096)
        c = dict(layers=log(1, 32), width=width, kv=max(1, width // rng.choice([1, 2, 4, 8])), ff=log(64, 14336),
                 vocab=log(50, 130000))
        if _numel(c) <= most:
            break
    dtype = "bf16" if op == "step" else rng.choice(["bf16", "bf16", "fp16", "fp32", "mixed"])
    scale = 1.0 if op == "norm" else 0.125 if op == "step" else rng.choice([1.0, 4.0])
    bound = 1e4 if op == "clip" and scale == 1.0 else rng.choice([0.5, 1.0, 2.0])
    norm = "2" if op == "step" else rng.choice(["2", "2", "1", "inf"])
    if op == "clip" and norm == "1":
        bound = 1e12 if scale == 1.0 else 50.0 * math.sqrt(_numel(c))
    if op == "clip" and norm == "inf" and scale != 1.0:
        bound = 1e-3
    return _case(None, op, **c, dtype=dtype, pad=rng.choice([1, 64]) if op != "step" else 64, norm=norm,
                 max_norm=bound, grad_scale=scale)


def _shapes(c):
    w, kv, ff = c["width"], c["kv"], c["ff"]
    block = [(w, w), (kv, w), (kv, w), (w, w), (ff, w), (ff, w), (w, ff), (w,), (w,)]
    return [(c["vocab"], w)] + block * c["layers"] + [(w,), (c["vocab"], w)]


def _numel(c):
    return sum(math.prod(s) for s in _shapes(c))


def _kinds(c):
    """The dtype name of each tensor."""
    if c["dtype"] == "mixed":
        return ["bf16" if len(s) > 1 else "fp32" for s in _shapes(c)]
    return [c["dtype"]] * len(_shapes(c))


def _packed(c, device, fill):
    """One buffer per dtype and a view of it for each tensor."""
    size, place = {}, []
    for shape, kind in zip(_shapes(c), _kinds(c)):
        at = size.get(kind, 0)
        place.append((kind, at, shape))
        size[kind] = at + -(-math.prod(shape) // c["pad"]) * c["pad"]
    flats = {kind: fill(n, DTYPES[kind]) for kind, n in size.items()}
    return flats, [flats[k][at:at + math.prod(s)].view(s) for k, at, s in place]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def noise(n, dtype):
        return torch.empty(n, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=gen)

    flats, grads = _packed(case, "cuda", noise)
    # each tensor has its own magnitude, and tokens that a batch lacks leave zero rows in the
    # gradient of the embedding table
    size = torch.empty(len(grads), device="cuda").uniform_(-3.5, -2.0, generator=gen)
    factors = (10.0 ** size).unbind()
    for g, f in zip(grads, factors):
        g.mul_(f.to(g.dtype))
    seen = torch.empty(grads[0].shape[0], 1, device="cuda").uniform_(0.0, 1.0, generator=gen) < 0.4
    grads[0].mul_(seen.to(grads[0].dtype))
    state = dict(case=case, flats=flats, grads=grads)
    if case["op"] == "norm":
        return state
    if case["op"] == "clip":
        params = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    else:
        # a resumed run: weights and both moments live in packed buffers
        weights, views = _packed(case, "cuda", lambda n, t: noise(n, t).mul_(0.02))
        first, ema = _packed(case, "cuda", lambda n, t: noise(n, t).mul_(1e-3))
        second, square = _packed(case, "cuda", lambda n, t: noise(n, t).square_().mul_(1e-6))
        params = [torch.nn.Parameter(v) for v in views]
        moments = [dict(step=100, ema=m, ema_squared=v) for m, v in zip(ema, square)]
        state.update(weights=weights["bf16"], first=first["bf16"], second=second["bf16"], moments=moments)
    for p, g in zip(params, grads):
        p.grad = g
    return dict(state, params=params)


def run(state):
    return {"norm": _norm, "clip": _clip, "step": _step}[state["case"]["op"]](state)


def _norm(state):
    order = float(state["case"]["norm"])
    if own:
        from muon_sr_b200 import get_total_norm
        total, each = get_total_norm(state["grads"], order, per_tensor=True)
        return {"total": total, "each": each}
    powers = _powers(state["grads"], order)
    each = powers.sqrt() if order == 2 else powers
    return {"total": _total(powers, order).float(), "each": each.float()}


def _powers(grads, order):
    """Sum of |g|^p of each tensor, or its largest |g| for infinity."""
    if order == 2:
        return torch.stack([g.float().square().sum() for g in grads]).double()
    if order == 1:
        return torch.stack([g.float().abs().sum() for g in grads]).double()
    return torch.stack([g.float().abs().max() for g in grads]).double()


def _total(powers, order):
    return powers.max() if order == math.inf else powers.sum().sqrt() if order == 2 else powers.sum()


def _factor(grads, order, c):
    """(norm of the scaled gradients, what every gradient is multiplied by)."""
    norm = _total(_powers(grads, order), order) * c["grad_scale"]
    coef = (c["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return norm.float(), (coef * c["grad_scale"]).float()


def _clip(state):
    c, order = state["case"], float(state["case"]["norm"])
    if own:
        from muon_sr_b200 import clip_grad_norm_
        norm = clip_grad_norm_(state["params"], c["max_norm"], order, grad_scale=c["grad_scale"])
        return {"norm": norm, "grads": state["flats"]}
    norm, factor = _factor(state["grads"], order, c)
    for g in state["grads"]:
        g.copy_(g.float() * factor)
    return {"norm": norm, "grads": state["flats"]}


def _step(state):
    c = state["case"]
    if own:
        opt = state.get("optimizer")
        if opt is None:  # the program's optimizer, resumed from the moments in hand
            from muon_sr_b200 import TritonAdamW
            opt = TritonAdamW(state["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)
            opt.state.update(zip(state["params"], state["moments"]))
            state["optimizer"] = opt
        opt.step(max_norm=c["max_norm"], grad_scale=c["grad_scale"])
        return _step_outputs(state, opt.grad_norm)
    norm, factor = _factor(state["grads"], 2.0, c)
    for i, (p, g, s) in enumerate(zip(state["params"], state["grads"], state["moments"])):
        _adamw(p.detach(), g, s, i, factor)
    return _step_outputs(state, norm)


def _step_outputs(state, norm):
    return {"norm": norm, "weights": state["weights"], "first": state["first"], "second": state["second"]}


def _adamw(p, g, s, index, factor):
    s["step"] += 1
    t = s["step"]
    seed = (t * 2654435761 ^ index * 1234567891) & 0xFFFFFFFF
    g = g.float() * factor
    m = s["ema"].float() * BETAS[0] + g * (1 - BETAS[0])
    v = s["ema_squared"].float() * BETAS[1] + g * (1 - BETAS[1]) * g
    denom = v.sqrt() / math.sqrt(1 - BETAS[1] ** t) + EPS
    w = p.float() * (1 - LR * DECAY)
    w = w - m * (LR / (1 - BETAS[0] ** t)) / denom
    for to, x, key in ((s["ema"], m, seed), (s["ema_squared"], v, seed + 1), (p, w, seed + 2)):
        to.copy_(_stochastic(x, key if seed >= 1 << 31 else _wrap(key)))


def _wrap(key):
    """A key that began below 2^31 counts in 32 bits with a sign."""
    return (key + (1 << 31)) % (1 << 32) - (1 << 31)


def _stochastic(x, key):
    """x rounded to bfloat16: the low 16 bits of word 0 of Philox4x32-10 (Salmon et al., 2011)
    at counter (element, 0, 0, 0) are added to x's bits, which are then cut."""
    k0, k1 = key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF
    mask = 0xFFFFFFFF
    c0 = torch.arange(x.numel(), dtype=torch.int64, device=x.device)
    c1 = c2 = c3 = torch.zeros((), dtype=torch.int64, device=x.device)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64: the bits of the full products
        c0, c1, c2, c3 = (b >> 32 & mask) ^ c1 ^ k0, b & mask, (a >> 32 & mask) ^ c3 ^ k1, a & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    bits = x.contiguous().view(torch.int32) + (c0 & 0xFFFF).to(torch.int32).view(x.shape)
    return (bits & -65536).view(torch.float32)


def work(case):
    n = sum(math.prod(s) * DTYPES[k].itemsize for s, k in zip(_shapes(case), _kinds(case)))
    count = _numel(case)
    if case["op"] == "norm":
        return {"bytes": n + 4 * len(_shapes(case)), "flops": 2 * count}
    if case["op"] == "clip":
        idle = case["max_norm"] >= 1e4 and case["grad_scale"] == 1.0
        return {"bytes": n if idle else 2 * n, "flops": 2 * count if idle else 3 * count}
    return {"bytes": 14 * count, "flops": 20 * count}


def exact(case, seed):
    """The definition in 64 bits; rounded outputs are given before their rounding."""
    state = prepare(case, seed)
    grads, p = state["grads"], float(case["norm"])
    if p == math.inf:
        each = torch.stack([g.abs().amax() for g in grads]).double()
        total = each.amax()
    else:
        power = torch.stack([torch.sum(g.double().abs().pow(p)) for g in grads])
        each, total = power.pow(1 / p), torch.sum(power).pow(1 / p)
    if case["op"] == "norm":
        return {"total": total, "each": each}
    norm = total * case["grad_scale"]
    factor = case["grad_scale"] * min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    if case["op"] == "clip":
        return {"norm": norm, "grads": {k: f.double() * factor if case["pad"] == 1 else _scaled(case, state, k, factor)
                                        for k, f in state["flats"].items()}}
    b1, b2 = BETAS
    t = 101
    outs = {"weights": state["weights"].double(), "first": state["first"].double(), "second": state["second"].double()}
    live = _live(case, state, "bf16")
    g = state["flats"]["bf16"].double() * factor
    m = b1 * outs["first"] + (1 - b1) * g
    v = b2 * outs["second"] + (1 - b2) * g ** 2
    w = outs["weights"] * (1 - LR * DECAY) - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + EPS)
    return {"norm": norm, "weights": torch.where(live, w, outs["weights"]),
            "first": torch.where(live, m, outs["first"]), "second": torch.where(live, v, outs["second"])}


def _live(case, state, kind):
    """Which elements of a packed buffer belong to a tensor (the rest is padding)."""
    flat = state["flats"][kind]
    live = torch.zeros(flat.numel(), dtype=torch.bool, device=flat.device)
    for g, k in zip(state["grads"], _kinds(case)):
        if k == kind:
            live[g.storage_offset():g.storage_offset() + g.numel()] = True
    return live


def _scaled(case, state, kind, factor):
    f = state["flats"][kind].double()
    return torch.where(_live(case, state, kind), f * factor, f)
