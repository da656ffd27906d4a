"""
What is measured of the operators that train the scattering head: AdamW over many tensors with 32-bit or 8-bit states,
routing of nodes to experts, and the experts' products.  `own = False` computes them in plain torch operations, `own =
True` calls esc_gnn_amd.  Sizes are the head's own (242 features, 256 hidden, 4096 graphs x 128 nodes, 32 graphs x 512
nodes) and generic larger ones.
"""
import math
import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 256                                   # elements that share a scale of an 8-bit state
TOP = {True: 15.0 * 2 ** 14, False: 14.0 * 2 ** 30}      # largest value of a code: signed (first moment), unsigned (second)


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the scattering head as DPTrainer holds it: eight small tensors, gradients clipped; launches are what counts
        {"name": "adamw32 head", "op": "adamw", "bits": 32, "type": "fp32", "layers": 0, "width": 256, "experts": 0, "clip": True},
        # a head with three middle layers of 16 experts, 1024 wide, fp32: 101 M parameters, bandwidth
        {"name": "adamw32 experts fp32", "op": "adamw", "bits": 32, "type": "fp32", "layers": 3, "width": 1024, "experts": 16, "clip": True},
        # bf16 parameters and gradients of odd sizes, no clipping
        {"name": "adamw32 odd bf16", "op": "adamw", "bits": 32, "type": "bf16", "layers": 9, "width": 999, "experts": 0, "clip": False},
        # the head with states in 8 bits
        {"name": "adamw8 head", "op": "adamw", "bits": 8, "type": "fp32", "layers": 0, "width": 256, "experts": 0, "clip": True},
        # the experts' head with states in 8 bits
        {"name": "adamw8 experts fp32", "op": "adamw", "bits": 8, "type": "fp32", "layers": 2, "width": 1024, "experts": 16, "clip": False},
        # one small graph answered: a few rows, scores with balance bias and groups
        {"name": "route few", "op": "route", "type": "fp32", "rows": 7, "experts": 64, "k": 4, "score": "sigmoid", "bias": True,
         "groups": 8, "keep": 3, "train": False},
        # every node of a 4096 x 128 batch to two of eight experts, forward and backward
        {"name": "route nodes", "op": "route", "type": "fp32", "rows": 524288, "experts": 8, "k": 2, "score": "softmax", "bias": False,
         "groups": 1, "keep": 1, "train": True},
        # many experts, bf16 logits, bias and groups, an odd number of rows, forward and backward
        {"name": "route groups", "op": "route", "type": "bf16", "rows": 65537, "experts": 256, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "keep": 4, "train": True},
        # one row through wide experts: the weights' bytes are all there is
        {"name": "experts one row bf16", "op": "experts", "type": "bf16", "rows": 1, "d": 1024, "h": 2048, "o": 1024, "experts": 64, "k": 4,
         "bias": True, "train": False},
        # the nodes of a 4096 x 128 batch through eight experts of the head's width, forward and backward
        {"name": "experts nodes bf16", "op": "experts", "type": "bf16", "rows": 524288, "d": 256, "h": 256, "o": 256, "experts": 8, "k": 2,
         "bias": True, "train": True},
        # a 32 x 512 batch straight from the 242 features (odd rows in memory), fp32, forward and backward
        {"name": "experts features fp32", "op": "experts", "type": "fp32", "rows": 16384, "d": 242, "h": 256, "o": 256, "experts": 8, "k": 2,
         "bias": True, "train": True},
        # many wide experts, 256 rows each on average, forward and backward
        {"name": "experts wide bf16", "op": "experts", "type": "bf16", "rows": 8192, "d": 1024, "h": 2048, "o": 1024, "experts": 64, "k": 2,
         "bias": False, "train": True},
    ]


def _between(rng, lo, hi):
    """a whole number in [lo, hi], spread over its logarithm; odd ones among them"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["adamw", "adamw", "route", "route", "experts", "experts"])
    kind = rng.choice(["fp32", "bf16", "fp16"])
    if op == "adamw":
        experts = rng.choice([0, 0, _between(rng, 2, 16)])
        return {"op": op, "bits": rng.choice([32, 8]), "type": kind, "layers": rng.randint(0, 2 if experts else 9),
                "width": _between(rng, 17, 1024), "experts": experts, "clip": rng.random() < 0.6}
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _between(rng, 2, 256 // groups)
        k = rng.randint(1, min(8, experts))
        keep = rng.randint(-(-k * groups // experts), groups)
        return {"op": op, "type": kind, "rows": _between(rng, 1, 524288 * 8 // max(experts, 8)), "experts": experts, "k": k,
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "keep": keep,
                "train": rng.random() < 0.6}
    experts = _between(rng, 2, 64)
    k = rng.randint(1, min(4, experts))
    d, h, o = (rng.choice([lambda: _between(rng, 17, 1024), lambda: 8 * _between(rng, 3, 128)])() for _ in range(3))
    most = max(1, min(262144, int(1.0e11 / (k * (d * h + h * o)))))      # at most about what the listed ones multiply
    return {"op": op, "type": kind, "rows": _between(rng, 1, most if kind != "fp32" else max(1, most // 4)), "d": d, "h": h, "o": o,
            "experts": experts, "k": k, "bias": rng.random() < 0.6, "train": rng.random() < 0.6}


# ------------------------------------------------------------------------------------------------ inputs
def _shapes(case):
    """the tensors of a scattering head: norm, input layer, middle layers (plain or experts), readout"""
    f, w, e = 242, case["width"], case["experts"]
    out = [(f,), (f,), (w, f), (w,)]
    if e:
        for _ in range(case["layers"]):
            out += [(e, w), (e, w, w), (e, w), (e, w, w), (e, w)]
    else:
        for _ in range(case["layers"] + 1):
            out += [(w, w), (w,)]
    return out + [(1, w), (1,)]


def _views(flat, shapes):
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += n
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)                                    # noqa: E731
    t = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "adamw":
        shapes = _shapes(case)
        sizes = [math.prod(x) for x in shapes]
        n = sum(sizes)
        # gradients differ in size from tensor to tensor and from element to element, some are exactly zero (unused features)
        scale = torch.repeat_interleave(torch.exp(1.5 * rnd(len(sizes))) * 1e-3, torch.tensor(sizes, device=DEV), output_size=n)
        wide = torch.exp(rnd(n))
        s["grad"] = (rnd(n) * scale * wide * (torch.rand(n, generator=g, device=DEV) > 0.02)).to(t)
        s["param"] = (rnd(n) * 0.05).to(t)
        m = 0.3 * rnd(n) * scale * wide
        v = (scale * wide).square() * torch.exp(0.3 * rnd(n))
        del wide, scale
        s["step"] = torch.full((1,), 100 + int(seed) % 50, dtype=torch.int32, device=DEV)
        s["params"], s["grads"] = _views(s["param"], shapes), _views(s["grad"], shapes)
        s["options"] = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01,
                        "max_grad_norm": 1.0 if case["clip"] else None, "seed": int(seed) % 1000}
        if case["bits"] == 32:
            s["m"], s["v"] = m, v
            s["ms"], s["vs"] = _views(m, shapes), _views(v, shapes)
        else:
            half = torch.full((1,), 1 << 15, dtype=torch.int64, device=DEV)
            s["ms"] = [_encode(x.reshape(-1), half, True) for x in _views(m, shapes)]
            s["vs"] = [_encode(x.reshape(-1), half, False) for x in _views(v, shapes)]
        return s
    if case["op"] == "route":
        rows, e = case["rows"], case["experts"]
        # popular and unpopular experts; a hundredth of the (row, expert) pairs is masked, and some rows have one expert left or none
        x = 1.5 * rnd(rows, e) + 0.7 * rnd(e)
        x = torch.where(torch.rand(rows, e, generator=g, device=DEV) < 0.01, -math.inf, x)
        u = torch.rand(rows, 1, generator=g, device=DEV)
        at = torch.arange(e, device=DEV)
        x = torch.where((u < 0.002) | ((u < 0.004) & (at != e // 2)), -math.inf, x)
        s["logits"] = x.to(t)
        s["bias"] = 0.05 * rnd(e) if case["bias"] else None
        s["up"] = rnd(rows, case["k"])
        return s
    rows, d, h, o, e, k = (case[q] for q in ("rows", "d", "h", "o", "experts", "k"))
    s["x"] = rnd(rows, d).to(t)
    s["w1"] = (rnd(e, h, d) / math.sqrt(d)).to(t)
    s["w2"] = (rnd(e, o, h) / math.sqrt(h)).to(t)
    s["b1"] = (0.1 * rnd(e, h)).to(t) if case["bias"] else None
    s["b2"] = (0.1 * rnd(e, o)).to(t) if case["bias"] else None
    at = torch.argsort(rnd(rows, e) + 0.5 * rnd(e), dim=1, descending=True)[:, :k] if rows * e <= 1 << 23 else \
        (rnd(rows, e) + 0.5 * rnd(e)).topk(k, dim=1).indices
    p = torch.rand(rows, k, generator=g, device=DEV) + 0.1
    s["weights"] = p / p.sum(1, keepdim=True)
    drop = torch.rand(rows, k, generator=g, device=DEV) < (0.002 if rows > 100 else 0.0)      # routed nowhere: expert -1, weight 0
    s["experts"] = torch.where(drop, -1, at).to(torch.int32).contiguous()
    s["weights"] = torch.where(drop, 0.0, s["weights"]).contiguous()
    s["up"] = rnd(rows, o).to(t)
    return s


# ------------------------------------------------------------------------------------------------ 8-bit states
def _hash(seed, t, blocks):
    """32 random bits for each element of tensors that have so many whole blocks, a function of (seed, step, ordinal of the tensor,
    element of the tensor) alone"""
    mask = 0xFFFFFFFF

    def mix(x):
        x = ((x ^ (x >> 16)) * 0x6C8E9CF5) & mask
        x = ((x ^ (x >> 13)) * 0x5851F42D) & mask
        return x ^ (x >> 16)

    key = mix((t.to(torch.int64) + (seed * 0x2545F491) % (mask + 1)) & mask)
    total, of = sum(blocks), torch.tensor([[i, f] for i, f in zip(range(len(blocks)), _starts(blocks))], device=DEV)
    of = torch.repeat_interleave(of, torch.tensor(blocks, device=DEV), dim=0, output_size=total)
    key = mix((key + of[:, 0] * 0x632BE5AB) & mask)[:, None]
    i = (torch.arange(total, device=DEV) - of[:, 1])[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)
    return mix(mix(((i >> 32) + key) & mask) ^ (i & mask)).view(-1)


def _starts(sizes):
    return [sum(sizes[:i]) for i in range(len(sizes))]


def _encode(x, r16, signed):
    """codes and scales of a flat fp32 state: blocks of 256, scale = largest magnitude / TOP, minifloats with 3 mantissa bits, rounded
    up where the dropped part exceeds 1 - r16 / 2^16"""
    n = x.numel()
    nb = -(-n // BLOCK)
    pad = torch.nn.functional.pad(x, (0, nb * BLOCK - n)).view(nb, BLOCK)
    size = torch.where(torch.isfinite(pad), pad.abs(), 0.0).amax(1)
    size = torch.where(size > 0, size.clamp(min=2.0 ** -90), size)
    inv = torch.where(size > 0, TOP[signed] / size, 0.0)
    y = (pad.abs() * inv[:, None]).clamp(max=TOP[signed]).view(-1)[:n]
    bits = ((y.view(torch.int32).to(torch.int64) + (r16 << 4)) >> 20) - (129 << 3)
    low = torch.floor(y + r16.to(torch.float32) * 2.0 ** -16).to(torch.int64)
    code = torch.where(y >= 8.0, bits, low)
    if signed:
        code = code.clamp(max=127)
        code = torch.where((x < 0) & (code > 0), code + 128, code)
        code = torch.where(torch.isfinite(x), code, 128)
    else:
        code = torch.where(x > 0, code.clamp(min=1, max=254), code)
        code = torch.where(torch.isfinite(x), code, 255)
    return code.to(torch.uint8), size * (1.0 / TOP[signed])


def _decode(code, scale, signed):
    c = code.to(torch.int32)
    a = (c & 127) if signed else c
    y = torch.where(a >= 8, ((a + (129 << 3)) << 20).view(torch.float32), a.to(torch.float32))
    if signed:
        y = torch.where(c == 128, math.nan, torch.where(c > 128, -y, y))
    else:
        y = torch.where(c == 255, math.nan, y)
    n = y.numel()
    return y * torch.repeat_interleave(scale, BLOCK, output_size=scale.numel() * BLOCK)[:n]


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_update(p, g, m, v, o, clip, bc1, bc2):
    """one tensor's (or a flat buffer's) update in fp32; returns the new p, m, v"""
    b1, b2 = o["betas"]
    g = g.float() * clip
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    x = p.float() * (1.0 - o["lr"] * o["weight_decay"])
    return x - (m * (o["lr"] / bc1).float()) / (torch.sqrt(v) * (1.0 / torch.sqrt(bc2)).float() + o["eps"]), m, v


def _plain_adamw(s):
    o = s["options"]
    s["step"] += 1
    t = s["step"].double()
    bc1, bc2 = (1.0 - torch.pow(torch.tensor(b, dtype=torch.float64, device=DEV), t) for b in o["betas"])
    norm, clip = None, 1.0
    if o["max_grad_norm"] is not None:
        norm = torch.sqrt(s["grad"].double().square().sum())
        clip = (o["max_grad_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    if s["case"]["bits"] == 32:
        p, m, v = _plain_update(s["param"], s["grad"], s["m"], s["v"], o, clip, bc1, bc2)
        s["param"].copy_(p)
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": s["param"], "m": s["m"], "v": s["v"], "step": s["step"], "norm": None if norm is None else norm.float()}

    # all tensors at once, each padded to whole blocks
    sizes = [x.numel() for x in s["params"]]
    blocks = [-(-n // BLOCK) for n in sizes]
    whole = lambda xs: torch.cat([torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % BLOCK)) for x in xs])      # noqa: E731
    m, v = (_decode(whole([c for c, _ in st]), torch.cat([z for _, z in st]), signed) for st, signed in ((s["ms"], True), (s["vs"], False)))
    p, m, v = _plain_update(whole(s["params"]), whole(s["grads"]), m, v, o, clip, bc1, bc2)
    r = _hash(o["seed"], s["step"], blocks)
    parts = [n * BLOCK for n in blocks]
    [x.view(-1).copy_(y[:n]) for x, y, n in zip(s["params"], p.split(parts), sizes)]
    out = {"p": s["param"], "step": s["step"], "norm": None if norm is None else norm.float()}
    out["m"] = _plain_store(s["ms"], m, r & 0xFFFF, True, blocks, sizes)
    out["v"] = _plain_store(s["vs"], v, r >> 16, False, blocks, sizes)
    return out


def _plain_store(states, x, r16, signed, blocks, sizes):
    """new codes and scales into the states' own buffers, and the values that they stand for"""
    code, scale = _encode(x, r16, signed)
    parts = [n * BLOCK for n in blocks]
    [c.copy_(y[:n]) for (c, _), y, n in zip(states, code.split(parts), sizes)]
    [z.copy_(y) for (_, z), y in zip(states, scale.split(blocks))]
    return [y[:n] for y, n in zip(_decode(code, scale, signed).split(parts), sizes)]


def _plain_route(s, logits):
    case = s["case"]
    rows, e = logits.shape
    k, groups = case["k"], case["groups"]
    x = logits.float()
    x64 = logits.detach().double()
    key = x64
    if case["bias"] or groups > 1:                  # values next to each other decide: in 64 bits
        key = torch.softmax(x64, 1) if case["score"] == "softmax" else torch.sigmoid(x64)
        key = torch.where(x64 == -math.inf, -math.inf, key + (s["bias"].double() if case["bias"] else 0.0))
        key = torch.where(torch.isnan(key), torch.where((x64 == -math.inf).all(1, keepdim=True), -math.inf, math.inf), key)
    if groups > 1:
        per = key.view(rows, groups, e // groups)
        best = per.sort(dim=2, descending=True).values[:, :, :2]
        total = torch.where(best == -math.inf, 0.0, best).sum(2)
        total = torch.where(best[:, :, 0] == -math.inf, -math.inf, total)
        place = total.sort(dim=1, descending=True, stable=True).indices[:, :case["keep"]]
        kept = torch.zeros(rows, groups, dtype=torch.bool, device=DEV).scatter_(1, place, True)
        key = torch.where(kept[:, :, None], per, -math.inf).view(rows, e)
    top = key.sort(dim=1, descending=True, stable=True)
    at, there = top.indices[:, :k], top.values[:, :k] > -math.inf
    if case["score"] == "softmax":
        chosen = torch.where(there, x.gather(1, at), -math.inf)
        m = torch.where(there[:, :1], chosen.detach().amax(1, keepdim=True), 0.0)
        w = torch.where(there, torch.exp(torch.where(there, chosen, 0.0) - m), 0.0)
    else:
        w = torch.where(there, torch.sigmoid(torch.where(there, x.gather(1, at), 0.0)), 0.0)
    w = w / (w.sum(1, keepdim=True) + 1e-20)
    return w, torch.where(there, at, -1).to(torch.int32)


def _plain_experts(s, x, weights, w1, b1, w2, b2):
    """rows sorted by expert into a padded batch of the experts in use, two batched products in fp32"""
    rows, k = s["experts"].shape
    flat = s["experts"].reshape(-1).long()
    pairs = torch.nonzero(flat >= 0).view(-1)
    used, inv = torch.unique(flat[pairs], return_inverse=True)
    order = torch.argsort(inv, stable=True)
    pairs, inv = pairs[order], inv[order]
    count = torch.bincount(inv, minlength=used.numel())
    first = torch.cumsum(count, 0) - count
    place = inv * int(count.max()) + torch.arange(pairs.numel(), device=DEV) - first[inv]
    cap = int(count.max())
    xs = torch.zeros(used.numel() * cap, x.shape[1], device=DEV).index_copy(0, place, x.float().index_select(0, pairs // k))
    u = torch.bmm(xs.view(used.numel(), cap, -1), w1.index_select(0, used).float().transpose(1, 2))
    if b1 is not None:
        u = u + b1.index_select(0, used).float()[:, None]
    y = torch.bmm(u * torch.sigmoid(u), w2.index_select(0, used).float().transpose(1, 2))
    if b2 is not None:
        y = y + b2.index_select(0, used).float()[:, None]
    y = y.reshape(used.numel() * cap, -1).index_select(0, place)
    y = y * weights.reshape(-1, 1).index_select(0, pairs)
    return torch.zeros(rows, y.shape[1], device=DEV).index_add(0, pairs // k, y).to(x.dtype)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        import esc_gnn_amd as E
    if case["op"] == "adamw":
        if not own:
            return _plain_adamw(s)
        norm = E.adamw_step(s["params"], s["grads"], s["ms"], s["vs"], s["step"], **s["options"])
        if case["bits"] == 32:
            return {"p": s["param"], "m": s["m"], "v": s["v"], "step": s["step"], "norm": norm}
        return {"p": s["param"], "m": [E.dequantize_state(c, z, True) for c, z in s["ms"]],
                "v": [E.dequantize_state(c, z, False) for c, z in s["vs"]], "step": s["step"], "norm": norm}
    if case["op"] == "route":
        x = s["logits"].detach().requires_grad_(case["train"])
        if own:
            w, at = E.route_experts(x, case["k"], score=case["score"], bias=s["bias"], groups=case["groups"], keep_groups=case["keep"])
        else:
            w, at = _plain_route(s, x)
        if not case["train"]:
            return {"weights": w, "experts": at}
        return {"weights": w.detach(), "experts": at, "dlogits": torch.autograd.grad(w, x, s["up"])[0]}
    names = [q for q in ("x", "weights", "w1", "b1", "w2", "b2") if s[q] is not None]
    a = {q: None if s[q] is None else s[q].detach().requires_grad_(case["train"]) for q in ("x", "weights", "w1", "b1", "w2", "b2")}
    if own:
        y = E.expert_mlp(a["x"], a["weights"], s["experts"], a["w1"], a["b1"], a["w2"], a["b2"])
    else:
        y = _plain_experts(s, a["x"], a["weights"], a["w1"], a["b1"], a["w2"], a["b2"])
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [a[q] for q in names], s["up"])
    return {"y": y.detach(), **{"d" + q: d for q, d in zip(names, grads)}}


def work(case):
    b = BYTES[case["type"]]
    if case["op"] == "adamw":
        n = sum(math.prod(x) for x in _shapes(case))
        # p twice, g once, the states read and written; 8-bit states come back as fp32 values too
        return {"bytes": n * (3 * b + (16 if case["bits"] == 32 else 4 + 8)), "flops": 14 * n}
    rows, e, k = case["rows"], case["experts"], case["k"]
    if case["op"] == "route":
        return {"bytes": rows * (e * b + 8 * k + ((e * b + 4 * k) if case["train"] else 0)), "flops": rows * e * (8 if case["train"] else 5)}
    d, h, o = case["d"], case["h"], case["o"]
    hit = e * (1.0 - (1.0 - 1.0 / e) ** (rows * k))                       # experts that a row is expected to reach
    weights = hit * (d * h + h * o + ((h + o) if case["bias"] else 0)) * b
    once = rows * (d + o) * b + rows * k * 8
    grads = e * (d * h + h * o + ((h + o) if case["bias"] else 0)) * b
    return {"bytes": int(once + weights + ((once + grads) if case["train"] else 0)),
            "flops": 2 * rows * k * (d * h + h * o) * (3 if case["train"] else 1)}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["op"] == "route":
        return _exact_route(s)
    return _exact_experts(s)


def _exact_adamw(s):
    o, t = s["options"], int(s["step"]) + 1
    b1, b2 = o["betas"]
    g = s["grad"].double()
    norm = float(torch.linalg.vector_norm(g))
    if o["max_grad_norm"] is not None and norm + 1e-6 > o["max_grad_norm"]:
        g = g * (o["max_grad_norm"] / (norm + 1e-6))
    if s["case"]["bits"] == 32:
        m0, v0 = s["m"].double(), s["v"].double()
    else:
        # the value of a code, from its fields; the new 8-bit states are roundings by drawn bits: no value of their own in 64 bits
        a = torch.arange(256, dtype=torch.float64, device=DEV)
        mag = torch.where(a < 8, a, (8 + a % 8) * torch.pow(2.0, torch.div(a, 8, rounding_mode="floor") - 1))
        sgn = torch.cat([mag[:128], -mag[:128]])
        wide = lambda z, n: z.double().repeat_interleave(BLOCK)[:n]                                 # noqa: E731
        m0 = torch.cat([sgn[c.long()] * wide(z, c.numel()) for c, z in s["ms"]])
        v0 = torch.cat([mag[c.long()] * wide(z, c.numel()) for c, z in s["vs"]])
    m = torch.lerp(g, m0, b1)
    v = torch.lerp(g * g, v0, b2)
    p = s["param"].double()
    p = p - o["lr"] * o["weight_decay"] * p - o["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + o["eps"])
    many = [None] * len(s["params"])
    kept = s["case"]["bits"] == 32
    return {"p": p, "m": m if kept else many, "v": v if kept else many, "step": t, "norm": None if o["max_grad_norm"] is None else norm}


def _exact_route(s):
    case = s["case"]
    x = s["logits"].double()
    _, at = _plain_route(s, s["logits"])            # which experts: whole numbers, compared as such
    at = at.long()
    there = (at >= 0).double()
    l = x.gather(1, at.clamp(min=0))
    l = torch.where(at >= 0, l, 0.0)
    if case["score"] == "softmax":
        top = torch.where(at >= 0, l, -math.inf).amax(1, keepdim=True)
        q = torch.where(at >= 0, torch.exp(torch.where(at >= 0, l - top, 0.0)), 0.0)
        slope = q
    else:
        q = there / (1 + torch.exp(-l))
        slope = q * (1 - q) * there
    z = q.sum(1, keepdim=True) + 1e-20
    out = {"weights": q / z, "experts": None}
    if case["train"]:
        up = s["up"].double()
        d = slope * (up - (up * q).sum(1, keepdim=True) / z) / z
        out["dlogits"] = torch.zeros_like(x).scatter_add_(1, at.clamp(min=0), d * there)
    return out


def _exact_experts(s):
    case = s["case"]
    x, p, w1, w2, up = (s[q].double() for q in ("x", "weights", "w1", "w2", "up"))
    b1, b2 = (None if s[q] is None else s[q].double() for q in ("b1", "b2"))
    y = torch.zeros(x.shape[0], case["o"], dtype=torch.float64, device=DEV)
    d = {"x": torch.zeros_like(x), "weights": torch.zeros_like(p), "w1": torch.zeros_like(w1), "w2": torch.zeros_like(w2),
         "b1": None if b1 is None else torch.zeros_like(b1), "b2": None if b2 is None else torch.zeros_like(b2)}
    for e in range(case["experts"]):
        row, slot = torch.nonzero(s["experts"] == e, as_tuple=True)
        if not row.numel():
            continue
        u = x[row] @ w1[e].t() + (0.0 if b1 is None else b1[e])
        q = 1 / (1 + torch.exp(-u))
        a = u * q
        z = a @ w2[e].t() + (0.0 if b2 is None else b2[e])
        c = p[row, slot][:, None]
        y.index_put_((row,), c * z, accumulate=True)
        if not case["train"]:
            continue
        r = up[row]
        d["weights"][row, slot] = (z * r).sum(1)
        d["w2"][e] = (c * r).t() @ a
        du = ((c * r) @ w2[e]) * (q * (1 + u * (1 - q)))
        d["w1"][e] = du.t() @ x[row]
        d["x"].index_put_((row,), du @ w1[e], accumulate=True)
        if b1 is not None:
            d["b1"][e], d["b2"][e] = du.sum(0), (c * r).sum(0)
    if not case["train"]:
        return {"y": y}
    return {"y": y, **{"d" + q: v for q, v in d.items() if v is not None}}
