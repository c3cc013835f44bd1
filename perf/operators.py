"""Cases and plain forms of the training operators: layer norm (forward, forward + backward), the gradient norm with its
clipping, and the AdamW step over many tensors with states in 32 or in 8 bits.

``run(state)`` is one pass through an operator: in plain torch operations where ``own`` is false, through
``ayolov2_amd`` where it is true.  ``exact(case, seed)`` evaluates the definition in float64.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-5                                          # layer norm
LR, BETA1, BETA2, ADAM_EPS, DECAY, MAX_NORM = 1e-3, 0.9, 0.999, 1e-8, 0.05, 1.0
BLOCK = 128                                         # elements that share an exponent in an 8-bit state


def listed():
    return [
        # one token on its way through a pre-norm block: the residual sum and its norm, nothing to keep
        dict(name="norm one token", op="layer_norm", rows=1, c=1024, dtype="bf16", wdtype="bf16", train=False, residual=True, pad=0, map=0),
        # inference: the norm in front of a block on the stride-16 feature map of sixteen 640 x 640 images
        dict(name="norm feature map", op="layer_norm", rows=16 * 40 * 40, c=256, dtype="fp16", wdtype="fp32", train=False, residual=False, pad=0, map=40),
        # a training step's norm on the stride-8 map: activations in fp16, master weights in fp32, a channel slice of a concat buffer
        dict(name="norm train map slice", op="layer_norm", rows=16 * 80 * 80, c=128, dtype="fp16", wdtype="fp32", train=True, residual=False, pad=128, map=80),
        # an odd width in exact precision: tail lanes, rows that start at no 16-byte boundary
        dict(name="norm train odd", op="layer_norm", rows=3001, c=1023, dtype="fp32", wdtype="fp32", train=True, residual=False, pad=4, map=0),
        # a training step's residual sum and norm on a long batch of tokens
        dict(name="norm train tokens", op="layer_norm", rows=16384, c=4096, dtype="bf16", wdtype="bf16", train=True, residual=True, pad=0, map=0),
        # clipping the few tensors of a fine-tuned head
        dict(name="clip head", op="clip", params=230_000, tensors=6, dtype="fp32"),
        # clipping every gradient of a large detector
        dict(name="clip large", op="clip", params=46_500_000, tensors=366, dtype="fp32"),
        # an optimiser step of a fine-tuned head
        dict(name="adamw head", op="adamw", params=230_000, tensors=6, dtype="fp32", bits=32),
        # an optimiser step of a small detector: many tensors, few of them large
        dict(name="adamw small model", op="adamw", params=7_200_000, tensors=177, dtype="fp32", bits=32),
        # 16-bit parameters with 32-bit states
        dict(name="adamw bf16", op="adamw", params=46_500_000, tensors=366, dtype="bf16", bits=32),
        # 8-bit states of the smallest model
        dict(name="adamw 8-bit nano", op="adamw", params=1_870_000, tensors=177, dtype="fp32", bits=8),
        # 8-bit states of the largest model
        dict(name="adamw 8-bit large", op="adamw", params=86_700_000, tensors=480, dtype="fp32", bits=8),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "clip", "adamw", "adamw"])
    if op == "layer_norm":
        c = _spread(rng, 16, 8192)
        if rng.random() < 0.6:
            c = max(16, c // 16 * 16)
        rows = min(_spread(rng, 1, 200_000), 64_000_000 // c)
        dtype = rng.choice(list(DTYPES))
        side = rng.choice([0, 0, 7, 20])
        if side:
            rows = max(1, rows // (side * side)) * side * side
            while rows * c > 64_000_000:
                rows -= side * side
            if rows < 1:
                rows, side = 1, 0
        return dict(op=op, rows=rows, c=c, dtype=dtype, wdtype=rng.choice([dtype, "fp32"]), train=rng.random() < 0.6,
                    residual=rng.random() < 0.4, pad=rng.choice([0, 0, 1, 64]), map=side)
    params = _spread(rng, 20_000, 46_000_000 if op == "clip" else 80_000_000)
    case = dict(op=op, params=params, tensors=rng.randint(3, 360), dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
    if op == "adamw":
        case["bits"] = rng.choice([32, 8])
        if case["bits"] == 32:
            case["params"] = min(params, 46_000_000)
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs
def _sizes(case):
    """Element counts of a model's tensors: weights that grow with depth, each with two vectors (a gain, a bias) beside it."""
    layers, extra = max(1, case["tensors"] // 3), case["tensors"] % 3
    raw = [2.0 ** (6.0 * i / layers) for i in range(layers)]
    out = []
    for r in raw:
        n = max(1, int(case["params"] * r / sum(raw)))
        c = max(1, int(math.sqrt(n / 9)))
        out += [n, c, c]
    return out + [255] * extra


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _layer_norm_inputs(case, seed):
    g = _gen(seed)
    rows, c, side, dt = case["rows"], case["c"], case["map"], DTYPES[case["dtype"]]
    shape = (rows // (side * side), side, side) if side else (rows,)

    def act(scale, shift=0.0):
        t = torch.randn(*shape, c + case["pad"], generator=g, device="cuda")
        t = (t * scale + shift).to(dt)[..., :c]
        return t.movedim(-1, 1) if side else t           # maps: logical (B, C, H, W), channels innermost in memory

    def vec(scale, shift):
        return (torch.randn(c, generator=g, device="cuda") * scale + shift).to(DTYPES[case["wdtype"]])

    s = {"case": case, "x": act(1.5, 0.3), "w": vec(0.2, 1.0), "b": vec(0.2, 0.0)}
    if case["residual"]:
        s["r"] = act(1.0)
    if case["train"]:
        s["gy"] = act(1.0)
        if case["residual"]:
            s["gs"] = act(0.5)
        for k in ("x", "r", "w", "b"):
            if k in s:
                s[k].requires_grad_(True)
    return s


def _tensors(case, seed):
    """Flat arenas [blocks, BLOCK] in which every tensor starts at a block, and the tensors as views of them."""
    g = _gen(seed)
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    starts = [0]
    for n in blocks:
        starts.append(starts[-1] + n)
    nb = starts[-1]
    s = {"case": case, "sizes": torch.tensor(sizes, device="cuda"), "blocks": torch.tensor(blocks, device="cuda"),
         "starts": torch.tensor(starts[:-1], device="cuda")}
    place = [(a * BLOCK, n) for a, n in zip(starts, sizes)]
    col = torch.arange(BLOCK, device="cuda")
    row = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), s["blocks"], output_size=nb)
    inside = ((torch.arange(nb, device="cuda") - s["starts"][row]) * BLOCK)[:, None] + col < s["sizes"][row][:, None]

    def arena(dtype, scale):
        # gradients and weights of different layers differ in size
        size = torch.exp2(torch.rand(len(sizes), generator=g, device="cuda") * 6 - 6)
        t = torch.randn(nb, BLOCK, generator=g, device="cuda") * (scale * size[row])[:, None]
        return torch.where(inside, t, 0.0).to(dtype)

    def views(flat):
        flat = flat.view(-1)
        return [flat[a:a + n] for a, n in place]

    dt = DTYPES[case["dtype"]]
    s["g"] = arena(dt, 1e-2)
    s["grads"] = views(s["g"])
    if case["op"] == "clip":
        return s
    s["p"] = arena(dt, 0.1)
    s["params"] = views(s["p"])
    s["t"] = torch.full((len(sizes),), float(100 + seed % 100), device="cuda")
    s["steps"] = list(s["t"].unbind())
    s["decay"] = torch.tensor([DECAY if k % 3 == 0 else 0.0 for k in range(len(sizes))], device="cuda")
    s["decays"] = [DECAY if k % 3 == 0 else 0.0 for k in range(len(sizes))]
    if case["bits"] == 32:
        s["m"], s["v"] = arena(torch.float32, 3e-3), arena(torch.float32, 1e-2).square_()
        s["ms"], s["vs"] = views(s["m"]), views(s["v"])
        return s

    def ints(lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")

    def exps(flat):
        return [flat[a:a + n] for a, n in zip(starts, blocks)]

    s["seed"] = seed % 100_000
    sign = ints(0, 2, (nb, BLOCK)) << 7
    s["mc"] = torch.where(inside, sign | ints(40, 120, (nb, BLOCK)), 0).to(torch.uint8)
    s["vc"] = torch.where(inside, ints(120, 248, (nb, BLOCK)), 0).to(torch.uint8)
    s["me"] = ints(112, 120, (nb,)).to(torch.uint8)
    s["ve"] = ints(100, 108, (nb,)).to(torch.uint8)
    s["ms"], s["vs"] = list(zip(views(s["mc"]), exps(s["me"]))), list(zip(views(s["vc"]), exps(s["ve"])))
    s["m"], s["v"] = torch.zeros(nb, BLOCK, device="cuda"), torch.zeros(nb, BLOCK, device="cuda")
    s["m_values"], s["v_values"] = views(s["m"]), views(s["v"])
    return s


def prepare(case, seed):
    return _layer_norm_inputs(case, seed) if case["op"] == "layer_norm" else _tensors(case, seed)


# ------------------------------------------------------------------------------------------------------------ plain forms
def _plain_layer_norm(s):
    case = s["case"]
    dim = 1 if case["map"] else -1
    shape = [1, -1, 1, 1] if case["map"] else [-1]
    x = s["x"].detach()
    dt = x.dtype
    total = x
    if case["residual"]:
        total = (x.float() + s["r"].detach().float()).to(dt)
    t = total.float()
    d = t - t.mean(dim, keepdim=True)
    rstd = torch.rsqrt(d.square().mean(dim, keepdim=True) + EPS)
    xh = d * rstd
    w, b = s["w"].detach().float().view(shape), s["b"].detach().float().view(shape)
    out = {"y": (xh * w + b).to(dt)}
    if case["residual"]:
        out["s"] = total
    if case["train"]:
        gy = s["gy"].float()
        gw = gy * w
        ds = rstd * (gw - gw.mean(dim, keepdim=True) - xh * (gw * xh).mean(dim, keepdim=True))
        if case["residual"]:
            ds = ds + s["gs"].float()
        rest = [k for k in range(gy.dim()) if k != dim % gy.dim()]
        out["dx"] = ds.to(dt)
        out["dw"] = (gy * xh).sum(rest).to(s["w"].dtype)
        out["db"] = gy.sum(rest).to(s["b"].dtype)
        if case["residual"]:
            out["dr"] = out["dx"]
    return out


def _plain_clip(s):
    norm = s["g"].float().square().sum().sqrt()
    s["g"].copy_(s["g"].float() * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0))
    return {"norm": norm, "g": s["g"]}


M32 = 0xFFFFFFFF


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def _pow2(e):
    """2 ** e in float64, of whole numbers."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _unpack(codes, exps, bias, signed):
    bits = (codes.int() & (0x7F if signed else 0xFF)) << 20
    x = (bits.view(torch.float32).double() * _pow2(exps.long() - bias)[:, None]).float()
    return torch.where(codes > 127, -x, x) if signed else x


def _pack(x, noise, bias, least, signed):
    """Stochastic rounding to 8 bits under the exponent of the block's largest value."""
    e = ((x.abs().amax(1).view(torch.int32) >> 23) & 255).clamp(min=least)
    y = (x.abs().double() * _pow2(bias - e)[:, None]).float()
    codes = (y.view(torch.int32) + ((noise << 4) | 8).int()) >> 20
    codes = codes | ((x < 0).int() << 7) if signed else torch.where(x > 0, codes.clamp(min=1), codes)
    return codes.to(torch.uint8), e.to(torch.uint8)


def _plain_adamw(s):
    case = s["case"]
    nb = s["g"].shape[0]
    row = torch.repeat_interleave(torch.arange(s["t"].numel(), device="cuda"), s["blocks"], output_size=nb)
    s["t"].add_(1)
    t = s["t"].double()
    step = (LR / (1 - BETA1 ** t)).float()[row][:, None]
    root = (1 / (1 - BETA2 ** t).sqrt()).float()[row][:, None]
    g = s["g"].float()
    if case["bits"] == 32:
        m, v = s["m"], s["v"]
        m.mul_(BETA1).add_(g * (1 - BETA1))
        v.mul_(BETA2).add_(g * g * (1 - BETA2))
    else:
        m = _unpack(s["mc"], s["me"], 14, True) * BETA1 + g * (1 - BETA1)
        v = _unpack(s["vc"], s["ve"], 30, False) * BETA2 + g * g * (1 - BETA2)
    p = s["p"].float()
    s["p"].copy_(p - (p * (LR * s["decay"])[row][:, None] + step * (m / (v.sqrt() * root + ADAM_EPS))))
    if case["bits"] == 8:
        k = torch.arange(s["t"].numel(), device="cuda") + 1
        key = _mix((_mix((s["seed"] + 0x9E3779B1 * s["t"].long()) & M32) + 0x9E3779B1 * k) & M32)
        i = ((torch.arange(nb, device="cuda") - s["starts"][row]) * BLOCK)[:, None] + torch.arange(BLOCK, device="cuda")
        h = _mix(((i * 0x9E3779B1) & M32) ^ key[row][:, None])
        mc, me = _pack(m, h >> 16, 14, 1, True)
        vc, ve = _pack(v, h & 0xFFFF, 30, 10, False)
        for kept, new in (("mc", mc), ("me", me), ("vc", vc), ("ve", ve)):
            s[kept].copy_(new)
        m, v = _unpack(mc, me, 14, True), _unpack(vc, ve, 30, False)
    return {"p": s["p"], "m": m, "v": v, "t": s["t"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_layer_norm, "clip": _own_clip, "adamw": _own_adamw}[op](state)
    with torch.no_grad():
        return {"layer_norm": _plain_layer_norm, "clip": _plain_clip, "adamw": _plain_adamw}[op](state)


# ------------------------------------------------------------------------------------------------------ the framework's own
def _own_layer_norm(s):
    from ayolov2_amd.functional import layer_norm
    case = s["case"]
    dim = 1 if case["map"] else -1
    if not case["train"]:
        with torch.no_grad():
            out = layer_norm(s["x"], s["w"], s["b"], EPS, residual=s.get("r"), dim=dim)
        return {"y": out[0], "s": out[1]} if case["residual"] else {"y": out}
    if not case["residual"]:
        y = layer_norm(s["x"], s["w"], s["b"], EPS, dim=dim)
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["gy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    y, t = layer_norm(s["x"], s["w"], s["b"], EPS, residual=s["r"], dim=dim)
    dx, dr, dw, db = torch.autograd.grad((y, t), (s["x"], s["r"], s["w"], s["b"]), (s["gy"], s["gs"]))
    return {"y": y, "s": t, "dx": dx, "dr": dr, "dw": dw, "db": db}


def _own_clip(s):
    from ayolov2_amd.optim import clip_grads_
    return {"norm": clip_grads_(s["grads"], MAX_NORM), "g": s["g"]}


def _own_adamw(s):
    from ayolov2_amd.optim import adamw_step, unpack_moments
    hyper = dict(lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=s["decays"])
    if s["case"]["bits"] == 32:
        adamw_step(s["params"], s["grads"], s["ms"], s["vs"], s["steps"], **hyper)
    else:
        adamw_step(s["params"], s["grads"], s["ms"], s["vs"], s["steps"], seed=s["seed"], **hyper)
        unpack_moments(s["ms"], signed=True, out=s["m_values"])
        unpack_moments(s["vs"], signed=False, out=s["v_values"])
    return {"p": s["p"], "m": s["m"], "v": s["v"], "t": s["t"]}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_layer_norm(case, s):
    d64 = {k: s[k].detach().double() for k in ("x", "r", "w", "b", "gy", "gs") if k in s}
    if case["map"]:
        for k in ("x", "r", "gy", "gs"):
            if k in d64:
                d64[k] = d64[k].permute(0, 2, 3, 1)
    t = d64["x"]
    out = {}
    if case["residual"]:
        out["s"] = t + d64["r"]
        t = out["s"].to(s["x"].dtype).double()           # the sum as it is kept: what is normed
    var, mu = torch.var_mean(t, -1, unbiased=False, keepdim=True)
    sd = (var + EPS).sqrt()
    xh = (t - mu) / sd
    out["y"] = xh * d64["w"] + d64["b"]
    if case["train"]:
        n = case["c"]
        a = d64["gy"] * d64["w"]
        ds = (a - a.sum(-1, keepdim=True) / n - xh * ((a * xh).sum(-1, keepdim=True) / n)) / sd
        if case["residual"]:
            ds = ds + d64["gs"]
            out["dr"] = ds
        out["dx"] = ds
        out["dw"] = (d64["gy"] * xh).flatten(0, -2).sum(0)
        out["db"] = d64["gy"].flatten(0, -2).sum(0)
    if case["map"]:
        out = {k: v.permute(0, 3, 1, 2) if v.dim() == 4 else v for k, v in out.items()}
    return out


def _exact_clip(case, s):
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    return {"norm": norm, "g": g * min(1.0, MAX_NORM / (float(norm) + 1e-6))}


def _exact_adamw(case, s):
    rows = torch.repeat_interleave(s["blocks"])
    t = (s["t"].double() + 1)[rows].unsqueeze(1)
    g, p = s["g"].double(), s["p"].double()
    if case["bits"] == 32:
        m0, v0 = s["m"].double(), s["v"].double()
    else:
        mc, vc = s["mc"].long(), s["vc"].long()
        me, ve = s["me"].long().unsqueeze(1), s["ve"].long().unsqueeze(1)
        e, f = (mc >> 3) & 15, mc & 7
        m0 = torch.where(e > 0, 8 + f, f).double() * torch.exp2((me - 144 + e.clamp(min=1)).double()) * (1 - 2 * (mc >> 7))
        e, f = vc >> 3, vc & 7
        v0 = torch.where(e > 0, 8 + f, f).double() * torch.exp2((ve - 160 + e.clamp(min=1)).double())
    m = BETA1 * m0 + (1 - BETA1) * g
    v = BETA2 * v0 + (1 - BETA2) * g ** 2
    mhat, vhat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    decay = s["decay"].double()[rows].unsqueeze(1)
    p = p * (1 - LR * decay) - LR * mhat / (vhat.sqrt() + ADAM_EPS)
    # a state rounded to 8 bits by random numbers has no value of its own in 64 bits
    return {"p": p, "m": m if case["bits"] == 32 else None, "v": v if case["bits"] == 32 else None, "t": s["t"].double() + 1}


def exact(case, seed):
    s = prepare(case, seed)
    return {"layer_norm": _exact_layer_norm, "clip": _exact_clip, "adamw": _exact_adamw}[case["op"]](case, s)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "layer_norm":
        n, b = case["rows"] * case["c"], BYTES[case["dtype"]]
        streams = (4 if case["residual"] else 2)                        # x (r) in, y (s) out
        flops = 8
        if case["train"]:
            streams += 3 if case["residual"] else 2                     # gy (gs) in, dx out; x is read once in all
            flops += 14
        return {"bytes": n * b * streams + 2 * case["c"] * BYTES[case["wdtype"]] * (2 if case["train"] else 1), "flops": flops * n}
    n, b = sum(_sizes(case)), BYTES[case["dtype"]]
    if case["op"] == "clip":
        return {"bytes": 2 * b * n, "flops": 3 * n}
    if case["bits"] == 32:
        return {"bytes": (3 * b + 16) * n, "flops": 16 * n}
    # 8-bit states read and written, and the values that they stand for written out
    return {"bytes": (3 * b + 4 + 8) * n + 4 * (n // BLOCK), "flops": 20 * n}
