"""Operators of an encoder's residual path and of the step that trains it, as they are measured.

  rotary    rotary positions of queries and keys: half and interleaved layouts, part of a head, frequencies scaled for
            contexts longer than the trained ones, key heads fewer than query heads; forward, and with its gradient
  sandwich  norm of a block's output, gate, residual scale, sum and the next block's norm in one operator; forward,
            and with all gradients
  adamw     one AdamW step over all tensors of a model, moments in 8 or in 32 bits

`own` false: the plain forms in elementary torch operations. `own` true: the calls of this package.

The 8-bit moments. 256 consecutive elements of a tensor are a block; a tensor starts a block. With E the exponent field of
(pattern of the block's largest magnitude + 2^20 - 1), a value is kept as the upper 12 bits of its fp32 pattern, less an offset:
    second moment   code = ((pattern + r) >> 20) - 8 max(E - 31, 0)       8 bits, 0 is zero, else at least 1
    first moment    code = ((pattern of |m| + r) >> 20) - 8 max(E - 15, 0)   7 bits below the sign
r is a random number of 20 bits, so that the kept value is the true one on average. A first moment below the smallest code becomes
that code with the probability that keeps its mean, else zero. r comes from a number given with each step and the element's place.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = torch.device("cuda:0")
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256


# ------------------------------------------------------------------------------------------ cases
def _rotary(name, tokens, q_heads, k_heads, width, rotated, dtype, interleaved, scaling, first, train):
    c = {"kind": "rotary", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "width": width, "rotated": rotated,
         "dtype": dtype, "interleaved": interleaved, "scaling": scaling, "first": first, "train": train}
    return dict(c, name=name) if name else c


def _sandwich(name, tokens, channels, dtype, gate, scaled, rms, train):
    c = {"kind": "sandwich", "tokens": tokens, "channels": channels, "dtype": dtype, "gate": gate, "scaled": scaled,
         "rms": rms, "train": train}
    return dict(c, name=name) if name else c


def _adamw(name, hidden, inter, layers, bits, params, grads, odd=0, shift=0):
    c = {"kind": "adamw", "hidden": hidden, "inter": inter, "layers": layers, "bits": bits, "params": params,
         "grads": grads, "odd": odd, "shift": shift}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one protein through the default student (8 heads of 64), q and k inside the packed projection: all latency
        _rotary("rotary_one", 236, 8, 8, 64, 64, "bf16", False, "none", 0, False),
        # training on the full micro-batch with a context extended fourfold
        _rotary("rotary_batch", 55424, 12, 12, 64, 64, "bf16", False, "yarn", 0, True),
        # a long concatenation of proteins, far positions, a quarter of a wide head, four queries to a key, neighbouring pairs
        _rotary("rotary_far", 32768, 16, 4, 128, 32, "fp16", True, "ntk", 900000, True),
        # ragged sizes in full precision: widths that fill no vector
        _rotary("rotary_odd", 4301, 5, 3, 70, 34, "fp32", False, "linear", 17, True),
        # the same protein: embedding call, gate per channel
        _sandwich("sandwich_one", 236, 512, "bf16", "channel", True, False, False),
        # the default encoder's full micro-batch with a learned gate for every token and channel
        _sandwich("sandwich_batch", 55424, 1024, "bf16", "sigmoid", True, False, True),
        # a 768-wide encoder on a smaller batch, RMSNorm, gate per channel
        _sandwich("sandwich_768", 17024, 768, "bf16", "channel", True, True, True),
        # full precision, a width that fills no vector, neither gate nor scale
        _sandwich("sandwich_odd", 4301, 1111, "fp32", "none", False, False, True),
        # the small encoder of a first experiment: where the launch counts
        _adamw("adamw_small_8", 256, 512, 3, 8, "fp32", "fp32"),
        # a 768-wide, 16-layer encoder: master weights, fp32 gradients, bf16 copy; both state widths
        _adamw("adamw_encoder_8", 768, 2048, 16, 8, "fp32", "fp32"),
        _adamw("adamw_encoder_32", 768, 2048, 16, 32, "fp32", "fp32"),
        # weights and gradients in bf16 without master weights, tensors of odd sizes at odd addresses
        _adamw("adamw_bf16_odd", 512, 1024, 12, 8, "bf16", "bf16", odd=7, shift=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "sandwich", "adamw"])
    if kind == "rotary":
        width = rng.choice([64, 64, 128, 80, 96, 32, rng.randint(9, 130)])
        rotated = width - width % 2 if rng.random() < 0.5 else 2 * rng.randint(1, width // 2)
        k_heads = rng.choice([1, 2, 3, 4, 5, 8, 12])
        q_heads = k_heads * rng.choice([1, 1, 2, 4])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 55424 * 24 * 64 // ((q_heads + k_heads) * width) // (2 if dtype == "fp32" else 1)
        return _rotary(None, _log_int(rng, 1, min(most, 200000)), q_heads, k_heads, width, rotated, dtype, rng.random() < 0.5,
                       rng.choice(["none", "linear", "ntk", "yarn"]), _log_int(rng, 1, 2000000), rng.random() < 0.6)
    if kind == "sandwich":
        channels = rng.choice([256, 512, 640, 768, 1024, 1280, 2048, 4096, _log_int(rng, 3, 4096), _log_int(rng, 3, 4096)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = int(55424 * 1024 / channels) // (2 if dtype == "fp32" else 1)
        return _sandwich(None, _log_int(rng, 1, min(most, 200000)), channels, dtype,
                         rng.choice(["none", "channel", "token", "sigmoid"]), rng.random() < 0.6, rng.random() < 0.5,
                         rng.random() < 0.7)
    hidden, inter, layers = rng.choice([(128, 256, 2), (256, 512, 3), (384, 768, 8), (512, 1024, 6), (640, 1280, 10),
                                        (768, 2048, 12), (rng.randint(20, 700), rng.randint(20, 1400), rng.randint(1, 9))])
    odd = rng.choice([0, 0, rng.randint(1, 9)])
    return _adamw(None, hidden, inter, layers, rng.choice([8, 8, 32]), rng.choice(["fp32", "fp32", "bf16"]),
                  rng.choice(["fp32", "bf16"]), odd, rng.choice([0, 0, 0, rng.randint(1, 5)]) if odd else 0)


# ---------------------------------------------------------------------------------------- prepare
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7fffffff)
    return g


def _frequencies(rotated, scaling):
    """(radians a position of each pair, fp64; factor on cos and sin) for contexts scaled by 4 from 1 024 trained positions."""
    i = torch.arange(0, rotated, 2, dtype=torch.float64, device=DEV) / rotated
    theta, s, factor = 10000.0, 4.0, 1.0
    if scaling == "ntk" and rotated > 2:
        theta *= s ** (rotated / (rotated - 2))
    w = theta ** -i
    if scaling == "linear":
        w = w / s
    if scaling == "yarn":       # pairs that turn more than 32 times in the trained context stay, those under once are slowed
        turns = 1024 * w / (2 * math.pi)
        at = ((torch.log(turns) - math.log(1.0)) / math.log(32.0)).clamp(0, 1)
        w = w / s * (1 - at) + w * at
        factor = 0.1 * math.log(s) + 1.0
    return w, factor


def _model_shapes(case):
    """[(shape, whether weight decay acts on it)] of an encoder's tensors; odd: sizes off by a little, as flat tensors."""
    h, i, odd = case["hidden"], case["inter"], case["odd"]
    shapes = [((32, h), True), ((32,), False), ((h,), False), ((h, h), True)]
    for _ in range(case["layers"]):
        shapes += [((3 * h, h), True), ((h, h), True), ((2 * i, h), True), ((h, i), True), ((h,), False), ((h,), False)]
    if odd:
        shapes = [((math.prod(x) + odd * (j % 5) + 1,), d) for j, (x, d) in enumerate(shapes)]
        shapes += [((k,), False) for k in (1, 3, 255, 256, 257)]
    return shapes


def _prepare_rotary(case, g):
    t, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["width"]
    dt = TYPES[case["dtype"]]
    packed = torch.randn(t, (hq + 2 * hk) * d, generator=g, device=DEV).to(dt)
    q, k = packed[:, :hq * d].view(t, hq, d), packed[:, hq * d:(hq + hk) * d].view(t, hk, d)
    lens = torch.randint(20, 1000, (t // 20 + 1,), generator=g, device=DEV)     # proteins one after the other
    ends = torch.cumsum(lens, 0)
    at = torch.arange(t, device=DEV)
    which = torch.searchsorted(ends, at, right=True)
    pos = (at - (ends - lens)[which] + case["first"]).to(torch.int32)
    w, factor = _frequencies(case["rotated"], case["scaling"])
    s = {"case": case, "q": q, "k": k, "pos": pos, "w": w, "factor": factor}
    if case["train"]:
        s["q"], s["k"] = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        s["dq"] = torch.randn(t, hq, d, generator=g, device=DEV).to(dt)
        s["dk"] = torch.randn(t, hk, d, generator=g, device=DEV).to(dt)
    return s


def _prepare_sandwich(case, g):
    t, c, dt = case["tokens"], case["channels"], TYPES[case["dtype"]]
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    s = {"case": case}
    # a residual stream some layers deep: a few channels much larger than the others
    wide = torch.where(torch.rand(c, generator=g, device=DEV) < 0.02, 8.0, 1.0)
    s["x"] = (1.5 * rnd(t, c) * wide).to(dt)
    s["f"] = (0.3 * rnd(t, c) + 0.05).to(dt)
    s["post"], s["next"] = (1 + 0.2 * rnd(c)).to(dt), (1 + 0.2 * rnd(c)).to(dt)
    s["gate"] = None
    if case["gate"] == "channel":
        s["gate"] = (0.3 + 0.1 * rnd(c)).to(dt)
    elif case["gate"] != "none":
        s["gate"] = rnd(t, c).to(dt)
    s["scale"] = (1 + 0.1 * rnd(c)).to(dt) if case["scaled"] else None
    if case["train"]:
        for n in ("x", "f", "post", "next", "gate", "scale"):
            if s[n] is not None:
                s[n].requires_grad_(True)
        s["dy"], s["dh"] = rnd(t, c).to(dt), rnd(t, c).to(dt)
    return s


def _prepare_adamw(case, g):
    shapes = _model_shapes(case)
    counts = [math.prod(s) for s, _ in shapes]
    blocks = [-(-n // BLOCK) for n in counts]
    total = sum(blocks) * BLOCK
    shift = case["shift"]
    pt, gt = TYPES[case["params"]], TYPES[case["grads"]]
    live = torch.zeros(total, dtype=torch.bool, device=DEV)
    first, at = [], 0
    for n, b in zip(counts, blocks):
        live[at:at + n] = True
        first.append(at)
        at += b * BLOCK
    flat = lambda dtype: torch.zeros(shift + total, dtype=dtype, device=DEV)[shift:]
    p, grad = flat(pt), flat(gt)
    # layers differ in the size of their gradients, and so do the elements of a tensor
    size = torch.exp(2 * torch.randn(total // BLOCK, 1, generator=g, device=DEV) - 7).expand(-1, BLOCK).reshape(-1)
    size = size * torch.exp(torch.randn(total, generator=g, device=DEV))
    p.copy_(0.03 * torch.randn(total, generator=g, device=DEV) * live)
    grad.copy_(size * torch.randn(total, generator=g, device=DEV) * live)
    m = 0.3 * size * torch.randn(total, generator=g, device=DEV) * live
    v = (size * (0.5 + torch.rand(total, generator=g, device=DEV))) ** 2 * live
    s = {"case": case, "p": p, "g": grad, "first": first, "counts": counts, "shapes": [x for x, _ in shapes],
         "decay": [d for _, d in shapes], "blocks": blocks}
    s["params"] = [p[a:a + n].view(x) for a, n, (x, _) in zip(first, counts, shapes)]
    s["grads"] = [grad[a:a + n].view(x) for a, n, (x, _) in zip(first, counts, shapes)]
    s["copy"] = s["copies"] = None
    if case["params"] == "fp32":
        s["copy"] = flat(torch.bfloat16)
        s["copies"] = [s["copy"][a:a + n].view(x) for a, n, (x, _) in zip(first, counts, shapes)]
    step, lr, b1, b2, eps, wd = 37, 1e-3, 0.9, 0.999, 1e-8, 0.01
    s["hyper"] = torch.tensor([lr, b1, b2, eps, wd, 1 - b1 ** step, 1 - b2 ** step, 0.25, 1.0], device=DEV)
    s["sumsq"] = grad.double().square().sum().float().reshape(1)
    s["rng"] = torch.randint(0, 2 ** 40, (1,), generator=g, device=DEV)
    if case["bits"] == 8:
        key = torch.randint(0, 2 ** 40, (1,), generator=g, device=DEV)
        r = _random_bits(total, key)
        (s["m"], e_m), (s["v"], e_v) = _encode(m, r & 0xfffff, True), _encode(v, r >> 12, False)
        s["scales"] = torch.stack((e_m, e_v))
    else:
        s["m"], s["v"], s["scales"] = m, v, None
    # which weight decay every block has
    s["decays"] = torch.repeat_interleave(torch.tensor(s["decay"], device=DEV), torch.tensor(blocks, device=DEV))
    return s


def prepare(case, seed):
    g = _generator(seed)
    return {"rotary": _prepare_rotary, "sandwich": _prepare_sandwich, "adamw": _prepare_adamw}[case["kind"]](case, g)


# ------------------------------------------------------------------------------------ plain forms
def _turn(x, c, s, rotated, interleaved):
    """x [T, H, D] in fp32 with its first `rotated` channels turned; c, s [T, rotated / 2]."""
    a, rest = x[..., :rotated], x[..., rotated:]
    x1, x2 = (a[..., 0::2], a[..., 1::2]) if interleaved else (a[..., :rotated // 2], a[..., rotated // 2:])
    c, s = c[:, None, :], s[:, None, :]
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    y = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((y, rest), -1)


def _plain_rotary(s):
    case = s["case"]
    dt, n, il = s["q"].dtype, case["rotated"], case["interleaved"]
    a = s["pos"].double()[:, None] * s["w"]
    c, sn = (s["factor"] * a.cos()).float(), (s["factor"] * a.sin()).float()
    out = {"q": _turn(s["q"].detach().float(), c, sn, n, il).to(dt), "k": _turn(s["k"].detach().float(), c, sn, n, il).to(dt)}
    if case["train"]:
        out["dq"] = _turn(s["dq"].float(), c, -sn, n, il).to(dt)
        out["dk"] = _turn(s["dk"].float(), c, -sn, n, il).to(dt)
    return out


def _unit(x, rms, eps):
    if not rms:
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)


def _plain_sandwich(s):
    case = s["case"]
    dt, rms = s["x"].dtype, case["rms"]
    names = [n for n in ("x", "f", "post", "next", "gate", "scale") if s[n] is not None]
    with torch.set_grad_enabled(case["train"]):
        a = {n: s[n].detach().float().requires_grad_(case["train"]) for n in names}
        n = _unit(a["f"], rms, 1e-5) * a["post"]
        if case["gate"] != "none":
            n = n * (torch.sigmoid(a["gate"]) if case["gate"] == "sigmoid" else a["gate"])
        y = (a["x"] * a["scale"] if case["scaled"] else a["x"]) + n
        h = _unit(y, rms, 1e-5) * a["next"]
        out = {"y": y.detach().to(dt), "h": h.detach().to(dt)}
        if case["train"]:
            grads = torch.autograd.grad((y, h), [a[n] for n in names], (s["dy"].float(), s["dh"].float()))
            out.update({"d" + n: d.to(dt) for n, d in zip(names, grads)})
    return out


def _mix(x):
    """A 32-bit mix of two multiplications and three shifts, on int64 tensors that hold 32 bits."""
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _random_bits(total, rng):
    """32 random bits for each element of `total`: from the step's number and the element's place."""
    key = _mix((rng & 0xffffffff) ^ _mix(rng >> 32))
    at = torch.arange(total, device=rng.device)
    return _mix((at & 0xffffffff) ^ _mix((key + (at >> 32)) & 0xffffffff))


def _base(e, signed):
    return (e.to(torch.int32) - (15 if signed else 31)).clamp(min=0)[:, None] << 3


def _encode(x, r, signed):
    """(codes, exponents) of fp32 values [blocks * 256] with random numbers of 20 bits."""
    bits = x.abs().view(torch.int32).view(-1, BLOCK)
    e = (bits.amax(1) + 0xfffff) >> 23
    base = _base(e, signed)
    r = r.to(torch.int32).view(-1, BLOCK)
    code = ((bits + r) >> 20) - base
    if signed:
        least = (base + 1) << 20                            # the pattern of code 1
        up = r.float() * (least.view(torch.float32) * 2.0 ** -20) < x.abs().view(-1, BLOCK)
        code = torch.where(bits < least, up.to(torch.int32), code)
        code = torch.where((code > 0) & torch.signbit(x).view(-1, BLOCK), code + 128, code)
    else:
        code = code.clamp(min=1)
    code = torch.where(bits == 0, 0, code)
    return code.to(torch.uint8).view(-1), e.to(torch.uint8)


def _decode(code, e, signed):
    code = code.view(-1, BLOCK).to(torch.int32)
    low = code & 127 if signed else code
    x = torch.where(low == 0, 0, (low + _base(e, signed)) << 20).view(torch.float32)
    if signed:
        x = torch.where(code >= 128, -x, x)
    return x.view(-1)


def _plain_adamw(s):
    lr, b1, b2, eps, wd, bc1, bc2, gs, most = s["hyper"]
    norm = s["sumsq"].sqrt() * gs
    factor = gs * torch.clamp(most / (norm + 1e-6), max=1.0)
    eight = s["scales"] is not None
    m, v = (_decode(s["m"], s["scales"][0], True), _decode(s["v"], s["scales"][1], False)) if eight else (s["m"], s["v"])
    g = s["g"].float() * factor
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    d = torch.where(s["decays"], 1 - lr * wd, 1.0)[:, None].expand(-1, BLOCK).reshape(-1)
    p = s["p"].float() * d - lr / bc1 * (m / (v.sqrt() / bc2.sqrt() + eps))
    s["p"].copy_(p)
    out = {"p": s["p"]}
    if s["copy"] is not None:
        s["copy"].copy_(p)
        out["copy"] = s["copy"]
    if eight:
        r = _random_bits(m.numel(), s["rng"])
        (cm, em), (cv, ev) = _encode(m, r & 0xfffff, True), _encode(v, r >> 12, False)
        s["m"].copy_(cm)
        s["v"].copy_(cv)
        s["scales"][0].copy_(em)
        s["scales"][1].copy_(ev)
        out["m"], out["v"] = _decode(cm, em, True).bfloat16(), _decode(cv, ev, False).bfloat16()
    else:
        out["m"], out["v"] = s["m"].copy_(m), s["v"].copy_(v)
    return out


# ------------------------------------------------------------------------------- the package's calls
def _own_rotary(s):
    from nanoplm_b200.ops import functional as ops
    case = s["case"]
    with torch.set_grad_enabled(case["train"]):
        q, k = ops.rotary(s["q"], s["k"], positions=s["pos"], frequencies=s["w"], factor=s["factor"],
                          interleaved=case["interleaved"])
        out = {"q": q.detach(), "k": k.detach()}
        if case["train"]:
            out["dq"], out["dk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return out


def _own_sandwich(s):
    from nanoplm_b200.ops import functional as ops
    case = s["case"]
    names = [n for n in ("x", "f", "post", "next", "gate", "scale") if s[n] is not None]
    with torch.set_grad_enabled(case["train"]):
        y, h = ops.sandwich_norm(s["x"], s["f"], s["post"], s["next"], gate=s["gate"], sigmoid=case["gate"] == "sigmoid",
                                 scale=s["scale"], eps=1e-5, rms=case["rms"])
        out = {"y": y.detach(), "h": h.detach()}
        if case["train"]:
            grads = torch.autograd.grad((y, h), [s[n] for n in names], (s["dy"], s["dh"]))
            out.update({"d" + n: d for n, d in zip(names, grads)})
    return out


def _own_adamw(s):
    from nanoplm_b200.ops import kernels as K
    K.adamw_tensors_(s["params"], s["grads"], s["m"], s["v"], s["hyper"], scales=s["scales"], rng=s["rng"],
                     copies=s["copies"], decay=s["decay"], sumsq=s["sumsq"])
    out = {"p": s["p"]}
    if s["copy"] is not None:
        out["copy"] = s["copy"]
    if s["scales"] is not None:
        out["m"], out["v"] = K.moment_values(s["m"], s["v"], s["scales"], torch.bfloat16)
    else:
        out["m"], out["v"] = s["m"], s["v"]
    return out


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "sandwich": _own_sandwich, "adamw": _own_adamw}[kind](state)
    return {"rotary": _plain_rotary, "sandwich": _plain_sandwich, "adamw": _plain_adamw}[kind](state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "rotary":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["tokens"] * (case["q_heads"] + case["k_heads"])
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * case["width"] * size + 4 * case["tokens"]),
                "flops": passes * 3 * n * case["rotated"]}
    if case["kind"] == "sandwich":
        size = 4 if case["dtype"] == "fp32" else 2
        full = case["gate"] in ("token", "sigmoid")
        n, arrays, ops = case["tokens"] * case["channels"], 4 + full, 16
        if case["train"]:
            arrays, ops = arrays + 6 + 2 * full, 56
        return {"bytes": n * arrays * size, "flops": n * ops}
    n = sum(math.prod(s) for s, _ in _model_shapes(case))
    per = 2 * (4 if case["params"] == "fp32" else 2) + (4 if case["grads"] == "fp32" else 2)
    per += 2 if case["params"] == "fp32" else 0
    per += 4 + 4 if case["bits"] == 8 else 16       # codes read and written, and the values that are handed out
    return {"bytes": n * per, "flops": 16 * n}


# ------------------------------------------------------------------------------------------ exact
def _exact_rotary(s):
    case = s["case"]
    half, n = case["rotated"] // 2, case["rotated"]
    angle = s["pos"].double()[:, None] * s["w"]
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None, :]
    places = torch.arange(n, device=DEV)
    re, im = (places[0::2], places[1::2]) if case["interleaved"] else (places[:half], places[half:])

    def turned(x, t):
        x = x.detach().double()
        z = torch.complex(x[..., re], x[..., im]) * t
        y = x.clone()
        y[..., re], y[..., im] = z.real, z.imag
        return y

    out = {"q": turned(s["q"], turn), "k": turned(s["k"], turn)}
    if case["train"]:
        out["dq"], out["dk"] = turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())
    return out


def _exact_sandwich(s):
    case = s["case"]
    rms, c = case["rms"], case["channels"]
    a = {n: (None if s[n] is None else s[n].detach().double()) for n in ("x", "f", "post", "next", "gate", "scale")}

    def stats(t):
        mean = torch.zeros_like(t[:, :1]) if rms else t.sum(1, keepdim=True) / c
        inv = (((t - mean) ** 2).sum(1, keepdim=True) / c + 1e-5) ** -0.5
        return (t - mean) * inv, inv

    def back(d, unit, inv):
        d1 = 0.0 if rms else d.sum(1, keepdim=True) / c
        return inv * (d - d1 - unit * ((d * unit).sum(1, keepdim=True) / c))

    uf, inv_f = stats(a["f"])
    n = uf * a["post"]
    g = 1.0 if a["gate"] is None else 1 / (1 + torch.exp(-a["gate"])) if case["gate"] == "sigmoid" else a["gate"]
    r = 1.0 if a["scale"] is None else a["scale"]
    y = r * a["x"] + g * n
    uy, inv_y = stats(y)
    out = {"y": y, "h": uy * a["next"]}
    if case["train"]:
        dy, dh = s["dy"].double(), s["dh"].double()
        t = dy + back(dh * a["next"], uy, inv_y)
        out["dx"], out["df"] = r * t, back(g * t * a["post"], uf, inv_f)
        out["dpost"], out["dnext"] = (g * t * uf).sum(0), (dh * uy).sum(0)
        if case["gate"] == "channel":
            out["dgate"] = (t * n).sum(0)
        elif case["gate"] == "token":
            out["dgate"] = t * n
        elif case["gate"] == "sigmoid":
            out["dgate"] = t * n * g * (1 - g)
        if case["scaled"]:
            out["dscale"] = (t * a["x"]).sum(0)
    return out


def _exact_moment(x, r, octaves, signed):
    """The kept value of every x (fp64, [blocks, 256]): between neighbours an eighth of an octave apart, by the random numbers r."""
    mag = x.abs()
    mant, expo = torch.frexp(mag)                       # mag = mant 2^expo, mant in [1/2, 1)
    eighths = mant * 16                                 # [8, 16): steps of an eighth of the octave
    top = (torch.where(mag > 0, expo + (eighths + (2 ** 20 - 1) / 2 ** 20 >= 16), -10 ** 6)).amax(1, keepdim=True)
    kept = torch.ldexp(torch.floor(eighths + r / 2.0 ** 20), expo - 4)
    least = torch.ldexp(torch.full_like(mag, 9.0), (top - octaves + 1 - 4).expand_as(expo))
    if signed:
        kept = torch.where(mag < least, torch.where(r / 2.0 ** 20 * least < mag, least, 0.0), kept)
    else:
        kept = torch.maximum(kept, least)
    return torch.where(mag > 0, kept, 0.0) * torch.sign(x)


def _exact_adamw(s):
    lr, b1, b2, eps, wd, bc1, bc2, gs, most = s["hyper"].double()
    eight = s["scales"] is not None
    if eight:       # the codes' values: mantissas of 3 bits, exponents above the block's lowest
        def value(code, e, octaves, signed):
            low = (code.view(-1, BLOCK) & (127 if signed else 255)).double()
            sign = torch.where(code.view(-1, BLOCK) >= 128, -1.0, 1.0) if signed else 1.0
            bottom = e.double()[:, None] - (octaves - 1) - 127
            x = sign * (1 + torch.remainder(low, 8) / 8) * torch.exp2(torch.floor(low / 8) + bottom)
            return torch.where(low == 0, 0.0, x).view(-1)
        m, v = value(s["m"], s["scales"][0], 16, True), value(s["v"], s["scales"][1], 32, False)
    else:
        m, v = s["m"].double(), s["v"].double()
    norm = s["sumsq"].double() ** 0.5 * gs
    g = s["g"].double() * gs * torch.minimum(torch.ones_like(norm), most / (norm + 1e-6))
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
    keep = (1 - lr * wd * s["decays"].double())[:, None].expand(-1, BLOCK).reshape(-1)
    p = keep * s["p"].double() - lr * (m / bc1) / ((v / bc2) ** 0.5 + eps)
    out = {"p": p}
    if s["copy"] is not None:
        out["copy"] = p
    if eight:
        r = _random_bits(m.numel(), s["rng"]).view(-1, BLOCK)
        m = _exact_moment(m.view(-1, BLOCK), (r & 0xfffff).double(), 16, True).view(-1)
        v = _exact_moment(v.view(-1, BLOCK), (r >> 12).double(), 32, False).view(-1)
    out["m"], out["v"] = m, v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "sandwich": _exact_sandwich, "adamw": _exact_adamw}[case["kind"]](s)
