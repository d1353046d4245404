"""The optimizer operators that follow the decoder losses in a training step, as measured cases.

``run`` computes one pass in its plain form (elementary torch operations in 32 bits) or, where ``own`` is
true, through ``flexsae_b200.optim``.  Notation: ``c`` the clipping factor, ``t`` the number of this step
(1 for the first), ``b1, b2`` the decay rates.

norm       ``sqrt(sum of g^2 over all gradients)``, one number for a list of tensors.

adamw      for every tensor of a list, in place:
               g = c g                         c = min(1, max_norm / (norm + 1e-6)), or 1 without clipping
               m = b1 m + (1 - b1) g           v = b2 v + (1 - b2) g^2
               p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
           With a 32-bit master copy, p is that copy and the parameter its rounding.

adamw8     the same with m held as e4m3 and v as e5m2, each times one scale for 256 consecutive values
           (SM = max|m| / 448, SV = max v / 57344, both 2^-20 larger so that the largest value stays in
           range).  The new m and v are rounded to 8 bits at random between their two neighbours, upwards
           with the probability that makes the rounding right on average; the random bits are a function of
           (seed, t, position of the tensor in the list, element).  p is computed before the rounding.

unit_rows  adamw on a [F, D] decoder whose rows are kept at unit length:
               g = g - (g.w / w.w) w  for every row, then adamw, then w = w / |w|.

The sparse autoencoder of a case is the four tensors w_enc [F, D], b_enc [F], w_dec [F, D], b_dec [D].
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 256
LR, B1, B2, EPS, WD = 1e-4, 0.9, 0.999, 1e-8, 0.01
E4M3_MAX, E5M2_MAX = 448.0, 57344.0
SCALE_M = (1.0 / E4M3_MAX) * (1.0 + 2.0 ** -20)
SCALE_V = (1.0 / E5M2_MAX) * (1.0 + 2.0 ** -20)
TINY = 2.0 ** -126


def case(name, op, F, D, dtype, saes=1, master=False, clip=False):
    return {"name": name, "op": op, "F": F, "D": D, "dtype": dtype, "saes": saes, "master": master, "clip": clip}


def listed():
    return [
        # a toy model of the unit tests: the call is all latency
        case("norm_tiny", "norm", 512, 64, "fp32"),
        # gradients of the benchmark's model (65536 features of width 2304), both halves
        case("norm_headline", "norm", 65536, 2304, "bf16"),
        # the same toy model through one optimizer step
        case("adamw_tiny", "adamw", 512, 64, "fp32"),
        # five models of different odd sizes trained side by side, one per layer: 20 tensors in one call
        case("adamw_five_ragged", "adamw", 5003, 517, "bf16", saes=5),
        # the benchmark's model held in bf16, with gradient clipping
        case("adamw_headline", "adamw", 65536, 2304, "bf16", clip=True),
        # the reference script's model (131072 features of width 1024) in fp32
        case("adamw_fp32", "adamw", 131072, 1024, "fp32"),
        # half-precision weights with a 32-bit master copy, clipped
        case("adamw_master", "adamw", 32768, 2304, "fp16", master=True, clip=True),
        # 8-bit states: toy model, odd sizes of three models, the benchmark's model
        case("adamw8_tiny", "adamw8", 512, 64, "bf16"),
        case("adamw8_ragged", "adamw8", 9001, 333, "fp32", saes=3),
        case("adamw8_headline", "adamw8", 65536, 2304, "bf16", clip=True),
        # decoder kept at unit rows: the CPU-sized configuration and the benchmark's decoder
        case("unit_rows_small", "unit_rows", 4096, 256, "fp32"),
        case("unit_rows_headline", "unit_rows", 65536, 2304, "bf16", clip=True),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "adamw", "adamw", "adamw8", "adamw8", "unit_rows"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    c = {"op": op, "dtype": dtype, "saes": 1 if op == "unit_rows" else rng.choice([1, 1, 2]),
         "master": op != "norm" and dtype != "fp32" and rng.random() < 0.3, "clip": op != "norm" and rng.random() < 0.5}
    c["D"] = _between(rng, 4, 8192 if op == "unit_rows" else 4096)
    most = 60_000_000 // c["saes"] // c["D"]
    c["F"] = _between(rng, 32, max(33, min(131072, most)))
    return c


def _shapes(case):
    got = []
    for i in range(case["saes"]):
        F, D = max(1, case["F"] // (i + 1)), max(1, case["D"] - 3 * i)
        got += [(F, D)] if case["op"] == "unit_rows" else [(F, D), (F,), (F, D), (D,)]
    return got


def _to_blocks(x):
    """A tensor's values as rows of BLOCK, the last row filled up with zeros."""
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = DTYPES[case["dtype"]], case["op"]

    def normal(shape, scale):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale)

    s = {"op": op, "grads": [], "params": [], "m": [], "v": [], "m_scale": [], "v_scale": [], "masters": [], "norm": None,
         "step": torch.full((), 1000, dtype=torch.int64, device="cuda"), "seed": seed & 0xFFFFFFFF, "max_norm": None}
    for shape in _shapes(case):
        grad = normal(shape, 1e-3)
        if len(shape) == 2:                                   # features that no row of the batch used
            idle = torch.rand(shape[0], 1, generator=g, device="cuda") < 0.1
            grad.masked_fill_(idle, 0.0)
        s["grads"].append(grad.to(dtype))
        if op == "norm":
            continue
        p = normal(shape, 1.0 / math.sqrt(shape[-1]) if len(shape) == 2 else 0.02)
        if op == "unit_rows":
            p = p / p.square().sum(1, keepdim=True).sqrt().clamp_min(1e-12)
        s["params"].append(p.to(dtype))
        if case["master"]:
            s["masters"].append(p)
        m, v = normal(shape, 3e-4), normal(shape, 1e-3).square_().add_(1e-8)
        if op != "adamw8":
            s["m"].append(m)
            s["v"].append(v)
            continue
        for x, keep, scales, factor, kind in ((m, "m", "m_scale", SCALE_M, torch.float8_e4m3fn), (v, "v", "v_scale", SCALE_V, torch.float8_e5m2)):
            rows = _to_blocks(x)
            scale = rows.abs().amax(1) * factor
            s[scales].append(scale)
            s[keep].append((rows / scale[:, None]).reshape(-1)[: x.numel()].view(shape).to(kind))
    if case["clip"]:
        s["norm"] = torch.stack([x.float().square().sum() for x in s["grads"]]).sum().sqrt()
        s["max_norm"] = 0.5 * float(s["norm"])                # the gradients are twice as long as allowed
    return s


# ---- the plain form ----------------------------------------------------------------------------------
def _factor(s):
    return 1.0 if s["norm"] is None else (s["max_norm"] / (s["norm"] + 1e-6)).clamp_max(1.0)


def _moments(grad, m, v):
    return B1 * m + (1.0 - B1) * grad, B2 * v + (1.0 - B2) * (grad * grad)


def _stepped(p, m, v, step):
    t = step.double()
    rate = (LR / (1.0 - B1 ** t)).float()
    root = (1.0 / (1.0 - B2 ** t).sqrt()).float()
    return p * (1.0 - LR * WD) - rate * (m / (v.sqrt() * root + EPS))


def _put(s, i, p):
    s["params"][i].copy_(p)
    if s["masters"]:
        s["masters"][i].copy_(p)


def _adamw_tensor(s, i, c):
    p = s["masters"][i] if s["masters"] else s["params"][i].float()
    grad = s["grads"][i].float() * c
    if s["op"] == "unit_rows":
        along = (grad * p).sum(1, keepdim=True) / (p * p).sum(1, keepdim=True)
        grad = grad - along * p
    m, v = _moments(grad, s["m"][i], s["v"][i])
    p = _stepped(p, m, v, s["step"])
    if s["op"] == "unit_rows":
        p = p / (p * p).sum(1, keepdim=True).sqrt()
    _put(s, i, p)
    s["m"][i].copy_(m)
    s["v"][i].copy_(v)


def _mix(x):
    """A 32-bit integer mixing function (two multiplications), on int64 tensors."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(seed, step, i, n, device):
    """The 32 random bits of every pair of elements of tensor i, repeated for both."""
    pair = torch.arange((n + 1) // 2, device=device)
    key = _mix((_mix((_mix(step & 0xFFFFFFFF) + i) & 0xFFFFFFFF) + seed) & 0xFFFFFFFF)
    return _mix((pair & 0xFFFFFFFF) ^ ((key + (pair >> 32)) & 0xFFFFFFFF)).repeat_interleave(2)[:n]


def _rounded(x, scale, random, drop, shift, floor):
    """Codes of x / scale: the value's bits, moved to the small format's exponent, plus random low bits, cut off."""
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    y = (_to_blocks(x) * inverse[:, None]).reshape(-1)[: x.numel()] * shift
    bits = torch.clamp_min(y.abs(), floor).view(torch.int32).to(torch.int64)
    return ((((bits + random) >> drop) | ((y < 0).to(torch.int64) << 7))).to(torch.uint8).view(x.shape)


def _scales(x, factor):
    s = _to_blocks(x).abs().amax(1) * factor
    return torch.where(s >= TINY, s, torch.zeros_like(s))


def _widened(code, scale):
    return (_to_blocks(code.float()) * scale[:, None]).reshape(-1)[: code.numel()].view(code.shape)


def _adamw8_tensor(s, i, c):
    p = s["masters"][i] if s["masters"] else s["params"][i].float()
    m, v = _moments(s["grads"][i].float() * c, _widened(s["m"][i], s["m_scale"][i]), _widened(s["v"][i], s["v_scale"][i]))
    _put(s, i, _stepped(p, m, v, s["step"]))
    h = _random_bits(s["seed"], s["step"], i, m.numel(), m.device)
    odd = torch.arange(m.numel(), device=m.device) % 2 == 1
    s["m_scale"][i].copy_(_scales(m, SCALE_M))
    s["v_scale"][i].copy_(_scales(v, SCALE_V))
    s["m"][i].view(torch.uint8).copy_(_rounded(m, s["m_scale"][i], torch.where(odd, h & 0xFFFFF, h >> 12), 20, 2.0 ** -120, 0.0))
    s["v"][i].view(torch.uint8).copy_(_rounded(v, s["v_scale"][i], torch.where(odd, h >> 11, h & 0x1FFFFF), 21, 2.0 ** -112, 2.0 ** -128))


def _outputs(s):
    out = {k: s[k] for k in ("params", "masters", "m", "v") if s[k]}
    return {**out, **({"m_scale": s["m_scale"], "v_scale": s["v_scale"]} if s["op"] == "adamw8" else {}), "step": s["step"]}


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "norm":
        return torch.stack([x.float().square().sum() for x in s["grads"]]).sum().sqrt()
    c = _factor(s)
    s["step"].add_(1)
    [(_adamw8_tensor if s["op"] == "adamw8" else _adamw_tensor)(s, i, c) for i in range(len(s["params"]))]
    return _outputs(s)


def _run_own(s):
    from flexsae_b200 import optim

    if s["op"] == "norm":
        return optim.grad_norm(s["grads"])
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, masters=s["masters"] or None, norm=s["norm"], max_norm=s["max_norm"])
    if s["op"] == "adamw8":
        optim.adamw8_step(s["params"], s["grads"], s["m"], s["m_scale"], s["v"], s["v_scale"], s["step"], seed=s["seed"], **kw)
    elif s["op"] == "unit_rows":
        optim.adamw_unit_rows_step(s["params"], s["grads"], s["m"], s["v"], s["step"], **kw)
    else:
        optim.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], **kw)
    return _outputs(s)


def work(case):
    n = sum(math.prod(x) for x in _shapes(case))
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        return {"bytes": n * size + 4, "flops": 2 * n}
    # the parameter read (from its master copy where there is one) and written, the gradient read, two states read and written
    per = size + (size + 8 if case["master"] else 2 * size)
    if case["op"] == "adamw8":
        blocks = sum(-(-math.prod(x) // BLOCK) for x in _shapes(case))
        return {"bytes": n * (per + 4) + 16 * blocks, "flops": 40 * n}
    return {"bytes": n * (per + 16), "flops": (24 if case["op"] == "unit_rows" else 16) * n}


# ---- the definition in 64 bits -------------------------------------------------------------------------
def _exact_random(seed, t, i, n):
    """The random bits again, with unsigned arithmetic modulo 2^32 kept in int64."""
    word = (1 << 32) - 1

    def mix(x):
        for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
            x = ((x ^ (x >> shift)) * factor) & word
        return x ^ (x >> 16)

    element = torch.arange(n, device="cuda")
    key = mix((mix((mix(t & word) + i) & word) + seed) & word)
    return mix(((element // 2) % 2 ** 32) ^ ((key + element // 2 ** 33) & word)), element % 2


def _exact_code(x, scale, random, drop, mantissa, least, lowest, dtype):
    """x / scale on the format's grid: the spacing at its size, then the next lower multiple of x / spacing plus a random fraction."""
    size = (x / torch.where(scale > 0, scale, torch.full_like(scale, math.inf))).abs().clamp_min(lowest)
    exponent = torch.frexp(size)[1].to(torch.float64) - 1.0
    spacing = torch.exp2(exponent.clamp_min(least) - mantissa)
    return (torch.floor(size / spacing + random.double() / 2.0 ** drop) * spacing * torch.where(x < 0, -1.0, 1.0)).to(dtype).double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        total = sum(float(x.double().square().sum()) for x in s["grads"])
        return torch.tensor(math.sqrt(total), dtype=torch.float64)
    t = int(s["step"]) + 1
    c = 1.0 if s["norm"] is None else min(1.0, s["max_norm"] / (float(s["norm"]) + 1e-6))
    out = {k: [] for k in ("params", "m", "v")}
    if s["masters"]:
        out["masters"] = []
    if case["op"] == "adamw8":
        out.update(m_scale=[], v_scale=[])
    for i, shape in enumerate(_shapes(case)):
        w = (s["masters"][i] if s["masters"] else s["params"][i]).double()
        grad = s["grads"][i].double() * c
        m, v = s["m"][i].double(), s["v"][i].double()
        if case["op"] == "adamw8":
            at = torch.arange(m.numel(), device="cuda").div(BLOCK, rounding_mode="floor").view(shape)
            m, v = m * s["m_scale"][i].double()[at], v * s["v_scale"][i].double()[at]
        if case["op"] == "unit_rows":
            grad = grad - w * (torch.einsum("fd,fd->f", grad, w) / torch.einsum("fd,fd->f", w, w))[:, None]
        m = m * B1 + grad * (1.0 - B1)
        v = v * B2 + grad.square() * (1.0 - B2)
        w = w * (1.0 - LR * WD) - LR * (m / (1.0 - B1 ** t)) / ((v / (1.0 - B2 ** t)).sqrt() + EPS)
        if case["op"] == "unit_rows":
            w = w / torch.linalg.vector_norm(w, dim=1, keepdim=True)
        out["params"].append(w)
        if s["masters"]:
            out["masters"].append(w)
        if case["op"] == "adamw8":
            blocks = s["m_scale"][i].numel()
            random, odd = _exact_random(s["seed"], t, i, m.numel())
            random, odd = random.view(shape), odd.view(shape).bool()
            largest = [torch.zeros(blocks, dtype=torch.float64, device="cuda").scatter_reduce(0, at.reshape(-1), x.abs().reshape(-1), "amax") for x in (m, v)]
            sm, sv = largest[0] * SCALE_M, largest[1] * SCALE_V
            sm, sv = sm * (sm >= TINY), sv * (sv >= TINY)
            out["m_scale"].append(sm)
            out["v_scale"].append(sv)
            m = _exact_code(m, sm[at], torch.where(odd, random % 2 ** 20, random // 2 ** 12), 20, 3, -6, 0.0, torch.float8_e4m3fn)
            v = _exact_code(v, sv[at], torch.where(odd, random // 2 ** 11, random % 2 ** 21), 21, 2, -14, 2.0 ** -16, torch.float8_e5m2)
        out["m"].append(m)
        out["v"].append(v)
    return {**out, "step": torch.tensor(t)}
