"""Oracle of the optimizer operators: AdamW, its unit-row form and the 8-bit states, in numpy.

``adamw`` works in 64 bits and is pinned to ``torch.optim.AdamW`` in float64.  The 8-bit states are
written out twice: ``moments32`` / ``codes`` follow the definition in 32-bit arithmetic, operation by
operation (the kernel has to agree bit for bit), and ``grid`` says which numbers the two formats have.
"""
from __future__ import annotations

from typing import Optional, Tuple

import numpy as np

BLOCK = 256


def clip_factor(norm: Optional[float], max_norm: Optional[float]) -> float:
    return 1.0 if norm is None or max_norm is None else min(1.0, max_norm / (norm + 1e-6))


def adamw(p, g, m, v, t: int, lr: float, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, clip: float = 1.0,
          unit_rows: bool = False) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
    """(p, m, v) after step ``t`` (1 for the first), all in float64."""
    p, g, m, v = (np.asarray(x, dtype=np.float64) for x in (p, g, m, v))
    g = g * clip
    if unit_rows:
        square = np.sum(p * p, axis=1, keepdims=True)
        g = g - np.divide(np.sum(g * p, axis=1, keepdims=True), square, out=np.zeros_like(square), where=square != 0) * p
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    p = p * (1 - lr * weight_decay) - lr / (1 - betas[0] ** t) * m / (np.sqrt(v) / np.sqrt(1 - betas[1] ** t) + eps)
    if unit_rows:
        length = np.sqrt(np.sum(p * p, axis=1, keepdims=True))
        p = np.divide(p, length, out=p.copy(), where=length != 0)
    return p, m, v


# ---- 8-bit states -------------------------------------------------------------------------------------
def grid(mantissa: int, bias: int, codes: int) -> np.ndarray:
    """Values of the codes 0 .. codes - 1 of an 8-bit float without sign: e4m3 = (3, 7, 127), e5m2 = (2, 15, 124)."""
    c = np.arange(codes)
    exponent, fraction = c >> mantissa, c & ((1 << mantissa) - 1)
    return np.where(exponent == 0, fraction * 2.0 ** (1 - bias - mantissa),
                    (1 + fraction / 2.0 ** mantissa) * 2.0 ** (exponent.astype(np.float64) - bias))


E4M3, E5M2 = grid(3, 7, 127), grid(2, 15, 124)


def widen(codes: np.ndarray, kind: str) -> np.ndarray:
    """float32 values of uint8 codes ("m": e4m3, "v": e5m2), NaN for 0x7f and infinity for an e5m2 0x7c."""
    table = E4M3 if kind == "m" else E5M2
    low = codes & 0x7F
    x = np.where(low < len(table), table[np.minimum(low, len(table) - 1)], np.where((low == 0x7C) & (kind == "v"), np.inf, np.nan)).astype(np.float32)
    return np.where(codes & 0x80, -x, x)


def mix(x):
    x = np.asarray(x, dtype=np.uint64) & np.uint64(0xFFFFFFFF)
    word = np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D)) & word
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x846CA68B)) & word
    return x ^ (x >> np.uint64(16))


def random_bits(seed: int, t: int, index: int, n: int, first: int = 0):
    """(20 bits for m, 21 bits for v) of the n elements from ``first`` on of tensor ``index``."""
    key = int(mix(int(mix(int(mix(t & 0xFFFFFFFF)) + index)) + seed))
    e = np.arange(first, first + n, dtype=np.uint64)
    pair = e >> np.uint64(1)
    h = mix((pair & np.uint64(0xFFFFFFFF)) ^ ((np.uint64(key) + (pair >> np.uint64(32))) & np.uint64(0xFFFFFFFF)))
    odd = (e & np.uint64(1)).astype(bool)
    return np.where(odd, h & np.uint64(0xFFFFF), h >> np.uint64(12)), np.where(odd, h >> np.uint64(11), h & np.uint64(0x1FFFFF))


def _by_block(x: np.ndarray) -> np.ndarray:
    return np.pad(x, (0, -len(x) % BLOCK)).reshape(-1, BLOCK)


def scales(x: np.ndarray, largest_code: float) -> np.ndarray:
    """float32 scale of every block: its largest finite absolute value / the format's largest number, 2^-20 larger.  A
    block of second moments whose finite values give none but that holds an infinity has the least one."""
    factor = np.float32((1.0 / largest_code) * (1.0 + 2.0 ** -20))
    a = np.abs(_by_block(x))
    s = np.max(np.where(np.isfinite(a), a, np.float32(0)), axis=1).astype(np.float32) * factor
    s = np.where(s >= np.float32(2.0 ** -126), s, np.float32(0))
    if largest_code == 57344.0:
        s = np.where((s == 0) & np.any(a == np.inf, axis=1), np.float32(2.0 ** -126), s)
    return s.astype(np.float32)


def codes(x: np.ndarray, scale: np.ndarray, random: np.ndarray, kind: str) -> np.ndarray:
    """uint8 codes of the float32 values ``x``: the pattern of x / scale, moved to the small format's exponent, plus
    the random bits, cut off."""
    drop, shift = (20, np.float32(2.0 ** -120)) if kind == "m" else (21, np.float32(2.0 ** -112))
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        inverse = np.where(scale > 0, np.float32(1) / scale, np.float32(0)).astype(np.float32)
        y = ((_by_block(x) * inverse[:, None]).reshape(-1)[: len(x)] * shift).astype(np.float32)
    size = np.abs(y)
    if kind == "v":
        size = np.fmax(size, np.float32(2.0 ** -128))
    c = (size.view(np.uint32).astype(np.uint64) + random.astype(np.uint64)) >> np.uint64(drop)
    c = np.where(np.isfinite(x), c, np.where((x == np.inf) & (kind == "v"), 0x7C, 0x7F)).astype(np.uint8)
    if kind == "m":
        c = np.where(np.isfinite(x) & np.signbit(y), c | 0x80, c)
    return c.astype(np.uint8)


def moments32(g: np.ndarray, m8, m_scale, v8, v_scale, betas=(0.9, 0.999), clip: np.float32 = np.float32(1)):
    """The new moments in 32-bit arithmetic, each operation rounded."""
    f = np.float32
    m = widen(m8, "m") * np.repeat(m_scale, BLOCK)[: len(m8)]
    v = widen(v8, "v") * np.repeat(v_scale, BLOCK)[: len(v8)]
    with np.errstate(over="ignore", invalid="ignore"):
        g = g.astype(f) * f(clip)
        return f(betas[0]) * m + f(1 - betas[0]) * g, f(betas[1]) * v + f(1 - betas[1]) * (g * g)


def adamw8_states(g, m8, m_scale, v8, v_scale, t: int, seed: int, index: int, betas=(0.9, 0.999), clip: float = 1.0, first: int = 0):
    """(m, v, m8, m_scale, v8, v_scale) after the step: the 32-bit moments and what is stored of them.  The arrays are
    the tensor's elements from ``first`` (a multiple of the block) on."""
    m, v = moments32(g, m8, m_scale, v8, v_scale, betas, np.float32(clip))
    rm, rv = random_bits(seed, t, index, len(g), first)
    sm, sv = scales(m, 448.0), scales(v, 57344.0)
    return m, v, codes(m, sm, rm, "m"), sm, codes(v, sv, rv, "v"), sv
