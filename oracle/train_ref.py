"""CPU restatement of the training operators (layer norm, gradient norm and clipping, AdamW with 32- and 8-bit moments): the
definitions in 64 bits, and the 8-bit moments' format in numpy.  Test oracle only; nothing in ayolov2_amd imports it."""
from __future__ import annotations

import numpy as np
import torch

BLOCK, M_BIAS, V_BIAS, M_LEAST, V_LEAST = 128, 14, 30, 1, 10
U32 = 2.0 ** -24                                       # half a step of fp32
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # half a step of the subnormals


def layer_norm(x, w, b, eps, r=None):
    """(y, s) in float64 over the last dimension; s = x + r rounded to x's type, as it is kept."""
    s = x if r is None else (x.float() + r.float()).to(x.dtype)
    t = s.double()
    mu = t.mean(-1, keepdim=True)
    var = ((t - mu) ** 2).mean(-1, keepdim=True)
    y = (t - mu) / torch.sqrt(var + eps)
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, s


def layer_norm_grads(s, w, eps, gy, gs=None):
    """(ds, dw, db) in float64 by the formula of the derivative."""
    t, g = s.double(), gy.double()
    n = t.shape[-1]
    mu = t.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((t - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (t - mu) * rstd
    gw = g if w is None else g * w.double()
    ds = rstd * (gw - gw.sum(-1, keepdim=True) / n - xh * (gw * xh).sum(-1, keepdim=True) / n)
    if gs is not None:
        ds = ds + gs.double()
    return ds, (g * xh).reshape(-1, n).sum(0), g.reshape(-1, n).sum(0)


def adamw(p, g, m, v, t, lr, b1, b2, eps, wd, factor=1.0):
    """One step in float64; t counts this step."""
    g = g.double() * factor
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g * g
    p = p.double()
    p = p - lr * wd * p - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p, m, v


def mix(x):
    x = np.asarray(x, dtype=np.uint32).copy()
    x ^= x >> np.uint32(16)
    x *= np.uint32(0x6A09E667)
    x ^= x >> np.uint32(15)
    x *= np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


def noise(seed: int, t: int, position: int, n: int, first: int = 0):
    """(16 bits for m, 16 bits for v) of elements first .. first + n - 1."""
    with np.errstate(over="ignore"):
        k = np.uint32(0x9E3779B1)
        one = lambda v: np.asarray([v & 0xFFFFFFFF], dtype=np.uint32)  # noqa: E731
        key = mix(mix(one(seed + 0x9E3779B1 * t)) + one(0x9E3779B1 * (position + 1)))
        h = mix((np.arange(first, first + n, dtype=np.uint64).astype(np.uint32) * k) ^ key)
    return h >> np.uint32(16), h & np.uint32(0xFFFF)


def decode(codes, exps, signed: bool):
    codes = np.asarray(codes, dtype=np.uint32)
    mag, top = (codes & 0x7F, 0x7F) if signed else (codes, 0xFF)
    e = np.repeat(np.asarray(exps, dtype=np.int64), BLOCK)[:len(codes)] - (M_BIAS if signed else V_BIAS)
    with np.errstate(over="ignore"):
        x = np.ldexp((mag << 20).astype(np.uint32).view(np.float32).astype(np.float64), e).astype(np.float32)
    x = np.where(mag == top, np.float32(np.nan), np.where(mag == top - 1, np.float32(np.inf), x))
    return np.where(codes & 0x80, -x, x).astype(np.float32) if signed else x.astype(np.float32)


def encode(x, r16, signed: bool):
    """(codes, exps) of float32 values under the rounding of the 16-bit numbers r16."""
    x = np.asarray(x, dtype=np.float32)
    n = len(x)
    bias, least, top = (M_BIAS, M_LEAST, 0x7F) if signed else (V_BIAS, V_LEAST, 0xFF)
    bits = x.view(np.uint32) & np.uint32(0x7FFFFFFF)
    field = (bits >> 23).astype(np.int64)
    field[field == 255] = 0
    nb = -(-n // BLOCK)
    exps = np.maximum(np.pad(field, (0, nb * BLOCK - n)).reshape(nb, BLOCK).max(1), least)
    with np.errstate(over="ignore", invalid="ignore"):
        y = np.ldexp(bits.view(np.float32).astype(np.float64), bias - np.repeat(exps, BLOCK)[:n]).astype(np.float32)
    code = (y.view(np.uint32) + ((r16.astype(np.uint32) << np.uint32(4)) | np.uint32(8))) >> np.uint32(20)
    if not signed:
        code = np.where((code == 0) & (bits != 0), np.uint32(1), code)
    code = np.where(bits == 0x7F800000, top - 1, np.where(bits > 0x7F800000, top, code))
    if signed:
        code = np.where(np.signbit(x) & ~np.isnan(x), code | 0x80, code)
    return code.astype(np.uint8), exps.astype(np.uint8)
