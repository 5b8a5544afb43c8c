"""64-bit restatements of the texel-layer operators (test infrastructure), from their
definitions in include/nt_capi.h."""
import math

import numpy as np
import torch

# half of the distance between neighbouring values, relative to a value
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # half the smallest step

_erf = np.vectorize(math.erf)


def activate(z, act):
    if act == "relu":
        return np.where(z < 0, 0.0, z)
    if act == "silu":
        return z / (1 + np.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
    return z


def slope(z, act):
    if act == "relu":
        return (z > 0).astype(np.float64)
    if act == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return np.ones_like(z)


def _spread(stat, c):
    return np.repeat(stat, c // stat.shape[1], axis=1)[:, None, None, :]


def group_norm(x, groups, gamma, beta, act, eps):
    """x [N][H][W][C] float64 -> (y, z, h, mean, rstd)"""
    n, hh, w, c = x.shape
    v = x.reshape(n, hh * w, groups, c // groups)
    mean = v.mean(axis=(1, 3))
    var = np.square(v - mean[:, None, :, None]).mean(axis=(1, 3))
    rstd = 1 / np.sqrt(var + eps)
    h = (x - _spread(mean, c)) * _spread(rstd, c)
    z = gamma * h + beta
    return activate(z, act), z, h, mean, rstd


def group_norm_backward(dy, x, mean, rstd, groups, gamma, beta, act):
    """-> (dx, dgamma, dbeta, and the sums of magnitudes that bound their rounding errors)"""
    n, hh, w, c = x.shape
    h = (x - _spread(mean, c)) * _spread(rstd, c)
    e = dy * slope(gamma * h + beta, act)
    per = (n, hh * w, groups, c // groups)
    s1, s2 = (gamma * e).reshape(per).mean(axis=(1, 3)), (gamma * e * h).reshape(per).mean(axis=(1, 3))
    a1, a2 = np.abs(gamma * dy).reshape(per).mean(axis=(1, 3)), np.abs(gamma * dy * h).reshape(per).mean(axis=(1, 3))
    r = _spread(rstd, c)
    dx = r * (gamma * e - _spread(s1, c) - h * _spread(s2, c))
    dx_size = r * (np.abs(gamma * dy) * (1 + np.abs(h)) + _spread(a1, c) + np.abs(h) * _spread(a2, c))
    axes = (0, 1, 2)
    return (dx, (e * h).sum(axis=axes), e.sum(axis=axes), dx_size,
            (np.abs(dy) * np.abs(h) * (1 + np.abs(h))).sum(axis=axes), (np.abs(dy) * (1 + np.abs(h))).sum(axis=axes))


# ---- 4-bit microscaled matrices -----------------------------------------------------------------

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([(m / 512 if e == 0 else (8 + m) * 2.0 ** (e - 10)) for e in range(16) for m in range(8)])
E4M3[127] = np.nan


def nearest(values, x):
    """Index of the nearest of the ascending `values` (index parity = last mantissa bit), ties to
    the even index, past the end the last one."""
    i = np.clip(np.searchsorted(values, x, side="right") - 1, 0, len(values) - 2)
    below, above = x - values[i], values[i + 1] - x
    return np.where((above < below) | ((above == below) & (i % 2 == 1)), i + 1, i)


def mx4_quantize(x, block):
    """x [rows][cols] float64 -> (codes [rows][cols], scale bytes [rows][blocks], values)"""
    rows, cols = x.shape
    blocks = -(-cols // block)
    v = np.zeros((rows, blocks * block))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, block)
    bad = ~np.isfinite(v).all(axis=2)
    a = np.abs(np.where(np.isfinite(v), v, 0)).max(axis=2)
    if block == 32:
        e = np.frexp(a)[1] - 1  # floor(log2)
        byte = np.where(a > 0, np.maximum(e - 2, -127) + 127, 0).astype(np.uint8)
        s = np.exp2(byte.astype(np.float64) - 127)
        byte[bad] = 0xff
    else:
        byte = nearest(E4M3[:127], (a.astype(np.float32) / np.float32(6)).astype(np.float64)).astype(np.uint8)
        s = E4M3[byte]
        byte[bad] = 0x7f
    u = np.where(s[:, :, None] > 0, np.abs(np.where(np.isfinite(v), v, 0)) / np.maximum(s[:, :, None], 1e-300), 0)
    codes = nearest(E2M1, u)
    values = np.copysign(E2M1[codes], v) * s[:, :, None]
    values[bad] = np.nan
    codes = codes + 8 * np.signbit(v)
    flat = lambda t: t.reshape(rows, -1)[:, :cols]
    return flat(codes).astype(np.uint8), byte, flat(values)


def mx4_pack(codes, byte, block):
    """-> (data [rows][pitch], scales) as NtMx4Matrix lays them out"""
    rows, cols = codes.shape
    wide = np.zeros((rows, -(-cols // 32) * 32), np.uint8)
    wide[:, :cols] = codes
    data = wide[:, 0::2] | (wide[:, 1::2] << 4)
    tiles = -(-cols // (4 * block))
    scales = np.zeros(-(-rows // 128) * tiles * 512, np.uint8)
    r, k = np.meshgrid(np.arange(rows), np.arange(byte.shape[1]), indexing="ij")
    scales[((r // 128) * tiles + k // 4) * 512 + 16 * (r % 32) + 4 * (r % 128 // 32) + k % 4] = byte
    return data, scales
