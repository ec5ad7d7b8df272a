"""Microscaled (OCP MX) quantisation, products and the residual + root-mean-square norm in numpy float64.

Elements are found by search in the table of the values that they can have (ties to the even code), scales in the list
of powers of two, so nothing here shares a formula with the kernels.
"""
from __future__ import annotations

import numpy as np

EMAX = {"mxfp4": 2, "mxfp8": 8}
TABLE = {
    "mxfp4": np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6]),
    "mxfp8": np.array([f * 2.0 ** -9 for f in range(8)] +
                      [(8 + f) * 2.0 ** (x - 10) for x in range(1, 16) for f in range(8)][:-1]),
}
POWERS = 2.0 ** np.arange(-127, 128)


def quantize(v, fmt):
    """v [rows, K] float64 -> (codes [rows, Kp] uint8 one element each, scale bytes [rows, Kp // 32]), Kp = K rounded up
    to a multiple of 128, with zeros beyond K."""
    rows, k = v.shape
    kp = -(-k // 128) * 128
    full = np.zeros((rows, kp))
    full[:, :k] = v
    blocks = full.reshape(rows, kp // 32, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(blocks).max(-1)
        fine = np.isfinite(top)
        at = np.searchsorted(POWERS, np.where(fine, top, 1.0), side="right") - 1
        byte = np.maximum(at - EMAX[fmt], 0)
        t = np.where(fine[..., None], blocks / POWERS[byte][..., None], 0.0)
    middle = (TABLE[fmt][1:] + TABLE[fmt][:-1]) / 2
    low, high = np.searchsorted(middle, np.abs(t)), np.searchsorted(middle, np.abs(t), side="right")
    code = np.where(low % 2 == 0, low, high)
    code = code | np.where(np.signbit(t), 8 if fmt == "mxfp4" else 128, 0)
    return code.reshape(rows, kp).astype(np.uint8), np.where(fine, byte, 255).astype(np.uint8)


def values(codes, scales, fmt, k):
    """What codes and scale bytes (as quantize gives them) stand for: [rows, k] float64."""
    sign = 8 if fmt == "mxfp4" else 128
    v = np.where(codes & sign, -1.0, 1.0) * TABLE[fmt][codes & (sign - 1)]
    s = np.where(scales == 255, np.nan, POWERS[np.minimum(scales, 254)])
    return (v * np.repeat(s, 32, axis=1))[:, :k]


def round_trip(v, fmt):
    return values(*quantize(v, fmt), fmt, v.shape[1])


def scale_tiles(scales):
    """Scale bytes [rows, Kp // 32] in the products' layout [ceil(rows / 128), Kp // 128, 32, 4, 4]."""
    rows, nb = scales.shape
    out = np.zeros((-(-rows // 128), nb // 4, 32, 4, 4), np.uint8)
    for r in range(rows):
        out[r // 128, :, r % 32, r % 128 // 32, :] = scales[r].reshape(-1, 4)
    return out


def residual_rmsnorm(h, o, bias, scale, gamma, eps):
    v = h if o is None else h + (o + (0.0 if bias is None else bias)) * (1.0 if scale is None else scale)
    return v, v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * gamma


def act(v, name):
    if name == "gelu":
        from scipy.special import erfc
        return 0.5 * v * erfc(-v / np.sqrt(2.0))
    return np.maximum(v, 0.0) if name == "relu" else v
