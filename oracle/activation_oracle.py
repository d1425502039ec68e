"""Numpy FP64 restatement of the 8-bit activation checkpoint operators."""
from __future__ import annotations

import math

import numpy as np

GROUP = 32
RANGES = {"float32": (-126, 121), "bfloat16": (-126, 121), "float16": (-24, 9)}


def checkpoint(x: np.ndarray, dtype: str):
    """(values int8 [rows, ld], exponents uint8 [rows, lde], x_hat float64) of
    x [rows, cols], given in FP64: per 32 columns the smallest e with
    max|x| <= 127 * 2^e, clamped to the range of `dtype`."""
    low, high = RANGES[dtype]
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    padded = np.zeros((rows, groups * GROUP))
    padded[:, :cols] = x
    parts = padded.reshape(rows, groups, GROUP)
    with np.errstate(invalid="ignore"):
        top = np.abs(parts).max(-1)
    good = np.isfinite(parts).all(-1)
    mantissa, power = np.frexp(np.where(good, top, 1.0))
    e = power - 7 + (mantissa > 127 / 128)
    e = np.clip(np.where(top == 0, low, e), low, high)
    scale = np.ldexp(1.0, e)[..., None]
    q = np.clip(np.rint(np.where(good[..., None], parts, 0.0) / scale), -127, 127)
    hat = np.where(good[..., None], q * scale, np.nan).reshape(rows, -1)[:, :cols]
    values = np.zeros((rows, -(-cols // 16) * 16), np.int8)
    width = min(values.shape[1], groups * GROUP)
    values[:, :width] = q.reshape(rows, -1)[:, :width]
    codes = np.full((rows, -(-cols // 128) * 4), 127, np.uint8)
    codes[:, :groups] = np.where(good, e + 127, 255)
    return values, codes, hat


_erfc = np.frompyfunc(math.erfc, 1, 1)


def gelu(x: np.ndarray, approximate: str):
    """(gelu(x), gelu'(x)) in FP64."""
    x = np.asarray(x, np.float64)
    if approximate == "tanh":
        c = math.sqrt(2 / math.pi)
        z = np.clip(x, -40, 40)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return x * (1 + t) / 2, (1 + t) / 2 + z * (1 - t * t) / 2 * c * (1 + 3 * 0.044715 * z * z)
    phi = 0.5 * _erfc(-x / math.sqrt(2)).astype(np.float64)
    return x * phi, phi + x * np.exp(-x * x / 2) / math.sqrt(2 * math.pi)
