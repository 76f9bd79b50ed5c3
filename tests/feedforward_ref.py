"""A feed-forward block's operators in plain numpy, 64 bits: what their tests
compare with.  Values in 8 bits follow include/ts_hip.h (ts_hip_pack8)."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative


def e4m3_values() -> np.ndarray:
    """What the 256 codes stand for (NaN: 0x7f, 0xff)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


def pitch_of(cols: int) -> int:
    return -(-cols // 128) * 128


def pack8(x):
    """(codes [rows, pitch], scales [pitch / 128, rows, 4]) of x, taken as 64 bits."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    pad = np.zeros((rows, pitch_of(cols)))
    pad[:, :cols] = x
    b = pad.reshape(rows, -1, 32)
    top = np.max(np.where(np.isnan(b), 0.0, np.abs(b)), axis=2)
    ks = np.full(top.shape, 119)
    for k in range(118, -118, -1):  # the smallest k that holds the block
        ks = np.where(top <= 448 * 2.0 ** k, k, ks)
    q = b * 2.0 ** -ks[:, :, None].astype(np.float64)
    q = np.clip(q, -448, 448)  # (NaN stays)
    a = np.abs(q)
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.where(np.isnan(a), 1.0, a), 2.0 ** -6))) - 3)
    r = np.minimum(np.rint(a / step) * step, 448.0)
    table = e4m3_values()[:127]
    codes = np.where(np.isnan(r), 127, np.searchsorted(table, np.where(np.isnan(r), 0.0, r)))
    codes = (codes | np.where(np.signbit(q), 128, 0)).astype(np.uint8).reshape(rows, -1)
    scales = (ks + 127).astype(np.uint8).reshape(rows, -1, 4).transpose(1, 0, 2)
    return codes, np.ascontiguousarray(scales)


def unpack8(codes, scales, cols):
    rows = codes.shape[0]
    k = scales.transpose(1, 0, 2).reshape(rows, -1, 1).astype(np.int64) - 127
    v = e4m3_values()[codes].reshape(rows, -1, 32) * 2.0 ** k.astype(np.float64)
    return v.reshape(rows, -1)[:, :cols]


def rms_norm(h, w, eps):
    h = np.asarray(h, np.float64)
    return h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * np.asarray(w, np.float64)


def rms_norm_grads(h, w, go, eps):
    h, w, go = (np.asarray(a, np.float64) for a in (h, w, go))
    r = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    g = go * w
    return r * g - h * r ** 3 * (g * h).mean(1, keepdims=True), (go * h * r).sum(0)


def act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return np.where(z > 0, z, 0.0)
    v = z if name == "silu" else 2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)
    q = np.exp(-np.abs(v))
    return z * np.where(v >= 0, 1 / (1 + q), q / (1 + q))


def act_slope(z, name):
    if name == "none":
        return np.ones_like(z)
    if name == "relu":
        return (z > 0).astype(np.float64)
    c = 2 * np.sqrt(2 / np.pi)
    v, dv = (z, 1.0) if name == "silu" else (c * (z + 0.044715 * z ** 3), c * (1 + 3 * 0.044715 * z ** 2))
    q = np.exp(-np.abs(v))
    s = np.where(v >= 0, 1 / (1 + q), q / (1 + q))
    return s + z * q / (1 + q) ** 2 * dv


def linear(x, w, b, name, res):
    """(y, z)"""
    z = np.asarray(x, np.float64) @ np.asarray(w, np.float64)
    if b is not None:
        z = z + b
    y = act(z, name)
    return (y if res is None else y + res), z


def linear_grads(kept, w, z, name, go):
    """dx, dw, db of a layer whose input is kept as `kept`, at the values z."""
    dz = np.asarray(go, np.float64) * act_slope(z, name)
    return dz @ np.asarray(w, np.float64).T, np.asarray(kept, np.float64).T @ dz, dz.sum(0)


# ---- how far fp32 may be off -----------------------------------------------------
# A product of K terms by either kind of kernel is within (K + 20) U of the sum of
# |a| |b| (fp32 instructions: a rounding a term; bf16 pieces: fewer).  |act'| <=
# 1.13 and |act''| <= 1.2 for both smooth activations; their own evaluation is
# within 16 U of max(|z|, 1) times what they multiply (an exponential, a
# reciprocal and a cubic, a few roundings each).

def product_bound(a, b):
    return (np.asarray(a).shape[1] + 20) * U * (np.abs(np.asarray(a, np.float64)) @ np.abs(np.asarray(b, np.float64)))


def linear_bound(x, w, b, name, res, z):
    e = product_bound(x, w) + U * np.abs(z)
    if name != "none":
        e = 1.13 * e + 16 * U * np.abs(z)
    return e + U * (np.abs(act(z, name)) + (0 if res is None else 2 * np.abs(res))) + 1e-37


def linear_grads_bound(kept, w, b, z, name, go):
    kept, w, go = (np.asarray(a, np.float64) for a in (kept, w, go))
    dz = go * act_slope(z, name)
    e = np.zeros_like(dz)
    if name != "none":
        ez = product_bound(kept, w) + U * np.abs(z)
        e = np.abs(go) * (1.2 * ez + 16 * U * np.maximum(np.abs(z), 1))
    a = np.abs(dz) + e
    n, k = w.shape[1], kept.shape[0]
    dx = (n + 20) * U * (a @ np.abs(w).T) + e @ np.abs(w).T
    dw = (k + 20) * U * (np.abs(kept).T @ a) + np.abs(kept).T @ e
    return dx + 1e-37, dw + 1e-37, (k + 20) * U * a.sum(0) + e.sum(0) + 1e-37


def relu_safe(x, w, b, kept):
    """Where relu's slope cannot turn within the products' rounding."""
    e = product_bound(kept, w)
    z = np.asarray(kept, np.float64) @ np.asarray(w, np.float64) + (0 if b is None else b)
    return np.abs(z) > 4 * e
