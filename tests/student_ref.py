"""A student's operators in plain numpy, 64 bits: what their tests compare with.
Values in 8 bits follow include/ts_hip.h (ts_hip_block8)."""
from __future__ import annotations

import numpy as np

from feedforward_ref import U, act, e4m3_values, pitch_of

LEAST, MOST = 2.0 ** -100, 448 * 2.0 ** 119


def scale_rows(rows, tiles):
    return -(-rows // 128) if tiles else rows


def block8(x, tiles=False):
    """(codes [rows, pitch], scales [pitch / 128, scale rows]) of x, taken as 64 bits."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    high = 128 if tiles else 1
    pad = np.zeros((scale_rows(rows, tiles) * high, pitch_of(cols)))
    pad[:rows, :cols] = x
    b = pad.reshape(pad.shape[0] // high, high, -1, 128)
    top = np.clip(np.max(np.where(np.isnan(b), 0.0, np.abs(b)), axis=(1, 3)), LEAST, MOST)
    scale = (top / 448).astype(np.float32)
    q = np.clip(b * (448 / top)[:, None, :, None], -448, 448)  # (NaN stays)
    a = np.where(np.isnan(q), 1.0, np.abs(q))
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    codes = np.searchsorted(e4m3_values()[:127], np.minimum(np.rint(a / step) * step, 448.0))
    codes = np.where(np.isnan(q), 127, codes) | np.where(np.signbit(q), 128, 0)
    return codes.astype(np.uint8).reshape(pad.shape)[:rows], np.ascontiguousarray(scale.T)


def unblock8(codes, scales, cols, tiles=False):
    """The values, in fp32 as they are given."""
    rows = codes.shape[0]
    by = scales.T[np.arange(rows) // (128 if tiles else 1)]
    v = e4m3_values()[codes].astype(np.float32).reshape(rows, -1, 128) * by[:, :, None]
    return v.reshape(rows, -1)[:, :cols]


def block8_values(codes, scales, cols, tiles=False):
    """The values in 64 bits."""
    rows = codes.shape[0]
    by = scales.T[np.arange(rows) // (128 if tiles else 1)].astype(np.float64)
    return (e4m3_values()[codes].reshape(rows, -1, 128) * by[:, :, None]).reshape(rows, -1)[:, :cols]


def linear(x, w, b, name, res):
    """(y, bound) of values in 64 bits, w [fan_out, fan_in].  The products of the codes are exact; their sums
    of K terms and those of the blocks within (K + 20) U of the sum of |x| |w| (feedforward_ref.product_bound),
    the product of two scales and its multiplication 2 U more."""
    z = x @ w.T + (0 if b is None else b)
    e = (x.shape[1] + 22) * U * (np.abs(x) @ np.abs(w).T) + U * np.abs(z)
    if name != "none":
        e = 1.13 * e + 16 * U * np.abs(z)
    y = act(z, name)
    e = e + U * np.abs(y)
    if res is not None:
        y = y + res
        e = e + U * np.abs(y)
    return y, e + 1e-37


# ---- layer norm ---------------------------------------------------------------------


def _parts(h, eps):
    h = np.asarray(h, np.float64)
    m = h.mean(1, keepdims=True)
    d = h - m
    m = m + d.mean(1, keepdims=True)  # the mean of far rows once more
    d = h - m
    r = 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    return m, r, d * r


def layer_norm(h, w, b, eps):
    return _parts(h, eps)[2] * np.asarray(w, np.float64) + (0 if b is None else np.asarray(b, np.float64))


def layer_norm_bound(h, w, b, eps):
    """u takes a rounding in each of its two differences, in r and in the last product, and m's second part is off by U^2 of m; y a
    rounding more."""
    m, r, u = _parts(h, eps)
    return (5 * U * np.abs(u) + U * U * np.abs(m) * r) * np.abs(w) + U * np.abs(layer_norm(h, w, b, eps)) + 1e-40


def layer_norm_grads(h, w, go, eps):
    """dh, dweight, dbias"""
    _, r, u = _parts(h, eps)
    go = np.asarray(go, np.float64)
    g = go * np.asarray(w, np.float64)
    return r * (g - g.mean(1, keepdims=True) - u * (g * u).mean(1, keepdims=True)), (go * u).sum(0), go.sum(0)


def layer_norm_grads_bound(h, w, go, eps):
    """dh = r (g - mean g - u mean(g u)): a rounding of g, of mean g, of each difference and of the product, u's
    own 4 and mean(g u)'s one, and r's two: under 9 U of the parts' magnitudes together; the f64 sums lose up to
    2^-28 of mean |g| beside them.  Sums over rows: u's 4, a workgroup's part and the result a rounding each."""
    m, r, u = _parts(h, eps)
    go = np.asarray(go, np.float64)
    g = go * np.asarray(w, np.float64)
    mg, mgu = np.abs(g.mean(1, keepdims=True)), np.abs((g * u).mean(1, keepdims=True))
    far = U * U * np.abs(m) * r
    size = np.abs(g) + mg + (np.abs(u) + far / U) * mgu
    dh = r * (9 * U * size + 2.0 ** -28 * np.abs(u) * np.abs(g).mean(1, keepdims=True))
    return dh + 1e-40, (np.abs(go) * (6 * U * np.abs(u) + far)).sum(0) + 1e-40, 3 * U * np.abs(go).sum(0) + 1e-40


# ---- distillation ---------------------------------------------------------------------


def _softmax(z, t):
    """(log p, p) of z / t over the last axis."""
    d = (z - z.max(-1, keepdims=True)) / t
    with np.errstate(divide="ignore"):
        lse = np.log(np.exp(d).sum(-1, keepdims=True))
    return d - lse, np.exp(d - lse)


def distillation(z, idx, teacher, t=1.0, labels=None, hard=0.0, weights=None):
    """(loss, dz, the bound of the loss, the bound of dz), row by row.

    An exponential 2^(c d) takes a rounding of d, of c and of their product, each U |c d| ln 2 of it, and the
    instruction's own 2 U: eps = (2.2 |c d| + 3) U = (3.2 |d| / t + 3) U.  A softmax's sum is off by the mean of
    its terms' eps and up to 70 U of fp32 additions in a lane (64 values and a few joins), a quotient by both and
    3 roundings.  Terms far below the largest may be flushed: 2^-120 of the coefficient."""
    z, teacher = np.asarray(z, np.float64), np.asarray(teacher, np.float64)
    rows = z.shape[0]
    w = np.full(rows, 1.0 / rows) if weights is None else np.asarray(weights, np.float64)
    dz, bz = np.zeros_like(z), np.zeros_like(z)
    loss = bound = 0.0
    for r in range(rows):
        live = (idx[r] >= 0) & (teacher[r] != -np.inf)
        label = -1 if labels is None or hard == 0 else labels[r]
        ks = idx[r][live]
        soft = (1 - hard) * (1 if ks.size else 0)
        if w[r] == 0 or (soft == 0 and label < 0):
            continue
        row = w[r] * (0.0 if soft == 0 else 1.0)
        d = z[r].max() - z[r]
        if soft:
            logp, p = _softmax(z[r], t)
            logq, q = _softmax(teacher[r][live], t)
            far = (teacher[r][live].max() - teacher[r][live]) / t
            e, ek = (3.2 * d / t + 3) * U, (3.2 * far + 3) * U
            es = (p * np.where(p > 0, e, 0)).sum() + 70 * U
            ea = (q * ek).sum() + 2 * U
            terms = np.where(q > 0, q * (logq - logp[ks]), 0.0)
            loss += row * soft * t * t * terms.sum()
            gap = (teacher[r][live] - z[r][ks]) / t
            gap = gap - (q * gap).sum()
            bound += abs(row) * soft * t * t * (es + ea + np.nansum(q * (ek + ea) * np.abs(gap)) + 4 * U * abs(terms.sum()))
            dz[r] += row * soft * t * p
            np.subtract.at(dz[r], ks, row * soft * t * q)
            bz[r] += abs(row) * soft * t * (p * np.where(p > 0, e + es + 4 * U, 0) + 2.0 ** -120)
            np.add.at(bz[r], ks, abs(row) * soft * t * q * (ek + ea + (4 + ks.size) * U))
        if label >= 0:
            logs, s = _softmax(z[r], 1.0)
            e = (3.2 * d + 3) * U
            es = (s * np.where(s > 0, e, 0)).sum() + 70 * U
            loss -= w[r] * hard * logs[label]
            bound += abs(w[r]) * hard * (es + 4 * U * abs(logs[label]))
            dz[r] += w[r] * hard * s
            dz[r][label] -= w[r] * hard
            bz[r] += abs(w[r]) * hard * (s * np.where(s > 0, e + es + 4 * U, 0) + 2.0 ** -120)
            bz[r][label] += abs(w[r]) * hard * 4 * U
    return loss, dz, bound + 2 * U * abs(loss) + 1e-37, bz + 2 * U * np.abs(dz) + 1e-37
