"""The wide affine layer from its formulas in float64, with bounds for 32-bit sums; and the calls.

Bounds. A sum of K products in 32 bits, each product exact or rounded once, is off by at most about 6 sqrt(K) 2^-24 of the
sum of the products' magnitudes (roundings of independent sign; six standard deviations of a bound that already takes every
rounding at its largest), and never by less than a few 2^-24 of it (the constant 4 for short sums). A gradient kept as n
16-bit numbers is off by the n-th power of the type's half step: bf16 three times for dw and twice for gx, f16 twice (its
second number lifted by 2^11, which leaves 2^-11 of half its smallest step).
"""
import ctypes as C

import numpy as np

from bullet_amd import lib

U = 2.0 ** -24
EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}          # half the smallest step


def sums(k):
    return (6 * np.sqrt(k) + 4) * U


def act(kind, z):
    if kind == "relu":
        return np.maximum(z, 0)
    if kind == "crelu":
        return np.clip(z, 0, 1)
    if kind == "screlu":
        return np.clip(z, 0, 1) ** 2
    if kind == "sqrrelu":
        return np.maximum(z, 0) ** 2
    return z


def slope(kind, a):
    if kind == "relu":
        return (a > 0) * 1.0
    if kind == "crelu":
        return ((a > 0) & (a < 1)) * 1.0
    if kind == "screlu":
        return ((a > 0) & (a < 1)) * 2.0 * np.sqrt(np.maximum(a, 0))
    if kind == "sqrrelu":
        return (a > 0) * 2.0 * np.sqrt(np.maximum(a, 0))
    return np.ones_like(a)


def forward(kind, w, bias, x, residual):
    """w [in][out], x [batch][in] -> y, saved and their bounds without the outputs' own rounding"""
    z = x @ w + (0 if bias is None else bias)
    dz = sums(x.shape[1] + 1) * (np.abs(x) @ np.abs(w) + (0 if bias is None else np.abs(bias)))
    a = act(kind, z)
    steep = {"screlu": 2.0, "sqrrelu": 2 * np.abs(z) + dz}.get(kind, 1.0)
    da = steep * dz + 2 * U * np.abs(a)
    if residual is None:
        return a, a, da, da
    return a + residual, a, da + 2 * U * np.abs(a + residual), da


def backward(kind, dtype, w, x, out, gy):
    s = slope(kind, out) if out is not None else np.ones_like(gy)
    gz = gy * s
    root = kind in ("screlu", "sqrrelu")
    n_w, n_x = {"f32": (1, 1), "bf16": (3, 2), "f16": (2, 2)}[dtype] if root else (1, 1)
    e_w, e_x = [4 * U + (0.0 if dtype == "f32" else EPS[dtype] ** n) if root else 0.0 for n in (n_w, n_x)]
    tiny = TINY["f16"] / 2048 if dtype == "f16" and root else 0.0
    dw, ax = x.T @ gz, np.abs(x)
    gx, aw = gz @ w.T, np.abs(w)
    g = np.abs(gz)
    ddw = (sums(n_w * x.shape[0]) + e_w) * (ax.T @ g) + 2 * tiny * ax.sum(0)[:, None]
    dgx = (sums(n_x * w.shape[1]) + e_x) * (g @ aw.T) + 2 * tiny * aw.sum(1)[None, :]
    return dict(dw=dw, dbias=gz.sum(0), gx=gx), dict(dw=ddw, dbias=(sums(x.shape[0]) + 4 * U) * g.sum(0), gx=dgx)


def check(got, want, tol, kind, what):
    err = np.abs(np.asarray(got, np.float64) - want)
    allow = tol + EPS[kind] * np.abs(want) * 1.01 + TINY[kind]
    bad = ~(err <= allow)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {np.asarray(got)[bad][0]!r} for "
                           f"{want[bad][0]!r}, allowed {allow[bad][0]:.3e}")


def desc(batch, in_, out, kind, act_="identity", w32=False, w_ld=None, x_ld=None, y_ld=None):
    return lib.AffineDesc(batch=batch, in_=in_, out=out, act=lib.ACT[act_], type=lib.TYPE[kind],
                          w_type=lib.TYPE["f32"] if w32 else lib.TYPE[kind], w_ld=w_ld or out, x_ld=x_ld or in_,
                          y_ld=y_ld or out)


def ptr(t):
    return None if t is None else t.data_ptr()


def call_forward(stream, d, w, bias, x, residual, y, saved, ws, ws_bytes):
    lib.check(lib.load().bt_affine_forward(stream, C.byref(d), ptr(w), ptr(bias), ptr(x), ptr(residual), ptr(y), ptr(saved),
                                           ptr(ws), ws_bytes))


def call_backward(stream, d, w, x, out, gy, dw, dbias, gx, ws, ws_bytes):
    lib.check(lib.load().bt_affine_backward(stream, C.byref(d), ptr(w), ptr(x), ptr(out), ptr(gy), ptr(dw), ptr(dbias), ptr(gx),
                                            ptr(ws), ws_bytes))
