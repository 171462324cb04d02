"""The policy and preference losses from their formulas, in float64 on the CPU, with the bounds that the kernels' 32-bit
row sums allow; and the calls, on torch-owned device memory.

Bounds. A row's sum of exponentials is taken in 32 bits: every term is off by at most 2^-21 of itself (argument, exp2 and
correction), and a lane adds at most 64 terms before a tree of at most 10 levels (74 roundings of 2^-24), so the sum, and
with it p, is off by less than S = 5e-6 of itself and l by less than S in absolute terms (rows of up to 2^14 elements; the
running sums of wider rows add width/2048 rescalings and additions of 8 terms a lane: S grows by width / 256 * 2^-24).
"""
import ctypes as C

import numpy as np

from bullet_amd import lib

EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -24}          # below the smallest step of each type
NAMES = {0: "f32", 1: "bf16", 2: "f16"}


def row_error(width):
    return 5e-6 + max(0, width - 2 ** 14) / 256 * 2.0 ** -24


def softmax_rows(z, mask, actions):
    """logs, p (0 where masked), counted; z float64 [n][width]"""
    legal = np.ones(z.shape, bool) if mask is None else mask != 0
    x = np.where(legal, z, -np.inf)
    n, width = z.shape
    ok = (actions >= 0) & (actions < width)
    at = np.where(ok, actions, 0)
    ok &= legal[np.arange(n), at]
    top = x.max(1)
    ok &= top > -np.inf
    base = np.where(np.isfinite(top), top, 0.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        x = x - base[:, None]  # (first: next to a logit of 1e38 the log of the sum would be lost, in 64 bits too)
        logs = x - np.log(np.exp(x).sum(1))[:, None]
        p = np.exp(logs)
    return logs, np.where(legal, p, 0.0), ok, at


def policy(z, mask, actions, old, adv, ref, weights, kl, low, high, klw):
    """-> dict of float64 results and of their bounds (without the output types' own rounding)"""
    n, width = z.shape
    S = row_error(width)
    logs, p, ok, at = softmax_rows(z, mask, actions)
    rows = np.arange(n)
    w = np.ones(n) if weights is None else weights.astype(np.float64)
    lp = np.where(ok, logs[rows, at], 0.0)
    adv = adv.astype(np.float64)
    lo, hi = 1.0 - np.float64(np.float32(low)), 1.0 + np.float64(np.float32(high))
    klw = np.float64(np.float32(klw))
    r = np.exp(lp - old.astype(np.float64))
    held = np.clip(r, lo, hi)
    free_gain, held_gain = r * adv, held * adv
    gain = np.minimum(free_gain, held_gain)
    slope = np.where(free_gain <= held_gain, -free_gain, 0.0)
    onehot = np.zeros_like(p)
    onehot[rows, at] = 1.0
    k, dk = np.zeros(n), np.zeros(n)
    g_full = np.zeros_like(p)
    bound = np.zeros_like(p)
    if kl == "taken":
        d = ref.astype(np.float64) - lp
        k, dk = np.expm1(d) - d, np.abs(np.expm1(d)) * S * 1.1 + np.exp(np.abs(d)) * S * S
        slope = slope - klw * np.expm1(d)
        bound += (w * klw * np.exp(d) * S * 1.1)[:, None] * (p + onehot)
    elif kl == "full":
        rl, q, _, _ = softmax_rows(ref, mask, np.zeros(n, int))
        with np.errstate(invalid="ignore"):
            diff = np.where(p > 0, logs - rl, 0.0)
        k = (p * diff).sum(1)
        raw = np.where(p > 0, np.abs(np.where(p > 0, z, 0) - np.where(p > 0, ref, 0)), 0.0)
        # cross / sum in 32 bits: each of its terms is off like the sum's, and so is the difference of the log-sums
        dk = 2 * S * ((p * raw).sum(1) + 1.0)
        g_full = klw * p * (diff - k[:, None])
        bound += (w * klw)[:, None] * p * (3 * S * np.abs(diff - k[:, None]) + dk[:, None] + S * 2 + 2.0 ** -22 * (raw + np.abs(k)[:, None]))
    grad = w[:, None] * (slope[:, None] * (onehot - p) + g_full)
    bound += np.abs(w * slope)[:, None] * (p + onehot) * 3 * S
    loss = w * (klw * k - gain)
    dloss = np.abs(w) * (klw * dk + np.abs(free_gain) * 1.1 * S)
    zero = lambda a: np.where(ok if a.ndim == 1 else ok[:, None], a, 0.0)  # noqa: E731
    out = dict(grad=zero(grad), row_loss=zero(loss), row_logp=zero(lp), row_kl=zero(k), loss=np.array([zero(loss).sum()]))
    tol = dict(grad=zero(bound), row_loss=zero(dloss), row_logp=zero(np.full(n, S)), row_kl=zero(dk),
               loss=np.array([zero(dloss).sum() + 2.0 ** -24 * np.abs(zero(loss)).sum()]))
    return out, tol, ok


def preference(z, mask, actions, offsets, ref, weights, beta, smoothing):
    n, width = z.shape
    S = row_error(width)
    logs, p, ok, at = softmax_rows(z, mask, actions)
    rows = np.arange(n)
    lp = np.where(ok, logs[rows, at], 0.0)
    pairs = len(ref) // 2
    w = np.ones(pairs) if weights is None else weights.astype(np.float64)
    beta, eps = np.float64(np.float32(beta)), np.float64(np.float32(smoothing))
    lines = [slice(offsets[k], offsets[k + 1]) for k in range(2 * pairs)]
    s = np.array([lp[x].sum() for x in lines])
    ds = np.array([ok[x].sum() * S for x in lines])
    m = s - ref.astype(np.float64)
    d = beta * (m[0::2] - m[1::2])
    dd = beta * (ds[0::2] + ds[1::2])
    loss = w * ((1 - eps) * np.logaddexp(0, -d) + eps * np.logaddexp(0, d))
    slope = w * beta * (eps - 1.0 / (1.0 + np.exp(d)))
    dslope = w * beta * dd * 0.25 + np.abs(slope) * 2.0 ** -23
    grad, bound = np.zeros_like(p), np.zeros_like(p)
    onehot = np.zeros_like(p)
    onehot[rows, at] = 1.0
    for k, x in enumerate(lines):
        c = slope[k // 2] * (1 if k % 2 == 0 else -1)
        grad[x] = np.where(ok[x, None], c * (onehot[x] - p[x]), 0.0)
        bound[x] = np.where(ok[x, None], (np.abs(c) * 2 * S + dslope[k // 2]) * (p[x] + onehot[x]), 0.0)
    out = dict(loss=np.array([loss.sum()]), pair_loss=loss, line_logp=s, grad=grad)
    tol = dict(loss=np.array([np.abs(w * dd).sum()]), pair_loss=np.abs(w) * dd, line_logp=ds, grad=bound)
    return out, tol


def check(got, want, tol, kind, what):
    """|got - want| <= tol + the rounding of the output's own type"""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    same_inf = np.isinf(want) & (got == want)
    err = np.abs(got - np.where(np.isinf(want), 0.0, want))
    allow = tol + EPS[kind] * np.abs(np.where(np.isinf(want), 0.0, want)) * 1.001 + TINY[kind]
    bad = ~(same_inf | (err <= allow))
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {got[bad][0]!r} for "
                           f"{want[bad][0]!r}, allowed {np.broadcast_to(allow, bad.shape)[bad][0]:.3e}")


def policy_desc(batch, width, kind, ld=None, mask_ld=None, kl="none", low=0.2, high=0.28, klw=0.05):
    return lib.PolicyDesc(batch=batch, width=width, type=lib.TYPE[kind], ld=ld or width, mask_ld=mask_ld or width,
                          kl=lib.KL[kl], clip_low=low, clip_high=high, kl_weight=klw)


def preference_desc(pairs, rows, width, kind, ld=None, mask_ld=None, beta=0.1, smoothing=0.05):
    return lib.PreferenceDesc(pairs=pairs, rows=rows, width=width, type=lib.TYPE[kind], ld=ld or width,
                              mask_ld=mask_ld or width, beta=beta, smoothing=smoothing)


def ptr(t):
    return None if t is None else t.data_ptr()


def call_policy(stream, d, z, mask, actions, old, adv, ref, weights, loss, grad, row_loss, row_logp, row_kl):
    lib.check(lib.load().bt_policy_loss(stream, C.byref(d), ptr(z), ptr(mask), ptr(actions), ptr(old), ptr(adv), ptr(ref),
                                        ptr(weights), ptr(loss), ptr(grad), ptr(row_loss), ptr(row_logp), ptr(row_kl)))


def call_preference(stream, d, z, mask, actions, offsets, ref, weights, loss, grad, pair_loss, line_logp, ws):
    lib.check(lib.load().bt_preference_loss(stream, C.byref(d), ptr(z), ptr(mask), ptr(actions), ptr(offsets), ptr(ref),
                                            ptr(weights), ptr(loss), ptr(grad), ptr(pair_loss), ptr(line_logp), ptr(ws),
                                            ws.numel()))
