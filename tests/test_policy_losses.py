"""bt_policy_loss / bt_preference_loss without a GPU: every refusal happens before anything is launched, and the float64
statement of the losses that the GPU tests compare with has the gradients that differences of its own losses have."""
import ctypes as C

import numpy as np
import pytest

import policy_ref as pr
from bullet_amd import lib


def L():
    """the library, loaded by the first call and not while tests are collected: torch's own HIP runtime has to be the
    process's first one where there is a GPU"""
    return lib.load()


P = 64  # stands for a buffer: aligned, never followed by a call that is refused


def policy(d, z=P, mask=P, actions=P, old=P, adv=P, ref=P, w=P, loss=P, grad=P * 2, row_loss=P, logp=P, kl=P):
    return L().bt_policy_loss(None, C.byref(d) if d is not None else None, z, mask, actions, old, adv, ref, w, loss, grad,
                            row_loss, logp, kl)


@pytest.mark.parametrize("change,args,message", [
    (dict(batch=0), {}, b"batch <= 0"), (dict(batch=-4), {}, b"batch <= 0"),
    (dict(width=0), {}, b"width <= 0"), (dict(ld=9), {}, b"leading dimension 9 < width 10"),
    (dict(mask_ld=9), {}, b"mask leading dimension 9"), (dict(type=3), {}, b"element type 3"), (dict(type=-1), {}, b"element type"),
    (dict(kl=3), {}, b"KL kind 3"), (dict(clip_low=-0.1), {}, b"clipping range"), (dict(clip_low=1.5), {}, b"clipping range"),
    (dict(clip_high=-1.0), {}, b"clipping range"), (dict(clip_high=float("nan")), {}, b"clipping range"),
    (dict(kl_weight=-1.0), {}, b"kl_weight"), (dict(kl_weight=float("inf")), {}, b"kl_weight"),
    ({}, dict(z=None), b"null pointer"), ({}, dict(actions=None), b"null pointer"), ({}, dict(old=None), b"null pointer"),
    ({}, dict(adv=None), b"null pointer"), ({}, dict(loss=None), b"null pointer"), ({}, dict(row_loss=None), b"null pointer"),
    (dict(kl=1), dict(ref=None), b"needs the reference policy"), (dict(kl=2), dict(ref=None), b"needs the reference policy"),
    ({}, dict(z=66), b"not aligned"), ({}, dict(grad=65), b"not aligned"), (dict(type=1), dict(z=65), b"not aligned"),
    (dict(kl=2), dict(ref=62), b"not aligned"), (dict(kl=2), dict(ref=P * 2), b"must not be the reference"),
])
def test_policy_loss_refuses(change, args, message):
    d = pr.policy_desc(4, 10, "f32")
    for k, v in change.items():
        setattr(d, k, v)
    assert policy(d, **args) == 1
    assert message in L().bt_last_error(), L().bt_last_error()


def test_policy_loss_refuses_a_null_descriptor():
    assert policy(None) == 1 and b"null pointer" in L().bt_last_error()


def preference(d, z=P, mask=P, actions=P, offsets=P, ref=P, w=P, loss=P, grad=P, pair_loss=P, line=P, ws=P, wsb=1 << 30):
    return L().bt_preference_loss(None, C.byref(d) if d is not None else None, z, mask, actions, offsets, ref, w, loss, grad,
                                pair_loss, line, ws, wsb)


@pytest.mark.parametrize("change,args,message", [
    (dict(pairs=0), {}, b"pairs = 0"), (dict(pairs=-1), {}, b"pairs = -1"), (dict(pairs=(1 << 29) + 1), {}, b"pairs ="),
    (dict(rows=-1), {}, b"rows < 0"), (dict(width=0), {}, b"width <= 0"), (dict(ld=9), {}, b"leading dimension 9"),
    (dict(mask_ld=1), {}, b"mask leading dimension 1"), (dict(type=7), {}, b"element type 7"),
    (dict(beta=-0.1), {}, b"beta"), (dict(beta=float("nan")), {}, b"beta"), (dict(smoothing=0.5), {}, b"smoothing"),
    (dict(smoothing=-0.1), {}, b"smoothing"), ({}, dict(z=None), b"null pointer"), ({}, dict(actions=None), b"null pointer"),
    ({}, dict(offsets=None), b"null pointer"), ({}, dict(ref=None), b"null pointer"), ({}, dict(loss=None), b"null pointer"),
    ({}, dict(pair_loss=None), b"null pointer"), ({}, dict(ws=None), b"null pointer"), ({}, dict(wsb=100), b"workspace too small"),
    ({}, dict(ws=66), b"not aligned to 4 bytes"), ({}, dict(z=65), b"not aligned"), ({}, dict(grad=66), b"not aligned"),
])
def test_preference_loss_refuses(change, args, message):
    d = pr.preference_desc(4, 30, 10, "f32")
    for k, v in change.items():
        setattr(d, k, v)
    assert preference(d, **args) == 1
    assert message in L().bt_last_error(), L().bt_last_error()


def test_preference_workspace():
    d = pr.preference_desc(4, 30, 10, "f32")
    assert L().bt_preference_loss_workspace_bytes(C.byref(d)) == 6 * 256
    d.ld = 3
    assert L().bt_preference_loss_workspace_bytes(C.byref(d)) == 0 and b"leading dimension 3" in L().bt_last_error()


@pytest.mark.parametrize("kl", ["none", "taken", "full"])
def test_policy_reference_gradient_is_that_of_differences(kl):
    rng = np.random.default_rng(3)
    n, width = 12, 7
    z = rng.standard_normal((n, width))
    mask = (rng.random((n, width)) < 0.7).astype(np.uint8)
    actions = rng.integers(-1, width, n)
    mask[np.arange(n), np.maximum(actions, 0)] = 1
    mask[3] = 0
    logp = pr.softmax_rows(z, mask, actions)[0][np.arange(n), np.maximum(actions, 0)]
    old = np.where(np.isfinite(logp), logp, 0) + 0.3 * rng.standard_normal(n)
    adv, w = rng.standard_normal(n), rng.random(n) + 0.5
    ref = old + 0.2 * rng.standard_normal(n) if kl == "taken" else z + rng.standard_normal((n, width))
    f = lambda zz: pr.policy(zz, mask, actions, old, adv, ref, w, kl, 0.2, 0.3, 0.4)[0]  # noqa: E731
    base = f(z)
    h = 1e-6
    for b in range(n):
        for j in range(width):
            up, down = z.copy(), z.copy()
            up[b, j] += h
            down[b, j] -= h
            slope = (f(up)["loss"][0] - f(down)["loss"][0]) / (2 * h)
            assert abs(slope - base["grad"][b, j]) < 1e-7, (b, j)


def test_preference_reference_gradient_is_that_of_differences():
    rng = np.random.default_rng(4)
    offsets = np.array([0, 2, 5, 5, 9])
    n, width = 9, 6
    z = rng.standard_normal((n, width))
    mask = (rng.random((n, width)) < 0.8).astype(np.uint8)
    actions = rng.integers(-1, width, n)
    mask[np.arange(n), np.maximum(actions, 0)] = 1
    ref, w = -2 * rng.random(4), rng.random(2) + 0.5
    f = lambda zz: pr.preference(zz, mask, actions, offsets, ref, w, 0.7, 0.1)[0]  # noqa: E731
    base = f(z)
    h = 1e-6
    for b in range(n):
        for j in range(width):
            up, down = z.copy(), z.copy()
            up[b, j] += h
            down[b, j] -= h
            slope = (f(up)["loss"][0] - f(down)["loss"][0]) / (2 * h)
            assert abs(slope - base["grad"][b, j]) < 1e-7, (b, j)
