"""bt_affine_* without a GPU: refusals happen before anything is launched; the float64 statement's gradients are those of
differences."""
import ctypes as C

import numpy as np
import pytest

import affine_ref as ar
from bullet_amd import lib


def L():
    """the library, loaded by the first call and not while tests are collected: torch's own HIP runtime has to be the
    process's first one where there is a GPU"""
    return lib.load()


A = [256 * (i + 1) for i in range(12)]  # stand for buffers: distinct, aligned, and never used by a call that is refused


def fwd(d, w=A[0], bias=A[1], x=A[2], res=A[3], y=A[4], saved=A[5], ws=A[6], wsb=1 << 40):
    return L().bt_affine_forward(None, C.byref(d) if d is not None else None, w, bias, x, res, y, saved, ws, wsb)


def bwd(d, w=A[0], x=A[1], out=A[2], gy=A[3], dw=A[4], db=A[5], gx=A[6], ws=A[7], wsb=1 << 40):
    return L().bt_affine_backward(None, C.byref(d) if d is not None else None, w, x, out, gy, dw, db, gx, ws, wsb)


SHAPES = [(dict(batch=0), b"0 x 8 -> 6"), (dict(in_=-1), b"4 x -1"), (dict(out=0), b"Mismatched sizes"),
          (dict(type=3), b"element type 3"), (dict(type=1, w_type=2), b"weights of type 2"), (dict(type=0, w_type=1), b"weights of type 1"),
          (dict(act=9), b"activation 9"), (dict(act=-1), b"activation"), (dict(w_ld=5), b"leading dimension"),
          (dict(x_ld=7), b"leading dimension"), (dict(y_ld=5), b"leading dimension"), (dict(batch=(1 << 30) + 1), b"too large")]


@pytest.mark.parametrize("change,message", SHAPES)
def test_shapes_are_refused(change, message):
    d = ar.desc(4, 8, 6, "f32")
    for k, v in change.items():
        setattr(d, k, v)
    for call in (fwd, bwd):
        assert call(d) == 1 and message in L().bt_last_error(), L().bt_last_error()
    assert L().bt_affine_forward_workspace_bytes(C.byref(d)) == 0 and message in L().bt_last_error()
    assert L().bt_affine_backward_workspace_bytes(C.byref(d)) == 0 and message in L().bt_last_error()


@pytest.mark.parametrize("batch,in_,out", [(1 << 30, 1, 1 << 20), (1 << 30, 1 << 30, 1), (1, 1 << 30, 1 << 30), (1 << 30,) * 3])
def test_matrices_beyond_any_memory_are_refused(batch, in_, out):
    d = ar.desc(batch, in_, out, "bf16", "relu")
    for size in (L().bt_affine_forward_workspace_bytes, L().bt_affine_backward_workspace_bytes):
        assert size(C.byref(d)) == 0 and b"too large" in L().bt_last_error()
    assert fwd(d) == 1 and bwd(d) == 1 and b"too large" in L().bt_last_error()


@pytest.mark.parametrize("batch,in_,out", [(1 << 30, 64, 64), (64, 1 << 30, 64), (64, 64, 1 << 30), (1 << 18,) * 3])
def test_workspaces_of_the_largest_matrices(batch, in_, out):
    """what is taken has a workspace, of at most the matrices' own bytes and 32 of f32 partial sums of either product"""
    d = ar.desc(batch, in_, out, "f16", "screlu", w32=True)
    mats = batch * in_ + batch * out + in_ * out
    for size in (L().bt_affine_forward_workspace_bytes, L().bt_affine_backward_workspace_bytes):
        assert 0 < size(C.byref(d)) <= 33 * 4 * mats * 2


@pytest.mark.parametrize("args,message", [
    (dict(w=None), b"null pointer"), (dict(x=None), b"null pointer"), (dict(y=None), b"null pointer"),
    (dict(w=258), b"not aligned"), (dict(x=770), b"not aligned"), (dict(y=1281), b"not aligned"), (dict(res=1025), b"not aligned"),
    (dict(saved=1537), b"not aligned"), (dict(bias=514), b"not aligned"), (dict(saved=A[4]), b"overlap"),
    (dict(saved=A[3]), b"overlap"), (dict(y=A[2]), b"overlap"),
])
def test_forward_refuses(args, message):
    assert fwd(ar.desc(4, 8, 6, "f32"), **args) == 1 and message in L().bt_last_error(), L().bt_last_error()


@pytest.mark.parametrize("args,message", [
    (dict(gy=None), b"null pointer"), (dict(x=None), b"null pointer"), (dict(w=None), b"null pointer"),
    (dict(out=None), b"null pointer"), (dict(dw=None, db=None, gx=None), b"null pointer"), (dict(ws=None), b"workspace too small"),
    (dict(wsb=1), b"workspace too small"), (dict(ws=A[7] + 8), b"workspace is not aligned"), (dict(x=514), b"not aligned"),
    (dict(dw=1282), b"not aligned"), (dict(gx=A[3]), b"overlaps"), (dict(gx=A[1]), b"overlaps"), (dict(dw=A[0]), b"overlaps"),
])
def test_backward_refuses(args, message):
    assert bwd(ar.desc(4, 8, 6, "f32", "relu"), **args) == 1 and message in L().bt_last_error(), L().bt_last_error()


def test_other_refusals():
    assert fwd(None) == 1 and bwd(None) == 1 and b"null pointer" in L().bt_last_error()
    assert bwd(ar.desc(4, 8, 6, "f16", "sqrrelu")) == 1 and b"range of f16" in L().bt_last_error()
    d = ar.desc(64, 256, 96, "bf16", "relu", w32=True)
    need = L().bt_affine_forward_workspace_bytes(C.byref(d))
    assert need >= 256 * 96 * 2
    assert fwd(d, wsb=need - 1) == 1 and b"workspace too small" in L().bt_last_error()
    assert fwd(d, ws=None) == 1 and b"workspace too small" in L().bt_last_error()
    assert fwd(d, ws=A[6] + 4) == 1 and b"workspace is not aligned" in L().bt_last_error()


@pytest.mark.parametrize("kind", ["identity", "relu", "crelu", "screlu", "sqrrelu"])
def test_reference_gradient_is_that_of_differences(kind):
    rng = np.random.default_rng(5)
    w, x, bias = rng.standard_normal((5, 4)), rng.random((6, 5)), 0.3 * rng.standard_normal(4)
    gy = rng.standard_normal((6, 4))
    f = lambda w, b, x: (ar.forward(kind, w, b, x, None)[0] * gy).sum()  # noqa: E731
    y = ar.forward(kind, w, bias, x, None)[0]
    got = ar.backward(kind, "f32", w, x, y, gy)[0]
    h = 1e-6
    for name, arr, args in (("dw", w, lambda v: (v, bias, x)), ("dbias", bias, lambda v: (w, v, x)), ("gx", x, lambda v: (w, bias, v))):
        for at in np.ndindex(arr.shape):
            up, down = arr.copy(), arr.copy()
            up[at] += h
            down[at] -= h
            assert abs((f(*args(up)) - f(*args(down))) / (2 * h) - got[name][at]) < 1e-6, (name, at)
