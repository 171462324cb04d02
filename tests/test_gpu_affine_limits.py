"""-m gpu: the wide affine layer where its values or its sizes are out of the ordinary: infinities and NaN, launches of more than
2^32 threads, and every tile size against float64 (affine_ref.py derives the bounds)."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

from bullet_amd import lib  # noqa: E402
import affine_ref as ar  # noqa: E402
import test_gpu_affine as tg  # noqa: E402

DT, INF = tg.DT, float("inf")


def forward(kind, act, w, x, y, bias=None, saved=None, residual=None, w32=False):
    (batch, in_), out = x.shape, w.shape[1]
    d = ar.desc(batch, in_, out, kind, act, w32)
    need = tg.L.bt_affine_forward_workspace_bytes(C.byref(d))
    ws = tg.space(need)
    ar.call_forward(tg.stream(), d, w, bias, x, residual, y, saved, ws, need)
    torch.cuda.synchronize()


def backward(kind, act, w, x, out, gy, dw, db, gx):
    (batch, in_), n = (x if x is not None else gx).shape, gy.shape[1]
    d = ar.desc(batch, in_, n, kind, act)
    need = tg.L.bt_affine_backward_workspace_bytes(C.byref(d))
    ws = tg.space(need)
    ar.call_backward(tg.stream(), d, w, x, out, gy, dw, db, gx, ws, need)
    torch.cuda.synchronize()


# ---------------------------------------------------------------- infinities and NaN
@pytest.mark.parametrize("kind", tg.KINDS)
def test_outputs_that_left_the_range_keep_their_slope(kind):
    """ReLU's slope is 1 at an output of infinity, which an f16 sum beyond 65504 becomes, as it is at every other positive one"""
    rng = np.random.default_rng(51)
    for batch, in_, out in ((1, 8, 8), (70, 50, 40), (130, 200, 96)):
        x, x64, _ = tg.place(rng.random((batch, in_)), kind, in_)
        w, w64, _ = tg.place(rng.standard_normal((in_, out)), kind, out)
        gy, g64, _ = tg.place(rng.standard_normal((batch, out)), kind, out)
        o = torch.from_numpy(rng.standard_normal((batch, out)).clip(0)).to(DT[kind]).cuda()
        o[batch // 2, 3], o[0, out - 1] = INF, INF
        dw, db, gx = torch.zeros(in_, out, device="cuda"), torch.zeros(out, device="cuda"), torch.zeros_like(x)
        backward(kind, "relu", w, x, o, gy, dw, db, gx)
        want, tol = ar.backward("relu", kind, w64, x64, o.double().cpu().numpy(), g64)
        ar.check(dw.double().cpu().numpy(), want["dw"], tol["dw"], "f32", "dw")
        ar.check(db.double().cpu().numpy(), want["dbias"], tol["dbias"], "f32", "dbias")
        ar.check(gx.double().cpu().numpy(), want["gx"], tol["gx"], kind, "gx")


def test_an_f16_sum_beyond_the_range_passes_its_gradient_on():
    """forward and backward together: 8 x 100 x 100 = 80000 is stored as infinity, and its unit's gradient goes through"""
    x, w = torch.full((6, 8), 100.0, device="cuda").half(), torch.full((8, 16), 100.0, device="cuda").half()
    w[:, 1::2] = -1.0
    y, gy = torch.zeros(6, 16, device="cuda").half(), torch.ones(6, 16, device="cuda").half()
    forward("f16", "relu", w, x, y)
    assert (y[:, ::2] == INF).all() and (y[:, 1::2] == 0).all()
    dw, db, gx = torch.zeros(8, 16, device="cuda"), torch.zeros(16, device="cuda"), torch.zeros_like(x)
    backward("f16", "relu", w, x, y, gy, dw, db, gx)
    assert (db[::2] == 6).all() and (db[1::2] == 0).all() and (dw[:, ::2] == 600).all() and (dw[:, 1::2] == 0).all()
    assert (gx == 800).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_squared_relu_at_infinity(kind):
    """its derivative, 2 sqrt(out), is infinite there: the unit's column of the gradients is, and no other"""
    o = torch.ones(5, 24, device="cuda", dtype=DT[kind])
    o[2, 7] = INF
    gy, db = torch.full_like(o, 0.5), torch.zeros(24, device="cuda")
    x, dw = torch.ones(5, 16, device="cuda", dtype=DT[kind]), torch.zeros(16, 24, device="cuda")
    backward(kind, "sqrrelu", None, x, o, gy, dw, db, None)
    rest = [c for c in range(24) if c != 7]
    assert db[7] == INF and (dw[:, 7] == INF).all() and (db[rest] == 5).all() and (dw[:, rest] == 5).all()


@pytest.mark.parametrize("act", ["identity", "relu", "crelu", "screlu", "sqrrelu"])
@pytest.mark.parametrize("kind", tg.KINDS)
def test_nan_shows_behind_every_activation(kind, act):
    """a NaN input makes its row of outputs NaN, a NaN weight its column; infinities become what the activation makes of them"""
    for batch, in_, out in ((1, 20, 40), (3, 300, 70), (70, 90, 150), (300, 513, 700)):
        x, w = torch.full((batch, in_), 0.5, device="cuda", dtype=DT[kind]), torch.zeros(in_, out, device="cuda", dtype=DT[kind])
        w[3, 7], w[5, 9], w[5, 10] = float("nan"), INF, -INF
        x[batch // 2, 1] = float("nan") if batch > 1 else 0.5
        y, res = torch.zeros(batch, out, device="cuda", dtype=DT[kind]), torch.zeros(batch, out, device="cuda", dtype=DT[kind])
        saved = torch.zeros_like(y)
        forward(kind, act, w, x, y, saved=saved, residual=res)
        want = torch.zeros(batch, out)
        want[:, 9] = 1.0 if act in ("crelu", "screlu") else INF
        want[:, 10] = -INF if act == "identity" else 0.0
        want[:, 7] = float("nan")
        if batch > 1:
            want[batch // 2] = float("nan")
        for t in (y, saved):
            t = t.float().cpu()
            assert torch.equal(t.isnan(), want.isnan()) and torch.equal(t.nan_to_num(7.0), want.nan_to_num(7.0)), (batch, in_, out)
