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


# ---------------------------------------------------------------- launches of more than 2^32 threads
def uniform(rows, cols, kind, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(rows, cols, dtype=DT[kind], device="cuda").uniform_(-1.0, 1.0, generator=g)


def compare(got, want, tol, kind, what):
    """as affine_ref.check, on the device"""
    allow = tol + ar.EPS[kind] * want.abs() * 1.01 + ar.TINY[kind]
    bad = int((~((got.double() - want).abs() <= allow)).sum())
    assert bad == 0, (what, bad)


def by_rows(rows, step=1 << 25):
    for a in range(0, rows, step):
        yield slice(a, min(rows, a + step))


@pytest.mark.parametrize("kind,batch,in_,out", [("f32", 1 << 29, 16, 4), ("bf16", 1 << 30, 8, 8), ("bf16", (1 << 30) - 3, 8, 8)])
def test_forward_of_more_rows_than_one_dimension_of_a_launch_has_threads(kind, batch, in_, out):
    x, w = uniform(batch, in_, kind, 1), uniform(in_, out, kind, 2)
    y = torch.full((batch, out), float("nan"), device="cuda", dtype=DT[kind])
    forward(kind, "relu", w, x, y)
    for r in by_rows(batch):
        a = x[r].double()
        compare(y[r], (a @ w.double()).clamp(min=0), ar.sums(in_ + 1) * (a.abs() @ w.double().abs()), kind, r)
    del x, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind,batch,in_,out", [("f32", 1 << 29, 16, 4)])
def test_backward_of_as_many_rows(kind, batch, in_, out):
    x, w, gy = uniform(batch, in_, kind, 1), uniform(in_, out, kind, 2), uniform(batch, out, kind, 3)
    dw, db, gx = torch.zeros(in_, out, device="cuda"), torch.zeros(out, device="cuda"), torch.zeros_like(x)
    backward(kind, "identity", w, x, None, gy, dw, db, gx)
    sums = dict(dw=0.0, adw=0.0, db=0.0, adb=0.0)
    for r in by_rows(batch):
        a, g = x[r].double(), gy[r].double()
        compare(gx[r], g @ w.double().t(), ar.sums(out) * (g.abs() @ w.double().abs().t()), kind, r)
        # (column by column: the library's product of 16 x 2^25 and 2^25 x 4 takes seconds)
        outer = [(a * g[:, o:o + 1]) for o in range(out)]
        for k, v in (("dw", torch.stack([p.sum(0) for p in outer], 1)), ("adw", torch.stack([p.abs_().sum(0) for p in outer], 1)),
                     ("db", g.sum(0)), ("adb", g.abs().sum(0))):
            sums[k] = sums[k] + v
    compare(dw, sums["dw"], ar.sums(batch) * sums["adw"], "f32", "dw")
    compare(db, sums["db"], (ar.sums(batch) + 4 * ar.U) * sums["adb"], "f32", "dbias")
    del x, gy, gx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_one_row_of_more_outputs_than_a_launch_has_workgroups_for(kind):
    out = (1 << 29) + 70
    x, w = uniform(1, 1, kind, 1), uniform(1, out, kind, 2)
    y = torch.full((1, out), float("nan"), device="cuda", dtype=DT[kind])
    forward(kind, "identity", w, x, y)
    want = (x.double() * w.double())
    compare(y, want, torch.zeros_like(want), kind, "y")
    db = torch.zeros(out, device="cuda")
    dw = torch.zeros(1, out, device="cuda")
    backward(kind, "identity", w, x, None, y, dw, db, None)
    compare(db, y.double()[0], 0.0, "f32", "dbias")
    compare(dw, x.double() * y.double(), 0.0, "f32", "dw")
    db.zero_()
    backward(kind, "identity", None, x, None, y, None, db, None)  # the column sums in a launch of their own
    compare(db, y.double()[0], 0.0, "f32", "dbias alone")
    del w, y, dw, db, want
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- every tile size
def variant(product, shape, kind, act="identity", w32=False, pad=0, direct=True):
    """tile and workgroups that share one (0 for the forward of few rows), as the library chooses them"""
    batch, in_, out = shape
    d = ar.desc(batch, in_, out, kind, act, w32, out + pad, in_ + pad, out + pad)
    tile, splits, both = C.c_int(), C.c_int(), C.c_int()
    lib.check(tg.L.bt_internal_affine_variant(C.byref(d), product, int(direct), C.byref(tile), C.byref(splits), C.byref(both)))
    return tile.value, splits.value


# bf16 and f16 shapes whose forward product takes 256 x 256 tiles: whole, with a ragged last tile in every direction, with
# two, three and many tiles of k, the last one ragged
FORWARD_256 = [(3841, 70, 4090), (3900, 130, 4000), (4096, 64, 4096), (3850, 448, 4003)]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("shape", FORWARD_256)
def test_forward_in_256_tiles(shape, kind):
    assert variant(0, shape, kind) == (256, 1)
    rng = np.random.default_rng(61)
    tg.run_forward(rng, *shape, kind, "screlu", residual=True)
    tg.run_forward(rng, *shape, kind, "identity", bias=False, pad=8)
    tg.run_forward(rng, *shape, kind, "crelu", residual=True, w32=True, pad=1)  # (both operands copied first)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_256_tiles_fall_back_to_128_through_registers(kind):
    """rows on 16 bytes behind a first element that is not"""
    for shape in ((3841, 70, 4088), (3904, 136, 4000)):
        assert variant(0, shape, kind, pad=8) == (256, 1) and variant(0, shape, kind, pad=8, direct=False) == (128, 1)
        tg.run_forward(np.random.default_rng(62), *shape, kind, "relu", residual=True, pad=8, shift=1)


# backward passes with 256 x 256 tiles, in three shares of both gradients or for grad_x alone: one summand of the gradient, two
# or three, and (f16) two in shares of their own
BACKWARD_256 = [((4200, 1000, 4200), "crelu", "bf16", (256, 3), (256, 3)), ((4200, 1000, 4200), "identity", "f16", (256, 3), (256, 3)),
                ((4200, 1000, 4200), "screlu", "bf16", (256, 3), (256, 3)), ((3900, 4000, 300), "relu", "bf16", (64, 1), (256, 1)),
                ((3900, 4000, 300), "screlu", "bf16", (128, 8), (256, 1)), ((3900, 4000, 300), "screlu", "f16", (64, 4), (256, 2))]


@pytest.mark.parametrize("shape,act,kind,dw,dx", BACKWARD_256)
def test_backward_in_256_tiles(shape, act, kind, dw, dx):
    assert variant(1, shape, kind, act) == dw and variant(2, shape, kind, act) == dx
    tg.run_backward(np.random.default_rng(63), *shape, kind, act)
