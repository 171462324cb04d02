"""-m gpu: the wide affine layer, forward and backward, against float64 (affine_ref.py derives the bounds)."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

from bullet_amd import lib  # noqa: E402
import affine_ref as ar  # noqa: E402

L = lib.load()
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
KINDS = ["f32", "bf16", "f16"]


def stream():
    return torch.cuda.current_stream().cuda_stream


def place(a, kind, ld, shift=0, fill=5.0):
    """rows `ld` apart, starting `shift` elements into an allocation that ends with the last row"""
    n, width = a.shape
    buf = torch.full((shift + (n - 1) * ld + width,), fill, dtype=DT[kind], device="cuda")
    view = buf[shift:].as_strided((n, width), (ld, 1))
    view.copy_(torch.from_numpy(np.ascontiguousarray(a)).to(DT[kind]))
    return view, view.double().cpu().numpy(), buf


def between(view, buf, shift, ld, fill=5.0):
    """everything in the allocation that is not an element of the matrix"""
    keep = torch.ones(buf.numel(), dtype=torch.bool, device="cuda")
    keep[shift:].as_strided(view.shape, (ld, 1)).fill_(False)
    return buf[keep]


def rounded(w, kind):
    return torch.from_numpy(w).to(DT[kind]).double().numpy()


def space(need):
    return torch.full((max(need, 1),), 0xFF, dtype=torch.uint8, device="cuda")


def make(rng, batch, in_, out, kind, w32, pad, shift):
    x_ld, y_ld, w_ld = in_ + pad, out + pad, out + (pad if pad != 1 else 3)
    x = place(np.clip(0.5 * rng.standard_normal((batch, in_)), 0, 1) + 0.1 * rng.standard_normal((batch, in_)), kind, x_ld, shift)
    w = place(rng.standard_normal((in_, out)) * 1.4 / np.sqrt(in_), "f32" if w32 else kind, w_ld, shift)
    return x, w, rounded(w[1], kind) if w32 else w[1], x_ld, y_ld, w_ld


def run_forward(rng, batch, in_, out, kind, act, residual=False, bias=True, w32=False, pad=0, shift=0, in_place=False):
    x, w, w64, x_ld, y_ld, w_ld = make(rng, batch, in_, out, kind, w32, pad, shift)
    b = (0.3 * rng.standard_normal(out)).astype(np.float32) if bias else None
    res = place(rng.standard_normal((batch, out)), kind, y_ld, shift) if residual else None
    y = res if in_place else place(np.full((batch, out), np.nan), kind, y_ld, shift)
    saved = place(np.full((batch, out), np.nan), kind, y_ld, shift) if residual else None
    d = ar.desc(batch, in_, out, kind, act, w32, w_ld, x_ld, y_ld)
    need = L.bt_affine_forward_workspace_bytes(C.byref(d))
    bt = None if b is None else torch.from_numpy(b).cuda()
    ar.call_forward(stream(), d, w[0], bt, x[0], res[0] if res else None, y[0], saved[0] if saved else None,
                    space(need) if need else None, need)
    torch.cuda.synchronize()
    want, a, tol, ta = ar.forward(act, w64, None if b is None else b.astype(np.float64), x[1], res[1] if res else None)
    what = f"{batch}x{in_}->{out} {kind} {act}"
    ar.check(y[0].double().cpu().numpy(), want, tol, kind, what + " y")
    if saved:
        ar.check(saved[0].double().cpu().numpy(), a, ta, kind, what + " saved")
    for t in (y, saved):
        if t and pad:
            assert (between(t[0], t[2], shift, y_ld) == 5.0).all(), what + ": written between rows"
    return y[0]


def run_backward(rng, batch, in_, out, kind, act, w32=False, pad=0, shift=0, want_dw=True, want_db=True, want_gx=True):
    x, w, w64, x_ld, y_ld, w_ld = make(rng, batch, in_, out, kind, w32, pad, shift)
    o = None
    if act != "identity":
        top = 1.0 if act in ("crelu", "screlu") else 3.0
        o = place(np.clip(rng.standard_normal((batch, out)) * 0.8, 0, top), kind, y_ld, shift)
    gy = place(0.05 * rng.standard_normal((batch, out)), kind, y_ld, shift)
    dw = place(np.full((in_, out), np.nan), "f32", w_ld, shift) if want_dw else None
    db = torch.full((out,), float("nan"), device="cuda") if want_db else None
    gx = place(np.full((batch, in_), np.nan), kind, x_ld, shift) if want_gx else None
    d = ar.desc(batch, in_, out, kind, act, w32, w_ld, x_ld, y_ld)
    need = L.bt_affine_backward_workspace_bytes(C.byref(d))
    ar.call_backward(stream(), d, w[0], x[0], o[0] if o else None, gy[0], dw[0] if dw else None, db, gx[0] if gx else None,
                     space(need), need)
    torch.cuda.synchronize()
    want, tol = ar.backward(act, kind, w64, x[1], o[1] if o else None, gy[1])
    what = f"{batch}x{in_}->{out} {kind} {act} "
    if dw:
        ar.check(dw[0].double().cpu().numpy(), want["dw"], tol["dw"], "f32", what + "dw")
        assert (between(dw[0], dw[2], shift, w_ld) == 5.0).all()
    if want_db:
        ar.check(db.double().cpu().numpy(), want["dbias"], tol["dbias"], "f32", what + "dbias")
    if gx:
        ar.check(gx[0].double().cpu().numpy(), want["gx"], tol["gx"], kind, what + "gx")
        if pad:
            assert (between(gx[0], gx[2], shift, x_ld) == 5.0).all()
    return dw, db, gx


# 1 x 1, less than a fragment, tile edges and their neighbours, long sums that are split, one row and few rows
SHAPES = [(1, 1, 1), (1, 300, 5), (2, 17, 130), (3, 5, 2), (7, 1030, 257), (16, 64, 64), (33, 31, 65), (64, 64, 128), (65, 127, 129),
          (128, 128, 128), (130, 200, 260), (200, 513, 333), (9, 2048, 96), (1, 2048, 1000), (8, 1500, 40), (700, 40, 1100)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_shapes(shape, kind):
    rng = np.random.default_rng(1)
    run_forward(rng, *shape, kind, "relu", residual=True)
    run_forward(rng, *shape, kind, "identity", bias=False, pad=8)
    run_forward(rng, *shape, kind, "screlu", pad=1, shift=1, w32=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward_shapes(shape, kind):
    rng = np.random.default_rng(2)
    run_backward(rng, *shape, kind, "crelu")
    run_backward(rng, *shape, kind, "identity", pad=8)
    run_backward(rng, *shape, kind, "screlu", pad=1, shift=1, w32=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ["identity", "relu", "crelu", "screlu", "sqrrelu"])
def test_activations(act, kind):
    rng = np.random.default_rng(3)
    for residual in (False, True):
        run_forward(rng, 70, 90, 150, kind, act, residual=residual)
    if not (kind == "f16" and act == "sqrrelu"):
        run_backward(rng, 70, 90, 150, kind, act)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(2100, 1100, 2200), (2049, 1000, 2056), (4099, 257, 2050)])
def test_large_tiles(shape, kind):
    """enough tiles for the largest variant, aligned and not, edges in every direction"""
    rng = np.random.default_rng(4)
    run_forward(rng, *shape, kind, "crelu", residual=True)
    run_forward(rng, *shape, kind, "crelu", pad=1, shift=1)
    run_backward(rng, *shape, kind, "screlu")
    run_backward(rng, *shape, kind, "identity", pad=5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,out", [(72, 80), (1160, 1608)])
def test_sums_of_few_tiles(batch, out, kind):
    """as many tiles of k as buffers, one less and a few more, whole and not, with few workgroups (three buffers) and many (two)"""
    tile = 32 if kind == "f32" else 64
    rng = np.random.default_rng(28)
    for tiles in (1, 2, 3, 4, 5, 6, 7):
        for k in (tiles * tile - 8, tiles * tile, tiles * tile + 3):
            run_forward(rng, batch, k, out, kind, "relu")
            if batch < 100:
                run_backward(rng, k, batch, out, kind, "crelu")
                run_backward(rng, batch, out, k, kind, "identity")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1000, 304, 4096), (990, 130, 4001), (2048, 64, 2048), (1030, 448, 4000)])
def test_tiles_that_just_fill_the_chip(shape, kind):
    rng = np.random.default_rng(29)
    run_forward(rng, *shape, kind, "screlu", residual=True)
    run_backward(rng, *shape, kind, "relu")


@pytest.mark.parametrize("kind", KINDS)
def test_parts_of_the_gradient(kind):
    for parts in (dict(want_dw=False), dict(want_db=False), dict(want_gx=False), dict(want_dw=False, want_gx=False),
                  dict(want_db=False, want_gx=False), dict(want_dw=False, want_db=False)):
        for act in ("identity", "screlu"):
            run_backward(np.random.default_rng(5), 130, 70, 100, kind, act, **parts)


def test_y_in_place_of_the_residual():
    for shape in ((50, 60, 70), (3, 900, 50), (2100, 1100, 2200)):
        a = run_forward(np.random.default_rng(6), *shape, "bf16", "relu", residual=True)
        b = run_forward(np.random.default_rng(6), *shape, "bf16", "relu", residual=True, in_place=True)
        assert torch.equal(a, b)


def test_long_sums_and_biases():
    rng = np.random.default_rng(7)
    run_backward(rng, 40000, 24, 40, "bf16", "crelu")
    run_backward(rng, 9001, 130, 9, "f32", "screlu", pad=1)
    run_forward(rng, 33, 20000, 70, "f16", "identity")


def test_results_repeat():
    for kind in ("f32", "bf16"):
        a = run_backward(np.random.default_rng(8), 1000, 300, 200, kind, "screlu")
        b = run_backward(np.random.default_rng(8), 1000, 300, 200, kind, "screlu")
        assert torch.equal(a[0][0], b[0][0]) and torch.equal(a[1], b[1]) and torch.equal(a[2][0], b[2][0])


def test_what_lies_beyond_the_operands_is_not_used():
    """NaN between the rows and behind every operand: k that is no multiple of a tile must not mix it in"""
    rng = np.random.default_rng(9)
    for kind in KINDS:
        for batch, in_, out, pad in ((70, 50, 40, 8), (130, 200, 136, 24), (5, 33, 20, 7)):
            ld = in_ + pad
            x, w = rng.standard_normal((batch, in_)), rng.standard_normal((in_, out)) / 8
            xt, x64, _ = place(x, kind, ld, 0, float("nan"))
            wt, w64, _ = place(w, kind, out + pad, 0, float("nan"))
            gy, g64, _ = place(rng.standard_normal((batch, out)), kind, out + pad, 0, float("nan"))
            d = ar.desc(batch, in_, out, kind, w_ld=out + pad, x_ld=ld, y_ld=out + pad)
            need, need_b = L.bt_affine_forward_workspace_bytes(C.byref(d)), L.bt_affine_backward_workspace_bytes(C.byref(d))
            y = torch.zeros(batch, out + pad, dtype=DT[kind], device="cuda")
            dw, db = torch.zeros(in_, out + pad, device="cuda"), torch.zeros(out, device="cuda")
            gx = torch.zeros(batch, ld, dtype=DT[kind], device="cuda")
            ar.call_forward(stream(), d, wt, None, xt, None, y, None, space(need), need)
            ar.call_backward(stream(), d, wt, xt, None, gy, dw, db, gx, space(need_b), need_b)
            want, _, tol, _ = ar.forward("identity", w64, None, x64, None)
            ar.check(y[:, :out].double().cpu().numpy(), want, tol, kind, "y")
            want, tol = ar.backward("identity", kind, w64, x64, None, g64)
            ar.check(dw[:, :out].double().cpu().numpy(), want["dw"], tol["dw"], "f32", "dw")
            ar.check(gx[:, :in_].double().cpu().numpy(), want["gx"], tol["gx"], kind, "gx")


def test_infinities_stay_in_their_rows_and_columns():
    x, w = torch.ones(130, 70, device="cuda"), torch.ones(70, 140, device="cuda")
    x[3, 5], w[7, 9] = float("inf"), float("nan")
    d = ar.desc(130, 70, 140, "f32")
    need = L.bt_affine_forward_workspace_bytes(C.byref(d))
    y = torch.zeros(130, 140, device="cuda")
    ar.call_forward(stream(), d, w, None, x, None, y, None, space(need), need)
    bad = ~torch.isfinite(y.cpu())
    want = torch.zeros(130, 140, dtype=torch.bool)
    want[3], want[:, 9] = True, True
    assert torch.equal(bad, want)


def test_offsets_beyond_32_bits():
    """x rows and y rows 2^31 - 8 elements apart"""
    ld, batch, in_, out = 2 ** 31 - 8, 3, 40, 24
    rng = np.random.default_rng(10)
    xb = torch.empty(2 * ld + in_, dtype=torch.bfloat16, device="cuda")
    yb = torch.empty(2 * ld + out, dtype=torch.bfloat16, device="cuda")
    x = torch.from_numpy(rng.standard_normal((batch, in_))).to(torch.bfloat16)
    w = torch.from_numpy(rng.standard_normal((in_, out))).to(torch.bfloat16).cuda()
    for r in range(batch):
        xb[r * ld:r * ld + in_] = x[r].cuda()
    d = ar.desc(batch, in_, out, "bf16", x_ld=ld, y_ld=ld)
    need, need_b = L.bt_affine_forward_workspace_bytes(C.byref(d)), L.bt_affine_backward_workspace_bytes(C.byref(d))
    ar.call_forward(stream(), d, w, None, xb, None, yb, None, space(need), need)
    y = torch.stack([yb[r * ld:r * ld + out] for r in range(batch)])
    want, _, tol, _ = ar.forward("identity", w.double().cpu().numpy(), None, x.double().numpy(), None)
    ar.check(y.double().cpu().numpy(), want, tol, "bf16", "y")
    dw, db = torch.zeros(in_, out, device="cuda"), torch.zeros(out, device="cuda")
    gx = torch.empty(2 * ld + in_, dtype=torch.bfloat16, device="cuda")
    ar.call_backward(stream(), d, w, xb, None, yb, dw, db, gx, space(need_b), need_b)
    want, tol = ar.backward("identity", "bf16", w.double().cpu().numpy(), x.double().numpy(), None, y.double().cpu().numpy())
    got = torch.stack([gx[r * ld:r * ld + in_] for r in range(batch)])
    ar.check(got.double().cpu().numpy(), want["gx"], tol["gx"], "bf16", "gx")
    ar.check(dw.double().cpu().numpy(), want["dw"], tol["dw"], "f32", "dw")
    del xb, yb, gx
    torch.cuda.empty_cache()


def test_replayed_from_a_graph_and_on_another_stream():
    rng = np.random.default_rng(11)
    for kind, batch, in_, out in (("bf16", 500, 300, 200), ("f32", 3, 1100, 64), ("f16", 2, 600, 90)):
        d = ar.desc(batch, in_, out, kind, "screlu", w32=True)
        need, need_b = L.bt_affine_forward_workspace_bytes(C.byref(d)), L.bt_affine_backward_workspace_bytes(C.byref(d))
        x = torch.zeros(batch, in_, dtype=DT[kind], device="cuda")
        w = torch.from_numpy(rng.standard_normal((in_, out)) / np.sqrt(in_)).float().cuda()
        gy = torch.from_numpy(rng.standard_normal((batch, out))).to(DT[kind]).cuda()
        ws, wsb = space(need), space(need_b)
        out_t = dict(y=torch.zeros(batch, out, dtype=DT[kind], device="cuda"), dw=torch.zeros(in_, out, device="cuda"),
                     db=torch.zeros(out, device="cuda"), gx=torch.zeros_like(x))

        def call(s):
            ar.call_forward(s, d, w, None, x, None, out_t["y"], None, ws, need)
            ar.call_backward(s, d, w, x, out_t["y"], gy, out_t["dw"], out_t["db"], out_t["gx"], wsb, need_b)

        call(stream())
        torch.cuda.synchronize()
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(stream())
        for step in range(3):
            x.copy_(torch.from_numpy(rng.random((batch, in_))).to(DT[kind]))
            call(stream())
            torch.cuda.synchronize()
            want = {k: v.clone() for k, v in out_t.items()}
            for how in ("replay", "stream"):
                for v in out_t.values():
                    v.fill_(float("nan"))
                torch.cuda.synchronize()
                graph.replay() if how == "replay" else call(side.cuda_stream)
                torch.cuda.synchronize()
                for k, v in out_t.items():
                    assert torch.equal(v, want[k]), (kind, step, how, k)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_on_16_bytes_behind_a_first_element_that_is_not(kind):
    rng = np.random.default_rng(12)
    for batch, in_, out in ((5, 40, 72), (140, 200, 264), (300, 72, 136)):
        run_forward(rng, batch, in_, out, kind, "crelu", residual=True, pad=8, shift=1)
        run_backward(rng, batch, in_, out, kind, "identity", pad=8, shift=1)
        run_backward(rng, batch, in_, out, kind, "screlu", pad=8, shift=3)


@pytest.mark.parametrize("kind", KINDS)
def test_few_rows(kind):
    """one position or a handful: the kernel without matrix cores, every width of its column chunks and tails of k"""
    rng = np.random.default_rng(13)
    for batch in (1, 2, 3, 4, 5, 8):
        for in_, out in ((1, 1), (7, 33), (2048, 64), (2049, 31), (513, 1000)):
            run_forward(rng, batch, in_, out, kind, "screlu", residual=batch % 2 == 0, w32=batch % 3 == 0, pad=batch % 4, shift=batch % 2)
