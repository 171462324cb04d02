"""-m gpu: the policy and preference losses against their float64 statement (policy_ref.py derives the bounds)."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

from bullet_amd import lib  # noqa: E402
import policy_ref as pr  # noqa: E402

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def place(a, kind, ld, shift=0, fill=5.0):
    """rows `ld` apart on the device, starting `shift` elements into an allocation -> (view of the buffer, values kept)"""
    n, width = a.shape
    buf = torch.full((n * ld + shift + 8,), fill, dtype=DT[kind], device="cuda")
    rows = buf[shift:shift + n * ld].view(n, ld)
    rows[:, :width] = torch.from_numpy(np.ascontiguousarray(a)).to(DT[kind]).cuda()
    return rows, rows[:, :width].double().cpu().numpy()


def dev(a, dtype=None):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a if dtype is None else a.astype(dtype))).cuda()


def moves(rng, n, width, legal):
    mask = None
    if legal is not None:
        mask = (rng.random((n, width)) < legal).astype(np.uint8) * rng.integers(1, 256, (n, width)).astype(np.uint8)
        mask[np.arange(n), rng.integers(0, width, n)] = 1
    if mask is None:
        actions = rng.integers(0, width, n)
    else:
        actions = np.array([rng.choice(np.flatnonzero(m)) for m in mask])
    return mask, actions.astype(np.int32)


def run_policy(rng, n, width, kind, kl, legal, pad=0, shift=0, weights=True, edges=True, in_place=False, scale=2.0):
    ld, mask_ld = width + pad, width + (3 if pad else 0)
    zt, z = place(scale * rng.standard_normal((n, width)), kind, ld, shift)
    mask, actions = moves(rng, n, width, legal)
    if edges and n >= 6:
        actions[1], actions[2] = -1, width  # padding, out of range
        if mask is not None:
            mask[4] = 0                      # no legal move
            mask[5, actions[5]] = 0          # the action itself is masked
            hole = np.argwhere(mask == 0)
            bad = np.array([np.nan, np.inf, -np.inf])
            for k, (r, c) in enumerate(hole[::3]):
                z[r, c] = bad[k % 3]
            zt[:, :width] = torch.from_numpy(z).to(DT[kind]).cuda()
    logs = pr.softmax_rows(z, mask, actions)[0]
    lp = np.nan_to_num(logs[np.arange(n), np.clip(actions, 0, width - 1)], nan=0.0, posinf=0.0, neginf=0.0)
    old = (lp + 0.3 * rng.standard_normal(n)).astype(np.float32)
    adv = rng.standard_normal(n).astype(np.float32)
    w = (0.5 + rng.random(n)).astype(np.float32) if weights else None
    ref_t = ref = None
    if kl == "taken":
        ref = (lp + 0.3 * rng.standard_normal(n)).astype(np.float32)
        ref_t = dev(ref)
    elif kl == "full":
        ref_t, ref = place(np.nan_to_num(z, nan=0.0, posinf=0.0, neginf=0.0) + rng.standard_normal((n, width)), kind, ld, shift)
    mt = None
    if mask is not None:
        mt = torch.full((n, mask_ld), 1, dtype=torch.uint8, device="cuda")
        mt[:, :width] = dev(mask)
    d = pr.policy_desc(n, width, kind, ld, mask_ld, kl)
    grad = zt if in_place else place(np.full((n, width), 9.0), kind, ld, shift)[0]
    loss = torch.full((1,), float("nan"), device="cuda")
    rows = [torch.full((n,), float("nan"), device="cuda") for _ in range(3)]
    pr.call_policy(stream(), d, zt, mt, dev(actions), dev(old), dev(adv), ref_t, dev(w), loss, grad, *rows)
    torch.cuda.synchronize()
    want, tol, ok = pr.policy(z, mask, actions, old, adv, ref, w, kl, 0.2, 0.28, 0.05)
    got_grad = grad[:, :width].double().cpu().numpy()
    for name, t in zip(("row_loss", "row_logp", "row_kl"), rows):
        pr.check(t.cpu().numpy(), want[name], tol[name], "f32", name)
        assert (t.cpu().numpy()[~ok] == 0).all(), name
    pr.check(loss.cpu().numpy(), want["loss"], tol["loss"], "f32", "loss_sum")
    pr.check(got_grad, want["grad"], tol["grad"], kind, "grad")
    assert (got_grad[~ok] == 0).all()
    if mask is not None:
        assert (got_grad[mask == 0] == 0).all()
    if pad:
        assert (grad[:, width:] == 5.0).all(), "elements between two rows were written"
    return got_grad


# one width per kernel shape (f32 chunks of 4, 16-bit chunks of 8) and its neighbours
WIDTHS = [1, 3, 8, 31, 32, 33, 65, 257, 511, 1027, 1880, 2049, 4097, 8200]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kl", ["none", "taken", "full"])
def test_policy_widths(kind, kl):
    rng = np.random.default_rng(11)
    for width in WIDTHS:
        run_policy(rng, 13, width, kind, kl, 0.3)


@pytest.mark.parametrize("kind,width", [("f32", 8193), ("f32", 20001), ("bf16", 16385), ("f16", 33333)])
@pytest.mark.parametrize("kl", ["taken", "full"])
def test_policy_rows_beyond_the_registers(kind, width, kl):
    rng = np.random.default_rng(12)
    run_policy(rng, 7, width, kind, kl, 0.02)
    run_policy(rng, 7, width, kind, kl, None, pad=5, shift=1)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 255, 1000])
def test_policy_batches(n):
    rng = np.random.default_rng(13)
    run_policy(rng, n, 3, "f32", "full", None)
    run_policy(rng, n, 150, "bf16", "taken", 0.2)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (5, 3), (8, 8)])
def test_policy_strides_and_alignment(kind, pad, shift):
    rng = np.random.default_rng(14)
    for width in (5, 64, 301, 1880, 4100):
        run_policy(rng, 9, width, kind, "full", 0.5, pad=pad, shift=shift)


def test_policy_without_mask_weights_or_row_outputs():
    rng = np.random.default_rng(15)
    run_policy(rng, 20, 100, "f32", "none", None, weights=False)
    n, width = 20, 100
    zt, z = place(rng.standard_normal((n, width)), "f32", width)
    actions, old, adv = rng.integers(0, width, n).astype(np.int32), -4 - rng.random(n), rng.standard_normal(n)
    old, adv = old.astype(np.float32), adv.astype(np.float32)
    loss, row = torch.zeros(1, device="cuda"), torch.zeros(n, device="cuda")
    pr.call_policy(stream(), pr.policy_desc(n, width, "f32"), zt, None, dev(actions), dev(old), dev(adv), None, None, loss,
                   None, row, None, None)
    want, tol, _ = pr.policy(z, None, actions, old, adv, None, None, "none", 0.2, 0.28, 0.05)
    pr.check(loss.cpu().numpy(), want["loss"], tol["loss"], "f32", "loss_sum")
    pr.check(row.cpu().numpy(), want["row_loss"], tol["row_loss"], "f32", "row_loss")


@pytest.mark.parametrize("width", [3, 200, 1880, 4100, 9000])
def test_policy_gradient_in_place_of_the_logits(width):
    a = run_policy(np.random.default_rng(16), 11, width, "f32", "full", 0.4)
    b = run_policy(np.random.default_rng(16), 11, width, "f32", "full", 0.4, in_place=True)
    assert np.array_equal(a, b)


def test_policy_values_at_the_ends_of_the_type():
    """masks made of the type's lowest value, rows of nothing else, infinities among legal moves"""
    low = float(np.finfo(np.float32).min)
    z = np.zeros((6, 40), np.float32)
    z[0, 3:] = low
    z[1, :] = low
    z[2, 5:] = -np.inf
    z[3, :] = -np.inf
    z[4, :] = 3e38
    z[5, ::2] = np.linspace(-200, 200, 20)
    actions = np.array([0, 7, 1, 2, 9, 38], np.int32)
    old, adv = np.full(6, -2.0, np.float32), np.array([1, -1, 1, 1, 1, -1], np.float32)
    rows = [torch.zeros(6, device="cuda") for _ in range(3)]
    loss, zt = torch.zeros(1, device="cuda"), dev(z)
    grad = torch.full_like(zt, 9.0)
    pr.call_policy(stream(), pr.policy_desc(6, 40, "f32", kl="full"), zt, None, dev(actions), dev(old), dev(adv), zt.clone(),
                   None, loss, grad, *rows)
    want, tol, _ = pr.policy(z.astype(np.float64), None, actions, old, adv, z.astype(np.float64), None, "full", 0.2, 0.28, 0.05)
    pr.check(grad.cpu().numpy(), want["grad"], tol["grad"], "f32", "grad")
    for name, t in zip(("row_loss", "row_logp", "row_kl"), rows):
        pr.check(t.cpu().numpy(), want[name], tol[name], "f32", name)


def test_policy_nan_stays_in_its_row():
    z = np.zeros((8, 50), np.float32)
    z[2, 9], z[5, 11] = np.nan, np.inf
    rows = [torch.zeros(8, device="cuda") for _ in range(3)]
    loss, grad = torch.zeros(1, device="cuda"), torch.zeros(8, 50, device="cuda")
    pr.call_policy(stream(), pr.policy_desc(8, 50, "f32"), dev(z), None, dev(np.zeros(8), np.int32),
                   dev(np.full(8, -4.0), np.float32), dev(np.ones(8), np.float32), None, None, loss, grad, *rows)
    bad = np.isnan(rows[0].cpu().numpy())
    assert bad.tolist() == [False, False, True, False, False, True, False, False]
    assert np.isnan(loss.item()) and np.isfinite(grad.cpu().numpy()[~bad]).all()


@pytest.mark.parametrize("width", [5, 50, 4100, 9000])
@pytest.mark.parametrize("kl", ["none", "taken", "full"])
def test_policy_rows_of_nothing_but_nan(kl, width):
    """a head that has diverged: its rows' losses are NaN, not the 0 of a row without moves; masked places keep gradient 0"""
    z = np.full((3, width), np.nan, np.float32)
    mask = np.zeros((3, width), np.uint8)
    mask[:, 1::2] = 1
    z[1] = 0.0
    z[2] = -np.inf
    for m in (None, mask):
        rows = [torch.zeros(3, device="cuda") for _ in range(3)]
        loss, grad = torch.zeros(1, device="cuda"), torch.full((3, width), 9.0, device="cuda")
        ref = None if kl == "none" else dev(np.full(3, -1.0), np.float32) if kl == "taken" else torch.zeros(3, width, device="cuda")
        pr.call_policy(stream(), pr.policy_desc(3, width, "f32", kl=kl), dev(z), dev(m), dev(np.full(3, 3), np.int32),
                       dev(np.full(3, -1.0), np.float32), dev(np.ones(3), np.float32), ref, None, loss, grad, *rows)
        g = grad.cpu().numpy()
        for t in rows[:2]:
            assert np.isnan(t[0].item()) and np.isfinite(t[1].item()) and t[2].item() == 0
        assert np.isnan(loss.item()) and np.isfinite(g[1]).all() and (g[2] == 0).all()
        legal = np.ones(width, bool) if m is None else m[0] != 0
        assert np.isnan(g[0, legal]).all() and (g[0, ~legal] == 0).all()


def test_policy_ratio_next_to_the_clipping_border():
    """ratios within a few 2^-24 of the border: which side they are on decides the whole gradient of the row"""
    rng = np.random.default_rng(17)
    n, width = 400, 300
    zt, z = place(2 * rng.standard_normal((n, width)), "f32", width)
    actions = rng.integers(0, width, n).astype(np.int32)
    lp = pr.softmax_rows(z, None, actions)[0][np.arange(n), actions]
    high = np.arange(n) % 2 == 0
    border = np.where(high, 1.0 + np.float64(np.float32(0.28)), 1.0 - np.float64(np.float32(0.2)))
    old = (lp - np.log(border)).astype(np.float32)
    adv = np.where(high, 1.0, -1.0).astype(np.float32)
    r = np.exp(lp - old.astype(np.float64))
    assert (np.abs(r / border - 1) < 5e-7).all() and (r > border).any() and (r < border).any()
    rows = [torch.zeros(n, device="cuda") for _ in range(3)]
    loss, grad = torch.zeros(1, device="cuda"), torch.zeros(n, width, device="cuda")
    pr.call_policy(stream(), pr.policy_desc(n, width, "f32"), zt, None, dev(actions), dev(old), dev(adv), None, None, loss,
                   grad, *rows)
    want, tol, _ = pr.policy(z, None, actions, old, adv, None, None, "none", 0.2, 0.28, 0.05)
    keep = np.abs(r / border - 1) > 1e-13
    pr.check(grad.cpu().numpy()[keep], want["grad"][keep], tol["grad"][keep], "f32", "grad")


def test_offsets_beyond_32_bits():
    """rows 2^31 - 8 elements apart: the third one starts 8 GB behind the first"""
    ld, width, n = 2 ** 31 - 8, 40, 3
    buf = torch.empty(2 * ld + width, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(18)
    z = torch.from_numpy(rng.standard_normal((n, width))).to(torch.bfloat16)
    for r in range(n):
        buf[r * ld:r * ld + width] = z[r].cuda()
    actions, old, adv = np.array([1, 2, 3], np.int32), np.full(n, -3.5, np.float32), np.ones(n, np.float32)
    loss, row = torch.zeros(1, device="cuda"), torch.zeros(n, device="cuda")
    pr.call_policy(stream(), pr.policy_desc(n, width, "bf16", ld=ld), buf, None, dev(actions), dev(old), dev(adv), None, None,
                   loss, buf, row, None, None)
    want, tol, _ = pr.policy(z.double().numpy(), None, actions, old, adv, None, None, "none", 0.2, 0.28, 0.05)
    got = torch.stack([buf[r * ld:r * ld + width] for r in range(n)]).double().cpu().numpy()
    pr.check(got, want["grad"], tol["grad"], "bf16", "grad")
    del buf
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- preference loss
def run_preference(rng, lens, width, kind, legal, front=0, tail=2, pad=0, shift=0, weights=True, in_place=False, edges=True):
    pairs = len(lens) // 2
    used = front + int(sum(lens))
    n = used + tail
    ld, mask_ld = width + pad, width + (1 if pad else 0)
    zt, z = place(2 * rng.standard_normal((n, width)), kind, ld, shift)
    mask, actions = moves(rng, n, width, legal)
    if edges:
        actions[::7] = -1
        if mask is not None:
            mask[5::11] = 0
    offsets = (front + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32)
    ref = (-3.0 * np.asarray(lens) + 2 * rng.standard_normal(2 * pairs)).astype(np.float32)
    w = (0.5 + rng.random(pairs)).astype(np.float32) if weights else None
    mt = None
    if mask is not None:
        mt = torch.zeros(n, mask_ld, dtype=torch.uint8, device="cuda")
        mt[:, :width] = dev(mask)
    d = pr.preference_desc(pairs, n, width, kind, ld, mask_ld)
    ws = torch.full((lib.load().bt_preference_loss_workspace_bytes(C.byref(d)),), 0xFF, dtype=torch.uint8, device="cuda")
    grad = zt if in_place else place(np.full((n, width), 9.0), kind, ld, shift)[0]
    before = grad.clone()
    loss, pl = torch.full((1,), float("nan"), device="cuda"), torch.full((pairs,), float("nan"), device="cuda")
    ll = torch.full((2 * pairs,), float("nan"), device="cuda")
    pr.call_preference(stream(), d, zt, mt, dev(actions), dev(offsets), dev(ref), dev(w), loss, grad, pl, ll, ws)
    torch.cuda.synchronize()
    want, tol = pr.preference(z, mask, actions, offsets, ref, w, 0.1, 0.05)
    pr.check(ll.cpu().numpy(), want["line_logp"], tol["line_logp"], "f32", "line_logp")
    pr.check(pl.cpu().numpy(), want["pair_loss"], tol["pair_loss"], "f32", "pair_loss")
    pr.check(loss.cpu().numpy(), want["loss"], tol["loss"], "f32", "loss_sum")
    got = grad[:, :width].double().cpu().numpy()
    pr.check(got[front:used], want["grad"][front:used], tol["grad"][front:used], kind, "grad")
    for part in (slice(0, front), slice(used, n)):
        assert torch.equal(grad[part], before[part]), "rows outside every line were written"
    if pad:
        assert torch.equal(grad[:, width:], before[:, width:])
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("width", WIDTHS + [20001])
def test_preference_widths(kind, width):
    run_preference(np.random.default_rng(21), [3, 1, 0, 4, 7, 7], width, kind, 0.4)


@pytest.mark.parametrize("lens", [[1, 1], [0, 0], [0, 5], [200, 1], [65, 64, 63, 0, 0, 0, 1, 130]])
def test_preference_lengths(lens):
    rng = np.random.default_rng(22)
    run_preference(rng, lens, 90, "f32", 0.5, front=3, tail=5)
    run_preference(rng, lens, 300, "bf16", None, tail=0, weights=False)


@pytest.mark.parametrize("pad,shift", [(1, 0), (0, 1), (5, 3), (8, 8)])
def test_preference_strides_and_alignment(pad, shift):
    for kind in ("f32", "bf16"):
        run_preference(np.random.default_rng(23), [4, 6, 3, 2], 517, kind, 0.3, pad=pad, shift=shift)


@pytest.mark.parametrize("width", [3, 500, 4100])
def test_preference_gradient_in_place_of_the_logits(width):
    a = run_preference(np.random.default_rng(24), [4, 6, 3, 2], width, "f32", 0.3, tail=0)
    b = run_preference(np.random.default_rng(24), [4, 6, 3, 2], width, "f32", 0.3, tail=0, in_place=True)
    assert np.array_equal(a, b)


def test_preference_many_pairs():
    rng = np.random.default_rng(25)
    run_preference(rng, list(rng.integers(0, 9, 2 * 301)), 66, "f32", 0.5)


def test_preference_extreme_margins():
    """margins of +-1e4: no overflow, the slope goes to its limits"""
    rng = np.random.default_rng(26)
    z, actions = rng.standard_normal((4, 30)), np.arange(4).astype(np.int32)
    ref = np.array([-1e5, 0.0, 1e5, 0.0], np.float32)
    offsets = np.arange(5).astype(np.int32)
    d = pr.preference_desc(2, 4, 30, "f32")
    ws = torch.zeros(lib.load().bt_preference_loss_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
    zt, loss, pl, ll = dev(z, np.float32), torch.zeros(1, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(4, device="cuda")
    grad = torch.zeros_like(zt)
    pr.call_preference(stream(), d, zt, None, dev(actions), dev(offsets), dev(ref), None, loss, grad, pl, ll, ws)
    want, tol = pr.preference(zt.double().cpu().numpy(), None, actions, offsets, ref, None, 0.1, 0.05)
    for name, t in (("loss", loss), ("pair_loss", pl), ("grad", grad)):
        pr.check(t.cpu().numpy(), want[name], tol[name], "f32", name)


@pytest.mark.parametrize("width", [5, 50, 4100, 20001])
def test_preference_rows_of_nothing_but_nan(width):
    """such a row makes its pair's loss and gradients NaN, and no other's"""
    n, offsets = 5, np.array([0, 1, 2, 3, 5], np.int32)
    z = np.zeros((n, width), np.float32)
    z[1] = np.nan
    z[4] = -np.inf  # a row without a move in the other pair
    mask = np.zeros((n, width), np.uint8)
    mask[:, 1::2] = 1
    d = pr.preference_desc(2, n, width, "f32")
    ws = torch.empty(lib.load().bt_preference_loss_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
    pair, line = torch.zeros(2, device="cuda"), torch.zeros(4, device="cuda")
    loss, grad = torch.zeros(1, device="cuda"), torch.full((n, width), 9.0, device="cuda")
    pr.call_preference(stream(), d, dev(z), dev(mask), dev(np.full(n, 3), np.int32), dev(offsets), torch.zeros(4, device="cuda"),
                       None, loss, grad, pair, line, ws)
    g, legal = grad.cpu().numpy(), mask[0] != 0
    assert np.isnan(pair.cpu().numpy()).tolist() == [True, False] and np.isnan(loss.item())
    assert np.isnan(line.cpu().numpy()).tolist() == [False, True, False, False]
    assert np.isnan(g[:2][:, legal]).all() and (g[:, ~legal] == 0).all()
    assert np.isfinite(g[2:]).all() and (g[4] == 0).all()


def test_preference_offsets_out_of_range_are_clamped():
    rng = np.random.default_rng(27)
    z, actions = rng.standard_normal((6, 30)), np.zeros(6, np.int32)
    d = pr.preference_desc(1, 6, 30, "f32")
    ws = torch.zeros(lib.load().bt_preference_loss_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
    zt = dev(z, np.float32)
    out = []
    for offsets in ([-5, 2, 900], [0, 2, 6]):
        loss, pl, ll = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros(2, device="cuda")
        grad = torch.zeros_like(zt)
        pr.call_preference(stream(), d, zt, None, dev(actions), dev(np.array(offsets), np.int32), dev(np.zeros(2), np.float32),
                           None, loss, grad, pl, ll, ws)
        out.append((loss.item(), grad.cpu().numpy()))
    assert out[0][0] == out[1][0] and np.array_equal(out[0][1], out[1][1])


def test_preference_without_rows_or_gradient():
    """no rows at all: every line is empty; and the losses alone"""
    for rows in (0, 5):
        d = pr.preference_desc(3, rows, 20, "f32")
        ws = torch.zeros(lib.load().bt_preference_loss_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
        z, actions = np.random.default_rng(28).standard_normal((max(rows, 1), 20)), np.zeros(max(rows, 1), np.int32)
        offsets = np.minimum(np.arange(7), rows).astype(np.int32)
        ref = np.linspace(-1, 1, 6).astype(np.float32)
        loss, pl, ll = torch.zeros(1, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(6, device="cuda")
        zt = dev(z, np.float32)
        pr.call_preference(stream(), d, zt, None, dev(actions), dev(offsets), dev(ref), None, loss, zt if rows == 0 else None,
                           pl, ll, ws)
        want, tol = pr.preference(zt.double().cpu().numpy(), None, actions, offsets, ref, None, 0.1, 0.05)
        for name, t in (("loss", loss), ("pair_loss", pl), ("line_logp", ll)):
            pr.check(t.cpu().numpy(), want[name], tol[name], "f32", name)
        assert np.array_equal(zt.cpu().numpy(), z.astype(np.float32))


# ---------------------------------------------------------------- streams and graphs
def test_losses_replayed_from_a_graph_and_on_another_stream():
    rng = np.random.default_rng(31)
    n, width = 37, 700
    zt, _ = place(rng.standard_normal((n, width)), "bf16", width)
    mask, actions = moves(rng, n, width, 0.2)
    mt, at, old, adv = dev(mask), dev(actions), dev(-3 - rng.random(n), np.float32), dev(rng.standard_normal(n), np.float32)
    offsets, ref = dev(np.array([0, 9, 20, 30, 37]), np.int32), dev(-20 * np.ones(4), np.float32)
    d, pd = pr.policy_desc(n, width, "bf16"), pr.preference_desc(2, n, width, "bf16")
    ws = torch.zeros(lib.load().bt_preference_loss_workspace_bytes(C.byref(pd)), dtype=torch.uint8, device="cuda")
    out = dict(loss=torch.zeros(1, device="cuda"), grad=torch.zeros_like(zt), row=torch.zeros(n, device="cuda"),
               loss2=torch.zeros(1, device="cuda"), grad2=torch.zeros_like(zt), pair=torch.zeros(2, device="cuda"))

    def call(s):
        pr.call_policy(s, d, zt, mt, at, old, adv, None, None, out["loss"], out["grad"], out["row"], None, None)
        pr.call_preference(s, pd, zt, mt, at, offsets, ref, None, out["loss2"], out["grad2"], out["pair"], None, ws)

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    call(stream())
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call(stream())
    for step in range(3):
        zt.copy_(torch.from_numpy(rng.standard_normal((n, width))).to(torch.bfloat16))
        call(stream())
        torch.cuda.synchronize()
        want = {k: v.clone() for k, v in out.items()}
        for how in ("replay", "stream"):
            for v in out.values():
                v.fill_(float("nan"))
            torch.cuda.synchronize()
            if how == "replay":
                graph.replay()
            else:
                call(side.cuda_stream)
            torch.cuda.synchronize()
            for k, v in out.items():
                assert torch.equal(v, want[k]), (step, how, k)
