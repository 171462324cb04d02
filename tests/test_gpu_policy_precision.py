"""-m gpu: how many digits the policy and preference losses keep, and what they make of infinite values: cases whose right answer
is known beyond the bounds that policy_ref.py allows for rows in general."""
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
INF = float("inf")


def stream():
    return torch.cuda.current_stream().cuda_stream


def dev(a, dtype=np.float32):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a).astype(dtype))).cuda()


def policy(z, actions, old, adv, kl="none", ref=None, mask=None, klw=0.05):
    """z: the logits on the device -> loss, grad, row_loss, row_logp, row_kl in float64"""
    n, width = z.shape
    kind = {v: k for k, v in DT.items()}[z.dtype]
    loss, grad = torch.full((1,), float("nan"), device="cuda"), torch.full_like(z, 9.0)
    rows = [torch.full((n,), float("nan"), device="cuda") for _ in range(3)]
    # (named: the call only queues work, and what it reads has to outlive it)
    at, ot, vt, mt = dev(actions, np.int32), dev(old), dev(adv), None if mask is None else dev(mask, np.uint8)
    pr.call_policy(stream(), pr.policy_desc(n, width, kind, kl=kl, klw=klw), z, mt, at, ot, vt, ref, None, loss, grad, *rows)
    torch.cuda.synchronize()
    return [t.double().cpu().numpy() for t in (loss, grad, *rows)]


def preference(z, actions, offsets, ref, beta=0.1, smoothing=0.05):
    """-> loss, grad, pair_loss, line_logp in float64"""
    n, width = z.shape
    kind = {v: k for k, v in DT.items()}[z.dtype]
    pairs = len(ref) // 2
    d = pr.preference_desc(pairs, n, width, kind, beta=beta, smoothing=smoothing)
    ws = torch.full((lib.load().bt_preference_loss_workspace_bytes(C.byref(d)),), 0xFF, dtype=torch.uint8, device="cuda")
    out = [torch.full((1,), float("nan"), device="cuda"), torch.full_like(z, 9.0), torch.full((pairs,), float("nan"), device="cuda"),
           torch.full((2 * pairs,), float("nan"), device="cuda")]
    at, ot, rt = dev(actions, np.int32), dev(offsets, np.int32), dev(ref)
    pr.call_preference(stream(), d, z, None, at, ot, rt, None, *out, ws)
    torch.cuda.synchronize()
    return [t.double().cpu().numpy() for t in out]


# ---------------------------------------------------------------- sums of long rows
def repeated(kind, width):
    """rows of one logit each below 512 logits of 0 at their front, one in every chunk that a lane reads first: from then on every
    term of a lane's sum is the same number -> logits on the device, the log-probability of move 4"""
    v = np.concatenate([np.arange(1, 49) / 8.0, np.array([0.15625, 5.09375, 3.65625, 5.40625])])
    z = torch.empty(len(v), width, dtype=DT[kind], device="cuda")
    z[:] = dev(-v).to(DT[kind])[:, None]
    z[:, :2048:4] = 0.0
    kept = z[:, 1].double().cpu().numpy()
    return z, -np.log(512 + (width - 512) * np.exp(kept))


# bound of a log-probability: as policy_ref.row_error without its share for the width, and one rounding to 32 bits
def logp_bound(lp):
    return 5e-6 + 2.0 ** -24 * np.abs(lp)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("width", [1 << 18, 1 << 20, (1 << 20) + 77])
def test_sums_of_long_rows_of_equal_logits(kind, width):
    z, lp = repeated(kind, width)
    n = len(lp)
    got = policy(z, np.full(n, 4), lp, np.ones(n))[3]
    assert (np.abs(got - lp) <= logp_bound(lp)).all(), np.abs(got - lp).max()
    offsets = np.arange(n + 1)  # a line for every row
    line = preference(z, np.full(n, 4), offsets, lp)[3]
    assert (np.abs(line - lp) <= logp_bound(lp)).all(), np.abs(line - lp).max()


@pytest.mark.parametrize("kl", ["none", "full"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_long_rows_next_to_the_clipping_border(kind, kl):
    """ratios 2e-5 and 4e-5 to either side of a border: the taken move's gradient is 0 on one side and the ratio's on the other"""
    z, lp = repeated(kind, 1 << 20)
    n = len(lp)
    klw = 0.0
    ref = z.clone() if kl == "full" else None
    for high, adv in ((True, 1.0), (False, -1.0)):
        border = 1.0 + np.float64(np.float32(0.28)) if high else 1.0 - np.float64(np.float32(0.2))
        for off in (2e-5, -2e-5, 4e-5, -4e-5):
            old = (lp - np.log(border * (1.0 + off))).astype(np.float32)
            r = np.exp(lp - old.astype(np.float64))  # (a step of old at 14 is 1e-6)
            assert (np.abs(r / border - 1.0 - off) < 2e-6).all()
            grad = policy(z, np.full(n, 4), old, np.full(n, adv), kl=kl, ref=ref, klw=klw)[1][:, 4]
            clipped = (off > 0) == high
            want = 0.0 if clipped else -r * adv * (1.0 - np.exp(lp))
            # (the ratio is off by the sum's 5e-6; the gradient is rounded to the logits' type)
            allow = np.abs(want) * (5e-6 + pr.EPS[kind] * 1.01)
            assert (np.abs(grad - want) <= allow).all(), (high, off, np.flatnonzero(np.abs(grad - want) > allow))


# ---------------------------------------------------------------- exponentials
@pytest.mark.parametrize("width", [7, 300, 1880, 7000, 20001])
def test_small_entries_of_a_gradient_keep_their_digits(width):
    """Beside two logits of 0, moves 0 (taken) and 1, a move of logit x has e^x times move 1's gradient. Move 1's e^0 is exactly 1,
    so the quotient is off by e^x alone and one rounding of the product: argument and correction together less than 2^-25, exp2 1 ulp
    (2^-23), the correction's rounding and the product's 2^-24 each."""
    rng = np.random.default_rng(41)
    x = -75.0 * rng.random((6, width)).astype(np.float32)
    x[:, :2] = 0.0
    z, n = dev(x), len(x)
    want = np.exp(x[:, 1:].astype(np.float64))
    bound = (2.0 ** -25 + 2.0 ** -23 + 2 * 2.0 ** -24) * 1.001
    lp = -np.log(np.exp(x.astype(np.float64)).sum(1))
    grads = dict(policy=policy(z, np.zeros(n), lp, np.ones(n))[1], preference=preference(z, np.zeros(n), np.arange(n + 1), lp)[1])
    for name, g in grads.items():
        off = np.abs(g[:, 1:] / g[:, 1:2] / want - 1.0)
        assert off.max() <= bound, (name, off.max(), x[:, 1:][off > bound][:3])


# ---------------------------------------------------------------- KL of the move taken
def series(x, first):
    """sum over k >= first of x^k / k!, for |x| <= 1, smallest terms first"""
    x, term, terms = np.asarray(x, np.longdouble), np.ones_like(x, np.longdouble), []
    for k in range(1, 30):
        term = term * x / k
        if k >= first:
            terms.append(term)
    return sum(reversed(terms))


def only_move(ref, klw=1.0, adv=None):
    """rows with one legal move: its log-probability is exactly 0 and its ratio 1, so the KL is that of d = ref"""
    n = len(ref)
    z = dev(np.random.default_rng(42).standard_normal((n, 9)))
    mask = np.zeros((n, 9))
    mask[:, 3] = 1
    return policy(z, np.full(n, 3), np.zeros(n), np.zeros(n) if adv is None else adv, kl="taken", ref=dev(ref), mask=mask, klw=klw)


def test_the_kl_estimate_is_never_negative_and_keeps_its_digits():
    """d from 1e-18 to 1 of either sign: KL = exp(d) - d - 1 = d^2 / 2 + ..., off by the output's rounding and 1e-12 (64-bit
    series and, beyond 0.3, differences of 1e-15 next to 0.04)"""
    d = np.float32(np.exp(np.random.default_rng(43).uniform(np.log(1e-18), 0.0, 3000)))
    d = np.concatenate([d, -d, np.float32([0.0, 0.2999999, 0.3, 0.3000001, -0.2999999, -0.3, -0.3000001, 0.34657359, -0.34657359])])
    _, _, row_loss, logp, kl = only_move(d)
    want = series(d, 2).astype(np.float64)
    assert (logp == 0).all() and (kl >= 0).all()
    assert (np.abs(kl - want) <= want * (2.0 ** -24 * 1.0001 + 1e-12) + 2.0 ** -149).all()
    assert (row_loss == kl).all()


@pytest.mark.parametrize("width", [40, 3000, 20001])
def test_a_move_that_has_become_impossible(width):
    """the move taken stands at -infinity among legal moves: l[a] = -infinity, ratio 0, KL = infinity and with it the loss, which a
    weight of 0 leaves out"""
    z = torch.zeros(2, width, device="cuda")
    z[0, 3] = -INF
    args = (z, np.full(2, 3), np.full(2, -np.log(width)), np.ones(2))
    loss, grad, row_loss, logp, kl = policy(*args, kl="taken", ref=dev([-1.0, -np.log(width)]))
    assert logp[0] == -INF and kl[0] == INF and row_loss[0] == INF and loss[0] == INF
    assert grad[0, 3] == -INF and (np.delete(grad[0], 3) == INF).all() and np.isfinite(grad[1]).all() and np.isfinite(row_loss[1])
    loss, grad, row_loss, logp, kl = policy(*args, kl="taken", ref=dev([-1.0, -np.log(width)]), klw=0.0)
    plain = policy(*args)
    assert kl[0] == INF and row_loss[0] == 0.0 and np.isfinite(loss).all() and np.isfinite(grad).all()
    assert np.array_equal(grad, plain[1]) and np.array_equal(row_loss, plain[2])


@pytest.mark.parametrize("width", [40, 3000, 20001])
def test_a_reference_policy_without_a_move_that_has_a_share(width):
    z = torch.zeros(2, width, device="cuda")
    ref = z.clone()
    ref[0, 7] = -INF
    args = (z, np.full(2, 3), np.full(2, -np.log(width)), np.ones(2))
    loss, _, row_loss, _, kl = policy(*args, kl="full", ref=ref)
    assert kl[0] == INF and row_loss[0] == INF and loss[0] == INF and np.isfinite(kl[1])
    loss, grad, row_loss, _, kl = policy(*args, kl="full", ref=ref, klw=0.0)
    plain = policy(*args)
    assert kl[0] == INF and np.array_equal(loss, plain[0]) and np.array_equal(grad, plain[1]) and np.array_equal(row_loss, plain[2])


# ---------------------------------------------------------------- what a row's gradient is scaled by
@pytest.mark.parametrize("width", [3, 7, 100, 1879, 5001, 20001])
def test_gradients_of_equal_logits_are_rounded_once(width):
    """p = 1 / width and every exponential is exactly 1, so that a gradient is a 64-bit scalar rounded to 32 bits"""
    n = 200
    rng = np.random.default_rng(44)
    z, actions = torch.zeros(n, width, device="cuda"), np.zeros(n)
    lp = -np.log(np.float64(width))
    old = np.float32(lp + 0.1 * rng.standard_normal(n))
    adv = rng.standard_normal(n).astype(np.float32)
    r, bound = np.exp(lp - old.astype(np.float64)), 2.0 ** -24 * 1.0001 + 1e-12
    free = (r * adv <= np.clip(r, 1 - np.float64(np.float32(0.2)), 1 + np.float64(np.float32(0.28))) * adv)
    want = np.where(free, r * adv / width, 0.0)[:, None]
    g = policy(z, actions, old, adv)[1][:, 1:]
    assert (np.abs(g - want) <= np.abs(want) * bound).all(), np.abs(g / want - 1).max()

    ref = np.float32(2.0 * rng.standard_normal(n))
    beta, eps = np.float64(np.float32(0.1)), np.float64(np.float32(0.05))
    d = beta * (ref[1::2].astype(np.float64) - ref[0::2])
    c = beta * (eps - 1.0 / (1.0 + np.exp(d)))
    want = (np.stack([-c, c], 1).reshape(-1) / width)[:, None]
    g = preference(z, actions, np.arange(n + 1), ref)[1][:, 1:]
    assert (np.abs(g - want) <= np.abs(want) * bound).all(), np.abs(g / want - 1).max()


# ---------------------------------------------------------------- infinite margins
@pytest.mark.parametrize("smoothing", [0.0, 0.05])
@pytest.mark.parametrize("line", [0, 1])
def test_a_line_with_an_impossible_move(line, smoothing):
    """one line's move stands at -infinity: the margin is infinite. The loss is 0 where the preferred line wins for sure, infinite
    where the other one does, and with smoothing infinite either way; no gradient is NaN, nor is anything of the other pair"""
    z = torch.zeros(4, 30, device="cuda")
    z[line, 5] = -INF
    loss, grad, pair, lp = preference(z, np.full(4, 5), np.arange(5), np.zeros(4), smoothing=smoothing)
    assert lp[line] == -INF and np.isfinite(np.delete(lp, line)).all()
    assert pair[0] == (0.0 if line == 1 and smoothing == 0.0 else INF)
    log2 = np.log(2.0)
    assert abs(pair[1] - log2) <= log2 * (2.0 ** -24 * 1.0001 + 1e-12) and loss[0] == pair.sum().astype(np.float32)
    beta, eps = np.float64(np.float32(0.1)), np.float64(np.float32(smoothing))
    c = beta * (eps - (1.0 if line == 0 else 0.0))  # the slope at its limits
    row = [c, -c][line]
    want = np.full(30, -row / 29)  # the row with the impossible move: p = 1 / 29 for the others
    want[5] = row
    assert (np.abs(grad[line] - want) <= np.abs(want) * (2.0 ** -24 * 1.0001 + 1e-12)).all()
    assert np.isfinite(grad).all()
