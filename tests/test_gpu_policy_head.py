"""-m gpu: a policy head trained as a program would do it, through every operator it needs: hidden layer -> residual layer ->
logits -> policy loss -> gradients -> bt_adamw on the f32 weights, and the preference loss on the same logits. Every
operator's outputs are checked in float64 against its formula on the inputs that it really got, so the bounds of
affine_ref / policy_ref apply; the whole chain's f32 gradients are checked against differences of the chain's loss."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

from bullet_amd import lib  # noqa: E402
import affine_ref as ar  # noqa: E402
import policy_ref as pr  # noqa: E402

L = lib.load()
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def f64(t):
    return None if t is None else t.double().cpu().numpy()


class Layer:
    def __init__(self, rng, batch, in_, out, kind, act):
        self.d, self.kind, self.act, self.shape = ar.desc(batch, in_, out, kind, act, w32=True), kind, act, (batch, in_, out)
        self.w = torch.from_numpy((rng.standard_normal((in_, out)) * 1.2 / np.sqrt(in_)).astype(np.float32)).cuda()
        self.b = torch.from_numpy((0.1 * rng.standard_normal(out)).astype(np.float32)).cuda()
        self.dw, self.db = torch.zeros_like(self.w), torch.zeros_like(self.b)
        self.m, self.v = [torch.zeros_like(t) for t in (self.w, self.b)], [torch.zeros_like(t) for t in (self.w, self.b)]
        self.nf, self.nb = L.bt_affine_forward_workspace_bytes(C.byref(self.d)), L.bt_affine_backward_workspace_bytes(C.byref(self.d))
        self.ws = torch.empty(max(self.nf, self.nb, 1), dtype=torch.uint8, device="cuda")

    def rounded(self):
        return f64(self.w.to(DT[self.kind]))

    def forward(self, x, residual=None, check=True):
        batch, in_, out = self.shape
        y = torch.empty(batch, out, dtype=DT[self.kind], device="cuda")
        self.x, self.a = x, y
        saved = None
        if residual is not None:
            self.a = saved = torch.empty_like(y)
        ar.call_forward(stream(), self.d, self.w, self.b, x, residual, y, saved, self.ws, self.nf)
        if check:
            want, a, tol, ta = ar.forward(self.act, self.rounded(), f64(self.b), f64(x), f64(residual))
            ar.check(f64(y), want, tol, self.kind, "y")
            ar.check(f64(self.a), a if saved is not None else want, ta if saved is not None else tol, self.kind, "saved")
        return y

    def backward(self, gy, check=True):
        gx = torch.empty_like(self.x)
        ar.call_backward(stream(), self.d, self.w, self.x, self.a, gy, self.dw, self.db, gx, self.ws, self.nb)
        if check:
            want, tol = ar.backward(self.act, self.kind, self.rounded(), f64(self.x), f64(self.a), f64(gy))
            ar.check(f64(self.dw), want["dw"], tol["dw"], "f32", "dw")
            ar.check(f64(self.db), want["dbias"], tol["dbias"], "f32", "dbias")
            ar.check(f64(gx), want["gx"], tol["gx"], self.kind, "gx")
        return gx


def adamw(layers, adj, lr):
    tensors = [(t, g, m, v) for la in layers for t, g, m, v in zip((la.w, la.b), (la.dw, la.db), la.m, la.v)]
    table = (lib.AdamwTensor * len(tensors))()
    for e, (t, g, m, v) in zip(table, tensors):
        e.grad, e.param, e.momentum, e.velocity, e.n = g.data_ptr(), t.data_ptr(), m.data_ptr(), v.data_ptr(), t.numel()
        e.decay, e.beta1, e.beta2, e.min_weight, e.max_weight = 0.01, 0.9, 0.999, -2.0, 2.0
    lib.check(L.bt_adamw(stream(), len(tensors), table, adj.data_ptr(), lr.data_ptr()))


def data(rng, batch, width):
    mask = (rng.random((batch, width)) < 0.2).astype(np.uint8)
    actions = rng.integers(0, width, batch).astype(np.int32)
    mask[np.arange(batch), actions] = 1
    actions[3], mask[5] = -1, 0
    return mask, actions


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_steps_of_a_policy_head(kind):
    rng = np.random.default_rng(41)
    batch, in_, hid, width = 203, 130, 96, 333
    l1, l2, l3 = Layer(rng, batch, in_, hid, kind, "screlu"), Layer(rng, batch, hid, hid, kind, "relu"), Layer(rng, batch, hid, width, kind, "identity")
    x = torch.from_numpy(np.clip(rng.standard_normal((batch, in_)), 0, 1)).to(DT[kind]).cuda()
    mask, actions = data(rng, batch, width)
    old, adv = (-4 - 0.3 * rng.random(batch)).astype(np.float32), rng.standard_normal(batch).astype(np.float32)
    ref = torch.from_numpy(rng.standard_normal((batch, width))).to(DT[kind]).cuda()
    mt, at, ot, vt = [torch.from_numpy(a).cuda() for a in (mask, actions, old, adv)]
    d = pr.policy_desc(batch, width, kind, kl="full")
    offsets = np.array([0, 40, 90, 150, 200], np.int32)
    line_ref = (-4.0 * np.diff(offsets)).astype(np.float32)
    pd = pr.preference_desc(2, batch, width, kind)
    offs, lr_t = torch.from_numpy(offsets).cuda(), torch.from_numpy(line_ref).cuda()
    ws = torch.empty(L.bt_preference_loss_workspace_bytes(C.byref(pd)), dtype=torch.uint8, device="cuda")
    loss, rows = torch.zeros(1, device="cuda"), [torch.zeros(batch, device="cuda") for _ in range(3)]
    pair, line = torch.zeros(2, device="cuda"), torch.zeros(4, device="cuda")
    adj, lr = torch.tensor([1.0 / batch], device="cuda"), torch.tensor([1e-3], device="cuda")
    for step in range(3):
        h1 = l1.forward(x)
        h2 = l2.forward(h1, residual=h1)
        z = l3.forward(h2)
        grad = torch.empty_like(z)
        before = l3.w.clone()
        if step % 2 == 0:
            pr.call_policy(stream(), d, z, mt, at, ot, vt, ref, None, loss, grad, *rows)
            want, tol, _ = pr.policy(f64(z), mask, actions, old, adv, f64(ref), None, "full", 0.2, 0.28, 0.05)
            pr.check(rows[0].cpu().numpy(), want["row_loss"], tol["row_loss"], "f32", "row_loss")
        else:
            grad.zero_()  # (rows behind the last line are left alone)
            pr.call_preference(stream(), pd, z, mt, at, offs, lr_t, None, loss, grad, pair, line, ws)
            want, tol = pr.preference(f64(z), mask, actions, offsets, line_ref, None, 0.1, 0.05)
            pr.check(pair.cpu().numpy(), want["pair_loss"], tol["pair_loss"], "f32", "pair_loss")
        pr.check(loss.cpu().numpy(), want["loss"], tol["loss"], "f32", "loss_sum")
        pr.check(f64(grad), want["grad"], tol["grad"], kind, "grad")
        g2 = l3.backward(grad)
        g1 = l2.backward(g2)
        l1.backward((g1 + g2).contiguous())  # the residual hands its gradient on unchanged
        adamw([l1, l2, l3], adj, lr)
        torch.cuda.synchronize()
        assert torch.isfinite(l1.w).all() and not torch.equal(before, l3.w)


def test_gradient_of_the_chain_is_that_of_differences():
    """f32, loss differences over a direction in each weight matrix: h = 1e-2 keeps the loss's rounding (2^-22 of about
    batch * 4) below 1e-2 of the slope's size while the third-order term, h^2 / 6, stays below 1e-4 of smooth activations"""
    rng = np.random.default_rng(42)
    batch, in_, hid, width = 64, 40, 48, 60
    l1, l2 = Layer(rng, batch, in_, hid, "f32", "identity"), Layer(rng, batch, hid, width, "f32", "identity")
    x = torch.from_numpy(rng.standard_normal((batch, in_))).float().cuda()
    mask, actions = data(rng, batch, width)
    old = np.zeros(batch, np.float32)  # ratios far below the range: the clipped branch is never the smaller one for adv > 0
    adv = (1 + rng.random(batch)).astype(np.float32) * 40
    mt, at, ot, vt = [torch.from_numpy(a).cuda() for a in (mask, actions, old, adv)]
    d = pr.policy_desc(batch, width, "f32")
    row = torch.zeros(batch, device="cuda")

    def loss_of(grad=None):
        z = l2.forward(l1.forward(x, check=False), check=False)
        out = torch.zeros(1, device="cuda")
        pr.call_policy(stream(), d, z, mt, at, ot, vt, None, None, out, grad, row, None, None)
        return float(row.double().sum())  # (the sum in 64 bits: differences are taken)

    grad = torch.empty(batch, width, device="cuda")
    loss_of(grad)
    l1.backward(l2.backward(grad, check=False), check=False)
    for la in (l1, l2):
        for t, g in ((la.w, la.dw), (la.b, la.db)):
            u = g / g.norm()  # along the gradient itself the slope is its norm
            keep, h = t.clone(), 1e-2
            t.copy_(keep + h * u)
            up = loss_of()
            t.copy_(keep - h * u)
            down = loss_of()
            t.copy_(keep)
            slope, norm = (up - down) / (2 * h), float(g.double().norm())
            assert abs(slope - norm) < 1e-2 * norm, (slope, norm)


def test_two_streams_at_once():
    """calls that overlap on two streams, each with its own workspace and outputs, give what they give alone"""
    rng = np.random.default_rng(43)
    jobs = []
    for kind, batch, in_, out in (("bf16", 3000, 700, 900), ("f32", 900, 500, 300)):
        la = Layer(rng, batch, in_, out, kind, "screlu")
        x = torch.from_numpy(rng.random((batch, in_))).to(DT[kind]).cuda()
        gy = torch.from_numpy(rng.standard_normal((batch, out))).to(DT[kind]).cuda()
        d, loss, row = pr.policy_desc(batch, out, kind), torch.zeros(1, device="cuda"), torch.zeros(batch, device="cuda")
        at = torch.zeros(batch, dtype=torch.int32, device="cuda")
        old, adv = torch.full((batch,), -6.0, device="cuda"), torch.ones(batch, device="cuda")
        grad = torch.empty(batch, out, dtype=DT[kind], device="cuda")

        def run(la=la, x=x, gy=gy, d=d, loss=loss, row=row, at=at, old=old, adv=adv, grad=grad):
            y = la.forward(x, check=False)
            pr.call_policy(stream(), d, y, None, at, old, adv, None, None, loss, grad, row, None, None)
            return [y, grad, row, la.backward(gy, check=False), la.dw, la.db]

        jobs.append(run)
    alone = []
    for run in jobs:
        alone.append([t.clone() for t in run()])
        torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, run in zip(side, jobs):
            with torch.cuda.stream(s):
                got.append(run())
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
