"""The wide affine layer, the clipped policy loss and the preference loss: cases that stand for their real use.

Shapes: 1024 / 2048 inputs are the accumulator widths this repository trains (1024, and 2 x 1024), 16384 positions its
default batch, 1880 / 4096 outputs a policy head of chess size, 3 outputs its win / draw / loss head.
"""
import ctypes as C
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    fwd, bwd, pol, pref = "affine_forward", "affine_backward", "policy_loss", "preference_loss"
    return [
        # one position at a time during search: the weights are all there is to read
        dict(name="affine_fwd_one", op=fwd, batch=1, inputs=2048, outputs=4096, type="bf16", act="relu", residual=False,
             w32=False, pad=0),
        # f32 hidden layer of a residual trunk, the type the rest of the framework trains in
        dict(name="affine_fwd_f32", op=fwd, batch=4096, inputs=1024, outputs=1024, type="f32", act="relu", residual=True,
             w32=True, pad=0),
        # nothing divides anything: odd widths, padded rows, f32 master weights rounded on the way in
        dict(name="affine_fwd_odd", op=fwd, batch=1537, inputs=1027, outputs=1881, type="f16", act="screlu", residual=True,
             w32=True, pad=3),
        # a whole training batch into a policy head
        dict(name="affine_fwd_head", op=fwd, batch=16384, inputs=2048, outputs=4096, type="bf16", act="identity",
             residual=False, w32=False, pad=0),
        # a small f32 step: the last, short batch of a file
        dict(name="affine_bwd_small", op=bwd, batch=200, inputs=512, outputs=333, type="f32", act="crelu", w32=True, pad=0),
        # a whole training batch through a hidden layer
        dict(name="affine_bwd_hidden", op=bwd, batch=16384, inputs=2048, outputs=2048, type="bf16", act="crelu", w32=False,
             pad=0),
        # and through the layer behind the accumulator, whose derivative is no longer 0 or 1
        dict(name="affine_bwd_screlu", op=bwd, batch=8192, inputs=1024, outputs=1880, type="bf16", act="screlu", w32=True,
             pad=0),
        # one small self-play update
        dict(name="policy_small", op=pol, batch=64, width=1880, type="f32", legal=35, kl="taken", pad=0),
        # a full batch, legal moves only, the whole reference policy
        dict(name="policy_batch", op=pol, batch=16384, width=1880, type="f32", legal=35, kl="full", pad=0),
        # wide bf16 rows without a mask (every entry a move)
        dict(name="policy_wide", op=pol, batch=8192, width=4096, type="bf16", legal=0, kl="taken", pad=0),
        # a handful of short lines
        dict(name="preference_small", op=pref, pairs=4, longest=20, width=1881, type="f32", legal=35, tail=3, pad=0),
        # many lines of very different lengths, with unused rows behind the last one
        dict(name="preference_large", op=pref, pairs=256, longest=64, width=1880, type="bf16", legal=35, tail=100, pad=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["affine_forward", "affine_backward", "policy_loss", "preference_loss"])
    kind, pad = rng.choice(["f32", "bf16", "f16"]), rng.choice([0, 0, 1, 5, 8])
    if op.startswith("affine"):
        batch, inputs, outputs = _log_int(rng, 1, 16384), _log_int(rng, 16, 2048), _log_int(rng, 3, 4096)
        if kind == "f32":  # the matrix rate for f32 is a sixteenth of the others'
            batch = min(batch, 4096)
        case = dict(op=op, batch=batch, inputs=inputs, outputs=outputs, type=kind,
                    act=rng.choice(["identity", "relu", "crelu", "screlu"]), w32=rng.random() < 0.5, pad=pad)
        if op == "affine_forward":
            case["residual"] = rng.random() < 0.5
        else:
            case["batch"], case["outputs"] = min(batch, 8192), min(outputs, 2048)
        return case
    width, legal = _log_int(rng, 3, 4096), rng.choice([0, 5, 35, 200])
    if op == "policy_loss":
        return dict(op=op, batch=_log_int(rng, 1, 8192), width=width, type=kind, legal=legal,
                    kl=rng.choice(["none", "taken", "full"]), pad=pad)
    return dict(op=op, pairs=_log_int(rng, 1, 200), longest=_log_int(rng, 1, 64), width=width, type=kind, legal=legal,
                tail=rng.choice([0, 1, 17]), pad=pad)


# ---------------------------------------------------------------------------------------------- inputs
class State:
    """What a user's program holds: the tensors of one call, the outputs' buffers and, with `own`, the descriptor."""


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _rows(values, ld, kind):
    """[n][width] values as rows `ld` apart (what lies between two rows is not the layer's)."""
    n, width = values.shape
    buf = torch.full((n, ld), 7.0, device="cuda", dtype=TYPES[kind])
    buf[:, :width] = values.to(TYPES[kind])
    return buf


def _prepare_affine(case, seed):
    g, s = _generator(seed), State()
    b, i, o, kind = case["batch"], case["inputs"], case["outputs"], case["type"]
    s.x_ld, s.y_ld, s.w_ld = i + case["pad"], o + case["pad"], o + case["pad"]
    # activations behind a clipped layer: in [0, 1], many of them 0
    s.x = _rows(_normal(g, b, i).mul_(0.5).clamp_(0.0, 1.0), s.x_ld, kind)
    # one column of `out` weights for each input, columns `w_ld` apart
    s.w = _rows(_normal(g, i, o).mul_(1.4 / math.sqrt(i)), s.w_ld, "f32" if case["w32"] else kind)
    s.bias = _normal(g, o).mul_(0.1)
    s.residual = s.out = None
    if case["op"] == "affine_forward":
        if case["residual"]:
            s.residual = _rows(_normal(g, b, o).mul_(0.5), s.y_ld, kind)
        s.y = torch.zeros(b, s.y_ld, device="cuda", dtype=TYPES[kind])
        # the activation's own output, kept for the backward pass where a residual hides it
        s.saved = torch.zeros_like(s.y) if s.residual is not None and case["act"] != "identity" else None
        return s
    s.gy = _rows(_normal(g, b, o).mul_(0.05), s.y_ld, kind)
    if case["act"] != "identity":
        out = _normal(g, b, o).mul_(0.7).clamp_(min=0.0)
        if case["act"] != "relu":
            out.clamp_(max=1.0)
        s.out = _rows(out * out if case["act"] == "screlu" else out, s.y_ld, kind)
    s.dw = torch.zeros(i, s.w_ld, device="cuda")
    s.dbias = torch.zeros(o, device="cuda")
    s.gx = torch.zeros(b, s.x_ld, device="cuda", dtype=TYPES[kind])
    return s


def _logits_and_moves(g, n, width, legal, ld, kind):
    """logits, legal-move mask (None: all) and the move taken in each row; every 50th row is padding (move -1) and every
    60th has no legal move."""
    z = _rows(_normal(g, n, width).mul_(2.0), ld, kind)
    rows = torch.arange(n, device="cuda")
    mask = None
    if legal:
        mask = _uniform(g, n, width) < min(1.0, legal / width)
        mask[rows, (rows * 7919) % width] = True
        score = _uniform(g, n, width).masked_fill_(~mask, -1.0)
        mask[rows % 60 == 59] = False
        mask = mask.to(torch.uint8)
    else:
        score = _uniform(g, n, width)
    moves = score.argmax(1).to(torch.int32)
    moves[rows % 50 == 49] = -1
    return z, mask, moves


def _row_logp(z, mask, width):
    x = z[:, :width].double()
    if mask is not None:
        x = x.masked_fill(mask == 0, -math.inf)
    return torch.log_softmax(x, 1)


def _prepare_policy(case, seed):
    g, s = _generator(seed), State()
    n, width, kind = case["batch"], case["width"], case["type"]
    s.ld = width + case["pad"]
    s.z, s.mask, s.moves = _logits_and_moves(g, n, width, case["legal"], s.ld, kind)
    at = s.moves.long().clamp(min=0)[:, None]
    logp = _row_logp(s.z, s.mask, width).gather(1, at)[:, 0].nan_to_num(0.0, 0.0, 0.0)
    # the policy that played the games is some updates old: ratios between about 0.5 and 2
    s.old = (logp + 0.25 * _normal(g, n)).float()
    s.adv = _normal(g, n)
    s.weights = 0.5 + _uniform(g, n)
    s.ref = None
    if case["kl"] == "taken":
        s.ref = (logp + 0.3 * _normal(g, n)).float()
    elif case["kl"] == "full":
        ref = s.z[:, :width].float() + 0.5 * _normal(g, n, width)
        s.ref = _rows(ref, s.ld, kind)
    s.low, s.high, s.kl_weight = 0.2, 0.28, 0.0 if case["kl"] == "none" else 0.05
    s.grad = torch.zeros(n, s.ld, device="cuda", dtype=TYPES[kind])
    s.loss, s.row_loss = torch.zeros(1, device="cuda"), torch.zeros(n, device="cuda")
    s.row_logp, s.row_kl = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    return s


def _all_lengths(case):
    """the lengths of a batch's lines, evenly from 1 to `longest`"""
    lines = 2 * case["pairs"]
    return [case["longest"] - (k * case["longest"]) // lines for k in range(lines)]


def _lengths(case, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    lens = torch.tensor(_all_lengths(case))
    return lens[torch.randperm(len(lens), generator=g)]


def _prepare_preference(case, seed):
    g, s = _generator(seed), State()
    width, kind, pairs = case["width"], case["type"], case["pairs"]
    lens = _lengths(case, seed)
    s.used = int(lens.sum())
    n = s.rows = s.used + case["tail"]
    s.offsets = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).to(torch.int32).cuda()
    s.ld = width + case["pad"]
    s.z, s.mask, s.moves = _logits_and_moves(g, n, width, case["legal"], s.ld, kind)
    at = s.moves.long().clamp(min=0)[:, None]
    logp = _row_logp(s.z, s.mask, width).gather(1, at)[:, 0].nan_to_num(0.0, 0.0, 0.0)
    logp = logp * (s.moves >= 0)
    sums = torch.cat([torch.zeros(1, device="cuda", dtype=torch.float64), logp.cumsum(0)])
    line = sums[s.offsets[1:].long()] - sums[s.offsets[:-1].long()]
    # the reference gives each line about the same probability
    s.ref = (line + 2.0 * _normal(g, 2 * pairs)).float()
    s.weights = 0.5 + _uniform(g, pairs)
    s.beta, s.smoothing = 0.1, 0.05
    s.grad = torch.zeros(n, s.ld, device="cuda", dtype=TYPES[kind])
    s.loss, s.pair_loss = torch.zeros(1, device="cuda"), torch.zeros(pairs, device="cuda")
    s.line_logp = torch.zeros(2 * pairs, device="cuda")
    return s


def prepare(case, seed):
    make = {"affine_forward": _prepare_affine, "affine_backward": _prepare_affine, "policy_loss": _prepare_policy,
            "preference_loss": _prepare_preference}[case["op"]]
    s = make(case, seed)
    s.case = case
    if own:
        _plan(s)
    return s


# ---------------------------------------------------------------------------------------------- plain form
def _act(kind, z):
    if kind == "relu":
        return z.clamp(min=0.0)
    if kind == "crelu":
        return z.clamp(0.0, 1.0)
    if kind == "screlu":
        c = z.clamp(0.0, 1.0)
        return c * c
    return z


def _act_slope(kind, a):
    """the activation's derivative, from its output"""
    if kind == "relu":
        return (a > 0).to(a.dtype)
    inside = ((a > 0) & (a < 1)).to(a.dtype)
    return inside * 2.0 * torch.sqrt(a) if kind == "screlu" else inside


def _weights(s):
    c = s.case
    w = s.w[:, :c["outputs"]]
    return w.to(TYPES[c["type"]]).float()


def _plain_affine_forward(s):
    c = s.case
    a = _act(c["act"], s.x[:, :c["inputs"]].float() @ _weights(s) + s.bias)
    dt = TYPES[c["type"]]
    if s.residual is None:
        return {"y": a.to(dt)}
    y = (a + s.residual[:, :c["outputs"]].float()).to(dt)
    return {"y": y} if s.saved is None else {"y": y, "saved": a.to(dt)}


def _plain_affine_backward(s):
    c = s.case
    gz = s.gy[:, :c["outputs"]].float()
    if s.out is not None:
        gz = gz * _act_slope(c["act"], s.out[:, :c["outputs"]].float())
    x = s.x[:, :c["inputs"]].float()
    return {"dw": x.t() @ gz, "dbias": gz.sum(0, dtype=torch.float64).float(), "gx": (gz @ _weights(s).t()).to(TYPES[c["type"]])}


def _plain_softmax(z, mask, width, moves):
    """log-probabilities (f32, masked places 0), probabilities, the counted rows and their moves; the row's sum is taken
    in 64 bits, since a ratio next to the clipping border is compared with it"""
    x = z[:, :width].float()
    legal = torch.ones_like(x, dtype=torch.bool) if mask is None else mask != 0
    x = torch.where(legal, x, -math.inf)
    counted = legal.any(1) & (moves >= 0) & (moves < width)
    at = moves.long().clamp(0, width - 1)[:, None]
    counted = counted & legal.gather(1, at)[:, 0]
    top = x.amax(1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    total = torch.exp(x.double() - top).sum(1, keepdim=True)
    lse = top + torch.log(total)
    logp = (x.gather(1, at).double() - lse)[:, 0]
    logs = torch.where(legal, x - lse.float(), 0.0)
    p = torch.where(legal, torch.exp(x - lse.float()), 0.0)
    return logs, p, counted, at, logp


def _plain_policy(s):
    c, width = s.case, s.case["width"]
    logs, p, counted, at, logp = _plain_softmax(s.z, s.mask, width, s.moves)
    r = torch.exp(logp - s.old)
    adv = s.adv.double()
    free, held = r * adv, r.clamp(1.0 - s.low, 1.0 + s.high) * adv
    loss = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, 0.0)
    kl = torch.zeros_like(logp)
    if c["kl"] == "taken":
        d = s.ref.double() - logp
        kl = torch.expm1(d) - d
        slope = slope - s.kl_weight * torch.expm1(d)
    onehot = torch.zeros_like(p).scatter_(1, at, 1.0)
    grad = slope.float()[:, None] * (onehot - p)
    if c["kl"] == "full":
        ref_logs = _plain_softmax(s.ref, s.mask, width, s.moves)[0]
        diff = logs - ref_logs
        kl32 = (p * diff).sum(1, keepdim=True)
        grad = grad + s.kl_weight * p * (diff - kl32)
        kl = kl32[:, 0].double()
    zero = torch.zeros_like(logp)
    row_loss = torch.where(counted, s.weights * (loss + s.kl_weight * kl), zero)
    grad = torch.where(counted[:, None], s.weights[:, None] * grad, 0.0)
    return {"loss": row_loss.sum().float().reshape(1), "row_loss": row_loss.float(), "grad": grad.to(TYPES[c["type"]]),
            "row_logp": torch.where(counted, logp, zero).float(), "row_kl": torch.where(counted, kl, zero).float()}


def _plain_preference(s):
    c = s.case
    logs, p, counted, at, logp = _plain_softmax(s.z[:s.used], s.mask[:s.used] if s.mask is not None else None, c["width"],
                                                s.moves[:s.used])
    off = s.offsets.long()
    line = torch.searchsorted(off, torch.arange(s.used, device="cuda"), right=True) - 1
    sums = torch.zeros(2 * c["pairs"], device="cuda", dtype=torch.float64)
    sums = sums.scatter_add_(0, line, torch.where(counted, logp, 0.0))
    margin = sums - s.ref
    d = s.beta * (margin[0::2] - margin[1::2])
    soft = torch.log1p(torch.exp(-d.abs()))  # -log sigmoid(d) = soft - min(d, 0)
    loss = (1.0 - s.smoothing) * (soft - d.clamp(max=0.0)) + s.smoothing * (soft + d.clamp(min=0.0))
    pair_loss = s.weights * loss
    slope = s.weights * s.beta * (1.0 / (1.0 + torch.exp(-d)) - (1.0 - s.smoothing))
    slope = torch.stack([slope, -slope], 1).reshape(-1)[line]
    onehot = torch.zeros_like(p).scatter_(1, at, 1.0)
    g = torch.where(counted, slope, 0.0).float()[:, None] * (onehot - p)
    s.grad[:s.used, :c["width"]] = torch.where(counted[:, None], g, 0.0).to(TYPES[c["type"]])
    return {"loss": pair_loss.sum().float().reshape(1), "pair_loss": pair_loss.float(), "line_logp": sums.float(),
            "grad": s.grad[:, :c["width"]]}


# ---------------------------------------------------------------------------------------------- the framework's operators
def _at(t):
    return None if t is None else t.data_ptr()


def _plan(s):
    """descriptor and workspace, made once by a user's program for one shape"""
    from bullet_amd import lib
    s.lib, s.L, c = lib, lib.load(), s.case
    kind = lib.TYPE[c["type"]]
    if c["op"].startswith("affine"):
        s.desc = lib.AffineDesc(batch=c["batch"], in_=c["inputs"], out=c["outputs"], act=lib.ACT[c["act"]], type=kind,
                                w_type=lib.TYPE["f32"] if c["w32"] else kind, w_ld=s.w_ld, x_ld=s.x_ld, y_ld=s.y_ld)
        size = (s.L.bt_affine_forward_workspace_bytes if c["op"] == "affine_forward" else
                s.L.bt_affine_backward_workspace_bytes)(C.byref(s.desc))
    elif c["op"] == "policy_loss":
        s.desc = lib.PolicyDesc(batch=c["batch"], width=c["width"], type=kind, ld=s.ld, mask_ld=c["width"],
                                kl=lib.KL[c["kl"]], clip_low=s.low, clip_high=s.high, kl_weight=s.kl_weight)
        size = 0
    else:
        s.desc = lib.PreferenceDesc(pairs=c["pairs"], rows=s.rows, width=c["width"], type=kind, ld=s.ld,
                                    mask_ld=c["width"], beta=s.beta, smoothing=s.smoothing)
        size = s.L.bt_preference_loss_workspace_bytes(C.byref(s.desc))
    s.workspace, s.workspace_bytes = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda"), size


def _own(s):
    c, stream = s.case, torch.cuda.current_stream().cuda_stream
    d, ws = C.byref(s.desc), s.workspace.data_ptr()
    if c["op"] == "affine_forward":
        s.lib.check(s.L.bt_affine_forward(stream, d, s.w.data_ptr(), s.bias.data_ptr(), s.x.data_ptr(), _at(s.residual),
                                          s.y.data_ptr(), _at(s.saved), ws, s.workspace_bytes))
        out = {"y": s.y[:, :c["outputs"]]}
        return out if s.saved is None else dict(out, saved=s.saved[:, :c["outputs"]])
    if c["op"] == "affine_backward":
        s.lib.check(s.L.bt_affine_backward(stream, d, s.w.data_ptr(), s.x.data_ptr(), _at(s.out), s.gy.data_ptr(),
                                           s.dw.data_ptr(), s.dbias.data_ptr(), s.gx.data_ptr(), ws, s.workspace_bytes))
        return {"dw": s.dw[:, :c["outputs"]], "dbias": s.dbias, "gx": s.gx[:, :c["inputs"]]}
    if c["op"] == "policy_loss":
        s.lib.check(s.L.bt_policy_loss(stream, d, s.z.data_ptr(), _at(s.mask), s.moves.data_ptr(), s.old.data_ptr(),
                                       s.adv.data_ptr(), _at(s.ref), s.weights.data_ptr(), s.loss.data_ptr(),
                                       s.grad.data_ptr(), s.row_loss.data_ptr(), s.row_logp.data_ptr(),
                                       s.row_kl.data_ptr()))
        return {"loss": s.loss, "row_loss": s.row_loss, "grad": s.grad[:, :c["width"]], "row_logp": s.row_logp,
                "row_kl": s.row_kl}
    s.lib.check(s.L.bt_preference_loss(stream, d, s.z.data_ptr(), _at(s.mask), s.moves.data_ptr(), s.offsets.data_ptr(),
                                       s.ref.data_ptr(), s.weights.data_ptr(), s.loss.data_ptr(), s.grad.data_ptr(),
                                       s.pair_loss.data_ptr(), s.line_logp.data_ptr(), ws, s.workspace_bytes))
    return {"loss": s.loss, "pair_loss": s.pair_loss, "line_logp": s.line_logp, "grad": s.grad[:, :c["width"]]}


def run(state):
    if own:
        return _own(state)
    return {"affine_forward": _plain_affine_forward, "affine_backward": _plain_affine_backward, "policy_loss": _plain_policy,
            "preference_loss": _plain_preference}[state.case["op"]](state)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    size = SIZE[case["type"]]
    if case["op"].startswith("affine"):
        b, i, o = case["batch"], case["inputs"], case["outputs"]
        w = i * o * (4 if case["w32"] else size)
        if case["op"] == "affine_forward":
            more = (case["residual"] + (case["residual"] and case["act"] != "identity")) * b * o * size
            return {"bytes": b * i * size + w + 4 * o + b * o * size + more, "flops": 2 * b * i * o}
        reads = b * i * size + w + b * o * size * (1 if case["act"] == "identity" else 2)
        return {"bytes": reads + 4 * i * o + 4 * o + b * i * size, "flops": 4 * b * i * o}
    width = case["width"]
    if case["op"] == "policy_loss":
        n = case["batch"]
        matrices = 3 if case["kl"] == "full" else 2
        taken = 4 if case["kl"] == "taken" else 0
        return {"bytes": n * (width * (size * matrices + (case["legal"] > 0)) + 28 + taken), "flops": 12 * n * width}
    n = sum(_all_lengths(case))  # the rows behind the last line are neither read nor written
    return {"bytes": n * (width * (2 * size + (case["legal"] > 0)) + 4) + 28 * case["pairs"], "flops": 8 * n * width}


# ---------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def _exact_affine_forward(s, c):
    w = s.w[:, :c["outputs"]].to(TYPES[c["type"]]).double()
    z = torch.addmm(s.bias.double(), s.x[:, :c["inputs"]].double(), w)
    if c["act"] == "relu":
        z = torch.relu(z)
    elif c["act"] == "crelu":
        z = torch.relu(z) - torch.relu(z - 1.0)
    elif c["act"] == "screlu":
        z = torch.minimum(torch.relu(z), torch.ones_like(z)).square()
    out = {"y": z}
    if s.residual is not None:
        out = {"y": z + s.residual[:, :c["outputs"]].double()}
        if c["act"] != "identity":
            out["saved"] = z
    return out


def _exact_affine_backward(s, c):
    """through the layer's function: the pre-activation that gives the kept output, differentiated by torch"""
    gy, x = s.gy[:, :c["outputs"]].double(), s.x[:, :c["inputs"]].double()
    w = s.w[:, :c["outputs"]].to(TYPES[c["type"]]).double()
    if s.out is not None:
        a = s.out[:, :c["outputs"]].double()
        slope = torch.where(a > 0, 1.0, 0.0).double()
        if c["act"] != "relu":
            slope = torch.where(a < 1, slope, 0.0)
        if c["act"] == "screlu":
            slope = slope * 2 * a.pow(0.5)
        gy = gy * slope
    return {"dw": (gy.t() @ x).t(), "dbias": gy.sum(0), "gx": gy @ w.t()}


def _exact_rows(z, mask, moves, width):
    """log-probabilities of the counted rows, as a function that can be differentiated"""
    legal = torch.ones_like(z, dtype=torch.bool) if mask is None else mask != 0
    ok = (moves >= 0) & (moves < width)
    at = moves.long() * ok
    ok = ok & legal[torch.arange(len(moves), device="cuda"), at]
    keep = torch.nonzero(ok)[:, 0]
    return keep, at[keep], legal[keep]


def _exact_logs(z, legal):
    low = torch.finfo(torch.float64).min / 4
    return torch.log_softmax(torch.where(legal, z, low), 1)


def _exact_policy(s, c):
    width, n = c["width"], c["batch"]
    keep, at, legal = _exact_rows(s.z[:, :width], s.mask, s.moves, width)
    z = s.z[:, :width].double().requires_grad_(True)
    logs = _exact_logs(z[keep], legal)
    logp = logs.gather(1, at[:, None])[:, 0]
    ratio = (logp - s.old[keep].double()).exp()
    adv = s.adv[keep].double()
    # the smaller of the free and the clipped gain, by cases of the advantage's sign
    gain = torch.where(adv >= 0, adv * ratio.clamp(max=1.0 + s.high), adv * ratio.clamp(min=1.0 - s.low))
    kl = torch.zeros_like(logp)
    if c["kl"] == "taken":
        d = s.ref[keep].double() - logp
        kl = d.exp() - d - 1.0
    elif c["kl"] == "full":
        ref = _exact_logs(s.ref[:, :width].double()[keep], legal)
        kl = torch.where(legal, logs.exp() * (logs - ref), 0.0).sum(1)
    rows = s.weights[keep].double() * (s.kl_weight * kl - gain)
    rows.sum().backward()

    def spread(v):
        return torch.zeros(n, device="cuda", dtype=torch.float64).index_copy(0, keep, v.detach())
    return {"loss": rows.sum().detach().reshape(1), "row_loss": spread(rows), "grad": z.grad, "row_logp": spread(logp),
            "row_kl": spread(kl)}


def _exact_preference(s, c):
    width = c["width"]
    used = s.used
    keep, at, legal = _exact_rows(s.z[:used, :width], s.mask[:used] if s.mask is not None else None, s.moves[:used], width)
    z = s.z[:, :width].double().requires_grad_(True)
    rows = torch.zeros(used, device="cuda", dtype=torch.float64)
    rows = rows.index_copy(0, keep, _exact_logs(z[keep], legal).gather(1, at[:, None])[:, 0])
    off = s.offsets.tolist()
    line = torch.stack([rows[a:b].sum() for a, b in zip(off[:-1], off[1:])])
    ratio = line - s.ref.double()
    d = s.beta * (ratio[0::2] - ratio[1::2])
    loss = -(1 - s.smoothing) * torch.nn.functional.logsigmoid(d) - s.smoothing * torch.nn.functional.logsigmoid(-d)
    pair = s.weights.double() * loss
    pair.sum().backward()
    return {"loss": pair.sum().detach().reshape(1), "pair_loss": pair.detach(), "line_logp": line.detach(), "grad": z.grad}


def exact(case, seed):
    make = {"affine_forward": (_prepare_affine, _exact_affine_forward),
            "affine_backward": (_prepare_affine, _exact_affine_backward),
            "policy_loss": (_prepare_policy, _exact_policy),
            "preference_loss": (_prepare_preference, _exact_preference)}[case["op"]]
    return make[1](make[0](case, seed), case)
