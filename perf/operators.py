"""The operators around a token model's blocks and at its vocabulary, case by case: what they are given, how they are called,
what they compute (plain torch in 32 bits), and what they should compute (64 bits).

A complex matrix is two fp32 planes.  `dz` is dL/dz, `dzs` its conjugate dL/d conj z (the loss is real).
  norm   y = v .* x / rms(x) in front of a block; behind it h = u + scale v .* f / rms(f) and, for the next block,
         y = w .* h / rms(h); forward, and backward down to the weights
  distil sum_j q_j (log q_j - log p[id_j]) over the teacher's top entries, p_k = |z_k|^2 / sum |z|^2, with the gradient at z
  head   logits z = x w^T of a vocabulary, loss -log p[label], most likely entry; with the gradients at x and w
"""
import math

import torch

own = False

EPS = 1e-6      # of the norms
SCALE = 0.35    # of the blocks' results on the residual path
FLOOR = 1e-15   # least |z|^2 and least probability that a loss takes the logarithm of


def listed():
    return [
        # one token on its way into a block: nothing but latency
        {"name": "norm forward, one token", "op": "norm_fwd", "rows": 1, "cols": 1024, "pad": 0, "row_gate": False, "join": False},
        # the activations of the token model of the benchmark, between two blocks
        {"name": "join forward 8192x1024", "op": "norm_fwd", "rows": 8192, "cols": 1024, "pad": 0, "row_gate": False, "join": True},
        {"name": "join backward 8192x1024", "op": "norm_bwd", "rows": 8192, "cols": 1024, "pad": 0, "row_gate": False, "join": True},
        # an odd width inside a wider buffer, a gate of its own for every row
        {"name": "norm backward 515x1001 gated", "op": "norm_bwd", "rows": 515, "cols": 1001, "pad": 2, "row_gate": True, "join": False},
        # the reduced token model of the tests
        {"name": "distil 96x512 top 8", "op": "distil", "rows": 96, "cols": 512, "top": 8, "pad": 0},
        # every token of the benchmark's batch, its vocabulary
        {"name": "distil 8192x32768 top 32", "op": "distil", "rows": 8192, "cols": 32768, "top": 32, "pad": 0},
        # a few long rows of an odd vocabulary
        {"name": "distil 3x100003 top 64", "op": "distil", "rows": 3, "cols": 100003, "top": 64, "pad": 0},
        # the next token of one sequence, and of a batch of 48
        {"name": "head scores 1x1024->32768", "op": "head_fwd", "rows": 1, "dim": 1024, "vocab": 32768},
        {"name": "head scores 48x1024->32768", "op": "head_fwd", "rows": 48, "dim": 1024, "vocab": 32768},
        # a training step: the reduced model of the tests, an odd one, the benchmark's
        {"name": "head step 96x64->512", "op": "head_bwd", "rows": 96, "dim": 64, "vocab": 512},
        {"name": "head step 1000x333->5003", "op": "head_bwd", "rows": 1000, "dim": 333, "vocab": 5003},
        {"name": "head step 8192x1024->32768", "op": "head_bwd", "rows": 8192, "dim": 1024, "vocab": 32768},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "distil", "head_fwd", "head_bwd"])
    if op in ("norm_fwd", "norm_bwd"):
        rows = _log(rng, 1, 16384)
        cols = _log(rng, 33, min(8192, 8192 * 1024 // rows))
        return {"op": op, "rows": rows, "cols": cols, "pad": rng.choice([0, 0, 1, 4]), "row_gate": rng.random() < 0.25, "join": rng.random() < 0.6}
    if op == "distil":
        rows = _log(rng, 1, 8192)
        cols = _log(rng, 256, min(131072, (1 << 28) // rows))
        return {"op": op, "rows": rows, "cols": cols, "top": rng.randint(1, 64), "pad": rng.choice([0, 0, 1, 4])}
    dim, vocab = _log(rng, 48, 2048), _log(rng, 256, 65536)
    if op == "head_fwd":
        return {"op": op, "rows": _log(rng, 1, 64), "dim": dim, "vocab": vocab}
    return {"op": op, "rows": _log(rng, 16, min(8192, max(17, (1 << 38) // (dim * vocab)))), "dim": dim, "vocab": vocab}


def _planes(g, rows, cols, ld, std):
    return [(torch.randn(rows, ld, device="cuda", generator=g) * std)[:, :cols] for _ in range(2)]


def _room(rows, cols, ld, count):
    return [torch.empty(rows, ld, device="cuda")[:, :cols] for _ in range(count)]


def _zipf(g, shape, n):
    """indices below n, the k-th with a weight of about 1 / k, as the tokens of a text"""
    return (torch.exp(torch.rand(shape, device="cuda", generator=g) * math.log(n)) - 1.0).long().clamp_(0, n - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, rows = case["op"], case["rows"]
    st = {"case": case}
    if op in ("norm_fwd", "norm_bwd"):
        cols, ld = case["cols"], case["cols"] + case["pad"]
        gates = rows if case["row_gate"] else 1
        st["x"] = _planes(g, rows, cols, ld, 0.7)                      # what the block computed, or its input
        st["v"] = _planes(g, gates, cols, ld, 0.3)
        st["v"][0] += 1.0
        if case["join"]:
            st["u"] = _planes(g, rows, cols, ld, 1.1)                  # the residual path
            st["w"] = _planes(g, 1, cols, ld, 0.2)
            st["w"][0] += 1.0
        inv = lambda p: (1.0 / torch.sqrt((p[0].double() ** 2 + p[1].double() ** 2).mean(1) + EPS)).float()  # noqa: E731
        if op == "norm_bwd":  # the forward pass has left these
            st["s"] = inv(st["x"])
            st["g"] = _planes(g, rows, cols, ld, 0.01)
            if case["join"]:
                k = SCALE * st["s"][:, None]
                a, b, c, d = st["v"][0], st["v"][1], st["x"][0], st["x"][1]
                st["h"] = _room(rows, cols, ld, 2)
                st["h"][0].copy_(st["u"][0] + k * (a * c - b * d))
                st["h"][1].copy_(st["u"][1] + k * (a * d + b * c))
                st["s2"] = inv(st["h"])
                st["gh"] = _planes(g, rows, cols, ld, 0.01)            # what reaches h along the residual path
                st["du"], st["dw"] = _room(rows, cols, ld, 2), _room(1, cols, ld, 4)
            st["dx"], st["dv"] = _room(rows, cols, ld, 2), _room(gates, cols, ld, 4)
        else:
            st["y"], st["so"] = _room(rows, cols, ld, 2), torch.empty(rows, device="cuda")
            if case["join"]:
                st["ho"], st["so2"] = _room(rows, cols, ld, 2), torch.empty(rows, device="cuda")
    elif op == "distil":
        cols, top = case["cols"], case["top"]
        st["z"] = _planes(g, rows, cols, cols + case["pad"], 1.0)
        best = (st["z"][0] ** 2 + st["z"][1] ** 2 + torch.rand(rows, cols, device="cuda", generator=g) * 4).topk(top, dim=1)
        st["ids"] = best.indices.int()                                 # a teacher that agrees in part
        q = torch.sort(torch.rand(rows, top, device="cuda", generator=g) ** 4 + 1e-4, dim=1, descending=True).values
        q = q / q.sum(1, keepdim=True) * 0.95                          # the rest of its probability lies elsewhere
        none = torch.rand(rows, device="cuda", generator=g) < 0.03     # rows of padding
        st["ids"][none] = -1
        q[none] = 0.0
        st["q"] = q.contiguous()
        st["s"], st["loss"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        st["dz"] = _room(rows, cols, cols + case["pad"], 2)
    else:
        dim, vocab = case["dim"], case["vocab"]
        st["w"] = _planes(g, vocab, dim, dim, (2 * dim) ** -0.5)
        st["x"] = _planes(g, rows, dim, dim, 0.5 ** 0.5)
        target = _zipf(g, (rows,), vocab)
        pull = 6.0 + 6.0 * torch.rand(rows, 1, device="cuda", generator=g)   # a model that has learnt: its token stands out
        st["x"][0] += pull * st["w"][0][target]
        st["x"][1] -= pull * st["w"][1][target]
        label = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.9, target, _zipf(g, (rows,), vocab))
        label[torch.rand(rows, device="cuda", generator=g) < 0.02] = -1      # padding, not trained on
        st["label"] = label.int()
        st["s"], st["loss"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        if op == "head_fwd":
            st["argmax"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        else:
            st["dx"], st["dw"] = _room(rows, dim, dim, 2), _room(vocab, dim, dim, 4)
    return st


# ------------------------------------------------------------------------------------------------ the framework's calls
class _Vec:
    """a vector on the device, as the framework's wrappers take one"""

    def __init__(self, t):
        self.ptr = t.data_ptr()


def _handles(st):
    """The planes of a state as the framework's matrices, made once as a program does that keeps its buffers."""
    from cnet_amd import capi, ops
    capi.init(0)

    def plane(t):
        return ops.Plane(t.data_ptr(), t.shape[0], t.shape[1], t.stride(0), t)

    def handle(v):
        if isinstance(v, torch.Tensor):
            return _Vec(v)
        return ops.CMat(plane(v[0]), plane(v[1])) if len(v) == 2 else ops.Grad([plane(t) for t in v])

    st["handles"] = dict({k: handle(v) for k, v in st.items() if k != "case"}, ops=ops)
    return st["handles"]


def _run_own(st):
    h = st.get("handles") or _handles(st)
    ops, case = h["ops"], st["case"]
    op = case["op"]
    if op == "norm_fwd":
        shared = not case["row_gate"]
        if case["join"]:
            ops.norm_join_fwd(h["u"], h["x"], h["v"], SCALE, h["ho"], h["so"], h["w"], h["y"], h["so2"], EPS, shared=shared)
            return st["y"], st["so"], st["ho"], st["so2"]
        ops.norm_gate_fwd(h["x"], h["v"], h["y"], h["so"], EPS, shared=shared)
        return st["y"], st["so"]
    if op == "norm_bwd":
        shared = not case["row_gate"]
        if case["join"]:
            ops.norm_join_bwd_sym(h["x"], h["s"], h["v"], SCALE, h["h"], h["s2"], h["w"], h["gh"], h["g"], h["du"], h["dx"], h["dv"], h["dw"],
                                  shared=shared, mirror=False)
            return st["du"], st["dx"], st["dv"], st["dw"]
        ops.norm_gate_bwd_sym(h["x"], h["s"], h["v"], h["g"], h["dx"], h["dv"], shared=shared, mirror=False)
        return st["dx"], st["dv"]
    if op == "distil":
        ops.distill_fwd_bwd_sym(h["z"], h["ids"], h["q"], case["top"], h["s"], h["loss"], h["dz"], mirror=False)
        return st["s"], st["loss"], st["dz"]
    if op == "head_fwd":
        ops.vocab_head_fwd(h["x"], h["w"], h["label"], h["s"], h["loss"], h["argmax"])
        return st["s"], st["loss"], st["argmax"]
    ops.vocab_head_fwd_bwd_sym(h["x"], h["w"], h["label"], h["s"], h["loss"], None, h["dx"], h["dw"], mirror_dx=False)
    return st["s"], st["loss"], st["dx"], st["dw"]


# ------------------------------------------------------------------------------------------------ plain forms
def _mul(a, b):
    return a[0] * b[0] - a[1] * b[1], a[0] * b[1] + a[1] * b[0]


def _inv_rms(x):
    return 1.0 / torch.sqrt((x[0] * x[0] + x[1] * x[1]).mean(1, keepdim=True) + EPS)


def _norm_back(x, s, v, g):
    """gradients (dz) at x and, row by row, at v, of y = v .* (x s); g = dL/dy"""
    n = x[0] * s, x[1] * s
    p = _mul(g, v)                                                # dL/dn
    t = (p[0] * n[0] - p[1] * n[1]).mean(1, keepdim=True)         # Re of sum(dL/dn n) over the width
    dx = s * (p[0] - n[0] * t), s * (p[1] + n[1] * t)
    return dx, _mul(g, n)


def _four(d, shared):
    """a weight's gradient, summed over the rows that share it, with its conjugate"""
    re, im = (d[0].sum(0, keepdim=True), d[1].sum(0, keepdim=True)) if shared else d
    return [re, im, re, -im]


def _logits(x, w):
    return x[0] @ w[0].T - x[1] @ w[1].T, x[0] @ w[1].T + x[1] @ w[0].T


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    op = case["op"]
    if op == "norm_fwd":
        x, v = st["x"], st["v"]
        s = _inv_rms(x)
        a = _mul(v, (x[0] * s, x[1] * s))
        if not case["join"]:
            return a, s[:, 0]
        h = st["u"][0] + SCALE * a[0], st["u"][1] + SCALE * a[1]
        s2 = _inv_rms(h)
        return _mul(st["w"], (h[0] * s2, h[1] * s2)), s[:, 0], h, s2[:, 0]
    if op == "norm_bwd":
        shared = not case["row_gate"]
        x, s, v, g = st["x"], st["s"][:, None], st["v"], st["g"]
        if not case["join"]:
            dx, dv = _norm_back(x, s, v, g)
            return dx, _four(dv, shared)
        dh, dw = _norm_back(st["h"], st["s2"][:, None], st["w"], g)
        dh = dh[0] + st["gh"][0], dh[1] + st["gh"][1]
        df, dv = _norm_back(x, s, v, (SCALE * dh[0], SCALE * dh[1]))
        return dh, df, _four(dv, shared), _four(dw, True)
    if op == "distil":
        z, q = st["z"], st["q"]
        there = st["ids"] >= 0
        ids = st["ids"].long().clamp(min=0)
        q = torch.where(there, q, torch.zeros_like(q))
        s = (z[0] * z[0] + z[1] * z[1]).sum(1, keepdim=True).clamp(min=FLOOR)
        zt = z[0].gather(1, ids), z[1].gather(1, ids)
        m = zt[0] * zt[0] + zt[1] * zt[1]
        terms = torch.where(q > 0, q * (torch.log(q) - torch.log((m / s).clamp(min=FLOOR))), torch.zeros_like(q))
        share = q.sum(1, keepdim=True) / s
        k = -q / m.clamp(min=FLOOR)
        re = (z[0] * share).scatter_add(1, ids, zt[0] * k)
        im = (z[1] * -share).scatter_add(1, ids, -zt[1] * k)
        return s[:, 0], terms.sum(1), (re, im)
    x, w, label = st["x"], st["w"], st["label"].long()
    z = _logits(x, w)
    p = z[0] * z[0] + z[1] * z[1]
    s = p.sum(1, keepdim=True).clamp(min=FLOOR)
    there, at = (label >= 0)[:, None], label.clamp(min=0)
    # (the label's logit in 64 bits: the gradient goes with its inverse, and an unlikely label has one near zero)
    zt = _mul((x[0].double(), x[1].double()), (w[0][at].double(), w[1][at].double()))
    zt = zt[0].sum(1, keepdim=True), zt[1].sum(1, keepdim=True)
    m = zt[0] * zt[0] + zt[1] * zt[1]
    loss = torch.where(there, -torch.log((m / s).clamp(min=FLOOR)), 0.0).float()
    if op == "head_fwd":
        return s[:, 0], loss[:, 0], p.argmax(1).int()
    # every logit's share of the norm, and apart from those thousands of small terms the label's one large term
    g = z[0] * (there / s), z[1] * -(there / s)
    k = there / m.clamp(min=FLOOR)
    c = (zt[0] * -k).float(), (zt[1] * k).float()
    del z, p
    to_w = _mul(c, (w[0][at], w[1][at]))
    dx = g[0] @ w[0] - g[1] @ w[1] + to_w[0], g[0] @ w[1] + g[1] @ w[0] + to_w[1]
    to_x = _mul(c, x)
    dw = g[0].T @ x[0] - g[1].T @ x[1], g[0].T @ x[1] + g[1].T @ x[0]
    dw[0].index_put_((at,), to_x[0], accumulate=True)
    dw[1].index_put_((at,), to_x[1], accumulate=True)
    return s[:, 0], loss[:, 0], dx, [dw[0], dw[1], dw[0], -dw[1]]


def work(case):
    op, rows = case["op"], case["rows"]
    if op in ("norm_fwd", "norm_bwd"):
        n, gates = rows * case["cols"], (rows if case["row_gate"] else 1) * case["cols"]
        if op == "norm_fwd":
            return {"bytes": 8 * ((4 if case["join"] else 2) * n + gates), "flops": (30 if case["join"] else 11) * n}
        return {"bytes": 8 * ((6 if case["join"] else 3) * n + 3 * gates), "flops": (62 if case["join"] else 27) * n}
    if op == "distil":
        return {"bytes": 16 * rows * case["cols"] + 8 * rows * case["top"], "flops": 6 * rows * case["cols"]}
    b, k, n = rows, case["dim"], case["vocab"]
    if op == "head_fwd":
        return {"bytes": 8 * (b * k + n * k), "flops": 8 * b * k * n}
    # x and w read, the gradient of x (one pair of planes) and of w (two) written; the logits, their gradient against w and
    # against x, or what the loss's quadratic norm makes of it: w^H w and the weighted x^H x (Hermitian: half of each) and one
    # product with each
    return {"bytes": 16 * b * k + 24 * n * k, "flops": 8 * min(3.0 * b * n * k, 1.5 * (b + n) * k * k)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _c(pair):
    return torch.complex(pair[0].double(), pair[1].double())


def _dz(grad):
    """autograd gives dL/dRe + i dL/dIm = 2 dL/d conj z; dL/dz is half of its conjugate"""
    d = grad.conj().resolve_conj() / 2
    return d.real, d.imag


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    rms = lambda c: torch.linalg.vector_norm(c, dim=1, keepdim=True).square().div(c.shape[1]).add(EPS).sqrt()  # noqa: E731
    if op in ("norm_fwd", "norm_bwd"):
        back = op == "norm_bwd"
        x, v = _c(st["x"]).requires_grad_(back), _c(st["v"]).requires_grad_(back)
        n = x / rms(x)
        if not case["join"]:
            y = v * n
            if not back:
                return (y.real, y.imag), (1 / rms(x))[:, 0]
            # the loss whose dz at y is g
            gx, gv = torch.autograd.grad(2 * (y * _c(st["g"])).real.sum(), [x, v])
            dv = _dz(gv)
            return _dz(gx), [dv[0], dv[1], dv[0], -dv[1]]
        u, w = _c(st["u"]).requires_grad_(back), _c(st["w"]).requires_grad_(back)
        if not back:
            h = u + SCALE * v * n
            y = w * h / rms(h)
            return (y.real, y.imag), (1 / rms(x))[:, 0], (h.real, h.imag), (1 / rms(h))[:, 0]
        # (h is an input of the backward pass, rounded to 32 bits: the gradient at it first, then through it)
        h = _c(st["h"]).requires_grad_(True)
        gh, gw = torch.autograd.grad(2 * (w * h / rms(h) * _c(st["g"])).real.sum(), [h, w])
        gh = gh + 2 * _c(st["gh"]).conj()
        gx, gv = torch.autograd.grad((SCALE * v * n * gh.conj()).real.sum(), [x, v])
        dv, dw = _dz(gv), _dz(gw)
        return _dz(gh), _dz(gx), [dv[0], dv[1], dv[0], -dv[1]], [dw[0], dw[1], dw[0], -dw[1]]
    if op == "distil":
        ids, q = st["ids"].long(), st["q"].double()
        q[ids < 0] = 0
        z = _c(st["z"]).requires_grad_(True)
        power = z.real.square() + z.imag.square()
        s = power.sum(1)
        logp = torch.log(power.gather(1, ids.clamp(min=0))) - torch.log(s)[:, None]
        loss = (torch.xlogy(q, q) - q * logp).sum(1)
        gz, = torch.autograd.grad(loss.sum(), z)
        return s.detach(), loss.detach(), _dz(gz)
    back = op == "head_bwd"
    x, w = _c(st["x"]).requires_grad_(back), _c(st["w"]).requires_grad_(back)
    label = st["label"].long()
    z = x @ w.T
    power = z.real.square() + z.imag.square()
    s = power.sum(1)
    loss = torch.log(s) - torch.log(power.gather(1, label.clamp(min=0)[:, None]))[:, 0]
    loss = torch.where(label >= 0, loss, torch.zeros_like(loss))
    if not back:
        return s, loss, power.argmax(1).int()
    gx, gw = torch.autograd.grad(loss.sum(), [x, w])
    dw = _dz(gw)
    return s.detach(), loss.detach(), _dz(gx), [dw[0], dw[1], dw[0], -dw[1]]
