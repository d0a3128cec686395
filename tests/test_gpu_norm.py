"""The norms around a block (cnet_norm_gate_*, cnet_norm_join_*) against the same formulas in 64 bits.

Tolerances count roundings of 2^-24 (half a step of fp32, relative).  A row's sum of `cols` terms takes at most
cols / 64 + 16 roundings on its longest path (a thread's own terms, then the lanes and wavefronts), a column's sum over the rows
at most as many as there are rows, and an element of the result a dozen more."""
import ctypes as C

import numpy as np
import pytest

from cnet_amd import capi, ops
from tests.gpu_util import gpu  # noqa: F401

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24
EPS, SCALE = 1e-6, 0.35
INVALID = -2
GUARD = 7.0


def padded(a, ld, off=0):
    """rows of `a` inside a buffer ld wide, `off` floats behind its start; everything else holds GUARD"""
    buf = np.full((a.shape[0] + 2, ld), GUARD, np.float32).reshape(-1)
    idx = ld + off + np.arange(a.shape[0])[:, None] * ld + np.arange(a.shape[1])[None, :]
    buf[idx] = a
    d = capi.to_device(buf.reshape(1, -1))
    p = ops.Plane(d.ptr + 4 * (ld + off), a.shape[0], a.shape[1], ld, d)
    p.idx = idx
    return p


def values(p):
    return p.owner.download().reshape(-1)[p.idx]


def untouched(p):
    rest = p.owner.download().reshape(-1)
    mask = np.ones(rest.size, bool)
    mask[p.idx] = False
    return bool(np.all(rest[mask] == GUARD))


def cmat(z, ld, off=0):
    return ops.CMat(padded(z.real.astype(np.float32), ld, off), padded(z.imag.astype(np.float32), ld, off))


def grad(shape, ld, off=0, fill=0.0):
    return ops.Grad([padded(np.full(shape, fill, np.float32), ld, off) for _ in range(4)])


def cval(m):
    return values(m.re).astype(np.float64) + 1j * values(m.im)


def dz_of(g):
    return values(g.planes[0]).astype(np.float64) + 1j * values(g.planes[1])


def dzs_of(g):
    return values(g.planes[2]).astype(np.float64) + 1j * values(g.planes[3])


def rnd(rng, rows, cols, std=1.0, mean=0.0):
    z = (mean + std * rng.standard_normal((rows, cols)) + 1j * std * rng.standard_normal((rows, cols)))
    return z.real.astype(np.float32).astype(np.float64) + 1j * z.imag.astype(np.float32)


def inv_rms(x, eps=EPS):
    return 1.0 / np.maximum(np.sqrt((np.abs(x) ** 2).mean(1, keepdims=True) + eps), 1e-15)


def back(x, s, v, g):
    """(dx, per-row dv, the bounds' magnitudes of both)"""
    n = x * s
    p = g * v
    t = (p * n).real.mean(1, keepdims=True)
    size = s * (np.abs(p) + np.abs(n) * (np.abs(p) * np.abs(n)).mean(1, keepdims=True))
    return s * (p - n.conj() * t), g * n, size, np.abs(g) * np.abs(n)


def close(got, want, size, roundings, what):
    err = np.abs(got - want)
    bound = roundings * HALF * size + 1e-37
    assert np.all(err <= bound), (what, float((err / (HALF * size + 1e-37)).max()), roundings)


def row_roundings(cols):
    return cols / 64 + 16


# rows, cols, leading dimension beyond cols, offset of the first element
SHAPES = [(1, 1, 0, 0), (1, 1024, 0, 0), (3, 7, 2, 1), (5, 64, 0, 0), (130, 333, 3, 1), (515, 1001, 2, 0), (66, 1000, 4, 0), (300, 1024, 0, 0),
          (37, 512, 0, 4), (9, 2048, 0, 0), (1100, 516, 0, 0), (4, 4096, 8, 0), (3, 4100, 0, 0), (2, 8192, 0, 0), (3, 9001, 0, 1), (2, 20000, 0, 0)]


@pytest.mark.parametrize("rows,cols,pad,off", SHAPES)
@pytest.mark.parametrize("shared", [True, False])
def test_norm_gate(gpu, rows, cols, pad, off, shared):
    rng = np.random.default_rng(rows * 7 + cols)
    ld = cols + pad + off
    x, v, g = rnd(rng, rows, cols, 0.7), rnd(rng, 1 if shared else rows, cols, 0.3, 1.0), rnd(rng, rows, cols, 0.01)
    X, V, G = cmat(x, ld, off), cmat(v, ld, off), cmat(g, ld, off)
    Y, s = cmat(0 * x, ld, off), capi.empty(rows)
    ops.norm_gate_fwd(X, V, Y, s, EPS, shared=shared)
    want_s = inv_rms(x)
    rr = row_roundings(cols)
    close(s.download()[:, None], want_s, want_s, rr, "s")
    close(cval(Y), v * x * want_s, np.abs(v) * np.abs(x) * want_s, rr + 12, "y")
    dX, dV = grad(x.shape, ld, off), grad(v.shape, ld, off)
    ops.norm_gate_bwd_sym(X, s, V, G, dX, dV, shared=shared)
    dx, dv, size, size_v = back(x, want_s, v, g)
    close(dz_of(dX), dx, size, 3 * rr + 16, "dx")
    assert np.array_equal(dzs_of(dX), dz_of(dX).conj()) and np.array_equal(dzs_of(dV), dz_of(dV).conj())
    if shared:
        dv, size_v = dv.sum(0, keepdims=True), size_v.sum(0, keepdims=True)
    close(dz_of(dV), dv, size_v, rr + 16 + (rows if shared else 0), "dv")
    first = dz_of(dX), dz_of(dV)
    # a second call adds onto what the first has left, without the dz* halves
    ops.norm_gate_bwd_sym(X, s, V, G, dX, dV, shared=shared, accumulate=1, accumulate_w=1, mirror=False, mirror_w=False)
    assert np.array_equal(dz_of(dX), 2 * first[0]) and np.array_equal(dz_of(dV), 2 * first[1])
    assert np.array_equal(dzs_of(dX), first[0].conj()) and np.array_equal(dzs_of(dV), first[1].conj())
    for p in [X.re, X.im, V.re, V.im, G.re, G.im, Y.re, Y.im] + dX.planes + dV.planes:
        assert untouched(p)


@pytest.mark.parametrize("rows,cols,pad,off", SHAPES)
@pytest.mark.parametrize("shared,second,residual", [(True, True, True), (False, True, True), (True, False, True), (True, True, False)])
def test_norm_join(gpu, rows, cols, pad, off, shared, second, residual):
    """second: the next block's norm is asked for; residual: a gradient reaches h along the residual path"""
    rng = np.random.default_rng(rows * 5 + cols)
    ld = cols + pad + off
    u, f, v = rnd(rng, rows, cols, 1.1), rnd(rng, rows, cols, 0.7), rnd(rng, 1 if shared else rows, cols, 0.3, 1.0)
    w, gh, gy = rnd(rng, 1, cols, 0.2, 1.0), rnd(rng, rows, cols, 0.01), rnd(rng, rows, cols, 0.01)
    U, F, V, W = cmat(u, ld, off), cmat(f, ld, off), cmat(v, ld, off), cmat(w, cols)
    H, Y, s, s2 = cmat(0 * u, ld, off), cmat(0 * u, ld, off), capi.empty(rows), capi.empty(rows)
    ops.norm_join_fwd(U, F, V, SCALE, H, s, W if second else None, Y if second else None, s2 if second else None, EPS, shared=shared)
    rr = row_roundings(cols)
    s_w = inv_rms(f)
    h = u + SCALE * v * f * s_w
    close(s.download()[:, None], s_w, s_w, rr, "s")
    size_h = np.abs(u) + SCALE * np.abs(v) * np.abs(f) * s_w
    close(cval(H), h, size_h, rr + 16, "h")
    hh = cval(H)             # the second half works on h as it was rounded
    s2_w = inv_rms(hh)
    if second:
        close(s2.download()[:, None], s2_w, s2_w, rr, "s2")
        close(cval(Y), w * hh * s2_w, np.abs(w) * np.abs(hh) * s2_w, rr + 12, "y")
    dU, dF, dV, dW = grad(u.shape, ld, off), grad(u.shape, ld, off), grad(v.shape, ld, off), grad(w.shape, cols)
    GH, GY = cmat(gh, ld, off), cmat(gy, ld, off)

    def run(accumulate, mirror):
        ops.norm_join_bwd_sym(F, s, V, SCALE, H if second else None, s2 if second else None, W if second else None, GH if residual else None,
                              GY if second else None, dU, dF, dV, dW if second else None, shared=shared, accumulate=accumulate,
                              accumulate_w=accumulate, mirror=mirror, mirror_w=mirror)
    run(0, True)
    dh, size = (gh, np.abs(gh)) if residual else (0 * gh, 0 * np.abs(gh))
    if second:
        d, dw, sz, size_w = back(hh, s2_w, w, gy)
        dh, size = dh + d, size + sz
        close(dz_of(dW), dw.sum(0, keepdims=True), size_w.sum(0, keepdims=True), rr + 16 + rows, "dw")
    else:
        assert np.all(dz_of(dW) == 0)
    close(dz_of(dU), dh, size, 3 * rr + 20, "du")
    df, dv, _, _ = back(f, s_w, SCALE * v, dh)
    _, _, size_f, size_v = back(np.abs(f), s_w, SCALE * np.abs(v), size)
    close(dz_of(dF), df, size_f, 8 * rr + 40, "df")
    dv, size_v = SCALE * dv, SCALE * size_v
    if shared:
        dv, size_v = dv.sum(0, keepdims=True), size_v.sum(0, keepdims=True)
    close(dz_of(dV), dv, size_v, 4 * rr + 40 + (rows if shared else 0), "dv")
    grads = [dU, dF, dV] + ([dW] if second else [])
    first = [dz_of(d) for d in grads]
    for d in grads:
        assert np.array_equal(dzs_of(d), dz_of(d).conj())
    run(1, False)
    for d, a in zip(grads, first):
        assert np.array_equal(dz_of(d), 2 * a) and np.array_equal(dzs_of(d), a.conj())
    for p in [H.re, H.im, Y.re, Y.im] + dU.planes + dF.planes + dV.planes + dW.planes:
        assert untouched(p)


def test_norm_join_gradient_against_differences(gpu):
    """L = sum |y - a|^2 + sum |h - b|^2 in 64 bits, moved along random directions of every input"""
    rng = np.random.default_rng(3)
    rows, cols = 6, 90
    u, f, v, w, a, b = (rnd(rng, r, cols) for r in (rows, rows, 1, 1, rows, rows))

    def forward(u, f, v, w):
        h = u + SCALE * v * f * inv_rms(f)
        return h, w * h * inv_rms(h)

    def loss(*args):
        h, y = forward(*args)
        return (np.abs(y - a) ** 2).sum() + (np.abs(h - b) ** 2).sum()
    U, F, V, W = (cmat(z, cols) for z in (u, f, v, w))
    H, Y, s, s2 = cmat(0 * u, cols), cmat(0 * u, cols), capi.empty(rows), capi.empty(rows)
    ops.norm_join_fwd(U, F, V, SCALE, H, s, W, Y, s2, EPS)
    gy, gh = (cval(Y) - a).conj(), (cval(H) - b).conj()      # dL/dz of |z|^2 is conj z
    dU, dF, dV, dW = grad(u.shape, cols), grad(u.shape, cols), grad(v.shape, cols), grad(w.shape, cols)
    ops.norm_join_bwd_sym(F, s, V, SCALE, H, s2, W, cmat(gh, cols), cmat(gy, cols), dU, dF, dV, dW)
    step = 1e-5
    for k, d in enumerate((dU, dF, dV, dW)):
        arg = [u, f, v, w]
        r = rnd(rng, *arg[k].shape)
        hi, lo = list(arg), list(arg)
        hi[k], lo[k] = arg[k] + step * r, arg[k] - step * r
        want = (loss(*hi) - loss(*lo)) / (2 * step)
        got = 2 * (dz_of(d) * r).sum().real
        # third order of the difference, and the fp32 gradient: 1e-4 of the terms' size
        assert abs(got - want) <= 1e-4 * 2 * (np.abs(dz_of(d)) * np.abs(r)).sum(), (k, got, want)


def test_norm_rows_of_zeros_nan_and_large_values(gpu):
    rows, cols = 6, 260
    rng = np.random.default_rng(9)
    x = rnd(rng, rows, cols)
    x[1] = 0                          # no length: y = 0 and a gradient of eps' scale, no NaN
    x[2, 7] = np.nan
    x[4] *= 1e15                      # |x|^2 = 1e30, its mean still a number
    x[5] *= 1e-12
    x = x.real.astype(np.float32).astype(np.float64) + 1j * x.imag.astype(np.float32)
    v, g = rnd(rng, rows, cols, 0.3, 1.0), rnd(rng, rows, cols)
    for eps in (0.0, EPS):
        X, V, Y, s = cmat(x, cols), cmat(v, cols), cmat(0 * x, cols), capi.empty(rows)
        ops.norm_gate_fwd(X, V, Y, s, eps, shared=False)
        dX, dV = grad(x.shape, cols), grad(x.shape, cols)
        ops.norm_gate_bwd_sym(X, s, V, cmat(g, cols), dX, dV, shared=False)
        ok = [0, 1, 3, 4, 5]
        want = inv_rms(x[ok], eps)
        close(cval(Y)[ok], v[ok] * x[ok] * want, np.abs(v[ok] * x[ok]) * want, 40, "y")
        dx, _, size, _ = back(x[ok], want, v[ok], g[ok])
        close(dz_of(dX)[ok], dx, size, 80, "dx")
        assert np.all(cval(Y)[1] == 0) and np.all(np.isnan(cval(Y)[2]))


def test_norm_same_bits_again_and_in_a_graph(gpu):
    rng = np.random.default_rng(11)
    rows, cols = 700, 1024
    F, V, H, W, GH, GY = (cmat(rnd(rng, r, cols), cols) for r in (rows, 1, rows, 1, rows, rows))
    U, Y = cmat(rnd(rng, rows, cols), cols), cmat(np.zeros((rows, cols)), cols)
    s, s2 = capi.empty(rows), capi.empty(rows)
    dU, dF, dV, dW = grad((rows, cols), cols), grad((rows, cols), cols), grad((1, cols), cols), grad((1, cols), cols)

    def step():
        ops.norm_join_fwd(U, F, V, SCALE, H, s, W, Y, s2, EPS)
        ops.norm_join_bwd_sym(F, s, V, SCALE, H, s2, W, GH, GY, dU, dF, dV, dW)

    def results():
        return [cval(Y), s.download(), s2.download()] + [dz_of(d) for d in (dU, dF, dV, dW)]
    step()
    want = results()
    capi.call("cnet_graph_begin")
    step()
    exe = C.c_void_p()
    capi.call("cnet_graph_end", C.byref(exe))
    for _ in range(3):
        for d in (dU, dF, dV, dW):
            for p in d.planes:
                p.owner.zero()
        big = [grad((2000, cols), cols), grad((1, cols), cols)]      # eager work in between, on a larger workspace
        ops.norm_gate_bwd_sym(cmat(np.ones((2000, cols)), cols), capi.zeros(2000), V, cmat(np.ones((2000, cols)), cols), *big)
        capi.sync()
        capi.call("cnet_graph_launch", exe)
        for a, b in zip(results(), want):
            assert np.array_equal(a, b)
    capi.call("cnet_graph_destroy", exe)


def test_norm_no_rows(gpu):
    cols = 33
    V, W, z = cmat(np.ones((1, cols)), cols), cmat(np.ones((1, cols)), cols), ops.CMat.empty(1, cols)
    none = ops.CMat(z.re.rows_from(0, 0), z.im.rows_from(0, 0))
    none.rows = 0
    none_g = ops.Grad([p.rows_from(0, 0) for p in grad((1, cols), cols).planes])
    s = capi.empty(1)
    ops.norm_gate_fwd(none, V, none, s, EPS)
    ops.norm_join_fwd(none, none, V, SCALE, none, s, W, none, s, EPS)
    dV, dW = grad((1, cols), cols, fill=3.0), grad((1, cols), cols, fill=3.0)
    ops.norm_join_bwd_sym(none, s, V, SCALE, none, s, W, none, none, none_g, none_g, dV, dW, accumulate_w=1)
    assert np.all(dz_of(dV) == 3 + 3j)
    ops.norm_join_bwd_sym(none, s, V, SCALE, none, s, W, none, none, none_g, none_g, dV, dW)
    assert all(not values(p).any() for p in dV.planes + dW.planes)
    dV = grad((1, cols), cols, fill=3.0)
    ops.norm_gate_bwd_sym(none, s, V, none, none_g, dV)
    assert all(not values(p).any() for p in dV.planes)


def test_norm_refusals(gpu):
    lib = capi.load()
    rows, cols = 4, 8
    x, v, y, g = (ops.CMat.empty(rows, cols, zero=True) for _ in range(4))
    s = capi.zeros(rows)
    d, dv = ops.Grad.empty(rows, cols), ops.Grad.empty(rows, cols)

    def fwd(x_im=x.im.ptr, ldx=8, ldv=8, y_re=y.re.ptr, ldy=8, rows=rows, cols=cols, eps=EPS):
        return lib.cnet_norm_gate_fwd(x.re.ptr, x_im, ldx, *v.p(), ldv, y_re, y.im.ptr, ldy, s.ptr, rows, cols, eps)
    assert fwd() == 0 and fwd(ldv=0) == 0 and fwd(rows=0) == 0
    assert INVALID == fwd(x_im=None) == fwd(ldx=7) == fwd(ldv=7) == fwd(y_re=None) == fwd(ldy=7) == fwd(rows=-1) == fwd(cols=0) == fwd(rows=1 << 22)
    assert INVALID == fwd(eps=-1.0) == fwd(eps=float("nan")) == fwd(eps=float("inf")) and b"cnet_norm_gate_fwd" in lib.cnet_last_error()

    def bwd(s_=s.ptr, g_im=g.im.ptr, ldg=8, dzs=d.planes[3].ptr, lddx=8, dv_re=dv.planes[0].ptr, lddv=8):
        return lib.cnet_norm_gate_bwd_sym(*x.p(), 8, s_, *v.p(), 8, g.re.ptr, g_im, ldg, *d.p()[:3], dzs, lddx, dv_re, *dv.p()[1:], lddv, rows, cols, 0, 0)
    assert bwd() == 0
    assert INVALID == bwd(s_=None) == bwd(g_im=None) == bwd(ldg=7) == bwd(dzs=None) == bwd(lddx=7) == bwd(dv_re=None) == bwd(lddv=7)

    def join(u_re=x.re.ptr, h_im=y.im.ptr, ldh=8, w=v.p(), y2=g.p(), ldy=8, eps=EPS):
        return lib.cnet_norm_join_fwd(u_re, x.im.ptr, 8, *x.p(), 8, *v.p(), 0, 1.0, y.re.ptr, h_im, ldh, s.ptr, *w, *y2, ldy, s.ptr, rows, cols, eps)
    none = (None, None)
    assert join() == 0 and join(w=none, y2=none, ldy=0) == 0
    assert INVALID == join(u_re=None) == join(h_im=None) == join(ldh=7) == join(w=none) == join(y2=none) == join(y2=(g.re.ptr, None)) == join(ldy=7)

    def jback(gh=g.p(), gy=g.p(), h_re=y.re.ptr, s2=s.ptr, w_im=v.im.ptr, du_im=d.planes[1].ptr, df_dzs=d.planes[3].ptr, dw=dv.p(), lddu=8):
        return lib.cnet_norm_join_bwd_sym(*x.p(), 8, s.ptr, *v.p(), 0, 1.0, h_re, y.im.ptr, 8, s2, v.re.ptr, w_im, *gh, 8, *gy, 8,
                                          d.planes[0].ptr, du_im, *d.p()[2:], lddu, *d.p()[:3], df_dzs, 8, *dv.p(), 8, *dw, rows, cols, 0, 0)
    assert jback() == 0 and jback(gh=none) == 0 and jback(gy=none, dw=(None,) * 4) == 0 and jback(gy=none, h_re=None, s2=None, w_im=None) == 0
    assert INVALID == jback(gh=none, gy=none) == jback(gh=(g.re.ptr, None)) == jback(h_re=None) == jback(s2=None) == jback(w_im=None)
    assert INVALID == jback(du_im=None) == jback(df_dzs=None) == jback(dw=(None,) * 4) == jback(lddu=7)
