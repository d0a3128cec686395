"""The norms around a block at the ends of single precision."""
import numpy as np
import pytest

from cnet_amd import capi, ops
from tests.gpu_util import gpu  # noqa: F401
from tests.test_gpu_norm import EPS, SCALE, back, close, cmat, cval, dz_of, grad, inv_rms, rnd, row_roundings

pytestmark = pytest.mark.gpu

# every kernel of the forward and the backward pass: by width, and by 128-bit accesses or not
WIDTHS = [(64, 0), (333, 0), (512, 4), (1001, 1), (2048, 0), (4096, 0), (4095, 0), (8192, 0), (16384, 0), (16500, 0)]


def rounded(z):
    return z.real.astype(np.float32).astype(np.float64) + 1j * z.imag.astype(np.float32)


@pytest.mark.parametrize("cols,pad", WIDTHS)
def test_norm_rows_whose_squares_leave_single_precision(gpu, cols, pad):
    """Rows of 1e19 to 1e38 are as finite as any: y has the rows' direction and length, and so have h and the gradients."""
    rng = np.random.default_rng(cols)
    rows = 6
    x, v, g = rnd(rng, rows, cols, 0.7), rnd(rng, 1, cols, 0.3, 1.0), rnd(rng, rows, cols, 0.01)
    w = rnd(rng, 1, cols, 0.2, 1.0)
    x = rounded(np.clip(x.real, -3, 3) * np.array([1e19, 3e19, 1e25, 1e30, 1e37, 1.0])[:, None]
                + 1j * np.clip(x.imag, -3, 3) * np.array([1e19, 3e19, 1e25, 1e30, 1e37, 1.0])[:, None])
    X, V, G, W = cmat(x, cols + pad), cmat(v, cols + pad), cmat(g, cols + pad), cmat(w, cols + pad)
    Y, s = cmat(0 * x, cols + pad), capi.empty(rows)
    ops.norm_gate_fwd(X, V, Y, s, EPS)
    want, rr = inv_rms(x), row_roundings(cols)
    close(s.download()[:, None], want, want, rr, "s")
    close(cval(Y), v * x * want, np.abs(v) * np.abs(x) * want, rr + 12, "y")
    dX, dV = grad(x.shape, cols + pad), grad(v.shape, cols + pad)
    ops.norm_gate_bwd_sym(X, s, V, G, dX, dV)
    dx, dv, size, size_v = back(x, want, v, g)
    close(dz_of(dX), dx, size, 3 * rr + 16, "dx")
    close(dz_of(dV), dv.sum(0, keepdims=True), size_v.sum(0, keepdims=True), rr + 16 + rows, "dv")
    # the residual path carries such a row into the second norm
    f = rnd(rng, rows, cols, 0.7)
    H, Y2, s1, s2 = cmat(0 * x, cols + pad), cmat(0 * x, cols + pad), capi.empty(rows), capi.empty(rows)
    ops.norm_join_fwd(X, cmat(f, cols + pad), V, SCALE, H, s1, W, Y2, s2, EPS)
    h = cval(H)
    want2 = inv_rms(h)
    close(s2.download()[:, None], want2, want2, rr, "s2")
    close(cval(Y2), w * h * want2, np.abs(w) * np.abs(h) * want2, rr + 12, "y2")
    assert np.abs(cval(Y2)).max(1).min() > 0.1


@pytest.mark.parametrize("cols,pad", WIDTHS)
def test_norm_gradient_of_rows_at_the_clamp(gpu, cols, pad):
    """A row whose rms is below 1e-15 (eps = 0) is scaled by 1e15 whatever it is: y is linear in it, and so is what comes back."""
    rng = np.random.default_rng(cols + 1)
    rows = 5
    size = np.array([6e-16, 3e-16, 0.7, 0.0, 2e-15])[:, None]           # clamped, clamped, not, a row of zeros, not
    x = rounded(rnd(rng, rows, cols, 0.7) * size)
    s_w = inv_rms(x, 0.0)
    held = (s_w >= 0.9999e15)[:, 0]
    assert list(held) == [True, True, False, True, False]
    v, w, g = rnd(rng, 1, cols, 0.3, 1.0), rnd(rng, 1, cols, 0.2, 1.0), rnd(rng, rows, cols)
    ld, rr = cols + pad, row_roundings(cols)
    X, V, Y, s = cmat(x, ld), cmat(v, ld), cmat(0 * x, ld), capi.empty(rows)
    ops.norm_gate_fwd(X, V, Y, s, 0.0)
    close(s.download()[:, None], s_w, s_w, rr, "s")
    dX, dV = grad(x.shape, ld), grad(v.shape, ld)
    ops.norm_gate_bwd_sym(X, s, V, cmat(g, ld), dX, dV)
    dx, dv, bound, size_v = back(x, s_w, v, g)
    dx = np.where(held[:, None], s_w * v * g, dx)                       # dL/dx of y = v x 1e15
    close(dz_of(dX), dx, bound, 3 * rr + 16, "dx")
    close(dz_of(dV), dv.sum(0, keepdims=True), size_v.sum(0, keepdims=True), rr + 16 + rows, "dv")
    # the join's second norm: h = u + scale v f s1 below the clamp in some rows
    scale = 2.0 ** -52
    f, u, gh = rnd(rng, rows, cols, 0.7), rounded(rnd(rng, rows, cols) * np.array([1e-16, 0.0, 1.0, 4e-16, 1e-3])[:, None]), rnd(rng, rows, cols)
    H, Y2, s1, s2 = cmat(0 * u, ld), cmat(0 * u, ld), capi.empty(rows), capi.empty(rows)
    F, W = cmat(f, ld), cmat(w, ld)
    ops.norm_join_fwd(cmat(u, ld), F, V, scale, H, s1, W, Y2, s2, 0.0)
    h = cval(H)
    s1_w, s2_w = inv_rms(f, 0.0), inv_rms(h, 0.0)
    held = (s2_w >= 0.9999e15)[:, 0]
    assert list(held) == [True, True, False, True, False]
    dU, dF, dV, dW = grad(u.shape, ld), grad(u.shape, ld), grad(v.shape, ld), grad(w.shape, ld)
    ops.norm_join_bwd_sym(F, s1, V, scale, H, s2, W, cmat(gh, ld), cmat(g, ld), dU, dF, dV, dW)
    dh, _, bound, _ = back(h, s2_w, w, g)
    dh = np.where(held[:, None], s2_w * w * g, dh) + gh
    bound = bound + np.abs(gh)
    close(dz_of(dU), dh, bound, 3 * rr + 20, "du")
    df, _, _, _ = back(f, s1_w, scale * v, dh)
    _, _, bound, _ = back(np.abs(f), s1_w, scale * np.abs(v), bound)
    close(dz_of(dF), df, bound, 8 * rr + 40, "df")


def test_norm_and_vocabulary_refuse_rows_that_32_bit_columns_cannot_walk(gpu):
    """A thread's next column has to stay within 32 bits behind the row's end: 2^30 columns and more are refused before anything is read."""
    lib, wide, p, invalid = capi.load(), 1 << 30, capi.zeros(4).ptr, -2
    for cols in (wide, (1 << 31) - 1):
        ld = 1 << 31
        assert lib.cnet_norm_gate_fwd(p, p, ld, p, p, 0, p, p, ld, None, 1, cols, EPS) == invalid
        assert lib.cnet_norm_gate_bwd_sym(p, p, ld, p, p, p, 0, p, p, ld, p, p, None, None, ld, p, p, None, None, ld, 1, cols, 0, 0) == invalid
        assert lib.cnet_norm_join_fwd(p, p, ld, p, p, ld, p, p, 0, 1.0, p, p, ld, None, None, None, None, None, 0, None, 1, cols, EPS) == invalid
        assert lib.cnet_norm_join_bwd_sym(p, p, ld, p, p, p, 0, 1.0, None, None, 0, None, None, None, p, p, ld, None, None, 0, p, p, None, None, ld,
                                          p, p, None, None, ld, p, p, None, None, ld, None, None, None, None, 1, cols, 0, 0) == invalid
        assert lib.cnet_distill_fwd(p, p, ld, p, p, 1, p, p, 1, cols) == invalid
        assert lib.cnet_distill_bwd_sym(p, p, ld, p, p, p, 1, p, p, None, None, ld, 1, cols) == invalid
        assert lib.cnet_distill_fwd_bwd_sym(p, p, ld, p, p, 1, p, p, p, p, None, None, ld, 1, cols) == invalid
        assert lib.cnet_vocab_head_fwd(p, p, ld, p, p, ld, p, p, p, p, 1, cols, 1) == invalid
        assert lib.cnet_vocab_head_fwd_bwd_sym(p, p, ld, p, p, ld, p, p, p, None, p, p, None, None, ld, 0, p, p, None, None, ld, 0, 1, cols, 1) == invalid
        assert b"cols < (1 << 30)" in lib.cnet_last_error() or b"K < (1 << 30)" in lib.cnet_last_error()
