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
