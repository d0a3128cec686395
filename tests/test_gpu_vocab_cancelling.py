"""The vocabulary head on rows of x in directions that the rows of w hardly have: sum |z|^2 is then far smaller than the terms that a
quadratic form of x makes it from.  Loss and gradients are compared with 64 bits."""
import numpy as np
import pytest

from cnet_amd import capi, ops
from tests.gpu_util import gpu  # noqa: F401
from tests.test_gpu_norm import cmat, dz_of, dzs_of, grad, rnd
from tests.test_gpu_vocab import head_ref

pytestmark = pytest.mark.gpu


def rounded(z):
    return z.real.astype(np.float32).astype(np.float64) + 1j * z.imag.astype(np.float32)


def rows_at(x, T, axis, share):
    """x moved along `axis` until sum |z|^2 = x T x^H is `share` of sum |x_i|^2 T_ii"""
    base = x - (x @ axis.conj())[:, None] * axis
    lo, hi = np.zeros(len(x)), np.full(len(x), np.linalg.norm(x, axis=1).max())
    for _ in range(60):
        mid = (lo + hi) / 2
        y = base + mid[:, None] * axis
        s = ((y.conj() @ T) * y).sum(1).real
        less = s < share * (np.abs(y) ** 2 @ T.diagonal().real)
        lo, hi = np.where(less, mid, lo), np.where(less, hi, mid)
    return base + hi[:, None] * axis


def test_vocab_head_rows_between_two_ways_are_written_once(gpu):
    """Rows whose sum is 1 / 64 of its terms to the last bits: whatever is decided about such a row is decided for all of it."""
    rng = np.random.default_rng(21)
    B, K, N = 4000, 64, 1000
    axis = np.ones(K) / np.sqrt(K)
    w = rounded(rnd(rng, N, 1) * axis + 1e-2 * rnd(rng, N, K, (2 * K) ** -0.5))
    x = rounded(rows_at(rnd(rng, B, K), w.conj().T @ w, axis, 1 / 64))
    labels = rng.integers(0, N, B).astype(np.int32)
    ref = head_ref(x, w, labels)
    s, loss, dX, dW = capi.empty(B), capi.empty(B), grad(x.shape, K, fill=0.0), grad(w.shape, K)
    for times in (1, 2):                                   # (the second call adds)
        ops.vocab_head_fwd_bwd_sym(cmat(x, K), cmat(w, K), ops.ints(labels), s, loss, None, dX, dW, accumulate_dx=1, accumulate_dw=times - 1)
        # fp32 products of rows whose terms cancel to a 64th: 2^-24 x 64 x (K + N) roundings are 4e-3; what is written twice or not at
        # all is off by the whole of a row's entry
        got, want = dz_of(dX), times * ref["dx"]
        assert np.all(np.linalg.norm(got - want, axis=1) <= 1e-2 * np.linalg.norm(want, axis=1))
        assert np.linalg.norm(dz_of(dW) - times * ref["dw"]) <= 1e-2 * np.linalg.norm(times * ref["dw"])
        assert np.array_equal(dzs_of(dX), got.conj())
    assert np.allclose(s.download(), ref["s"], rtol=1e-2)
