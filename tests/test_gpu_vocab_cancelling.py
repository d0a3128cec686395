"""The vocabulary head on rows of x in directions that the rows of w hardly have: sum |z|^2 is then far smaller than the terms that a
quadratic form of x makes it from.  Loss and gradients are compared with 64 bits."""
import os
import subprocess
import sys

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


HALF = 2.0 ** -24
HALF64 = 2.0 ** -53


def shared_axis(B, K, N, weak, seed=15):
    """rows of w that are one strong direction plus a little noise; a third of the rows of x orthogonal to it, a third at 1/50 of their terms,
    a third as they come"""
    rng = np.random.default_rng(seed)
    axis = np.ones(K) / np.sqrt(K)
    w = rounded(rnd(rng, N, 1) * axis + weak * rnd(rng, N, K, (2 * K) ** -0.5))
    x = rnd(rng, B, K)
    x[::3] -= (x[::3] @ axis)[:, None] * axis
    x[1::3] = rows_at(x[1::3], w.conj().T @ w, axis, 1 / 50)
    labels = rng.integers(0, N, B).astype(np.int32)
    labels[5] = -1
    labels[B // 2:B // 2 + 20] = 3
    return rounded(x), w, labels


def shared_rows(B, K, N, weak, seed=16):
    """the other way round: a batch along one direction, and rows of w that are orthogonal to it"""
    rng = np.random.default_rng(seed)
    axis = np.ones(K) / np.sqrt(K)
    x = rounded(rnd(rng, B, 1) * axis * 3 + weak * rnd(rng, B, K))
    w = rnd(rng, N, K, (2 * K) ** -0.5)
    w[::2] -= (w[::2] @ axis)[:, None] * axis
    labels = (rng.integers(0, N // 2, B) * 2 + 1).astype(np.int32)
    labels[5] = -1
    return x, rounded(w), labels


def sizes(x, w, labels):
    """What each row's roundings are measured against: of dx and dw without any cancellation inside (conj(z) w / S as it comes out, and the
    label's term), and D / S, the terms of sum |z|^2 as a quadratic form of x against what is left of them."""
    ref = head_ref(x, w, labels)
    z = x @ w.T
    live = (labels >= 0)[:, None] / ref["s"][:, None]
    ref["y"] = np.abs(z.conj() @ w) * live
    ref["z_dw"] = (np.abs(z) * live).T @ np.abs(x)
    ref["lost"] = (np.abs(x) ** 2 @ (np.abs(w) ** 2).sum(0)) / ref["s"]
    T = (np.abs(w) ** 2).sum(0)
    ref["terms_dx"] = np.sqrt(ref["lost"][:, None] * T[None, :] / ref["s"][:, None]) * (labels >= 0)[:, None]
    P = ((np.abs(x) ** 2) * live).sum(0)
    ref["terms_dw"] = np.sqrt((np.abs(w) ** 2 @ P)[:, None] * P[None, :])
    return ref


def direct(x, w, labels, ref):
    """the same gradients from logits in single precision (numpy's), the label's term apart and in 64 bits"""
    x32, w32 = x.astype(np.complex64), w.astype(np.complex64)
    z = x32 @ w32.T
    live = (labels >= 0)[:, None]
    s = np.maximum((z.real.astype(np.float64) ** 2 + z.imag.astype(np.float64) ** 2).sum(1), 1e-15)[:, None]
    g = (z.conj() / s.astype(np.float32) * live).astype(np.complex64)
    at = np.where(labels >= 0, labels, 0)
    dx = (g @ w32).astype(np.complex128) - ref["c"][:, None] * w[at]
    dw = (g.T @ x32).astype(np.complex128)
    np.subtract.at(dw, at, ref["c"][:, None] * x)
    return s[:, 0], dx, dw


def norms(a):
    return np.linalg.norm(a, axis=1)


def as_direct(err, scale):
    """What fp32 logits may be off by, row by row, from what numpy's are off by.  One row's error is one draw and may be near zero (of 200 rows
    some 16 lie within a tenth of the deviation), so a multiple of it bounds nothing; over `scale`, which they grow with, all rows'
    errors are of one size, and four times the largest of them bounds each."""
    some = scale > 0
    return 4 * (err[some] / scale[some]).max() * scale


def cancelling_check(x, w, labels, gram, pad=0, off=0, argmax=False):
    """gram: the call goes through w^H w, whose results are as good as rounded once; otherwise as good as those of fp32 logits."""
    B, K, N = len(x), x.shape[1], len(w)
    ref = sizes(x, w, labels)
    X, W, L = cmat(x, K + pad + off, off), cmat(w, K + pad + off, off), ops.ints(labels)
    s, loss, am = capi.empty(B), capi.empty(B), capi.empty(B, np.int32) if argmax else None
    dX, dW = grad(x.shape, K + pad + off, off), grad(w.shape, K + pad + off, off)
    ops.vocab_head_fwd_bwd_sym(X, W, L, s, loss, am, dX, dW)
    s32, dx32, dw32 = direct(x, w, labels, ref)
    # sums in double: sqrt of their length in roundings of 2^-53, at three times its deviation, on the terms; then 2^-24 for s
    in_double = 3 * np.sqrt(K + N) * HALF64
    off_s = HALF + in_double * ref["lost"]
    # (the sum over fp32 logits: relative error by the square root of D / S)
    loose_s = off_s + as_direct(np.abs(s32 - ref["s"]) / ref["s"] + HALF, np.sqrt(ref["lost"]))
    err = np.abs(s.download() - ref["s"]) / ref["s"]
    assert np.all(err <= (off_s if gram else loose_s)), (err / off_s).max()
    ok = labels >= 0
    err = np.abs(loss.download() - ref["loss"])[ok]
    assert np.all(err <= ((off_s if gram else loose_s) + 4 * HALF * (1 + np.abs(ref["loss"])))[ok])
    # dx: y rounded, 1 / S (with S's error), their product, c, its product (2), the difference
    size = norms(ref["y"] + ref["label_dx"])
    allowed = 6 * HALF * size + off_s * norms(ref["y"]) + in_double * norms(ref["terms_dx"])
    err = norms(dz_of(dX) - ref["dx"])
    bound = allowed if gram else allowed + as_direct(norms(dx32 - ref["dx"]) + HALF * size, norms(ref["y"]) * np.sqrt(ref["lost"])) + 16 * HALF * size
    assert np.all(err <= bound), (float((err / bound).max()), int((err / bound).argmax()))
    # dw: rounded, the label's rows summed up (their number in roundings) and subtracted
    count = np.bincount(labels[ok], minlength=N)
    size = norms(ref["z_dw"] + ref["label_dw"])
    weights = (np.abs(x @ w.T) * ((labels >= 0) * off_s / ref["s"])[:, None]).T @ np.abs(x)
    allowed = 3 * HALF * size + (6 + count) * HALF * norms(ref["label_dw"]) + norms(weights) + 3 * np.sqrt(K + B) * HALF64 * norms(ref["terms_dw"])
    err = norms(dz_of(dW) - ref["dw"])
    bound = allowed if gram else allowed + as_direct(norms(dw32 - ref["dw"]) + HALF * size, norms(ref["terms_dw"])) + 16 * HALF * size
    assert np.all(err <= bound), (float((err / bound).max()), int((err / bound).argmax()))
    assert not dz_of(dX)[labels < 0].any()
    # the forward pass alone, with and without the argmax
    for best in (None, capi.empty(B, np.int32)):
        s2, loss2 = capi.empty(B), capi.empty(B)
        ops.vocab_head_fwd(X, W, L, s2, loss2, best)
        err = np.abs(s2.download() - ref["s"]) / ref["s"]
        # (the argmax needs the logits, and up to 64 rows are scored in one pass over w whatever the override: fp32 logits)
        allowed = off_s if gram and best is None and B > 64 else loose_s
        assert np.all(err <= allowed), (err / allowed).max()
        assert np.all(np.abs(loss2.download() - ref["loss"])[ok] <= (allowed + 4 * HALF * (1 + np.abs(ref["loss"])))[ok])


WEAK = [1e-1, 1e-2, 1e-3, 1e-5]
# B, K, N, padding of the leading dimensions, offset of the first element
CANCELLING = [(600, 64, 1000, 0, 0), (300, 160, 16000, 0, 0), (2000, 100, 3001, 3, 1)]


@pytest.mark.parametrize("B,K,N,pad,off", CANCELLING)
@pytest.mark.parametrize("weak", WEAK)
@pytest.mark.parametrize("argmax", [False, True])
def test_vocab_head_gradients_where_the_terms_of_a_row_cancel(gpu, B, K, N, pad, off, weak, argmax):
    cancelling_check(*shared_axis(B, K, N, weak), False, pad, off, argmax)


@pytest.mark.parametrize("B,K,N,pad,off", CANCELLING)
@pytest.mark.parametrize("weak", [1e-1, 1e-2, 1e-3])
def test_vocab_head_gradients_where_the_terms_of_an_entry_cancel(gpu, B, K, N, pad, off, weak):
    cancelling_check(*shared_rows(B, K, N, weak), False, pad, off)


def test_vocab_head_through_the_gram_matrix_is_rounded_once(gpu):
    """whatever the sizes (CNET_HEAD_GRAM is read once, so in a process of its own), and whatever cancels"""
    script = os.path.join(os.path.dirname(os.path.abspath(__file__)), "gpu_vocab_cancelling_check.py")
    res = subprocess.run([sys.executable, script], env={**os.environ, "CNET_HEAD_GRAM": "1"}, capture_output=True, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip().endswith("ok"), res.stdout[-500:] + res.stderr[-2000:]
