"""The losses of a vocabulary (cnet_distill_*, cnet_vocab_head_*) against their definitions in 64 bits.

Tolerances count roundings of 2^-24 (half a step of fp32, relative) against sums of absolute values.  A sum of n products takes at
most n roundings on its longest path; being as often up as down, they add up to about the square root of that over a whole
array, which is what `near` asks of the 2-norm (three times it), and no single element exceeds the longest path."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from cnet_amd import capi, ops
from tests.gpu_util import gpu  # noqa: F401
from tests.test_gpu_norm import HALF, INVALID, cmat, cval, close, dz_of, dzs_of, grad, rnd, untouched

pytestmark = pytest.mark.gpu

LEAST = 1e-15


def near(got, want, size, roundings, what):
    close(got, want, size, 2 * roundings, what)
    err, bound = np.linalg.norm(got - want), 3 * np.sqrt(2 * roundings) * HALF * np.linalg.norm(size)
    assert err <= bound, (what, err, bound)


# ------------------------------------------------------------------------------------------------ distillation
def distill_ref(z, ids, q):
    cols = z.shape[1]
    power = np.abs(z) ** 2
    s = np.maximum(power.sum(1), LEAST)
    q = np.where(ids >= 0, q, 0.0).astype(np.float64)
    loss, size = np.zeros(len(z)), np.zeros(len(z))
    k = np.repeat((q.sum(1) / s)[:, None], cols, 1)
    for r in range(len(z)):
        for j in range(ids.shape[1]):
            i = ids[r, j]
            if i < 0 or q[r, j] == 0:
                continue
            if i >= cols:
                loss[r] = np.nan
                continue
            p = max(power[r, i] / s[r], LEAST)
            loss[r] += q[r, j] * np.log(q[r, j] / p)
            size[r] += q[r, j] * (1 + abs(np.log(q[r, j] / p)))
            k[r, i] -= q[r, j] / max(power[r, i], LEAST)
    return s, loss, z.conj() * k, size


def teacher(rng, rows, cols, top, pad=True):
    ids = np.stack([rng.permutation(max(cols, top))[:top] % cols for _ in range(rows)]).astype(np.int32)
    q = rng.random((rows, top)).astype(np.float32) ** 3 + np.float32(1e-3)
    q = (q / q.sum(1, keepdims=True) * 0.9).astype(np.float32)
    if pad and top > 1:
        ids[rows // 2, top // 2:] = -1                   # padding behind a shorter list
        q[rows // 3, 0] = 0                              # an entry without weight
    if rows > 2:
        ids[2] = -1                                      # a row of padding
    return ids, q


DISTILL = [(1, 1, 1, 0, 0), (1, 5, 3, 0, 1), (4, 64, 8, 0, 0), (7, 333, 9, 3, 1), (96, 512, 8, 0, 0), (5, 1001, 64, 2, 0), (300, 700, 4, 4, 0),
           (3, 4096, 300, 0, 0), (6, 8200, 1024, 0, 0), (3, 20000, 7, 0, 0), (2, 33000, 50, 0, 0), (1, 100003, 64, 0, 0), (5, 131072, 16, 4, 4),
           (1030, 36, 2, 0, 0), (65, 32772, 5, 0, 0), (66, 33001, 33, 0, 0), (64, 9000, 3, 0, 0), (63, 9001, 3, 0, 0), (2, 300000, 9, 0, 0)]


@pytest.mark.parametrize("rows,cols,top,pad,off", DISTILL)
def test_distill(gpu, rows, cols, top, pad, off):
    rng = np.random.default_rng(rows + cols + top)
    ld = cols + pad + off
    z = rnd(rng, rows, cols)
    ids, q = teacher(rng, rows, cols, top)
    if cols > 4 and top > 2:
        ids[0, 0] = ids[0, 2] = 3                        # the same index twice
        z[0, ids[0, 1]] = 0                              # an entry the student gives no probability at all
    s_w, loss_w, dz_w, size = distill_ref(z, ids, q)
    Z, I, Q = cmat(z, ld, off), ops.ints(ids), capi.to_device(q)
    s, loss, dz = capi.empty(rows), capi.empty(rows), grad(z.shape, ld, off)
    ops.distill_fwd_bwd_sym(Z, I, Q, top, s, loss, dz)
    close(s.download(), s_w, s_w, 2, "s")
    close(loss.download(), loss_w, size, top + 16, "loss")
    k = np.abs(z) * (np.abs(np.where(ids >= 0, q, 0)).sum(1) / s_w)[:, None]
    close(dz_of(dz), dz_w, np.abs(dz_w) + 2 * k, top + 16, "dz")
    assert np.array_equal(dzs_of(dz), dz_of(dz).conj())
    both = s.download(), loss.download(), dz_of(dz)
    # the two halves alone: the same bits, the dz* half left as it was
    s2, loss2, dz2 = capi.empty(rows), capi.empty(rows), grad(z.shape, ld, off, fill=5.0)
    ops.distill_fwd(Z, I, Q, top, s2, loss2)
    ops.distill_bwd_sym(Z, s2, I, Q, top, dz2, mirror=False)
    assert np.array_equal(s2.download(), both[0]) and np.array_equal(loss2.download(), both[1]) and np.array_equal(dz_of(dz2), both[2])
    assert np.all(dzs_of(dz2) == 5 + 5j)
    for p in [Z.re, Z.im] + dz.planes + dz2.planes:
        assert untouched(p)


def test_distill_with_one_entry_is_cross_entropy(gpu):
    rng = np.random.default_rng(2)
    rows, cols = 9, 700
    z = rnd(rng, rows, cols)
    labels = rng.integers(0, cols, rows).astype(np.int32)
    labels[3] = cols + 5                                  # outside the row: a NaN loss, no label entry
    Z, L = cmat(z, cols), ops.ints(labels)
    s, loss, dz = capi.empty(rows), capi.empty(rows), grad(z.shape, cols)
    ops.distill_fwd_bwd_sym(Z, L, capi.to_device(np.ones((rows, 1), np.float32)), 1, s, loss, dz)
    s2, loss2, am, dz2 = capi.empty(rows), capi.empty(rows), capi.empty(rows, np.int32), grad(z.shape, cols)
    ops.cross_entropy_fwd_bwd_sym(Z, L, s2, loss2, am, dz2)
    a, b = loss.download(), loss2.download()
    assert np.isnan(a[3]) and np.isnan(b[3])
    ok = np.arange(rows) != 3
    assert np.array_equal(s.download(), s2.download())
    close(a[ok], b[ok].astype(np.float64), 1 + np.abs(b[ok]), 8, "loss")
    close(dz_of(dz), dz_of(dz2), np.abs(dz_of(dz2)) + np.abs(z) / s.download()[:, None], 10, "dz")


def test_distill_gradient_against_differences(gpu):
    rng = np.random.default_rng(4)
    rows, cols, top = 4, 60, 6
    z = rnd(rng, rows, cols)
    ids, q = teacher(rng, rows, cols, top, pad=False)
    s, loss, dz = capi.empty(rows), capi.empty(rows), grad(z.shape, cols)
    ops.distill_fwd_bwd_sym(cmat(z, cols), ops.ints(ids), capi.to_device(q), top, s, loss, dz)
    r = rnd(rng, rows, cols)
    step = 1e-6
    want = (distill_ref(z + step * r, ids, q)[1] - distill_ref(z - step * r, ids, q)[1]).sum() / (2 * step)
    got = 2 * (dz_of(dz) * r).sum().real
    assert abs(got - want) <= 1e-5 * (np.abs(dz_of(dz)) * np.abs(r)).sum()


def test_distill_rows_of_zeros_nan_and_extremes(gpu):
    rng = np.random.default_rng(5)
    rows, cols, top = 5, 130, 3
    z = rnd(rng, rows, cols)
    z[0] = 0                                              # both clamps
    z[1, 4] = np.nan
    z[3] *= 1e-9
    z[4] *= 1e17
    z = z.real.astype(np.float32).astype(np.float64) + 1j * z.imag.astype(np.float32)
    ids, q = teacher(rng, rows, cols, top, pad=False)
    s_w, loss_w, dz_w, size = distill_ref(z, ids, q)
    s, loss, dz = capi.empty(rows), capi.empty(rows), grad(z.shape, cols)
    ops.distill_fwd_bwd_sym(cmat(z, cols), ops.ints(ids), capi.to_device(q), top, s, loss, dz)
    for r in (0, 2, 3, 4):
        close(s.download()[r], s_w[r], s_w[r], 2, r)
        close(loss.download()[r], loss_w[r], size[r], 20, r)
        close(dz_of(dz)[r], dz_w[r], np.abs(dz_w[r]) * 2 + np.abs(z[r]) / s_w[r], 20, r)
    assert np.isnan(s.download()[1])


# ------------------------------------------------------------------------------------------------ vocabulary head
def head_ref(x, w, labels):
    """s, loss, argmax, dx, dw and what their roundings are measured against"""
    z = x @ w.T
    power = np.abs(z) ** 2
    s = np.maximum(power.sum(1), LEAST)
    size_z = np.abs(x) @ np.abs(w).T
    known, live = (labels >= 0) & (labels < len(w)), labels >= 0
    at = np.where(known, labels, 0)
    zl = z[np.arange(len(x)), at]
    m = np.maximum(np.abs(zl) ** 2, LEAST)
    loss = np.where(live, np.where(known, -np.log(np.maximum(m / s, LEAST)), np.nan), 0.0)
    c = np.where(known, zl.conj() / m, 0)
    g = z.conj() * (live / s)[:, None]
    g[np.arange(len(x)), at] -= c
    size_g = size_z * (live / s)[:, None]
    size_c = np.zeros_like(size_g)
    size_c[np.arange(len(x)), at] = np.abs(c)
    return dict(s=s, loss=loss, argmax=power.argmax(1), dx=g @ w, dw=g.T @ x, size_s=(power + 2 * np.abs(z) * size_z).sum(1), size_z=size_z,
                size_dx=size_g @ np.abs(w), size_dw=size_g.T @ np.abs(x), label_dx=size_c @ np.abs(w), label_dw=size_c.T @ np.abs(x), power=power,
                # what an error of the label's logit (its products are summed in double) does: relative 2^-24 of the exact terms
                c=c)


def head_data(rng, B, K, N, std=1.0):
    x, w = rnd(rng, B, K, std), rnd(rng, N, K, (2 * K) ** -0.5)
    labels = rng.integers(0, N, B).astype(np.int32)
    if B > 3:
        labels[1] = -1                                    # not trained on
        labels[2] = labels[3]                             # one label twice
    if B > 100:
        labels[40:90] = labels[40]                        # a frequent token
    if B > 8:
        labels[7] = N + 3                                 # outside the vocabulary
    return x, w, labels


def check_argmax(got, ref):
    """the index of a largest entry: of all that are within the logits' roundings of the largest"""
    best = ref["power"].max(1)
    mine = ref["power"][np.arange(len(got)), got]
    slack = 8 * np.sqrt(best) * ref["size_z"].max(1) * 40 * HALF
    assert np.all(mine >= best - slack)


def head_check(B, K, N, pad=0, off=0, argmax=True, data=None):
    rng = np.random.default_rng(B * 3 + K * 5 + N)
    x, w, labels = data or head_data(rng, B, K, N)
    ld = K + pad + off
    ref = head_ref(x, w, labels)
    X, W, L = cmat(x, ld, off), cmat(w, ld, off), ops.ints(labels)
    n = 2 * (K + N) + 64                                   # roundings on the longest path of a sum over both
    ok = np.isfinite(ref["loss"])

    def close_loss(loss, want, rows):
        # the label's logit has its products summed in double; what s is off by (its longest path, above) is off in the logarithm
        bad = np.abs(loss - want) > (2 * (2 * K + 32) * HALF * ref["size_s"] / ref["s"])[rows] + 8 * HALF * (1 + np.abs(want))
        assert not bad.any(), (loss[bad][:5], want[bad][:5])

    def check(s, loss, am):
        near(s, ref["s"], ref["size_s"], 2 * K + 32, "s")
        assert np.array_equal(np.isnan(loss), ~ok)
        close_loss(loss[ok], ref["loss"][ok], ok)
        if am is not None:
            check_argmax(am, ref)
        assert np.all(loss[labels < 0] == 0)
    s, loss, am = capi.empty(B), capi.empty(B), capi.empty(B, np.int32)
    ops.vocab_head_fwd(X, W, L, s, loss, am)
    check(s.download(), loss.download(), am.download())
    # scoring: no labels, the loss of the most likely entry
    s1, loss1, am1 = capi.empty(B), capi.empty(B), capi.empty(B, np.int32)
    ops.vocab_head_fwd(X, W, None, s1, loss1, am1)
    assert np.array_equal(am1.download(), am.download()) and np.array_equal(s1.download(), s.download())
    p = ref["power"][np.arange(B), am.download()] / ref["s"]
    close_loss(loss1.download(), -np.log(np.maximum(p, LEAST)), np.arange(B))
    # a training step
    s2, loss2, am2 = capi.empty(B), capi.empty(B), capi.empty(B, np.int32)
    dX, dW = grad(x.shape, ld, off), grad(w.shape, ld, off)
    ops.vocab_head_fwd_bwd_sym(X, W, L, s2, loss2, am2 if argmax else None, dX, dW)
    check(s2.download(), loss2.download(), am2.download() if argmax else None)
    label_n = 24 + np.bincount(labels[(labels >= 0) & (labels < N)], minlength=N).max()
    near(dz_of(dX), ref["dx"], ref["size_dx"] + label_n / n * ref["label_dx"], n, "dx")
    near(dz_of(dW), ref["dw"], ref["size_dw"] + label_n / n * ref["label_dw"], n + 2 * B, "dw")
    assert np.array_equal(dzs_of(dX), dz_of(dX).conj()) and np.array_equal(dzs_of(dW), dz_of(dW).conj())
    assert not np.any(dz_of(dX)[labels < 0])
    # a second call: the same bits again into other planes without the dz* halves, and added onto what is there
    dX2, dW2 = grad(x.shape, ld, off, fill=5.0), grad(w.shape, ld, off, fill=5.0)
    ops.vocab_head_fwd_bwd_sym(X, W, L, s2, loss2, am2 if argmax else None, dX2, dW2, mirror_dx=False, mirror_dw=False)
    assert np.array_equal(dz_of(dX2), dz_of(dX))
    near(dz_of(dW2), dz_of(dW), ref["size_dw"] + label_n / n * ref["label_dw"], n + 2 * B, "dw again")
    assert np.all(dzs_of(dX2) == 5 + 5j) and np.all(dzs_of(dW2) == 5 + 5j)
    first = dz_of(dX), dz_of(dW)
    ops.vocab_head_fwd_bwd_sym(X, W, L, s2, loss2, am2 if argmax else None, dX, dW, accumulate_dx=1, accumulate_dw=1)
    # (a product that goes out in two launches adds its parts to what is there one after the other: (a + b) + c in place of
    # a + (b + c), so the doubled sum may be rounded differently)
    near(dz_of(dX), 2 * first[0], 4 * (ref["size_dx"] + label_n / n * ref["label_dx"]), n, "dx twice")
    near(dz_of(dW), 2 * first[1], 4 * (ref["size_dw"] + label_n / n * ref["label_dw"]), n + 2 * B, "dw twice")
    assert np.array_equal(dzs_of(dW), dz_of(dW).conj())
    for pl in [X.re, X.im, W.re, W.im] + dX.planes + dW.planes + dX2.planes + dW2.planes:
        assert untouched(pl)


# B, K, N, padding of the leading dimensions, offset of the first element
HEAD = [(1, 1, 1, 0, 0), (3, 5, 7, 0, 0), (1, 64, 512, 0, 0), (2, 1024, 300, 0, 0), (16, 128, 1001, 0, 0), (17, 33, 130, 2, 1), (48, 256, 2000, 4, 0),
        (65, 100, 1000, 0, 0), (96, 64, 512, 0, 0), (513, 40, 300, 0, 0), (300, 96, 700, 0, 4), (700, 333, 1100, 3, 0), (1500, 64, 1024, 0, 0),
        (130, 512, 4099, 0, 0), (2100, 17, 19, 0, 0), (9000, 8, 40, 0, 0), (8200, 20, 3, 1, 0), (40, 1300, 64, 0, 0)]


@pytest.mark.parametrize("B,K,N,pad,off", HEAD)
@pytest.mark.parametrize("argmax", [True, False])
def test_vocab_head(gpu, B, K, N, pad, off, argmax):
    head_check(B, K, N, pad, off, argmax)


@pytest.mark.parametrize("env", [{"CNET_HEAD_GRAM": "0", "CNET_HEAD_PIECE_MB": "1"}, {"CNET_HEAD_GRAM": "1", "CNET_HEAD_PIECE_MB": "1"},
                                 {"CNET_HEAD_GRAM": "0"}, {"CNET_HEAD_GRAM": "1", "CNET_CGEMM_3M": "1"}])
def test_vocab_head_every_way(gpu, env):
    """through pieces of the logits, through the Gram matrix, and through whole logits, whatever the sizes"""
    script = os.path.join(os.path.dirname(os.path.abspath(__file__)), "gpu_vocab_head_check.py")
    res = subprocess.run([sys.executable, script], env={**os.environ, **env}, capture_output=True, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip().endswith("ok"), res.stdout[-500:] + res.stderr[-2000:]


@pytest.mark.parametrize("B,K,N,pad,off", [(900, 528, 1601, 0, 0), (700, 333, 4001, 3, 1), (4100, 320, 700, 0, 4), (400, 129, 24100, 0, 0)])
def test_vocab_head_half_of_a_gram_matrix(gpu, B, K, N, pad, off):
    """sizes at which T = w^H w, or P = x^H x / S, is formed above its diagonal and turned over; w in whole chunks of 16 rows and not"""
    head_check(B, K, N, pad, off, argmax=False)


def weak_data(B, K, N, weak, every=3):
    """rows of w that are one strong direction plus a little noise; every third row of x is orthogonal to that"""
    rng = np.random.default_rng(15)
    x, w, labels = head_data(rng, B, K, N)
    axis = np.ones(K) / np.sqrt(K)
    w = rnd(rng, N, 1) * axis + weak * w
    x[::every] -= (x[::every] @ axis)[:, None] * axis
    x, w = (z.real.astype(np.float32).astype(np.float64) + 1j * z.imag.astype(np.float32) for z in (x, w))
    labels[7] = 1
    return x, w, labels


@pytest.mark.parametrize("B,K,N", [(600, 64, 1000), (300, 160, 16000)])
@pytest.mark.parametrize("weak", [1e-1, 1e-3, 1e-6])
def test_vocab_head_rows_in_directions_that_the_weights_hardly_have(gpu, weak, B, K, N):
    """There the Gram matrix gives sum |z|^2 as a difference of large terms, and the rows are computed again from w."""
    head_check(B, K, N, argmax=False, data=weak_data(B, K, N, weak))


@pytest.mark.parametrize("B,K,N", [(70, 8, 9000), (200, 6, 30000), (5000, 4, 9), (101, 700, 4000)])
def test_vocab_head_a_label_of_little_probability_keeps_its_digits(gpu, B, K, N):
    """Where the label's logit is small its term, conj(z_l) / |z_l|^2, outweighs everything else in dx and dw.  It takes part in a few
    operations of its own (the logit, |z_l|^2, the division, the product, for dw the sum of the rows with that label), not in as many
    roundings as the sum over the vocabulary or the batch."""
    rng = np.random.default_rng(B + N)
    x, w = rnd(rng, B, K), rnd(rng, N, K, (2 * K) ** -0.5)
    labels = rng.integers(0, N, B).astype(np.int32)
    l = w[labels]
    x -= ((x * l).sum(1) / (np.abs(l) ** 2).sum(1) * (1 - 1e-5))[:, None] * l.conj()
    x = x.real.astype(np.float32).astype(np.float64) + 1j * x.imag.astype(np.float32)
    ref = head_ref(x, w, labels)
    X, W, L = cmat(x, K), cmat(w, K), ops.ints(labels)
    s, loss = capi.empty(B), capi.empty(B)
    dX, dW = grad(x.shape, K), grad(w.shape, K)
    ops.vocab_head_fwd_bwd_sym(X, W, L, s, loss, None, dX, dW)
    n = 2 * (K + N) + 64
    # c: two roundings of z_l, three of |z_l|^2 with z_l's twice, one division; three of the complex product, one of the sum
    term, same = 12, np.bincount(labels, minlength=N)[:, None]
    err, bound = np.abs(dz_of(dX) - ref["dx"]), HALF * (term * ref["label_dx"] + 2 * n * ref["size_dx"])
    assert np.all(err <= bound), (err / bound).max()
    err, bound = np.abs(dz_of(dW) - ref["dw"]), HALF * ((term + np.minimum(same, 64 + same / 64)) * ref["label_dw"] + 2 * (n + B) * ref["size_dw"])
    assert np.all(err <= bound), (err / bound).max()
    assert np.median(2 * n * ref["size_dx"] / ref["label_dx"]) < 16      # the label's share is what the bounds are about


@pytest.mark.parametrize("B,K,N,pad,off", [(1, 40, 17000, 0, 0), (3, 5, 20001, 0, 0), (16, 64, 16500, 4, 0), (17, 33, 9001, 2, 1), (32, 100, 8300, 0, 0),
                                           (40, 30, 6001, 0, 0), (48, 48, 5600, 0, 4), (63, 1, 4200, 0, 0), (64, 130, 4100, 0, 0), (1, 1024, 32768, 0, 0)])
def test_vocab_head_few_rows_against_a_large_vocabulary(gpu, B, K, N, pad, off):
    rng = np.random.default_rng(B + K + N)
    x, w, labels = head_data(rng, B, K, N)
    if N > 5000:
        w[4999] = w[137]                                  # the same entry twice: the lower index
        x[0] = 3 * w[137].conj()
    x, w = (z.real.astype(np.float32).astype(np.float64) + 1j * z.imag.astype(np.float32) for z in (x, w))
    ref = head_ref(x, w, labels)
    X, W = cmat(x, K + pad + off, off), cmat(w, K + pad + off, off)
    s, loss, am = capi.empty(B), capi.empty(B), capi.empty(B, np.int32)
    ops.vocab_head_fwd(X, W, ops.ints(labels), s, loss, am)
    near(s.download(), ref["s"], ref["size_s"], 2 * K + 32, "s")
    ok = np.isfinite(ref["loss"])
    assert np.array_equal(np.isnan(loss.download()), ~ok)
    bound = 2 * (2 * K + 32) * HALF * ref["size_s"] / ref["s"] + 8 * HALF * (1 + np.abs(ref["loss"]))
    assert np.all(np.abs(loss.download() - ref["loss"])[ok] <= bound[ok])
    check_argmax(am.download(), ref)
    assert N <= 5000 or K < 30 or am.download()[0] == 137
    loss1, am1 = capi.empty(B), capi.empty(B, np.int32)
    ops.vocab_head_fwd(X, W, None, s, loss1, am1)
    assert np.array_equal(am1.download(), am.download())
    p = ref["power"][np.arange(B), am.download()] / ref["s"]
    assert np.all(np.abs(loss1.download() + np.log(p)) <= np.nanmax(bound) + 8 * HALF * (1 + np.abs(np.log(p))))


def test_vocab_head_gives_what_the_separate_calls_give(gpu):
    """Linear, CrossEntropy and their backward passes over kept logits"""
    rng = np.random.default_rng(8)
    B, K, N = 200, 72, 900
    x, w, labels = head_data(rng, B, K, N)
    labels[7] = labels[1] = 5                              # (what the two treat differently: a row left out)
    ref = head_ref(x, w, labels)
    X, W, L = cmat(x, K), cmat(w, K), ops.ints(labels)
    z, s, loss, am, dz = ops.CMat.empty(B, N), capi.empty(B), capi.empty(B), capi.empty(B, np.int32), ops.Grad.empty(B, N)
    dX, dW = grad(x.shape, K), grad(w.shape, K)
    ops.linear_fwd(X, W, z)
    ops.cross_entropy_fwd_bwd_sym(z, L, s, loss, am, dz)
    ops.linear_bwd_sym(dz, X, W, dX, dW)
    s2, loss2, am2, dX2, dW2 = capi.empty(B), capi.empty(B), capi.empty(B, np.int32), grad(x.shape, K), grad(w.shape, K)
    ops.vocab_head_fwd_bwd_sym(X, W, L, s2, loss2, am2, dX2, dW2)
    assert np.array_equal(am.download(), am2.download())
    assert np.allclose(s.download(), s2.download(), rtol=1e-5) and np.allclose(loss.download(), loss2.download(), rtol=1e-4, atol=1e-4)
    n = 2 * (K + N) + 64
    # (the separate calls take the label's logit as the product rounded it: K roundings against the gradient's 1 / z)
    k = (2 * K + 32) * np.abs(ref["c"])[:, None] * ref["size_z"].max(1)[:, None]
    near(dz_of(dX2), dz_of(dX), ref["size_dx"] + k / n * ref["label_dx"], 2 * n, "dx")
    assert np.linalg.norm(dz_of(dW2) - dz_of(dW)) <= 1e-3 * np.linalg.norm(dz_of(dW))


def test_vocab_head_gradient_against_differences(gpu):
    rng = np.random.default_rng(6)
    B, K, N = 12, 24, 90
    x, w, labels = head_data(rng, B, K, N)
    labels[7] = 1
    dX, dW = grad(x.shape, K), grad(w.shape, K)
    ops.vocab_head_fwd_bwd_sym(cmat(x, K), cmat(w, K), ops.ints(labels), capi.empty(B), capi.empty(B), None, dX, dW)
    step = 1e-6
    for d, arg in ((dX, 0), (dW, 1)):
        r = rnd(rng, *(x, w)[arg].shape)
        hi, lo = [x, w], [x, w]
        hi[arg], lo[arg] = hi[arg] + step * r, lo[arg] - step * r
        want = (head_ref(*hi, labels)["loss"].sum() - head_ref(*lo, labels)["loss"].sum()) / (2 * step)
        got = 2 * (dz_of(d) * r).sum().real
        assert abs(got - want) <= 1e-5 * (np.abs(dz_of(d)) * np.abs(r)).sum(), (arg, got, want)


@pytest.mark.parametrize("B,K,N", [(5, 12, 40), (400, 12, 40)])
def test_vocab_head_rows_of_zeros_and_no_labels_at_all(gpu, B, K, N):
    rng = np.random.default_rng(12)
    x, w, labels = head_data(rng, B, K, N)
    x[0] = 0                                              # every logit zero: both clamps, no NaN
    labels[0] = 3
    s, loss, dX, dW = capi.empty(B), capi.empty(B), grad(x.shape, K), grad(w.shape, K)
    ops.vocab_head_fwd_bwd_sym(cmat(x, K), cmat(w, K), ops.ints(labels), s, loss, None, dX, dW)
    assert s.download()[0] == np.float32(LEAST) and loss.download()[0] == np.float32(-np.log(LEAST))
    assert not dz_of(dX)[0].any() and np.all(np.isfinite(dz_of(dW)))
    ops.vocab_head_fwd_bwd_sym(cmat(x, K), cmat(w, K), ops.ints(np.full(B, -1, np.int32)), s, loss, None, dX, dW)
    assert not loss.download().any() and not dz_of(dX).any() and not dz_of(dW).any()


def test_vocab_head_a_row_of_nan_stays_in_its_row(gpu):
    rng = np.random.default_rng(13)
    B, K, N = 20, 48, 300
    x, w, labels = head_data(rng, B, K, N)
    labels[7] = 2
    ref = head_ref(x, w, labels)
    bad = x.copy()
    bad[4, 3] = np.nan
    s, loss, am = capi.empty(B), capi.empty(B), capi.empty(B, np.int32)
    ops.vocab_head_fwd(cmat(bad, K), cmat(w, K), ops.ints(labels), s, loss, am)
    ok = np.arange(B) != 4
    assert np.allclose(s.download()[ok], ref["s"][ok], rtol=1e-5) and np.array_equal(am.download()[ok], ref["argmax"][ok])
    assert 0 <= am.download()[4] < N


@pytest.mark.parametrize("B,K,N", [(20, 48, 300), (300, 40, 260), (100, 300, 1001), (700, 333, 1100), (60, 7, 5000), (200, 300, 4500), (700, 333, 4001)])
def test_vocab_head_rows_left_out_may_hold_anything(gpu, B, K, N):
    """NaN and infinities in rows without a label touch neither the other rows nor the gradient of the weights"""
    rng = np.random.default_rng(16)
    x, w, labels = head_data(rng, B, K, N)
    labels[7] = 2
    labels[10:15] = -1
    ref = head_ref(x, w, labels)
    bad = x.copy()
    bad[1], bad[10], bad[12, 3] = np.nan, np.inf, -np.inf
    s, loss, dX, dW = capi.empty(B), capi.empty(B), grad(x.shape, K), grad(w.shape, K)
    with np.errstate(invalid="ignore"):
        X = cmat(bad, K)
    ops.vocab_head_fwd_bwd_sym(X, cmat(w, K), ops.ints(labels), s, loss, None, dX, dW)
    n = 2 * (K + N) + 64
    label_n = 24 + np.bincount(labels[labels >= 0], minlength=N).max()
    near(dz_of(dX), ref["dx"], ref["size_dx"] + label_n / n * ref["label_dx"], n, "dx")
    near(dz_of(dW), ref["dw"], ref["size_dw"] + label_n / n * ref["label_dw"], n + 2 * B, "dw")
    assert not loss.download()[labels < 0].any()


@pytest.mark.parametrize("B,K,N,argmax", [(260, 64, 1000, True), (700, 333, 4001, False), (60, 7, 5000, False), (17, 33, 9001, True)])
def test_vocab_head_in_a_graph(gpu, B, K, N, argmax):
    rng = np.random.default_rng(14)
    x, w, labels = head_data(rng, B, K, N)
    X, W, L = cmat(x, K), cmat(w, K), ops.ints(labels)
    s, loss, am, dX, dW = capi.empty(B), capi.empty(B), capi.empty(B, np.int32), grad(x.shape, K), grad(w.shape, K)

    best = capi.empty(B)

    def step():
        ops.vocab_head_fwd_bwd_sym(X, W, L, s, loss, am if argmax else None, dX, dW)
        ops.vocab_head_fwd(X, W, None, s, best, am)

    def results():
        return [s.download(), loss.download(), best.download(), am.download(), dz_of(dX), dz_of(dW)]
    step()
    want = results()
    exes = []
    for _ in range(2):                                     # two recordings share the library's buffers
        capi.call("cnet_graph_begin")
        step()
        exes.append(C.c_void_p())
        capi.call("cnet_graph_end", C.byref(exes[-1]))
    x2, w2, l2 = head_data(rng, 900, 96, 3000)
    for k in range(4):
        for p in dX.planes + dW.planes:
            p.owner.zero()
        big = cmat(x2, 96), cmat(w2, 96), ops.ints(l2), capi.empty(900), capi.empty(900)     # eager work that needs more room
        ops.vocab_head_fwd_bwd_sym(*big, None, grad(x2.shape, 96), grad(w2.shape, 96))
        capi.sync()
        capi.call("cnet_graph_launch", exes[k % 2])
        for a, b in zip(results(), want):
            assert np.array_equal(a, b, equal_nan=True)
    for e in exes:
        capi.call("cnet_graph_destroy", e)


def test_vocab_head_no_rows(gpu):
    K, N = 9, 21
    z, w = ops.CMat.empty(1, K), ops.CMat.empty(N, K, zero=True)
    none = ops.CMat(z.re.rows_from(0, 0), z.im.rows_from(0, 0))
    none_g = ops.Grad([z.re.rows_from(0, 0)] * 4)
    L, s = ops.ints([0]), capi.empty(1)
    am = capi.empty(1, np.int32)
    ops.vocab_head_fwd(none, w, L, s, s, am)
    dW = grad((N, K), K + 2, fill=3.0)
    ops.vocab_head_fwd_bwd_sym(none, w, L, s, s, am, none_g, dW, accumulate_dw=1)
    assert np.all(dz_of(dW) == 3 + 3j)
    ops.vocab_head_fwd_bwd_sym(none, w, L, s, s, am, none_g, dW)
    assert not dz_of(dW).any() and not dzs_of(dW).any() and all(untouched(p) for p in dW.planes)


def test_vocab_refusals(gpu):
    lib = capi.load()
    rows, cols, top = 4, 8, 2
    z, g = ops.CMat.empty(rows, cols, zero=True), ops.Grad.empty(rows, cols, zero=True)
    ids, q, s = ops.ints(np.zeros((rows, top))), capi.zeros((rows, top)), capi.zeros(rows)

    def distill(z_im=z.im.ptr, ldz=8, ids=ids.ptr, q=q.ptr, top=top, s=s.ptr, loss=s.ptr, dz=g.p(), lddz=8, rows=rows, cols=cols):
        out = [lib.cnet_distill_fwd_bwd_sym(z.re.ptr, z_im, ldz, ids, q, top, s, loss, *dz, lddz, rows, cols)]
        if dz == g.p() and lddz == 8:
            out.append(lib.cnet_distill_fwd(z.re.ptr, z_im, ldz, ids, q, top, s, loss, rows, cols))
        if loss is not None:
            out.append(lib.cnet_distill_bwd_sym(z.re.ptr, z_im, ldz, s, ids, q, top, *dz, lddz, rows, cols))
        assert len(set(out)) == 1, out
        return out[0]
    assert distill() == 0 and distill(rows=0) == 0 and distill(dz=(*g.p()[:2], None, None)) == 0
    assert INVALID == distill(z_im=None) == distill(ldz=7) == distill(ids=None) == distill(q=None) == distill(top=0) == distill(top=1025)
    assert INVALID == distill(s=None) == distill(loss=None) == distill(lddz=7) == distill(dz=(*g.p()[:3], None)) == distill(rows=-1) == distill(cols=0)
    assert b"cnet_distill" in lib.cnet_last_error()

    x, w, lab, am = ops.CMat.empty(rows, cols, zero=True), ops.CMat.empty(5, cols, zero=True), ops.ints(np.zeros(rows)), capi.empty(rows, np.int32)
    dx, dw = ops.Grad.empty(rows, cols), ops.Grad.empty(5, cols)

    def fwd(x_im=x.im.ptr, ldx=8, ldw=8, labels=lab.ptr, s=s.ptr, loss=s.ptr, am=am.ptr, B=rows, K=cols, N=5):
        return lib.cnet_vocab_head_fwd(x.re.ptr, x_im, ldx, *w.p(), ldw, labels, s, loss, am, B, K, N)
    loss2 = capi.empty(rows)
    assert fwd(loss=loss2.ptr) == 0 and fwd(loss=loss2.ptr, am=None) == 0 and fwd(loss=None) == 0 and fwd(labels=None, loss=loss2.ptr) == 0 and fwd(B=0) == 0
    assert INVALID == fwd(B=1 << 24) == fwd(N=1 << 28) == distill(rows=1 << 22)
    assert INVALID == fwd(x_im=None) == fwd(ldx=7) == fwd(ldw=7) == fwd(s=None) == fwd(loss=None, am=None) == fwd(B=-1) == fwd(K=0) == fwd(N=0)

    def step(labels=lab.ptr, loss=loss2.ptr, am=am.ptr, dx_im=dx.p()[1], dxs=dx.p()[3], lddx=8, dw_re=dw.p()[0], dws=dw.p()[2], lddw=8, ldx=8):
        return lib.cnet_vocab_head_fwd_bwd_sym(*x.p(), ldx, *w.p(), 8, labels, s.ptr, loss, am, dx.p()[0], dx_im, dx.p()[2], dxs, lddx, 0,
                                               dw_re, dw.p()[1], dws, dw.p()[3], lddw, 0, rows, cols, 5)
    assert step() == 0 and step(am=None) == 0
    assert INVALID == step(labels=None) == step(loss=None) == step(dx_im=None) == step(dxs=None) == step(lddx=7) == step(ldx=7)
    assert INVALID == step(dw_re=None) == step(dws=None) == step(lddw=7)
