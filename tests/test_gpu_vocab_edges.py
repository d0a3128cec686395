"""The losses of a vocabulary at what their documentation allows besides the ordinary: NaN among a row's logits, padding rows that hold
anything, entries without weight."""
import numpy as np
import pytest

from cnet_amd import capi, ops
from tests.gpu_util import gpu  # noqa: F401
from tests.test_gpu_norm import cmat, cval, dz_of, dzs_of, grad, rnd
from tests.test_gpu_vocab import head_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,N,at", [(1, 17000, 0), (1, 17000, 16), (5, 17000, 4992), (17, 9000, 64 * 70), (64, 9000, 35), (65, 9000, 35),
                                    (40, 9000, 8999), (130, 300, 16)])
def test_vocab_head_argmax_beside_a_logit_of_nan(gpu, B, N, at):
    """One entry of the vocabulary is NaN: the largest of the others is found all the same, next to it too, however many rows there are."""
    rng = np.random.default_rng(N + at)
    K = 48
    x, w = rnd(rng, B, K), rnd(rng, N, K, (2 * K) ** -0.5)
    near = [k for k in range(at - 16, at + 17) if 0 <= k < N and k != at]
    for r in range(B):                                     # every row's largest logit lies within 16 of the entry, on either side
        x[r] += 6 * w[near[r % len(near)]].conj() / np.linalg.norm(w[near[r % len(near)]])
    x = x.real.astype(np.float32).astype(np.float64) + 1j * x.imag.astype(np.float32)
    power = head_ref(x, w, np.zeros(B, np.int32))["power"]
    power[:, at] = -1
    want = power.argmax(1)
    bad = w.copy()
    bad[at] = np.nan
    s, loss, am = capi.empty(B), capi.empty(B), capi.empty(B, np.int32)
    ops.vocab_head_fwd(cmat(x, K), cmat(bad, K), None, s, loss, am)
    got = am.download()
    gap = np.sort(power, axis=1)
    sure = gap[:, -1] > gap[:, -2] * (1 + 1e-4)            # (two logits as large to within their roundings: either)
    assert sure.sum() >= 0.9 * B and np.array_equal(got[sure], want[sure])
    assert np.all(np.isnan(s.download())) and np.all(np.isnan(loss.download()))


# every way a row can go: a wavefront's, a workgroup's of each width, longer than its registers, dealt out to several workgroups
DISTIL_WAYS = [(6, 300, 5), (6, 513, 5), (6, 1200, 70), (6, 4000, 5), (6, 8191, 5), (70, 9001, 5), (70, 20000, 3), (66, 33000, 9), (6, 9001, 5), (3, 100003, 64)]


@pytest.mark.parametrize("rows,cols,top", DISTIL_WAYS)
@pytest.mark.parametrize("pad", [0, 1])
def test_distill_rows_of_padding_may_hold_anything(gpu, rows, cols, top, pad):
    """A row without an entry has loss 0 and gradient 0, with NaN and infinities in it as well; the rows beside it are what they were."""
    rng = np.random.default_rng(cols + top)
    z = rnd(rng, rows, cols)
    ids = np.stack([rng.permutation(cols)[:top] for _ in range(rows)]).astype(np.int32)
    q = rng.random((rows, top)).astype(np.float32) + np.float32(0.1)
    ids[1:3] = -1
    q[1] = 0
    q[2] = np.nan                                          # (the weight of no entry at all)
    I, Q = ops.ints(ids), capi.to_device(q)

    def run(z):
        with np.errstate(invalid="ignore"):
            Z = cmat(z, cols + pad)
        s, loss, dz, dz2 = capi.empty(rows), capi.empty(rows), grad(z.shape, cols + pad, fill=5.0), grad(z.shape, cols + pad, fill=5.0)
        ops.distill_fwd_bwd_sym(Z, I, Q, top, s, loss, dz)
        ops.distill_bwd_sym(Z, s, I, Q, top, dz2)
        assert np.array_equal(dz_of(dz), dz_of(dz2)) and np.array_equal(dzs_of(dz2), dz_of(dz2).conj())
        return loss.download(), dz_of(dz)
    good = run(z)
    z[1], z[2, ::7], z[2, 1] = np.nan, np.inf, -np.inf
    loss, dz = run(z)
    assert np.all(loss[1:3] == 0) and np.all(dz[1:3] == 0)
    assert np.array_equal(loss, good[0]) and np.array_equal(dz, good[1])
