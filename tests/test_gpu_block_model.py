"""A deep complex token model of norms, gates, Linears and the vocabulary's losses, run as one: every gradient against automatic
differentiation of the same formulas in complex128 on the CPU, and a short run of SGD steps on it."""
import numpy as np
import pytest
import torch

from cnet_amd import capi, ops
from cnet_amd.workloads import BlockTokenModel
from tests.gpu_util import gpu, rel_c, TOL  # noqa: F401

pytestmark = pytest.mark.gpu

B, S, D, H, V, L = 3, 20, 24, 40, 70, 3
SCALE, EPS = 0.5, 1e-6


def parameters(seed):
    rng = np.random.default_rng(seed)

    def n(rows, cols, std, mean=0.0):
        a = std * rng.standard_normal((2, rows, cols))
        a[0] += mean
        return a.astype(np.float32)
    return {"table": n(V, D, 1.0), "head": n(V, D, D ** -0.5), "norm": [n(1, D, 0.2, 1.0) for _ in range(L + 1)],
            "gate": [n(1, D, 0.3, 1.0) for _ in range(L)], "after": [n(1, D, 0.2, 1.0) for _ in range(L)],
            "w1": [n(H, D, D ** -0.5) for _ in range(L)], "w2": [n(D, H, H ** -0.5) for _ in range(L)]}


def plain(params, ids, labels, teacher):
    """(losses, most likely tokens, parameters with their gradients) in complex128"""
    def c(a):
        return torch.complex(torch.tensor(a[0], dtype=torch.float64), torch.tensor(a[1], dtype=torch.float64)).requires_grad_(True)
    p = {k: [c(x) for x in v] if isinstance(v, list) else c(v) for k, v in params.items()}
    q = np.arange(S)
    F = torch.tensor(np.exp(-2j * np.pi * np.outer(q, q) / S) / np.sqrt(S))

    def norm(z):
        return z / torch.sqrt((z.abs() ** 2).mean(-1, keepdim=True) + EPS)

    def gelu(z):
        f = torch.nn.functional.gelu
        return torch.complex(f(z.real, approximate="tanh"), f(z.imag, approximate="tanh"))
    h = p["table"][torch.tensor(ids).long()]
    y = p["norm"][0] * norm(h)
    for k in range(L):
        m = torch.einsum("pq,bqd->bpd", F, y)
        f = gelu((p["gate"][k] * m) @ p["w1"][k].T) @ p["w2"][k].T
        h = h + SCALE * p["after"][k] * norm(f)
        y = p["norm"][k + 1] * norm(h)
    z = (y @ p["head"].T).reshape(B * S, V)
    power = z.real ** 2 + z.imag ** 2
    logp = torch.log(power) - torch.log(power.sum(1, keepdim=True))
    if teacher is None:
        at = torch.tensor(labels).reshape(-1).long()
        loss = torch.where(at >= 0, -logp.gather(1, at.clamp(min=0)[:, None])[:, 0], torch.zeros(B * S, dtype=torch.float64))
    else:
        t, w = torch.tensor(teacher[0]).long(), torch.tensor(teacher[1], dtype=torch.float64)
        w = torch.where(t >= 0, w, torch.zeros_like(w))
        loss = (torch.xlogy(w, w) - w * logp.gather(1, t.clamp(min=0))).sum(1)
    loss.sum().backward()
    return loss.detach().numpy(), power.argmax(1).numpy(), p


def data(seed):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, V, (B, S)).astype(np.int32)
    ids[0, 3] = ids[1, 5] = ids[2, 7]
    labels = np.concatenate([ids[:, 1:], np.full((B, 1), -1, np.int32)], axis=1)
    top = np.stack([rng.permutation(V)[:6] for _ in range(B * S)]).astype(np.int32)
    w = rng.random((B * S, 6)).astype(np.float32)
    w /= w.sum(1, keepdims=True)
    top[5:9] = -1
    return ids, labels, (top, w)


@pytest.mark.parametrize("distil", [False, True])
def test_block_model_gradients(gpu, distil):
    params = parameters(1)
    ids, labels, teacher = data(2)
    model = BlockTokenModel(B, S, D, H, V, L, params, SCALE, EPS).set_tokens(ids)
    if distil:
        model.set_teacher(*teacher)
    loss, best, p = plain(params, ids, labels, teacher if distil else None)
    for _ in range(2):                                     # a second step on the same planes
        model.step()
        assert np.allclose(model.loss.download(), loss, rtol=1e-4, atol=1e-4)
        for k, v in model.grads.items():
            for got, want in zip(v if isinstance(v, list) else [v], p[k] if isinstance(p[k], list) else [p[k]]):
                g = want.grad.numpy() / 2                  # dL/d conj z
                h = got.host()
                assert rel_c(h[2:4], (g.real, g.imag)) < TOL, k
                if k != "table":
                    assert np.array_equal(h[0], h[2]) and np.array_equal(h[1], -h[3]), k
    model.score()
    assert np.array_equal(model.argmax.download(), best)


def test_block_model_learns_a_batch(gpu):
    ids, _, _ = data(3)
    model = BlockTokenModel(B, S, D, H, V, L, parameters(4), SCALE, EPS).set_tokens(ids)
    for _ in range(3):
        model.step()
        for k, v in model.grads.items():
            for g, w in zip(v if isinstance(v, list) else [v], model.p[k] if isinstance(model.p[k], list) else [model.p[k]]):
                ops.sgd_update(w, g.planes[2], g.planes[3], 1e-3)
    assert np.all(np.isfinite(model.loss.download()))
    capi.sync()
