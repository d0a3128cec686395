"""The norms around a block and the distillation loss on fixed inputs; `results()` returns every output array by name, `digests()` a hash of each.

tests/test_gpu_block_policies.py runs this file in processes of their own with CNET_STREAM_MIN_MB=0 (every launch counts as streaming) and
CNET_STREAM_POLICY = 1, 2, 3 (the library reads both once per process), and compares the hashes with those of the plain accesses."""
import hashlib
import json
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from cnet_amd import capi, ops  # noqa: E402
from tests.test_gpu_norm import EPS, SCALE, cmat, cval, dz_of, dzs_of, grad, rnd  # noqa: E402

NORMS = [(37, 64), (13, 500), (9, 1024), (7, 2048), (5, 4096), (3, 8192), (3, 16384), (6, 333)]
# rows, columns, entries: one wavefront, one workgroup of each width and a row longer than the registers
DISTIL = [(9, 512, 8), (7, 2048, 70), (5, 4096, 9), (66, 8192, 5), (65, 16384, 3), (65, 32768, 40), (64, 40000, 50), (6, 777, 5)]


def results():
    out = {}
    for rows, cols in NORMS:
        rng = np.random.default_rng(rows + cols)
        u, f, g, gh = (cmat(rnd(rng, rows, cols), cols) for _ in range(4))
        w = cmat(rnd(rng, 1, cols, 0.2, 1.0), cols)
        for shared in (True, False):
            v = cmat(rnd(rng, 1 if shared else rows, cols, 0.3, 1.0), cols)
            y, h, s, s2 = cmat(np.zeros((rows, cols)), cols), cmat(np.zeros((rows, cols)), cols), capi.empty(rows), capi.empty(rows)
            name = "norm %dx%d %s" % (rows, cols, shared)
            ops.norm_gate_fwd(f, v, y, s, EPS, shared=shared)
            dx, dv = grad((rows, cols), cols, fill=0.5), grad((1 if shared else rows, cols), cols, fill=0.5)
            for acc in (0, 1):
                ops.norm_gate_bwd_sym(f, s, v, g, dx, dv, shared=shared, accumulate=acc, accumulate_w=acc, mirror=not acc)
            out[name + " gate"] = [cval(y), s.download(), dz_of(dx), dzs_of(dx), dz_of(dv), dzs_of(dv)]
            ops.norm_join_fwd(u, f, v, SCALE, h, s, w, y, s2, EPS, shared=shared)
            du, df, dw = grad((rows, cols), cols), grad((rows, cols), cols), grad((1, cols), cols)
            for acc in (0, 1):
                ops.norm_join_bwd_sym(f, s, v, SCALE, h, s2, w, gh, g, du, df, dv, dw, shared=shared, accumulate=acc, accumulate_w=acc, mirror=not acc)
            out[name + " join"] = [cval(h), cval(y), s.download(), s2.download()] + [q(d) for d in (du, df, dv, dw) for q in (dz_of, dzs_of)]
    for rows, cols, top in DISTIL:
        rng = np.random.default_rng(rows + cols + top)
        z = rnd(rng, rows, cols)
        ids = rng.integers(0, cols, (rows, top)).astype(np.int32)
        ids[1, top // 2:] = -1
        ids[2] = -1
        ids[0, 0] = ids[0, top - 1]                        # the same index twice
        q = (rng.random((rows, top)) + 0.01).astype(np.float32)
        Z, I, Q = cmat(z, cols), ops.ints(ids), capi.to_device(q)
        for mirror in (True, False):
            s, loss, dz = capi.empty(rows), capi.empty(rows), grad(z.shape, cols, fill=5.0)
            ops.distill_fwd_bwd_sym(Z, I, Q, top, s, loss, dz, mirror=mirror)
            out["distil %dx%d %s" % (rows, cols, mirror)] = [s.download(), loss.download(), dz_of(dz), dzs_of(dz)]
        s, loss = capi.empty(rows), capi.empty(rows)
        ops.distill_fwd(Z, I, Q, top, s, loss)
        out["distil %dx%d forward" % (rows, cols)] = [s.download(), loss.download()]
    return out


def digests():
    found = {}
    for name, arrays in results().items():
        h = hashlib.sha256()
        for a in arrays:
            h.update(np.ascontiguousarray(a).tobytes())
        found[name] = h.hexdigest()
    return found


if __name__ == "__main__":
    capi.init(0)
    print("DIGESTS " + json.dumps(digests()))
