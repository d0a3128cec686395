"""Run by tests/test_gpu_vocab_launches.py in processes of their own, with tuning overrides in the environment (the library reads them once):
a small training step of the vocabulary head, its results against 64 bits, and how many kernels one call queues."""
import ctypes as C
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from cnet_amd import capi, ops  # noqa: E402
from tests.test_gpu_norm import cmat, grad  # noqa: E402
from tests.test_gpu_vocab import head_check, head_data  # noqa: E402

SHAPE = (96, 64, 512)


def kernels_of(call):
    """the kernels that `call` queues, from a recording of the library's stream"""
    hip = C.CDLL("libamdhip64.so.7")
    stream, graph, count = C.c_void_p(capi.load().cnet_stream()), C.c_void_p(), C.c_size_t()
    call()                                                 # (workspaces grow outside a recording)
    capi.sync()
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    call()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphGetNodes(graph, None, C.byref(count)) == 0
    nodes = (C.c_void_p * count.value)()
    assert hip.hipGraphGetNodes(graph, nodes, C.byref(count)) == 0
    kinds = []
    for n in nodes:
        kind = C.c_int()
        assert hip.hipGraphNodeGetType(C.c_void_p(n), C.byref(kind)) == 0
        kinds.append(kind.value)
    assert hip.hipGraphDestroy(graph) == 0
    return kinds.count(0)


def main():
    capi.init(0)
    B, K, N = SHAPE
    for argmax in (True, False):
        head_check(B, K, N, argmax=argmax)
    head_check(17, 33, 130, 2, 1)
    x, w, labels = head_data(np.random.default_rng(1), B, K, N)
    X, W, L = cmat(x, K), cmat(w, K), ops.ints(labels)
    s, loss, am, dX, dW = capi.empty(B), capi.empty(B), capi.empty(B, np.int32), grad(x.shape, K), grad(w.shape, K)
    print("KERNELS", kernels_of(lambda: ops.vocab_head_fwd_bwd_sym(X, W, L, s, loss, am, dX, dW)))


if __name__ == "__main__":
    main()
