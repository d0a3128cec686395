"""Run by tests/test_gpu_vocab_cancelling.py in a process of its own, with CNET_HEAD_GRAM=1 in the environment: the vocabulary head through the
Gram matrix of w on shapes that would take another way, on ordinary rows and on rows and entries whose terms cancel."""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from cnet_amd import capi  # noqa: E402
from tests.test_gpu_vocab import head_data  # noqa: E402
from tests.test_gpu_vocab_cancelling import CANCELLING, WEAK, cancelling_check, rounded, shared_axis, shared_rows  # noqa: E402


def main():
    capi.init(0)
    # blocks of 64, chunks of 16 and what does not fill them; one row, one column, one entry; more rows than one block of ordered labels
    for B, K, N, pad, off in ((1, 1, 1, 0, 0), (3, 5, 7, 0, 0), (64, 64, 64, 0, 0), (65, 63, 129, 1, 0), (17, 33, 130, 2, 1), (300, 96, 1700, 0, 0),
                              (700, 61, 1100, 3, 0), (9000, 8, 100, 0, 0), (203, 700, 1001, 0, 0), (330, 1001, 600, 0, 4), (90, 16, 40000, 0, 0)):
        rng = np.random.default_rng(B + K + N)
        x, w, labels = head_data(rng, B, K, N)
        labels[labels >= N] = 0
        for argmax in (False, True):
            print(B, K, N, argmax, flush=True)
            cancelling_check(rounded(x), rounded(w), labels, True, pad, off, argmax)
    # leading dimensions whose offsets inside a block of 64 rows pass 32 bits
    x, w, labels = head_data(np.random.default_rng(3), 2, 5, 3)
    print("far", flush=True)
    cancelling_check(rounded(x), rounded(w), labels, True, 1 << 23)
    for B, K, N, pad, off in CANCELLING + [(129, 72, 65, 4, 0), (40, 130, 9000, 0, 0)]:
        for weak in WEAK:
            print(B, K, N, weak, flush=True)
            cancelling_check(*shared_axis(B, K, N, weak), True, pad, off)
            cancelling_check(*shared_rows(B, K, N, weak), True, pad, off, argmax=True)


if __name__ == "__main__":
    main()
    print("ok")
