"""Run by tests/test_gpu_vocab.py in a process of its own, with CNET_HEAD_GRAM and CNET_HEAD_PIECE_MB in the environment (the
library reads them once, at the first call of the head): every way through the vocabulary head on shapes that would take another."""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from cnet_amd import capi  # noqa: E402
from tests.test_gpu_vocab import head_check  # noqa: E402


def main():
    capi.init(0)
    for B, K, N, pad, off in ((1, 5, 9, 0, 0), (17, 33, 130, 2, 1), (300, 96, 1700, 0, 0), (700, 61, 1100, 3, 0), (9000, 8, 100, 0, 0), (400, 576, 900, 0, 0), (203, 700, 1001, 0, 0), (330, 1001, 600, 0, 0),
                              (500, 600, 1200, 0, 0)):
        for argmax in (True, False):
            print(B, K, N, argmax, flush=True)
            head_check(B, K, N, pad, off, argmax)


if __name__ == "__main__":
    main()
    print("ok")
