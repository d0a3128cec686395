"""Run by tests/test_gpu_vocab.py in a process of its own, with CNET_HEAD_GRAM and CNET_HEAD_PIECE_MB in the environment (the
library reads them once, at the first call of the head): every way through the vocabulary head on shapes that would take another."""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from cnet_amd import capi  # noqa: E402
from tests.test_gpu_vocab import head_check, weak_data  # noqa: E402


def main():
    capi.init(0)
    for B, K, N, pad, off in ((1, 5, 9, 0, 0), (17, 33, 130, 2, 1), (300, 96, 1700, 0, 0), (700, 61, 1100, 3, 0), (9000, 8, 100, 0, 0), (400, 576, 900, 0, 0), (203, 700, 1001, 0, 0), (330, 1001, 600, 0, 0),
                              (500, 600, 1200, 0, 0)):
        for argmax in (True, False):
            print(B, K, N, argmax, flush=True)
            head_check(B, K, N, pad, off, argmax)
    # rows whose sum is formed again from w: in two blocks of rows, all of them, a few beside the end, unaligned
    for B, K, N, pad, off, every in ((4300, 24, 100, 0, 0, 3), (150, 200, 400, 0, 0, 1), (129, 72, 65, 4, 0, 128), (500, 61, 900, 2, 1, 2), (40, 130, 9000, 0, 0, 1)):
        print(B, K, N, "weak", flush=True)
        head_check(B, K, N, pad, off, False, weak_data(B, K, N, 1e-3, every))


if __name__ == "__main__":
    main()
    print("ok")
