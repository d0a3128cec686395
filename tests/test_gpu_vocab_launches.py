"""The vocabulary head's small step under the overrides of the small products (include/cnet_hip.h): two products in one launch or in two,
any number of wavefronts."""
import os
import subprocess
import sys

import pytest

from tests.gpu_util import gpu  # noqa: F401

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def kernels(overrides):
    env = {k: v for k, v in os.environ.items() if not k.startswith("CNET_CGEMM_")}
    r = subprocess.run([sys.executable, os.path.join(HERE, "gpu_head_launches_check.py")], env={**env, **overrides}, capture_output=True, text=True,
                       timeout=100, cwd=os.path.dirname(HERE))
    assert r.returncode == 0, r.stdout[-1000:] + r.stderr[-3000:]
    line = [l for l in r.stdout.splitlines() if l.startswith("KERNELS ")]
    return int(line[-1].split()[1])


def test_the_head_obeys_the_overrides_of_the_small_products(gpu):
    joint = kernels({})
    assert kernels({"CNET_CGEMM_SKINNY_TWO": "0"}) == joint + 1
    for w in ("4", "8", "16"):
        assert kernels({"CNET_CGEMM_SKINNY_W": w}) == joint
