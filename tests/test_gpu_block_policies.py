"""The cache policies of the norms and of the distillation loss (plain; hint on loads and stores; hinted stores; hinted loads and device-scope
stores) move the same bits, also where a row's entries overwrite what other wavefronts have just stored with a hint.  A launch picks its policy by
its footprint, which small shapes reach through the overrides, read once per process: see tests/gpu_block_policy_check.py."""
import json
import os
import subprocess
import sys

import pytest

from tests import gpu_block_policy_check as check
from tests.gpu_util import gpu  # noqa: F401

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def plain(gpu):
    if os.environ.get("CNET_STREAM_MIN_MB") or os.environ.get("CNET_STREAM_POLICY"):
        pytest.skip("this process already runs under a policy override")
    return check.digests()


@pytest.mark.parametrize("policy", [1, 2, 3])
def test_every_policy_gives_the_same_bits(plain, policy):
    env = dict(os.environ, CNET_STREAM_MIN_MB="0", CNET_STREAM_POLICY=str(policy))
    r = subprocess.run([sys.executable, os.path.join(HERE, "gpu_block_policy_check.py")], env=env, capture_output=True, text=True, timeout=100,
                       cwd=os.path.dirname(HERE))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    line = [l for l in r.stdout.splitlines() if l.startswith("DIGESTS ")]
    got = json.loads(line[-1][len("DIGESTS "):])
    assert len(plain) == 4 * len(check.NORMS) + 3 * len(check.DISTIL) and set(got) == set(plain)
    differ = sorted(k for k in plain if got[k] != plain[k])
    assert not differ, (policy, differ)
