"""The error text of a refused call names the function that was called, not one that it calls inside."""
from cnet_amd import capi

import pytest

NOT_INITIALIZED = -1


def test_refused_calls_name_themselves():
    lib = capi.load()
    if lib.cnet_stream():
        pytest.skip("the library is initialised in this process")
    seen = 0
    for name, kinds in capi.SIGNATURES.items():
        if not name.startswith(("cnet_clinear_bwd", "cnet_norm_", "cnet_distill_", "cnet_vocab_")):
            continue
        if getattr(lib, name)(*[k() for k in kinds]) == NOT_INITIALIZED:
            seen += 1
            assert lib.cnet_last_error().decode().startswith(name + ":"), lib.cnet_last_error()
    assert seen >= 14
