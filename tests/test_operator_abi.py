"""CPU-only: the entry points of the 8-bit cache, the mixture of experts and the
log probabilities answer missing handles with an error, not a crash."""
import ctypes as C

import pytest

from tensorlogic_amd import _lib as L

N = None


@pytest.mark.parametrize("name,args", [
    ("tlhip_token_logprobs", (N, N, N, 0, N, N, N, N)),
    ("tlhip_token_logprobs", (N, N, N, 5, N, N, N, N)),
    ("tlhip_moe", (N, N, N, N, N, N, 1, 1, N)),
    ("tlhip_kvcache_create_q8", (N, 1, 64, 1, 64, C.byref(C.c_void_p()))),
    ("tlhip_kvcache_create_q8", (N, 1, 64, 1, 64, N)),
])
def test_missing_handles(name, args):
    assert getattr(L.lib(), name)(*args) != 0
    assert L.lib().tlhip_last_error()
