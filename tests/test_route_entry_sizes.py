"""Token counts that the routing entry point refuses before it computes with them (no GPU)."""

import ctypes

import pytest

from loraforge_amd import _lib


@pytest.mark.parametrize("tokens,top", [(2**62, 4), (2**58, 64), (2**63 - 1, 2), (2**61, 8), (2**31, 1), (2**31 - 2**16, 1), (-1, 1)])
def test_token_counts_past_32_bits_are_refused(tokens, top):
    """Also those whose choices, counted in 64 bits, wrap round to a small number."""
    lib, p = _lib.library(), ctypes.c_void_p(16)
    status = lib.lf_route_experts(p, 0, tokens, 64, 64, top, 1, p, p, p, p, p, p, 1 << 40, None)
    assert status == _lib.LF_EINVAL
    assert 0 <= tokens < 2**31 or lib.lf_route_experts_workspace_size(tokens, 64) == -1
