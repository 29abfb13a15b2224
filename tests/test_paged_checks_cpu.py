"""Refusals of the paged C entries that no kernel can make good: addresses that it would fault on."""
import ctypes as C

import pytest

from test_paged_cpu import _append_params, _cache_params


@pytest.mark.parametrize("kw", [dict(cu_q=0x1002, total_q=2), dict(lse=0x1002), dict(status=0x1002)])
def test_attention_refuses_addresses(kw):
    from miniattn import _lib
    assert _lib.lib.miniattn_fwd_cache(C.byref(_cache_params(**kw)), None, 0, None) == _lib.EINVAL
    assert "4-byte aligned" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(cu_q=0x1002, total=2), dict(status=0x1002)])
def test_append_refuses_addresses(kw):
    from miniattn import _lib
    assert _lib.lib.miniattn_paged_append(C.byref(_append_params(**kw)), None) == _lib.EINVAL
    assert "4-byte aligned" in _lib.last_error()
