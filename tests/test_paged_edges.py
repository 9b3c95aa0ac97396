"""The paged cache's calls beside the ordinary ones, without a GPU."""
import ctypes

import pytest

from mkx import _lib

from test_paged import P16, SIZES, _attend_args


@pytest.mark.parametrize("over,status", SIZES + [(dict(q=None), _lib.EINVAL), (dict(ws=P16 + 16), _lib.EINVAL), (dict(out=P16), _lib.EINVAL)])
def test_attention_of_granted_requests_refuses(over, status):
    L = _lib.lib()
    assert L.mkx_page_attend_granted(ctypes.byref(_attend_args(**over)), P16, None) == status, L.mkx_last_error()
    assert "mkx_page_attend_granted:" in L.mkx_last_error().decode()
    assert L.mkx_page_attend_granted(None, P16, None) == _lib.EINVAL
    assert L.mkx_page_attend_granted(ctypes.byref(_attend_args(T=0)), P16, None) == _lib.OK
