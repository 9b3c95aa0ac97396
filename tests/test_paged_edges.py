"""The paged cache's calls beside the ordinary ones, without a GPU."""
import ctypes
import os
import re

import pytest

from mkx import _lib

from test_paged import P16, ROOT, SIZES, _attend_args, _rope_args


@pytest.mark.parametrize("over,status", SIZES + [(dict(q=None), _lib.EINVAL), (dict(ws=P16 + 16), _lib.EINVAL), (dict(out=P16), _lib.EINVAL)])
def test_attention_of_granted_requests_refuses(over, status):
    L = _lib.lib()
    assert L.mkx_page_attend_granted(ctypes.byref(_attend_args(**over)), P16, None) == status, L.mkx_last_error()
    assert "mkx_page_attend_granted:" in L.mkx_last_error().decode()
    assert L.mkx_page_attend_granted(None, P16, None) == _lib.EINVAL
    assert L.mkx_page_attend_granted(ctypes.byref(_attend_args(T=0)), P16, None) == _lib.OK


@pytest.mark.parametrize("over,status", [
    (dict(dtype=2 | _lib.ROPE_POS64), _lib.EUNSUPPORTED), (dict(dtype=_lib.BF16 | 4 * _lib.ROPE_POS64), _lib.EUNSUPPORTED),
    (dict(dtype=_lib.FP16 | _lib.ROPE_POS64, pos=P16 + 4), _lib.EINVAL), (dict(pos=P16 + 2), _lib.EINVAL), (dict(dtype=_lib.BF16 | _lib.ROPE_POS64, pos_stride=3), _lib.EINVAL)])
def test_rope_of_64_bit_positions_refuses(over, status):
    L = _lib.lib()
    assert L.mkx_rope_axes(ctypes.byref(_rope_args(**over)), None) == status, L.mkx_last_error()
    assert L.mkx_rope_axes(ctypes.byref(_rope_args(T=0, dtype=_lib.FP16 | _lib.ROPE_POS64)), None) == _lib.OK


@pytest.mark.parametrize("over,status", [
    (dict(dtype=2 | _lib.ROPE_NORM32), _lib.EUNSUPPORTED), (dict(dtype=_lib.BF16 | _lib.ROPE_NORM32, q_norm=P16 + 8), _lib.EINVAL),
    (dict(dtype=_lib.FP16 | _lib.ROPE_NORM32 | _lib.ROPE_POS64, k_norm=P16 + 4), _lib.EINVAL)])
def test_rope_of_32_bit_weights_refuses(over, status):
    L = _lib.lib()
    assert L.mkx_rope_axes(ctypes.byref(_rope_args(**over)), None) == status, L.mkx_last_error()
    assert L.mkx_rope_axes(ctypes.byref(_rope_args(T=0, dtype=_lib.FP16 | _lib.ROPE_NORM32)), None) == _lib.OK


def test_rope_flags_are_the_headers():
    text = open(os.path.join(ROOT, "include", "mkx.h")).read()
    for name in ("ROPE_POS64", "ROPE_NORM32"):
        assert int(re.search(rf"#define MKX_{name} (\d+)", text).group(1)) == getattr(_lib, name)
