"""The paged cache's calls beside the ordinary ones, without a GPU."""
import ctypes
import os
import random
import re
import subprocess

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


@pytest.mark.parametrize("over", [
    dict(q_out=P16 + 2 * 64, v=9 * P16), dict(q_out=P16 - 2 * 64, v=9 * P16), dict(q_out=P16 + 2 * 128, v=9 * P16), dict(q_out=P16 + 2 * 3 * 128, v=9 * P16),
    dict(q_out=3 * P16 - 2 * 128, v=9 * P16), dict(q_out=9 * P16 + 2 * 64, v=9 * P16), dict(q_out=5 * P16, v=9 * P16, slots=None, k_out=3 * P16 + 2 * 128),
    dict(q_out=5 * P16, v=9 * P16, slots=None, k_out=P16 + 2 * 64), dict(q_out=5 * P16, v=9 * P16, slots=None, k_out=5 * P16 + 2 * 64)])
def test_rope_refuses_outputs_that_share_elements(over):
    L = _lib.lib()
    assert L.mkx_rope_axes(ctypes.byref(_rope_args(**over)), None) == _lib.EINVAL
    assert "shares elements" in L.mkx_last_error().decode()


@pytest.mark.parametrize("out", [P16 + 2 * 128, P16 - 2 * 128, P16 + 2 * 512, P16 + 2 * 3 * 512 + 2 * 384])
def test_attention_refuses_an_out_that_shares_elements_with_q(out):
    L = _lib.lib()
    assert L.mkx_page_attend(ctypes.byref(_attend_args(out=out)), None) == _lib.EINVAL
    assert "shares elements" in L.mkx_last_error().decode()


def test_shared_elements_against_a_count_of_them(tmp_path):
    """No pair of views that share nothing is called shared, and every pair that does is, where a stride spans the other axis."""
    (tmp_path / "o.cpp").write_text(
        '#include "mkx_overlap.h"\nextern "C" int share(int64_t p, int64_t xn, int64_t xt, int64_t xh, int64_t q, int64_t yn, int64_t yt, int64_t yh, int64_t T, '
        "int64_t hd) { return mkx::share_elements({(void*)p, xn, xt, xh}, {(void*)q, yn, yt, yh}, T, hd); }\n")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "reki-megakernel_amd", "csrc"), str(tmp_path / "o.cpp"), "-o",
                    str(tmp_path / "o.so")], check=True)
    share = ctypes.CDLL(str(tmp_path / "o.so")).share
    share.argtypes = [ctypes.c_int64] * 10
    rng = random.Random(3)
    counts = [0, 0]
    for _ in range(6000):
        T, N, hd = rng.randint(1, 5), rng.randint(1, 5), 8
        xn, yn = rng.randint(1, N), rng.randint(1, N)
        sh = 8 * rng.randint(1, 2)
        st = sh * N + 8 * rng.randint(0, 1)
        if rng.random() < 0.4:
            st = 8 * rng.randint(1, 2)
            sh = st * T + 8 * rng.randint(0, 2)
        xh, yh = (rng.choice([sh, 8 * rng.randint(0, 9)]) if n == 1 else sh for n in (xn, yn))
        by = 8 * rng.randint(-50, 50)
        held = [{base + t * st + h * s + c for t in range(T) for h in range(n) for c in range(hd)} for base, n, s in ((1 << 20, xn, xh), ((1 << 20) + by, yn, yh))]
        got, truth = bool(share(2 << 20, xn, st, xh, (2 << 20) + 2 * by, yn, st, yh, T, hd)), bool(held[0] & held[1])
        known = xn > 1 or yn > 1 or xh == yh == sh  # one head each: their own strides are not looked at
        assert got == truth or (not got and not known), (T, xn, yn, st, xh, yh, by)
        counts[truth] += 1
    assert min(counts) > 500
