"""Outputs on top of inputs: what the header names is taken, and what would lose a result or read rows that are written already is
refused before anything is launched. (Without a device a call that is taken ends at its launch, with status 3.)"""
import ctypes

import pytest

from nanoengine_amd import _lib

P, f = None, ctypes.c_float


def at(n):
    return ctypes.c_void_p(1 << 20 | n << 12)


@pytest.fixture(scope="module")
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the arguments are no memory")
    if not _lib.LIB_PATH.exists():
        from nanoengine_amd import build
        build.build()
    return _lib.load()


def norm(lib, x, residual, total, out, rows=4, x_s=256, residual_s=256, total_s=256, out_s=256):
    return lib.dsa_rms_norm(x, x_s, residual, residual_s, total, total_s, at(9), 0, f(1e-6), rows, 256, out, out_s, P, 0, P, 0, 0, P)


def test_norm(lib):
    x, r, o, t = at(1), at(2), at(3), at(4)
    for args in ((x, P, P, o), (x, P, P, x), (x, r, r, o), (x, r, x, o), (x, r, t, x), (x, r, r, x), (x, r, t, o)):
        assert norm(lib, *args) == 3, lib.dsa_last_error()
    # the sum and the norm in one place: one of them would be lost
    assert norm(lib, x, r, x, x) == 1 and norm(lib, x, r, o, o) == 1 and b"residual_out" in lib.dsa_last_error()
    # in place with rows elsewhere: a row's output would lie on another row's input
    for args, stride in (((x, P, P, x), dict(out_s=320)), ((x, P, P, x), dict(x_s=320)), ((x, r, r, o), dict(total_s=264)),
                         ((x, r, x, o), dict(x_s=264))):
        assert norm(lib, *args, **stride) == 1, (args, stride)
        assert norm(lib, *args, rows=1, **stride) == 3


def rope(lib, q, q_out, k=P, k_out=P, tokens=4, heads=3, q_s=(640, 64), qo_s=(640, 64), k_s=(64, 64), ko_s=(64, 64), k_heads=0):
    return lib.dsa_rope(q, *q_s, heads, q_out, *qo_s, k, *k_s, k_heads, k_out, *ko_s, tokens, 64, at(8), 100, at(9), 0, 1, 1, P)


def test_rope(lib):
    q, k, o = at(1), at(2), at(3)
    assert rope(lib, q, q) == 3 and rope(lib, q, o, q_s=(0, 0)) == 3 and rope(lib, q, o, qo_s=(192, 64)) == 3
    assert rope(lib, q, q, qo_s=(192, 64)) == 1 and b"in place" in lib.dsa_last_error()
    assert rope(lib, q, q, q_s=(640, 128)) == 1 and rope(lib, q, q, q_s=(640, 0)) == 1
    # one token or one head: its stride says nothing
    assert rope(lib, q, q, tokens=1, qo_s=(192, 64)) == 3 and rope(lib, q, q, heads=1, q_s=(640, 0)) == 3
    assert rope(lib, q, q, k, k, k_heads=1) == 3 and rope(lib, q, q, k, k, k_heads=1, k_s=(128, 64)) == 1
