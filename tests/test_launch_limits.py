"""Calls of more threads than a launch holds (2^32 - 1) are refused by the limit that the header names, before anything is launched; the
largest ones below it get past the check, to the launch, which these null devices cannot make."""
import ctypes

import pytest

from nanoengine_amd import _lib

ONE, P, f = ctypes.c_void_p(16), None, ctypes.c_float


@pytest.fixture(scope="module")
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the arguments are no memory")
    if not _lib.LIB_PATH.exists():
        from nanoengine_amd import build
        build.build()
    return _lib.load()


def norm(rows, dim):
    return "dsa_rms_norm", [ONE, dim, P, 0, P, 0, ONE, 0, f(1e-6), rows, dim, ONE, dim, P, 0, P, 0, 0, P]


def quant(rows, dim):
    return "dsa_act_quant", [ONE, dim, rows, dim, ONE, dim, ONE, -(-dim // 128), 0, P]


def rope(tokens, heads, k_heads, rot):
    return "dsa_rope", [ONE, heads * rot, rot, heads, ONE, heads * rot, rot, ONE, k_heads * rot, rot, k_heads, ONE, k_heads * rot, rot,
                        tokens, rot, ONE, 100, ONE, 0, 1, 1, P]


def product(m, n, k):
    return "dsa_fp8_gemm", [ONE, k, ONE, -(-k // 128), ONE, k, ONE, -(-k // 128), 0, m, n, k, ONE, n, 0, P, 0, P]


@pytest.mark.parametrize("call,args", [(norm, (2 ** 22, 8192)), (norm, (2 ** 22, 4097)), (norm, (2 ** 23, 4096)), (norm, (2 ** 24, 2048)),
                                       (norm, (2 ** 26, 512)), (norm, (2 ** 31 - 1, 8)), (quant, (2 ** 28, 128)), (quant, (2 ** 21, 16384)),
                                       (quant, (2 ** 31 - 1, 1)), (rope, (2 ** 28, 4, 1, 64)), (rope, (2 ** 26, 1, 0, 512)),
                                       (product, (1, 2 ** 29, 16)), (product, (8, 2 ** 31 - 1, 128))])
def test_past_a_launch(lib, call, args):
    name, a = call(*args)
    assert getattr(lib, name)(*a) == 2, lib.dsa_last_error()
    assert b"2^32" in lib.dsa_last_error()


@pytest.mark.parametrize("call,args", [(norm, (2 ** 22 - 1, 8192)), (norm, (2 ** 23 - 1, 4096)), (norm, (2 ** 24 - 1, 2048)),
                                       (norm, (2 ** 26 - 4, 512)), (quant, (2 ** 28 - 16, 128)), (rope, (2 ** 28 - 32, 4, 1, 64)),
                                       (product, (1, 2 ** 29 - 32, 16))])
def test_below_it(lib, call, args):
    name, a = call(*args)
    assert getattr(lib, name)(*a) == 3, lib.dsa_last_error()  # (no device)
