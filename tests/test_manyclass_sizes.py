"""Workspace sizes of shapes that no call takes: refused, where the bytes would not fit 64 bits or the call would refuse them; no GPU."""
import ctypes as C

import pytest

from admm_amd import capi


@pytest.fixture(scope="module")
def L():
    from admm_amd import build
    build.build_lib()
    return capi.load()


def size(fn, *args):
    n = C.c_uint64(12345)
    rc = fn(*args, C.byref(n))
    return rc, n.value


@pytest.mark.parametrize("rows,cols,fits", [(1 << 39, 1 << 30, False), (1 << 39, (1 << 31) - 256, False), (1 << 16, 1 << 30, False), (1 << 15, 1 << 30, True),
                                            ((1 << 40) - 1, 32, True), (1 << 39, 5000, False), (1 << 20, 1 << 20, True)])
def test_sample(L, rows, cols, fits):
    """the product that a matrix of logits may have: fewer than 2^46 elements"""
    rc, n = size(L.admm_sample_workspace, rows, cols)
    assert (rc == 0) == fits
    if fits:
        assert n < rows * cols * 4 + (1 << 24)
    else:
        assert "logits" in L.admm_last_error().decode()


@pytest.mark.parametrize("nnz,cols,fits", [((1 << 32) - 256, 1 << 39, False), ((1 << 32) - 256, 1 << 34, False), (1 << 20, 1 << 38, False), (1000, 1 << 36, False),
                                           ((1 << 32) - 256, 65535 * 64 * 8, True), (1000, 65535 * 64 * 8, True), (1000, 65535 * 64 * 8 + 1, False), (16, 1 << 39, True),
                                           (0, 1 << 39, True)])
def test_embed_grad(L, nnz, cols, fits):
    """as many columns as the gradient takes (65535 tiles of 64 lanes of 8); where no workspace is needed, any number"""
    bags = capi.BagsStruct(1 << 20, 1 << 20, None, 1000, nnz, capi.I64)
    rc, n = size(L.admm_embed_grad_workspace, C.byref(bags), cols)
    assert (rc == 0) == fits
    if not fits:
        assert "columns" in L.admm_last_error().decode()
    elif nnz > 16:
        chunk = 8 if nnz * cols <= 1 << 23 else 16 if nnz * cols <= 1 << 25 else 32
        assert n == (nnz + chunk - 1) // chunk * 2 * ((cols + 7) // 8 * 8) * 4
    else:
        assert n == 0
