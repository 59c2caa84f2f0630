"""What the many-class entry points (admm_embed, admm_embed_order, admm_embed_grad, admm_softmax_loss, admm_sample) refuse,
and the sizes of their workspaces: all of it is decided on the host, before anything is launched, so no GPU is needed.  The
context is a block of zeros that a refused call never looks into."""
import ctypes as C

import pytest

from admm_amd import capi

F32, BF16, F16, I32, I64 = range(5)
P = 1 << 20  # a pretended device address


@pytest.fixture(scope="module")
def L():
    from admm_amd import build
    build.build_lib()
    return capi.load()


@pytest.fixture(scope="module")
def ctx():
    return C.create_string_buffer(1 << 14)


def mat(rows, cols, type=F32, stride=None, at=P):
    return capi.MatStruct(at, rows, cols, cols if stride is None else stride, type)


def bags(n, id_type=I64, rowptr=None, val=None, nnz=None, ids=P):
    return capi.BagsStruct(ids, rowptr, val, n, n if nnz is None else nnz, id_type)


def refused(L, rc, text):
    assert rc == -1, rc
    assert text in L.admm_last_error().decode(), L.admm_last_error()


def test_embed(L, ctx):
    def call(b, t, o, c=ctx):
        return L.admm_embed(c, C.byref(b) if b else None, C.byref(t) if t else None, 1.0, C.byref(o) if o else None)
    far = P + (1 << 30)
    table, out = mat(10, 8), mat(4, 8, at=far)
    refused(L, call(bags(4), table, out, None), "ctx is NULL")
    refused(L, call(None, table, out), "bags is NULL")
    refused(L, call(bags(4), None, out), "table is NULL")
    refused(L, call(bags(4), table, None), "out is NULL")
    refused(L, call(bags(4, id_type=F32), table, out), "ids of type")
    refused(L, call(bags(4, ids=None), table, out), "ids is NULL")
    refused(L, call(bags(4, ids=P + 4), table, out), "not aligned")
    refused(L, call(bags(4, nnz=5), table, out), "without row pointers")
    refused(L, call(bags(4, val=P), table, out), "factors need row pointers")
    refused(L, call(bags(4, rowptr=P, nnz=2**32 - 1), table, out), "2^32")
    refused(L, call(bags(4), mat(0, 8), out), "table of 0 rows")
    refused(L, call(bags(4), mat(2**32 - 1, 8), out), "a table of")
    refused(L, call(bags(4), mat(1 << 39, 1 << 10), out), "too large")
    refused(L, call(bags(4), mat(10, 8, type=I32), out), "has type")
    refused(L, call(bags(4), mat(10, 8, stride=7), out), "apart")
    refused(L, call(bags(4), mat(10, 8, at=P + 2), out), "not aligned")
    refused(L, call(bags(4), mat(10, 8, at=None), out), "no memory")
    refused(L, call(bags(4), table, mat(3, 8, at=far)), "out is 3 x 8")
    refused(L, call(bags(4), table, mat(4, 7, at=far)), "out is 4 x 7")
    refused(L, call(bags(4), table, mat(4, 8, type=BF16, at=far)), "the table's type")
    refused(L, call(bags(4), mat(10, 8, type=F16), mat(4, 8, type=BF16, at=far)), "the table's type")
    refused(L, call(bags(4), table, mat(4, 8, at=P + 9 * 8 * 4)), "overlaps")
    assert call(bags(0, ids=None), table, mat(0, 8, at=None)) == 0
    assert call(bags(4), mat(10, 0), mat(4, 0)) == 0


def test_embed_grad(L, ctx):
    far = P + (1 << 30)
    n = C.c_uint64()
    b = bags(100)
    assert L.admm_embed_order_bytes(C.byref(b), 50, C.byref(n)) == 0
    size = n.value
    assert 2 * 4 * 100 <= size < 1 << 16
    refused(L, L.admm_embed_order_bytes(C.byref(b), 0, C.byref(n)), "table of 0 rows")
    refused(L, L.admm_embed_order_bytes(C.byref(b), 50, None), "bytes is NULL")
    refused(L, L.admm_embed_order(None, C.byref(b), 50, P, size), "ctx is NULL")
    refused(L, L.admm_embed_order(ctx, C.byref(b), 50, None, size), "order is NULL")
    refused(L, L.admm_embed_order(ctx, C.byref(b), 50, P + 128, size), "256 bytes")
    refused(L, L.admm_embed_order(ctx, C.byref(b), 50, P, size - 1), "are needed")
    empty = bags(0)
    assert L.admm_embed_order(ctx, C.byref(empty), 50, None, 0) == 0
    assert L.admm_embed_grad_workspace(C.byref(b), 8, C.byref(n)) == 0
    need = n.value
    assert need > 0

    def call(g, t, order=P, bytes=size, ws=P, wn=need, bb=b, acc=0):
        return L.admm_embed_grad(ctx, C.byref(bb), order, bytes, C.byref(g), 1.0, acc, C.byref(t), ws, wn)
    g, t = mat(100, 8), mat(50, 8, at=far)
    refused(L, call(mat(99, 8), t), "grad_out is 99 x 8")
    refused(L, call(mat(100, 9), t), "grad_out is 100 x 9")
    refused(L, call(g, mat(50, 8, type=BF16, at=far)), "grad_out's type")
    refused(L, call(g, mat(50, 8)), "overlaps")
    refused(L, call(g, t, order=None), "order is NULL")
    refused(L, call(g, t, bytes=size - 1), "are needed")
    refused(L, call(g, t, ws=None), "workspace is NULL")
    refused(L, call(g, t, wn=need - 1), "workspace is NULL")
    refused(L, call(g, mat(0, 8, at=far)), "table of 0 rows")
    assert call(g, t, bb=empty, order=None, ws=None, acc=1) == 0  # nothing to add


def test_softmax_loss(L, ctx):
    far = P + (1 << 30)

    def call(x, labels=P, kind=I64, loss=P, g=None):
        return L.admm_softmax_loss(ctx, C.byref(x), labels, kind, None, 1.0, loss, None, C.byref(g) if g else None, far, 1 << 40)
    x = mat(10, 8)
    refused(L, call(x, kind=BF16), "labels of type")
    refused(L, call(x, labels=None), "labels or loss is NULL")
    refused(L, call(x, loss=None), "labels or loss is NULL")
    refused(L, call(mat(10, 0)), "no classes")
    refused(L, call(x, g=mat(9, 8, at=far)), "another shape")
    refused(L, call(x, g=mat(10, 8, type=BF16, at=far)), "another shape or type")
    refused(L, call(x, g=mat(10, 8, at=P + 4)), "overlaps")
    refused(L, call(x, g=mat(10, 8, stride=16)), "overlaps")
    assert call(mat(0, 8)) == 0
    n = C.c_uint64()
    assert L.admm_softmax_loss_workspace(10, 8, C.byref(n)) == 0
    refused(L, L.admm_softmax_loss_workspace(10, 8, None), "bytes is NULL")
    refused(L, L.admm_softmax_loss_workspace(1 << 50, 8, C.byref(n)), "logits")


def test_sample(L, ctx):
    def call(x, u=P, token=P, ws=P, wn=1 << 40):
        return L.admm_sample(ctx, C.byref(x), None, u, token, None, ws, wn)
    refused(L, call(mat(4, 8), u=None), "uniform or token is NULL")
    refused(L, call(mat(4, 8), token=None), "uniform or token is NULL")
    refused(L, call(mat(4, 0)), "0 classes")
    refused(L, call(mat(1, 1 << 31)), "classes")
    assert call(mat(0, 8)) == 0
    n = C.c_uint64()
    refused(L, L.admm_sample_workspace(1, 1 << 31, C.byref(n)), "logits")
    refused(L, L.admm_sample_workspace(1, 10, None), "bytes is NULL")


def test_csr_bags(L):
    out = capi.BagsStruct()
    refused(L, L.admm_csr_bags(None, C.byref(out)), "NULL argument")
