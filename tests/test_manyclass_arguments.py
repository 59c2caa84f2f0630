"""Arguments of the many-class calls of the Python binding that are refused, or taken for what they are, before anything is
queued: on the recording runtime, without a GPU."""
import textwrap

from test_host_devices import MANY, recorder, run  # noqa: F401

REFUSED = """
def refused(call, text):
    rec.rec_clear()
    try:
        call()
    except capi.AdmmError as e:
        assert text in str(e), (text, str(e))
    else:
        raise AssertionError("not refused: " + text)
    assert not [c for c in calls() if c[0] == "hipLaunchKernel"], calls()
"""


def check(recorder, body):  # noqa: F811
    run(recorder, "ctx = capi.Context(0, stream=0x6000)" + MANY + REFUSED + textwrap.dedent(body))


def test_labels_in_a_buffer_say_their_type(recorder):  # noqa: F811
    """a buffer of bytes could hold labels of three types: it has to say which, and the library is told that one"""
    check(recorder, """
    x, loss = mat(4, 8), vec(4)
    refused(lambda: ctx.softmax_loss(x, ctx.buf(32), loss), "type")
    refused(lambda: ctx.softmax_loss(x, ctx.buf(16), loss), "type")
    refused(lambda: ctx.softmax_loss(x, ctx.buf(32, type=capi.BF16), loss), "type")
    refused(lambda: ctx.softmax_loss(x, ctx.buf(31, type=capi.I64), loss), "31 bytes")
    refused(lambda: ctx.sample(x, ctx.buf(16, type=capi.I32), ctx.buf(16)), "uniform")
    refused(lambda: ctx.buf(16, type=9), "type 9")
    seen, library = [], ctx.L.admm_softmax_loss

    class Spy:
        def __getattr__(self, name):
            if name != "admm_softmax_loss":
                return getattr(L, name)
            return lambda *a: seen.append(a[3]) or library(*a)
    ctx.L = Spy()
    for kind, size in ((capi.I32, 16), (capi.I64, 32), (capi.F32, 16)):
        ctx.softmax_loss(x, ctx.buf(size, type=kind), loss)
    assert seen == [capi.I32, capi.I64, capi.F32], seen
    ctx.L = L
    ctx.sample(x, ctx.buf(16), ctx.buf(16, type=capi.I32))   # one type only: it need not be said
    """)


def test_bags_of_a_set_that_is_gone(recorder):  # noqa: F811
    """the arrays of a sample set's bags are the set's: after destroy nothing reads them; the gradient, which takes only
    counts from its bags, goes on with an order that was made before"""
    check(recorder, """
    csr = ctx.csr_upload(np.array([0, 2, 3], np.uint64), np.array([0, 5, 7]), None, np.array([0, 1.]), 64)
    bags = csr.bags()
    table, out, grad = mat(64, 8), mat(2, 8), mat(64, 8)
    rec.rec_clear()
    ctx.embed(bags, table, out)
    order = ctx.embed_order(bags, 64)
    assert len([c for c in calls() if c[0] == "hipLaunchKernel"]) >= 2
    csr.destroy()
    refused(lambda: ctx.embed(bags, table, out), "destroyed")
    refused(lambda: ctx.embed_order(bags, 64, order), "destroyed")
    refused(lambda: ctx.embed_order(bags, 64), "destroyed")
    refused(lambda: csr.bags(), "destroyed")
    ctx.embed_grad(bags, order, out, grad)
    refused(lambda: ctx.embed(None, table, out), "bags")
    refused(lambda: ctx.embed(vec(4), table, out), "bags")
    """)


def test_memory_of_another_contexts_gpu(recorder):  # noqa: F811
    """vectors, buffers, bags and matrices that are known to lie on another GPU are refused, as tensors are"""
    check(recorder, """
    other = capi.Context(1, stream=0x7000)
    csr = other.csr_upload(np.array([0, 2, 3], np.uint64), np.array([0, 5, 7]), None, np.array([0, 1.]), 64)
    x, loss, lab, u, tok, far = mat(4, 8), vec(4), vec(4), vec(4), ctx.buf(16), other.vec(4096)
    table, out, grad, mine = mat(64, 8), mat(2, 8), mat(64, 8), ids(2)
    refused(lambda: ctx.embed(csr.bags(), table, out), "bags")
    refused(lambda: ctx.embed_order(csr.bags(), 64), "bags")
    order = other.embed_order(csr.bags(), 64)
    refused(lambda: ctx.embed_grad(csr.bags(), order, out, grad), "bags")
    refused(lambda: ctx.embed_grad(mine, order, out, grad), "order")
    refused(lambda: ctx.embed_order(mine, 64, other.buf(1 << 16)), "order")
    refused(lambda: ctx.softmax_loss(x, far, loss), "labels")
    refused(lambda: ctx.softmax_loss(x, lab, far), "loss")
    refused(lambda: ctx.softmax_loss(x, lab, loss, weight=far), "weight")
    refused(lambda: ctx.sample(x, u, other.buf(16)), "token")
    refused(lambda: ctx.sample(x, u, tok, workspace=other.buf(1 << 16)), "workspace")
    there = capi.DeviceMat(far.ptr.value, 4, 8, device=1)
    refused(lambda: ctx.sample(there, u, tok), "logits")
    refused(lambda: ctx.embed(mine, there, mat(2, 8)), "table")
    ctx.sample(x, u, tok)
    other.sample(there, far, other.buf(16))
    ctx.embed(mine, mat(4, 8), mat(2, 8))      # bags and matrices from pointers may be anywhere: the caller knows
    """)


def test_freed_vectors_are_not_absent_ones(recorder):  # noqa: F811
    """a weight, temperature or filter whose memory was freed is not taken for one that was not given"""
    check(recorder, """
    x, loss, lab, u, tok = mat(4, 8), vec(4), vec(4), vec(4), ctx.buf(16)
    gone, k = vec(4), ctx.buf(16)
    gone.free(), k.free()
    refused(lambda: ctx.softmax_loss(x, lab, loss, weight=gone), "weight")
    refused(lambda: ctx.softmax_loss(x, lab, loss, lse=gone), "lse")
    for name in ("logprob", "temperature", "top_p", "min_p"):
        refused(lambda: ctx.sample(x, u, tok, **{name: gone}), name)
    refused(lambda: ctx.sample(x, u, tok, top_k=k), "top_k")
    refused(lambda: ctx.embed_order(ids(4), 8, k), "order")
    refused(lambda: ctx.sample(x, u, tok, workspace=k), "workspace")
    none = capi.DeviceVec.from_ptr(ctx, 0, 0)
    ctx.softmax_loss(capi.DeviceMat(0, 0, 8), none, none, weight=none)   # nothing of nothing
    """)


def test_bags_of_something_else(recorder):  # noqa: F811
    """row pointers and factors that are no tensors are refused as ids are"""
    check(recorder, """
    class Tensor:
        def __init__(self, n, dtype):
            self.n, self.dtype, self.mem, self.shape = n, dtype, vec(2 * n + 2), (n,)
        data_ptr = lambda self: self.mem.ptr.value
        numel = lambda self: self.n
        get_device = lambda self: 0
        is_contiguous = lambda self: True
        stride = lambda self: (1,)
    capi._ARRAYS.update({"i64": capi.I64, "f32": capi.F32})
    t = Tensor(4, "i64")
    ctx.embed(ctx.bags(t), mat(8, 2), mat(4, 2))
    ctx.embed(ctx.bags(t, Tensor(3, "i64"), Tensor(4, "f32")), mat(8, 2), mat(2, 2))
    for other in (np.zeros(3, np.int64), [0, 2, 4], vec(4)):
        refused(lambda: ctx.bags(t, other), "rowptr")
    refused(lambda: ctx.bags(t, Tensor(3, "f32")), "rowptr")
    refused(lambda: ctx.bags(t, Tensor(0, "i64")), "rowptr")
    refused(lambda: ctx.bags(np.zeros(3, np.int64)), "ids")
    refused(lambda: ctx.bags(t, Tensor(3, "i64"), np.ones(4, np.float32)), "val")
    """)
