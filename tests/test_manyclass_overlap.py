"""Matrices that lie side by side in rows of one stride do not overlap, whatever the spans from their first to their last
element do; all others that share memory are refused.  On the recording runtime, without a GPU."""
from test_host_devices import recorder  # noqa: F401
from test_manyclass_arguments import check


def test_matrices_side_by_side(recorder):  # noqa: F811
    check(recorder, """
    base = vec(1 << 14).ptr.value
    base += -base % 256
    b, labels = ids(6), vec(6)
    loss = vec(6)

    def at(offset, cols, stride=100, rows=6, type=capi.F32):
        return capi.DeviceMat(base + offset, rows, cols, type, stride)

    def softmax(x, g):
        ctx.softmax_loss(x, labels, loss, grad=g)
    order = ctx.embed_order(b, 6)
    for call in (softmax, lambda x, g: ctx.embed(b, x, g), lambda x, g: ctx.embed_grad(b, order, x, g)):
        rec.rec_clear()
        call(at(0, 50), at(200, 50))                    # halves of the same rows, either first
        call(at(200, 50), at(0, 50))
        call(at(12, 25), at(112, 25))
        call(at(0, 50), at(200 + 400, 50))              # a row further on
        call(at(200 + 800, 50), at(0, 50))
        assert len([c for c in calls() if c[0] == "hipLaunchKernel"]) >= 5, calls()
        for x, g in ((at(0, 51), at(200, 51)),          # one column of both
                     (at(0, 50), at(196, 50)),
                     (at(200, 50), at(4, 50)),
                     (at(0, 50), at(220, 50)),          # into the next row
                     (at(0, 50), at(200, 50, 99)),      # another stride
                     (at(0, 50), at(400, 50))):         # the same columns of other rows
            refused(lambda: call(x, g), "overlaps")
    # one row among many; another type of the same row length in bytes
    one = ids(1)
    ctx.embed(one, at(0, 50), at(200 + 400, 50, rows=1))
    ctx.embed(one, at(0, 50, rows=1), at(200, 50, stride=100))
    ctx.embed(b, at(0, 50, 200, type=capi.BF16), at(200, 50))
    refused(lambda: ctx.embed(b, at(0, 50, 200, type=capi.BF16), at(96, 50)), "overlaps")
    refused(lambda: ctx.embed(one, at(0, 50), at(96, 50, rows=1)), "overlaps")
    refused(lambda: ctx.embed(one, at(0, 50, rows=1), at(96, 50, rows=1)), "overlaps")
    """)
