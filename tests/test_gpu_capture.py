"""Vectors that are allocated while the context's stream is captured into a HIP graph."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("mode", ["relaxed", "thread_local", "global"])
@pytest.mark.parametrize("n", [1, 1000, 300_001])
def test_a_vector_allocated_under_capture(mode, n):
    """zero at every replay, and usable by what is captured behind it"""
    from admm_amd import capi
    side = torch.cuda.Stream()
    ctx = capi.Context(0, stream=side.cuda_stream)
    x = ctx.vec(n, np.arange(n, dtype=np.float32))
    y = ctx.vec(n, np.ones(n, np.float32))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode=mode):
        v, out = ctx.vec(n), ctx.vec(n)
        ctx.payload(x, y, 2.0, out)
    for turn in range(4):
        torch.cuda.synchronize()
        v.upload(np.full(n, 3.0, np.float32))
        out.zero()
        ctx.sync()
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(v.download(), np.zeros(n, np.float32))
        got = out.download()
        if turn == 0:
            first = got
            eager = ctx.vec(n)
            ctx.payload(x, y, 2.0, eager)
            np.testing.assert_array_equal(got, eager.download())
        np.testing.assert_array_equal(got, first)
    del graph
    for u in (x, y, v, out, eager):
        u.free()
    ctx.close()
