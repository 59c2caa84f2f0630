"""What the library's host side does with devices and streams, on a runtime that records its calls (hip_recorder.c): two devices,
no GPU.  Every test runs in a process of its own, because the recorder takes the HIP runtime's place in it."""
import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    from admm_amd import build
    build.build_lib()
    so = str(tmp_path_factory.mktemp("rec") / "hip_recorder.so")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", "-w", "-I/opt/rocm/include", os.path.join(ROOT, "tests", "hip_recorder.c"), "-o", so])
    return so


PRELUDE = """
import ctypes as C, sys
import numpy as np
rec = C.CDLL(%r, mode=C.RTLD_GLOBAL)
rec.rec_name.restype = C.c_char_p
rec.rec_stream.restype = C.c_void_p
sys.path.insert(0, %r)
from admm_amd import capi
L = capi.load()

def calls():
    return [(rec.rec_name(i).decode(), rec.rec_device(i), rec.rec_stream(i)) for i in range(rec.rec_count())]

def current():
    d = C.c_int()
    rec.hipGetDevice(C.byref(d))
    return d.value
"""


def run(recorder, body):
    out = subprocess.run([sys.executable, "-c", PRELUDE % (recorder, ROOT) + textwrap.dedent(body)], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-4000:]
    return out.stdout


def test_the_default_stream_is_that_of_the_contexts_device(recorder):
    """a context on device 1's default stream, called while device 0 is current: the default stream is a device's own, so
    everything has to be queued, and waited for, with device 1 current"""
    run(recorder, """
    ctx = capi.Context(1, stream=capi.DEFAULT_STREAM)
    n = 64
    v = [ctx.vec(n) for _ in range(6)]
    rows = np.array([0, 2, 3], np.uint64)
    csr = ctx.csr_upload(rows, np.array([0, 5, 7]), None, np.array([0, 1.]), n)
    host = np.zeros(n, np.float32)
    ctx.timing_enable(True)
    many = {  # (calls on built copies are left out: the copies' sizes come from kernels)
        "sync": lambda: ctx.sync(),
        "vec": lambda: ctx.vec(n),
        "upload": lambda: v[0].upload(host),
        "download": lambda: v[0].download(),
        "zero": lambda: v[0].zero(),
        "copy": lambda: v[0].copy_from(v[1]),
        "payload": lambda: ctx.payload(v[0], v[1], 0.1, v[2]),
        "global_update": lambda: L.admm_global_update(ctx.h, v[0].ptr, 1, 0.1, 0.1, 0.1, v[1].ptr, n),
        "dual_update": lambda: L.admm_dual_update(ctx.h, v[0].ptr, v[1].ptr, v[2].ptr, 0.1, n),
        "consensus": lambda: L.admm_consensus(ctx.h, v[0].ptr, 1, 0.1, 0.1, 0.1, v[1].ptr, v[2].ptr, v[3].ptr, n, None, None),
        "consensus with sums": lambda: L.admm_consensus(ctx.h, v[0].ptr, 1, 0.1, 0.1, 0.1, v[1].ptr, v[2].ptr, v[3].ptr, n, C.byref(C.c_double()), None),
        "timing_get": lambda: ctx.timing_get(capi.K_ELEMENTWISE),
        "timing_reset": lambda: (ctx.payload(v[0], v[1], 0.1, v[2]), rec.hipSetDevice(0), ctx.timing_reset()),
        "timing off": lambda: (ctx.payload(v[0], v[1], 0.1, v[2]), rec.hipSetDevice(0), ctx.timing_enable(False)),
        "download set": lambda: csr.download(),
        "copy_labels": lambda: L.admm_csr_copy_labels(csr.h, v[0].ptr),
        "build_transposed": lambda: L.admm_csr_build_transposed(csr.h, 0, 0),
        "predict": lambda: L.admm_predict(csr.h, (C.c_void_p * 1)(v[0].ptr), 1, v[1].ptr),
        "metrics": lambda: L.admm_metrics(csr.h, (C.c_void_p * 1)(v[0].ptr), 1, C.byref(C.c_double()), C.byref(C.c_double()), None),
        "ftrl_pass by row": lambda: L.admm_ftrl_pass(csr.h, *[x.ptr for x in v[:5]], 0.1, 1.0, 0.1, 0.1, 1),
        "ftrl_pass_multi": lambda: ctx.ftrl_pass_multi([csr], [v[0]], [v[1]], [v[2]], [v[3]], [v[4]], 0.1, 1.0, 0.1, 0.1),
        "embed": lambda: ctx.embed(csr.bags(), capi.DeviceMat(v[0].ptr.value, n, 1), capi.DeviceMat(v[1].ptr.value, 2, 1)),
        "free": lambda: v[5].free(),
        "relabel": lambda: L.admm_csr_relabel_by_frequency(csr.h),
        "destroy": lambda: csr.destroy(),
        "close": lambda: ctx.close(),
    }
    for name, call in many.items():
        rec.hipSetDevice(0)
        rec.rec_clear()
        call()
        seen = [c for c in calls() if c[0] != "hipMalloc"]
        wrong = [c for c in seen if c[1] != 1]
        assert not wrong, (name, wrong)
        assert seen or name == "vec", (name, L.admm_last_error())
    """)


def test_contexts_with_a_stream_of_their_own_do_not_touch_the_current_device(recorder):
    """calls that never set the device (their stream says where they go) still do not"""
    run(recorder, """
    ctx = capi.Context(1, stream=0x6000)
    v = [ctx.vec(16) for _ in range(3)]
    rec.hipSetDevice(0)
    v[0].zero(); v[0].copy_from(v[1]); ctx.payload(v[0], v[1], 0.1, v[2]); ctx.sync()
    v[0].upload(np.zeros(16, np.float32))
    assert current() == 0
    assert all(c[2] == 0x6000 for c in calls() if c[0] not in ("hipMalloc", "hipMemcpy"))
    """)


MANY = """
def vec(n):
    return ctx.vec(n)

def mat(rows, cols):
    return capi.DeviceMat(vec(rows * cols).ptr.value, rows, cols)

def ids(n):
    return capi.Bags(vec(2 * n).ptr.value, None, None, n, n, capi.I64)
"""


MANY_ALLOC = """
ctx = capi.Context(1, stream=stream)
""" + MANY + """
x, u, tok, b = mat(3, 5000), vec(3), capi.DeviceBuf(ctx, 12), ids(100)
src, to, loss, lab = mat(100, 8), mat(50, 8), vec(3), vec(3)
wide = mat(3, 200000)
rec.hipSetDevice(0)
rec.rec_clear()
ctx.sample(x, u, tok)
assert current() == 0, "sample"
order = ctx.embed_order(b, 50)
assert current() == 0, "embed_order"
ctx.embed_grad(b, order, src, to)
assert current() == 0, "embed_grad"
ctx.softmax_loss(wide, lab, loss)
assert current() == 0, "softmax_loss"
seen = calls()
assert sum(c[0] == "hipMalloc" for c in seen) >= 2 and all(c[1] == 1 for c in seen), seen
"""


def test_calls_without_a_workspace_leave_the_current_device(recorder):
    """the context's own workspace, and an order that embed_order makes, are allocated on the context's device; the calling
    thread's stays what it was"""
    run(recorder, "stream = 0x6000" + MANY_ALLOC)
    run(recorder, "stream = capi.DEFAULT_STREAM" + MANY_ALLOC)


def test_the_workspace_does_not_grow_under_capture(recorder):
    """what a graph uses is allocated before its capture: growing is refused, and nothing is allocated or queued; a call whose
    workspace is there is not"""
    run(recorder, """
    ctx = capi.Context(1, stream=0x6000)
    """ + textwrap.indent(MANY, "    ") + """
    x, u, tok, b = mat(3, 5000), vec(3), capi.DeviceBuf(ctx, 12), ids(100)
    for status in (1, 2, 4):   # captured, capture invalidated, not to be asked for
        rec.rec_capture(status)
        rec.rec_clear()
        for call in (lambda: ctx.sample(x, u, tok), lambda: ctx.embed_order(b, 50)):
            try:
                call()
            except capi.AdmmError as e:
                assert "captured" in str(e), e
            else:
                raise AssertionError("not refused")
        assert not calls(), calls()
        assert rec.hipSetDevice(1) == 0
    rec.rec_capture(0)
    ctx.sample(x, u, tok)
    rec.rec_capture(1)
    ctx.sample(x, u, tok)
    rec.rec_capture(0)
    ctx.close()
    """)


def test_a_refused_growth_keeps_the_workspace(recorder):
    """a call that needs more than there is, under capture: refused, and the calls that have enough go on"""
    run(recorder, """
    ctx = capi.Context(1, stream=0x6000)
    """ + textwrap.indent(MANY, "    ") + """
    x, u, tok = mat(3, 5000), vec(3), capi.DeviceBuf(ctx, 12)
    big, bu, btok = mat(400, 5000), vec(400), capi.DeviceBuf(ctx, 1600)
    ctx.sample(x, u, tok)
    had = ctx._scratch.ptr.value
    rec.rec_capture(1)
    try:
        ctx.sample(big, bu, btok)
    except capi.AdmmError as e:
        assert "captured" in str(e), e
    else:
        raise AssertionError("not refused")
    ctx.sample(x, u, tok)
    rec.rec_capture(0)
    assert ctx._scratch.ptr.value == had
    ctx.sample(big, bu, btok)
    assert ctx._scratch.ptr.value != had and [b.ptr.value for b in ctx._retired] == [had]
    ctx.close()
    """)


def test_vectors_may_be_allocated_under_capture(recorder):
    """admm_vec_alloc while the stream is captured: the thread's capture mode allows the allocation and is what it was
    afterwards, and what zeroes the vector is a kernel, not a memset, in the graph"""
    run(recorder, """
    ctx = capi.Context(1, stream=0x6000)
    rec.rec_capture(1)
    rec.rec_clear()
    v = ctx.vec(64)
    assert [c[0] for c in calls()] == ["hipMalloc, relaxed", "hipLaunchKernel"], calls()
    assert calls()[1][2] == 0x6000 and rec.rec_thread_mode() == 0
    for status in (2, 4):   # a capture that has failed, another stream's that keeps this one from being used
        rec.rec_capture(status)
        rec.rec_clear()
        try:
            ctx.vec(64)
        except capi.AdmmError as e:
            assert "captured" in str(e), e
        else:
            raise AssertionError("not refused")
        assert not calls(), calls()
    rec.rec_capture(0)
    rec.rec_clear()
    ctx.vec(64)
    assert [c[0] for c in calls()] == ["hipMalloc", "hipMemsetAsync"], calls()
    ctx.close()
    """)
