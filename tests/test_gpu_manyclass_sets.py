"""Bags of a sample set whose rows are renumbered or freed after they were asked for."""
import numpy as np
import pytest

from conftest import make_synth_csr

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def make(ctx, dim):
    raw = make_synth_csr(500, dim, 12, seed=3, binary=False)
    return ctx.csr_upload(raw.rowptr, raw.col, raw.val, np.zeros(500, np.float32), dim)


@pytest.mark.parametrize("what", ["destroy", "relabel", "lean"])
def test_bags_go_stale(what):
    from admm_amd import capi
    ctx, dim = capi.Context(0, stream=capi.DEFAULT_STREAM), 600
    csr = make(ctx, dim)
    bags = csr.bags()
    table, out = torch.randn(dim, 5, device="cuda"), torch.empty(500, 5, device="cuda")
    grad = [torch.empty(dim, 5, device="cuda") for _ in range(2)]
    ctx.embed(bags, table, out)
    before = out.clone()
    order = ctx.embed_order(bags, dim)
    ctx.embed_grad(bags, order, before, grad[0])
    if what == "destroy":
        csr.destroy()
    else:
        if what == "lean":
            csr.set_lean()
        csr.relabel_by_frequency()
        csr.build_transposed()
    for call in (lambda: ctx.embed(bags, table, out), lambda: ctx.embed_order(bags, dim), lambda: ctx.embed_order(bags, dim, order)):
        with pytest.raises(capi.AdmmError, match="destroyed|relabelled|rows"):
            call()
    ctx.embed_grad(bags, order, before, grad[1])   # its order holds copies, in the old numbers
    torch.cuda.synchronize()
    assert torch.equal(out, before) and torch.equal(grad[0], grad[1])
    order.free()
    csr.destroy()
    ctx.close()


def test_bags_follow_a_set_that_stays():
    """what leaves the rows where they are, or builds copies of them, leaves the bags usable"""
    from admm_amd import capi
    ctx, dim = capi.Context(0, stream=capi.DEFAULT_STREAM), 600
    csr = make(ctx, dim)
    bags = csr.bags()
    table, out = torch.randn(dim, 5, device="cuda"), torch.empty(500, 5, device="cuda")
    ctx.embed(bags, table, out)
    before = out.clone()
    csr.build_transposed()
    out.zero_()
    ctx.embed(bags, table, out)
    assert torch.equal(out, before)
    csr.destroy()
    ctx.close()
