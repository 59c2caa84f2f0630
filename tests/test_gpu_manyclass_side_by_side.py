"""Operands and results as columns of one buffer, against the same calls on buffers of their own with the same strides and
alignment (a float sum's order follows the 16-byte granules of its row): equal bits, and nothing outside the columns is touched."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    from admm_amd import capi
    c = capi.Context(0, stream=capi.DEFAULT_STREAM)
    yield c
    c.close()


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,gap", [(1, 7, 0), (33, 7, 0), (33, 64, 0), (40, 255, 3), (9, 5000, 1), (140, 9001, 0), (3, 70001, 2)])
def test_halves_of_the_same_rows(ctx, kind, rows, cols, gap):
    g = torch.Generator(device="cuda")
    g.manual_seed(rows * 131 + cols)
    values = (torch.randn(rows, cols, generator=g, device="cuda") * 3).to(kind)
    labels = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    ids = torch.randint(-1, rows, (rows,), generator=g, device="cuda")
    bags = ctx.bags(ids)
    order = ctx.embed_order(bags, rows)
    loss = torch.empty(rows, device="cuda")

    def softmax(x, to):
        ctx.softmax_loss(x, labels, loss, grad=to)

    def lookup(x, to):
        ctx.embed(bags, x, to, scale=0.5)

    def gradient(x, to):
        ctx.embed_grad(bags, order, x, to)
    def buffer():
        return torch.full((rows, 2 * cols + gap), 7.0, device="cuda").to(kind)
    halves = (slice(0, cols), slice(cols + gap, 2 * cols + gap))
    for call in (softmax, lookup, gradient):
        for here, there in (halves, halves[::-1]):
            source, want, both = buffer(), buffer(), buffer()
            source[:, here] = values
            call(source[:, here], want[:, there])
            both[:, here] = values
            call(both[:, here], both[:, there])
            assert torch.equal(both[:, there], want[:, there]) and torch.equal(both[:, here], values)
            assert torch.all(both[:, cols:cols + gap] == 7.0)
    order.free()
