"""Softmax rows that are nearly sure of their label: the loss and every element of the gradient are right relative to themselves,
not to 1, whatever is left to the other classes."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from admm_amd import capi
    c = capi.Context(0, stream=capi.DEFAULT_STREAM)
    yield c
    c.close()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols,pad", [(40, 2, 0), (40, 3, 0), (40, 17, 1), (40, 300, 0), (40, 1500, 0), (131, 4099, 0), (131, 9001, 3), (131, 33001, 0),
                                           (131, 70003, 1), (131, 131100, 0), (3, 40000, 0), (4, 140001, 1)])
def test_confident_rows(ctx, kind, rows, cols, pad, in_place):
    g = torch.Generator(device="cuda")
    g.manual_seed(rows * 31 + cols)
    mem = torch.zeros(rows, cols + pad, device="cuda", dtype=kind)
    x = mem[:, :cols]
    x.copy_((torch.randn(rows, cols, generator=g, device="cuda") * 2).to(kind))
    labels = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    labels[0], labels[1] = 0, cols - 1
    at = torch.arange(rows, device="cuda")
    # from an even chance to 10^-12 for all other classes together
    lead = torch.linspace(0, 28, rows, device="cuda") + math.log(cols) + 2
    x[at, labels] = lead.to(kind)
    x[2, labels[2]] = -math.inf                     # a masked label
    if cols > 2:
        x[rows - 1, (int(labels[rows - 1]) + 1) % cols] = -math.inf
    src = x.double()
    rest = src.clone()
    rest[at, labels] = -math.inf
    others = torch.logsumexp(rest, 1)               # of the classes that are not the label's
    xt = src[at, labels]
    lse = torch.logaddexp(others, xt)
    want_loss = torch.where(xt == -math.inf, math.inf, torch.nn.functional.softplus(others - xt, threshold=1000))
    want = torch.exp(src - lse[:, None])
    want[at, labels] = -torch.exp(others - lse)
    scale = 2.0 ** 10 if kind == torch.float16 else 1.0 / 64
    loss = torch.empty(rows, device="cuda")
    grad = x if in_place else torch.empty(rows, cols, device="cuda", dtype=kind)
    big = float(torch.where(torch.isfinite(src), src.abs(), 0.0).max()) * 1.4427 + math.log2(cols) + 1
    ctx.softmax_loss(x, labels, loss, grad=grad, grad_scale=scale)
    # relative error of a power: its exponent is off by 2^-24 of itself and of m L, and L by 2^-25, exp2 by two units; of a sum: a
    # rounding per addition of a thread's, the wave's and the block's; of the quotient and the products: a rounding each
    rel = U * (5 * big + 64 + 8 * cols / 1024 + 24)
    # bf16: subnormals may count as zero, as the float powers below 2^-126 do
    tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[kind]
    off = (grad.double() - want * scale).abs() - ((want * scale).abs() * (rel + 8 * U + torch.finfo(kind).eps / 2 * 1.01) + tiny)
    assert float(off.max()) <= 0, (float(off.max()), torch.nonzero(off > 0)[:5].tolist())
    fin = torch.isfinite(want_loss)
    assert torch.equal(loss[~fin].double(), want_loss[~fin])
    # up to an even chance the loss is log(1 + others / label's), beyond it a difference of numbers of that size
    sure = fin & (want_loss < 0.5)
    assert float(((loss.double() - want_loss).abs() - want_loss * (rel + 8 * U))[sure].max()) <= 0
    assert float(((loss.double() - want_loss).abs() - (2 * rel + want_loss * 4 * U))[fin].max()) <= 0
