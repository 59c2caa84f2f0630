"""Softmax rows with logits to both sides of 2^30, where the factor of the exponents changes from log2 e to 1."""
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


def neighbours(kind):
    """(smaller, larger) magnitudes around 2^30: close together, and a tenth to either side"""
    top = 2.0 ** 30
    step = 64.0 if kind == torch.float32 else 2.0 ** 22   # the type's step below 2^30
    return [(top - step, top), (top - step, top + 2 * step), (0.9 * top, 1.1 * top), (0.5 * top, 2.5 * top), (1000.0, top)]


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(5, 300), (5, 1800), (131, 3000), (131, 9000), (131, 33001), (131, 66000), (131, 131089), (3, 40000), (3, 140001)])
def test_logits_around_the_switch(ctx, kind, rows, cols):
    g = torch.Generator(device="cuda")
    g.manual_seed(rows * 7 + cols)
    half = cols // 2
    for near, far in neighbours(kind):
        near, far = (float(torch.tensor(v, dtype=kind)) for v in (near, far))
        assert near < far
        for low, high in ((near, far), (-far, -near), (-far, near)):
            x = torch.empty(rows, cols, device="cuda", dtype=kind)
            x[0::3] = low          # the larger ones behind, in front, scattered
            x[0::3, half:] = high
            x[1::3] = high
            x[1::3, half:] = low
            spread = torch.rand(rows, cols, generator=g, device="cuda") < 0.5
            spread[:, 0], spread[:, 1] = True, False
            x[2::3] = torch.where(spread, torch.tensor(high, dtype=kind, device="cuda"), torch.tensor(low, dtype=kind, device="cuda"))[2::3]
            on = x == high
            many = on.sum(1).double()
            labels = torch.randint(0, cols, (rows,), generator=g, device="cuda")
            loss, lse, grad = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x)
            ctx.softmax_loss(x, labels, loss, grad=grad, lse=lse)
            what = (kind, low, high)
            step = high - low      # at least 64: what is lower weighs at most 2^-64
            at = on.gather(1, labels[:, None])[:, 0]
            want = torch.where(at, 0.0, step) + torch.log(many)
            # equal powers: a rounding per addition, of a thread's, the wave's and the block's, and the powers' own logarithm, at most
            # 64, which is in the sum and in the label's exponent; the label's difference and its two factors are rounded, and log2 e
            sums = U * (64 + cols / 256)
            assert torch.all((loss.double() - want).abs() <= sums + U * (8 * 64 + 8 * math.log(cols)) + torch.where(at, 0.0, step) * 6 * U), what
            assert torch.all((lse.double() - (high + torch.log(many))).abs() <= sums + U * (4 * abs(high) + 8 * 64 + 8 * math.log(cols))), what
            p = on.double() / many[:, None]
            p[torch.arange(rows, device="cuda"), labels] -= 1.0
            bound = p.abs() * (torch.finfo(kind).eps / 2 * 1.01 + 4 * U) + (sums + 4 * U) / many[:, None] * on + 2.0 ** -63
            assert torch.all((grad.double() - p).abs() <= bound), what
