"""The many-class operators at sizes where the row gradient takes other paths (tiles of 2048 entries, chunks of 16 and 32, four
passes of the sort, more than 64 KB of LDS), and a softmax of more than 2^32 logits whose every element shows.

The gradient's operands are small integers, halves among their products, so that every sum is a multiple of 1/2 below 2^23: any
order of additions gives the same float, and results are compared for equality."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    from admm_amd import capi
    c = capi.Context(0, stream=capi.DEFAULT_STREAM)
    yield c
    c.close()


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make(n, vocab, rows, how, dtype, factors, g):
    """ids (a few of them padding, 40 % of them one id where `how` says so), row pointers, factors, the entries' rows"""
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    if how == "heavy":
        ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.4, vocab // 3, ids)
    elif how == "few":
        ids = ids % 3 * (vocab // 3)
    ids[::1001] = -1
    ids[5::2003] = vocab
    rowptr = val = None
    row = torch.arange(n, device="cuda")
    if rows != n:
        rowptr = torch.sort(torch.randint(0, n + 1, (rows + 1,), generator=g, device="cuda"))[0]
        rowptr[0], rowptr[-1] = 0, n
        row = torch.searchsorted(rowptr, row, right=True) - 1
    if factors:
        val = torch.randint(0, 4, (n,), generator=g, device="cuda") * 0.5  # 0, 1/2, 1, 3/2
    return ids.to(dtype), rowptr, val, row


def want_of(ids, val, row, src, vocab, old):
    """on the host, a column at a time (sums over few ids by atomics on the GPU take minutes)"""
    there = (ids >= 0) & (ids < vocab)
    at = ids[there].long().cpu().numpy()
    row = row[there].cpu().numpy()
    factor = None if val is None else val[there].double().cpu().numpy()
    src = src.double().cpu().numpy()
    want = old.double().cpu().numpy()
    for c in range(src.shape[1]):
        terms = src[row, c]
        want[:, c] += np.bincount(at, weights=terms if factor is None else terms * factor, minlength=vocab)
    return torch.from_numpy(want).cuda()


CASES = [
    # entries, table rows, rows, columns, how, ids, factors
    ((1 << 20) + 4097, 70001, None, 4, "heavy", torch.int64, False),        # tiles of 2048, three passes
    ((1 << 20) + 4097, 70001, 30000, 4, "heavy", torch.int32, True),
    ((1 << 20) + 1, 200, None, 4, "even", torch.int32, False),              # one pass
    (1100003, 1 << 20, 27000, 16, "even", torch.int32, True),               # 2^23 to 2^25 sums: chunks of 16
    (1100003, 1 << 20, 27000, 16, "heavy", torch.int64, True),
    (600001, 5000, None, 40, "heavy", torch.int64, False),
    (70001, 30000, None, 520, "heavy", torch.int64, False),                 # more than 2^25 sums: chunks of 32
    (70001, 30000, 900, 520, "few", torch.int32, True),
    (8500003, 100000, 200000, 4, "heavy", torch.int32, True),               # 256 groups of lanes: 101 KB of LDS
    (8500003, 100000, None, 4, "few", torch.int32, False),                  # 68 KB
    (30001, (1 << 24) + 1001, None, 1, "even", torch.int64, False),         # four passes of the sort
    ((1 << 20) + 77, (1 << 24) + 1001, 9000, 1, "heavy", torch.int32, True),
]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_row_gradient_of_many_entries(ctx, case, accumulate):
    n, vocab, rows, cols, how, dtype, factors = CASES[case]
    g = generator(100 + case)
    rows = n if rows is None else rows
    ids, rowptr, val, row = make(n, vocab, rows, how, dtype, factors, g)
    src = torch.randint(-2, 3, (rows, cols), generator=g, device="cuda").float()
    if case % 3 == 0:
        src = src.bfloat16()
    old = torch.randint(-100, 101, (vocab, cols), generator=g, device="cuda").float()
    grad = old.clone()
    bags = ctx.bags(ids, rowptr, val)
    order = torch.empty(ctx.embed_order_bytes(bags, vocab), dtype=torch.uint8, device="cuda")
    ctx.embed_order(bags, vocab, order)
    ctx.embed_grad(bags, order, src, grad, accumulate=accumulate)
    want = want_of(ids, val, row, src, vocab, old if accumulate else torch.zeros_like(old))
    assert float(want.abs().max()) < 2 ** 23
    assert torch.equal(grad.double(), want), (int((grad.double() != want).sum()), case)


@pytest.mark.parametrize("n,vocab,cols", [(10001, 5000, 8), (16384, 200000, 24), (8500003, 50000, 4)])
def test_row_gradient_captured(ctx, n, vocab, cols):
    """kernels that ask for more than 64 KB of LDS, in a graph: replays on changing ids against the eager calls"""
    from admm_amd import capi
    g = generator(n)
    side = torch.cuda.Stream()
    other = capi.Context(0, stream=side.cuda_stream)
    rows = 4000
    ids, rowptr, val, _ = make(n, vocab, rows, "heavy", torch.int32, True, g)
    src = torch.randint(-2, 3, (rows, cols), generator=g, device="cuda").float()
    out = [torch.empty(vocab, cols, device="cuda") for _ in range(2)]
    bags = ctx.bags(ids, rowptr, val)
    size = ctx.embed_order_bytes(bags, vocab)
    order = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    ws = [torch.empty(1 << 28, dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.embed_order(bags, vocab, order[0])
        other.embed_grad(bags, order[0], src, out[0], workspace=ws[0])
    for _ in range(3):
        ids.copy_(ids[torch.randperm(n, generator=g, device="cuda")])
        out[0].fill_(5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ctx.embed_order(bags, vocab, order[1])
        ctx.embed_grad(bags, order[1], src, out[1], workspace=ws[1])
        assert torch.equal(out[0], out[1])
    del graph
    other.close()


def test_softmax_of_more_than_32_bits_of_logits(ctx):
    """every element of the gradient is of the size of 1 and written over its logit, so that one left out or misplaced shows"""
    rows, cols = 33000, 130200
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    peak = torch.arange(rows, device="cuda") * 7919 % cols
    x[torch.arange(rows, device="cuda"), peak] = 3.0
    loss = torch.empty(rows, device="cuda")
    ctx.softmax_loss(x, peak, loss, grad=x, grad_scale=float(cols))
    total = cols - 1 + math.exp(3.0)
    U = 2.0 ** -24
    # a probability: the exponent is off by 2^-24 of 4.4 twice, exp2 by two units, the sum by a rounding per addition (64 granules
    # a thread of eight, the wave's and the block's); its rounding to bf16 is 2^-8
    rel = U * (2 * 4.4 + 4 + 8 * 64 + 24)
    assert float((loss.double() - (math.log(total) - 3.0)).abs().max()) <= rel + 4 * U * 12
    rest, top = cols / total, cols * (math.exp(3.0) / total - 1.0)
    for b in range(0, rows, 1000):
        part = x[b:b + 1000]
        at = torch.arange(part.shape[0], device="cuda")
        label = part[at, peak[b:b + 1000]].double()
        assert float((label - top).abs().max()) <= abs(top) * (2.0 ** -8 + rel)
        part[at, peak[b:b + 1000]] = rest
        # compared as what they are: in bf16 the distance to the expected value is exact
        assert float((part.float() - rest).abs().max()) <= rest * (2.0 ** -8 + rel) * (1 + 2.0 ** -20)
