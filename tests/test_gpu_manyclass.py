"""The many-class operators against their definitions in 64 bits: row lookup of a weight matrix and its gradient by sorted
ids, softmax loss with its gradient, sampling.  Tolerances count roundings: one of a value to type t is off by at most
finfo(t).eps / 2 of it (and half of its smallest subnormal), a float sum of n terms by n 2^-24 of the terms' magnitudes."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
U = 2.0 ** -24  # half a step of a float at 1

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}  # bf16: subnormals may count as zero


@pytest.fixture(scope="module")
def ctx():
    from admm_amd import capi
    c = capi.Context(0, stream=capi.DEFAULT_STREAM)
    yield c
    c.close()


def rng(*key):
    g = torch.Generator(device="cuda")
    g.manual_seed(abs(hash(tuple(key))) % (1 << 31) if not all(isinstance(k, int) for k in key) else sum(k * 7919 ** i for i, k in enumerate(key)) % (1 << 31))
    return g


def within(got, want, bound, what):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), what
    assert torch.isfinite(got[fin]).all(), what
    off = (got - want).abs() - bound
    off = off[fin]
    if off.numel():
        assert float(off.max()) <= 0, (what, float(off.max()), float((got - want)[fin].abs().max()))


def strided(rows, cols, kind, pad, shift, g, scale=1.0):
    """a matrix whose rows lie cols + pad apart and begin `shift` elements into memory"""
    mem = torch.full((rows * (cols + pad) + shift + 8,), 7.0, device="cuda").to(kind)
    m = mem[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    m.copy_((torch.randn(rows, cols, generator=g, device="cuda") * scale).to(kind))
    return m, mem


# ---- lookup -------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind,out_kind", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,vocab,cols,pad,shift", [(1, 1, 1, 0, 0), (5, 7, 3, 0, 1), (8, 100, 64, 0, 0), (33, 50, 257, 0, 0),
                                                       (33, 50, 250, 6, 0), (257, 300, 1024, 8, 4), (70, 9, 4100, 0, 0)])
def test_embed_rows(ctx, kind, out_kind, rows, vocab, cols, pad, shift):
    g = rng(1, rows, vocab, cols)
    table, _ = strided(vocab, cols, TYPES[kind], pad, shift, g)
    table[0, :] = math.nan  # what padding must not pick up
    out, mem = strided(rows + 2, cols, TYPES[out_kind], pad, shift, g)
    before = out.clone()
    for dtype in (torch.int32, torch.int64):
        ids = torch.randint(min(1, vocab - 1), vocab, (rows,), generator=g, device="cuda", dtype=dtype)
        ids[::5] = -1
        if rows > 3:
            ids[3], ids[2] = vocab, torch.iinfo(dtype).max
        there = (ids >= 0) & (ids < vocab)
        out.copy_(before)
        ctx.embed(ctx.bags(ids), table, out, scale=1.75)
        want = torch.where(there[:, None], table[torch.where(there, ids, 0).long()].double() * 1.75, 0.0)
        bound = want.abs().nan_to_num() * (torch.finfo(TYPES[out_kind]).eps / 2 * (1 + U) + U) + TINY[out_kind]
        within(out[:rows], want, bound, dtype)
        assert torch.equal(out[rows:], before[rows:])  # rows behind the last are left alone
        if pad:
            assert torch.all(mem[shift:shift + (rows + 2) * (cols + pad)].view(rows + 2, cols + pad)[:, cols:] == 7.0)


def make_bags(lengths, vocab, g, dtype=torch.int32, values=True):
    lengths = torch.as_tensor(lengths, dtype=torch.int64, device="cuda")
    rowptr = torch.zeros(lengths.numel() + 1, dtype=torch.int64, device="cuda")
    rowptr[1:] = torch.cumsum(lengths, 0)
    nnz = int(rowptr[-1])
    u = torch.rand(nnz, generator=g, device="cuda", dtype=torch.float64)
    ids = torch.clamp((vocab ** u - 1).long(), 0, vocab - 1).to(dtype)
    val = torch.rand(nnz, generator=g, device="cuda") * 2 - 0.5 if values else None
    row = torch.repeat_interleave(torch.arange(lengths.numel(), device="cuda"), lengths)
    return ids, rowptr, val, row


BAGS = [[0], [1], [3, 0, 0, 5], [40] * 70 + [0] * 3, [700, 0, 900, 1], [5000], list(range(130))]


def bag_sums(table, ids, val, row, nrows, vocab, scale):
    """the sum and the sum of the magnitudes per row, in 64 bits"""
    there = (ids >= 0) & (ids < vocab)
    ids, row = ids.long()[there], row[there]
    val = torch.ones(ids.numel(), dtype=torch.float64, device="cuda") if val is None else val[there].double()
    terms = table[ids].double() * val[:, None] * scale
    want = torch.zeros(nrows, table.shape[1], dtype=torch.float64, device="cuda").index_put_((row,), terms, accumulate=True)
    size = torch.zeros_like(want).index_put_((row,), terms.abs(), accumulate=True)
    return want, size


@pytest.mark.parametrize("kind,out_kind", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("cols", [1, 3, 16, 64, 100, 1030])
@pytest.mark.parametrize("which", range(len(BAGS)))
def test_embed_bags(ctx, kind, out_kind, cols, which):
    g, vocab = rng(2, cols, which), 200
    table, _ = strided(vocab, cols, TYPES[kind], which % 3, which % 2, g)
    for values in (False, True):
        ids, rowptr, val, row = make_bags(BAGS[which], vocab, g, values=values)
        if ids.numel() > 2:
            ids[1] = -1
        nrows = rowptr.numel() - 1
        out = torch.full((nrows + 1, cols), 3.0, device="cuda", dtype=TYPES[out_kind])
        ctx.embed(ctx.bags(ids, rowptr, val), table, out, scale=-0.5)
        want, size = bag_sums(table, ids, val, row, nrows, vocab, -0.5)
        longest = max(BAGS[which])
        bound = size * (longest + 3) * U + (want.abs() + size * (longest + 3) * U) * torch.finfo(TYPES[out_kind]).eps / 2 + TINY[out_kind]
        within(out[:nrows], want, bound, values)
        assert torch.all(out[nrows:] == 3.0)


def test_embed_bags_that_point_outside(ctx):
    """row pointers beyond the entries (or running backwards) read nothing beyond them"""
    table = torch.randn(10, 8, device="cuda")
    ids = torch.zeros(16, dtype=torch.int32, device="cuda")
    rowptr = torch.tensor([0, 2, 1, 1 << 40, 1 << 41], device="cuda")
    out = torch.zeros(4, 8, device="cuda")
    ctx.embed(ctx.bags(ids, rowptr), table, out)
    want = torch.stack([table[0] * 2, table[0] * 0, table[0] * 15, table[0] * 0])
    within(out, want, want.abs().double() * 20 * U, "rows")
    order = ctx.embed_order(ctx.bags(ids, rowptr), 10)
    grad = torch.zeros(10, 8, device="cuda")
    ctx.embed_grad(ctx.bags(ids, rowptr), order, torch.ones(4, 8, device="cuda"), grad)
    assert torch.all(grad[1:] == 0) and torch.isfinite(grad).all()


# ---- its gradient -------------------------------------------------------------------------------

def check_grad(ctx, ids, rowptr, val, row, nrows, vocab, cols, kind, out_kind, accumulate, g, pad=0, shift=0):
    src, _ = strided(nrows + 1, cols, TYPES[kind], pad, shift, g, 0.5)
    grad, mem = strided(vocab, cols, TYPES[out_kind], pad, shift, g)
    old = grad.double().clone()
    bags = ctx.bags(ids, rowptr, val)
    order = ctx.embed_order(bags, vocab)
    ctx.embed_grad(bags, order, src, grad, scale=1.5, accumulate=accumulate)
    there = (ids >= 0) & (ids < vocab)
    at, frm = ids.long()[there], row[there]
    w = torch.ones(at.numel(), dtype=torch.float64, device="cuda") if val is None else val[there].double()
    terms = src[frm].double() * w[:, None] * 1.5
    want = torch.zeros(vocab, cols, dtype=torch.float64, device="cuda").index_put_((at,), terms, accumulate=True)
    size = torch.zeros_like(want).index_put_((at,), terms.abs(), accumulate=True)
    count = torch.bincount(at, minlength=vocab).double()[:, None] + 3
    if accumulate:
        want, size = want + old, size + old.abs()
    bound = size * count * U + (want.abs() + size * count * U) * torch.finfo(TYPES[out_kind]).eps / 2 + TINY[out_kind]
    within(grad, want, bound, (ids.numel(), vocab, cols))
    if accumulate:
        absent = torch.bincount(at, minlength=vocab) == 0
        assert torch.equal(grad[absent].double(), old[absent])
    if pad:
        assert torch.all(mem[shift:shift + vocab * (cols + pad)].view(vocab, cols + pad)[:, cols:] == 7.0)
    again = torch.empty_like(grad).copy_(old)
    ctx.embed_grad(bags, order, src, again, scale=1.5, accumulate=accumulate)
    assert torch.equal(again.view(-1).view(torch.uint8), grad.contiguous().view(-1).view(torch.uint8))  # same bits again
    order.free()


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 128, 129, 1000, 8192, 8193, 20001])
@pytest.mark.parametrize("how", ["zipf", "same", "distinct", "padding", "two"])
def test_embed_grad_tokens(ctx, rows, how):
    g = rng(3, rows)
    vocab = 70001 if how == "distinct" else 500
    if how == "distinct":
        ids = torch.randperm(vocab, generator=g, device="cuda")[:rows]
    elif how == "same":
        ids = torch.full((rows,), 17, dtype=torch.int64, device="cuda")
    elif how == "padding":
        ids = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    elif how == "two":
        ids = torch.where(torch.arange(rows, device="cuda") % 3 == 0, 499, 0)
    else:
        ids = make_bags([rows], vocab, g, torch.int64)[0]
        ids[::7] = -1
    row = torch.arange(rows, device="cuda")
    check_grad(ctx, ids, None, None, row, rows, vocab, 40, "f32", "f32", rows % 2 == 0, g)
    check_grad(ctx, ids.int(), None, None, row, rows, vocab, 24, "bf16", "bf16", rows % 2 == 1, g)


@pytest.mark.parametrize("kind,out_kind", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("vocab,cols,pad,shift", [(1, 1, 0, 0), (2, 3, 1, 1), (50, 16, 0, 0), (257, 64, 8, 4), (300, 100, 0, 0),
                                                  (100, 257, 0, 1), (63, 1024, 0, 0), (64, 2100, 4, 0), (1 << 20, 4, 0, 0)])
def test_embed_grad_shapes(ctx, kind, out_kind, vocab, cols, pad, shift):
    g = rng(4, vocab, cols)
    for accumulate in (False, True):
        ids = make_bags([333], vocab, g, torch.int32)[0]
        check_grad(ctx, ids, None, None, torch.arange(333, device="cuda"), 333, vocab, cols, kind, out_kind, accumulate, g, pad, shift)


@pytest.mark.parametrize("which", range(len(BAGS)))
@pytest.mark.parametrize("cols", [1, 16, 70])
def test_embed_grad_bags(ctx, which, cols):
    g = rng(5, which, cols)
    for values in (False, True):
        ids, rowptr, val, row = make_bags(BAGS[which], 300, g, values=values)
        check_grad(ctx, ids, rowptr, val, row, rowptr.numel() - 1, 300, cols, "f32", "f32", values, g)


def test_embed_grad_many_entries(ctx):
    """several passes of the sort over many tiles, runs of tens of thousands of entries"""
    g = rng(6, 1)
    ids, rowptr, val, row = make_bags([40] * 9000, 1 << 20, g)
    check_grad(ctx, ids, rowptr, val, row, 9000, 1 << 20, 16, "f32", "f32", False, g)
    ids[:] = torch.where(torch.rand(ids.numel(), generator=g, device="cuda") < 0.4, 5, ids)
    check_grad(ctx, ids, rowptr, val, row, 9000, 1 << 20, 8, "f32", "f32", True, g)


def test_embed_grad_is_the_gradient(ctx):
    """sum(out * r) is linear in the table: its differences in a few directions, in 64 bits of the outputs"""
    g = rng(7, 1)
    ids, rowptr, val, row = make_bags([5, 0, 9, 30], 40, g)
    bags = ctx.bags(ids, rowptr, val)
    r = torch.randn(4, 12, generator=g, device="cuda")
    grad = torch.empty(40, 12, device="cuda")
    ctx.embed_grad(bags, ctx.embed_order(bags, 40), r, grad, scale=2.0)
    table = torch.randn(40, 12, generator=g, device="cuda")
    for _ in range(4):
        d = torch.randn(40, 12, generator=g, device="cuda")
        out = []
        for t in (table + d, table - d):
            o = torch.empty(4, 12, device="cuda")
            ctx.embed(bags, t, o, scale=2.0)
            out.append(float((o.double() * r.double()).sum()))
        want = float((grad.double() * d.double()).sum())
        # 44 entries of 12 columns, each term below 2 * 2 * 4 * 4 * 4 = 128 in magnitude and off by 40 roundings
        assert abs((out[0] - out[1]) / 2 - want) <= 44 * 12 * 128 * 40 * U


# ---- softmax loss -------------------------------------------------------------------------------

def check_softmax(ctx, x, labels, weight=None, grad_scale=1.0, grad=None, loss_only=False):
    rows, cols = x.shape
    kind = x.dtype
    src = x.double()
    w = torch.ones(rows, dtype=torch.float64, device="cuda") if weight is None else weight.double()
    t = labels.double().trunc().long() if labels.is_floating_point() else labels.long()
    on = (t >= 0) & (t < cols) & (w != 0)
    lse = torch.logsumexp(src, 1)
    at = torch.where(on, t, 0)
    xt = src.gather(1, at[:, None])[:, 0]
    none = lse == -math.inf
    want_loss = torch.where(on, w * torch.where(none, math.inf, lse - xt), 0.0)
    p = torch.where(none[:, None], 0.0, torch.exp(src - lse[:, None]))
    delta = torch.zeros_like(src).scatter_(1, at[:, None], 1.0)
    want_grad = torch.where(on[:, None], torch.where(none[:, None], 0.0, (p - delta) * (w * grad_scale)[:, None]), 0.0)
    loss, lse_out = torch.full((rows,), 9.0, device="cuda"), torch.full((rows,), 9.0, device="cuda")
    g = None if loss_only else torch.empty(rows, cols, device="cuda", dtype=kind) if grad is None else grad
    ctx.softmax_loss(x, labels, loss, grad=g, lse=lse_out, weight=weight, grad_scale=grad_scale)
    # relative error of a probability: the exponent x L - m L is off by 2^-24 of itself, of m L and of lse L, and L by 2^-25;
    # the exponentials' sum by a rounding per addition of a thread's and the block's; exp2 by two units
    big = torch.where(torch.isfinite(src), src.abs(), 0.0).amax(1) * 1.4427 + math.log2(cols) + 1
    rel = U * (5 * big + 64 + 8 * cols / 1024 + 24)
    within(lse_out, lse, 2 * rel + lse.abs().nan_to_num(posinf=0, neginf=0) * 3 * U, "lse")
    within(loss, want_loss, w.abs() * (2 * rel + (lse - xt).abs().nan_to_num(posinf=0) * 3 * U), "loss")
    if g is not None:
        name = [k for k in TYPES if TYPES[k] == kind][0]
        s = (w * grad_scale).abs()[:, None]
        exact = s * (p * rel[:, None] + (p + delta) * 3 * U)
        within(g, want_grad, (exact + want_grad.abs() * torch.finfo(kind).eps / 2 * 1.01 + TINY[name]).nan_to_num(), "grad")
    lone = torch.full((rows,), 9.0, device="cuda")
    if g is None or g.data_ptr() != x.data_ptr():
        ctx.softmax_loss(x, labels, lone, weight=weight, grad_scale=grad_scale)  # without lse: rows not trained on are not read
        assert torch.equal(lone.view(torch.int32), loss.view(torch.int32))


def make_logits(rows, cols, kind, g, spread=3.0):
    return (torch.randn(rows, cols, generator=g, device="cuda") * spread).to(TYPES[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (130, 3), (65, 16), (70, 17), (9, 100), (5, 1000), (6, 1024), (7, 2049),
                                       (3, 4100), (5, 33000), (2, 70001), (3, 140000)])
def test_softmax_loss(ctx, kind, rows, cols):
    g = rng(8, rows, cols)
    x = make_logits(rows, cols, kind, g)
    labels = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    check_softmax(ctx, x, labels)
    labels[::3] = -100
    labels[rows // 2] = cols
    weight = torch.rand(rows, generator=g, device="cuda") + 0.5
    weight[rows // 3] = 0
    check_softmax(ctx, x, labels.int(), weight, 0.125)
    check_softmax(ctx, x, labels.float() + 0.25, loss_only=True)
    x[torch.rand(rows, cols, generator=g, device="cuda") < 0.3] = -math.inf  # masked classes, the label's among them
    check_softmax(ctx, x, labels)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols", [4099, 9000, 16385, 33001, 65600, 131089])
def test_softmax_loss_many_long_rows(ctx, kind, cols):
    """rows enough that each has a workgroup of its own: in registers of several sizes, and read twice"""
    g = rng(18, cols)
    rows = 131
    x = make_logits(rows, cols, kind, g)
    labels = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    labels[::9] = -1
    labels[1], labels[2] = 0, cols - 1
    x[3, ::2] = -math.inf
    x[4, :] = -math.inf
    x[5, : cols - 1] = torch.finfo(x.dtype).min
    x[6, cols // 3] = math.nan
    x[7, 1] = math.inf
    loss, grad = torch.empty(rows, device="cuda"), torch.empty_like(x)
    ctx.softmax_loss(x, labels, loss, grad=grad)
    assert loss[4] == math.inf and torch.all(grad[4] == 0)
    for r in (6, 7):
        assert torch.isnan(loss[r]) and torch.isnan(grad[r]).all()
    x[6:8] = 0
    check_softmax(ctx, x, labels)
    check_softmax(ctx, x, labels, grad=x)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols", [5, 16, 300, 5000, 9001, 70000])
def test_softmax_loss_rows_without_classes_or_with_nan(ctx, kind, cols):
    g = rng(9, cols)
    x = make_logits(7, cols, kind, g)
    labels = torch.randint(0, cols, (7,), generator=g, device="cuda")
    x[1] = -math.inf
    x[2, cols // 2] = math.nan
    x[3, cols - 1] = math.inf
    x[4] = torch.finfo(x.dtype).min
    x[5, 1:] = torch.finfo(x.dtype).min
    labels[6] = -1
    x[6] = math.nan  # not trained on: its logits do not matter
    loss, grad = torch.empty(7, device="cuda"), torch.empty_like(x)
    ctx.softmax_loss(x, labels, loss, grad=grad)
    assert loss[1] == math.inf and torch.all(grad[1] == 0)
    assert torch.isnan(loss[2]) and torch.isnan(grad[2]).all()
    assert torch.isnan(loss[3]) and torch.isnan(grad[3]).all()
    assert abs(float(loss[4]) - math.log(cols)) < 1e-5 * (1 + math.log(cols))
    assert loss[6] == 0 and torch.all(grad[6] == 0)
    check_softmax(ctx, x[[0, 5]].contiguous(), torch.zeros(2, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(2, 300), (131, 3000), (131, 9000), (131, 33001), (131, 131089), (3, 40000)])
def test_softmax_loss_where_the_shift_of_huge_logits_changes(ctx, kind, rows, cols):
    """logits to both sides of 2^126 within a row, a larger one behind a smaller one; the loss is within the logits' own steps"""
    g = rng(41, rows, cols)
    x = make_logits(rows, cols, kind, g)
    near, far = torch.tensor(0.9 * 2.0 ** 126, dtype=TYPES[kind]), torch.tensor(1.1 * 2.0 ** 126, dtype=TYPES[kind])
    x[0, : cols // 2], x[0, cols // 2:] = near, far
    x[1, : cols // 2], x[1, cols // 2:] = -far, -near
    x[rows - 1], x[rows - 1, cols - 2] = near, far
    labels = torch.zeros(rows, dtype=torch.int64, device="cuda")
    labels[rows - 1] = cols - 2
    loss, grad = torch.empty(rows, device="cuda"), torch.empty_like(x)
    ctx.softmax_loss(x, labels, loss, grad=grad)
    step = float(far) - float(near)
    many = cols - cols // 2
    U32 = torch.finfo(torch.float32).eps / 2
    for r in {0, 1} - {rows - 1}:  # the label is one of the smaller: the rest share the probability
        # both logits' products with L and their difference are rounded: 2^-24 each of at most 2^127 L
        assert abs(float(loss[r]) - step) <= 8 * U32 * 2.0 ** 127.6, (r, float(loss[r]), step)
        want = torch.zeros(cols, device="cuda", dtype=torch.float64)
        want[cols // 2:] = 1.0 / many
        want[0] -= 1
        # a sum of equal powers: a rounding per addition, of a thread's, the wave's and the block's
        bound = want.abs() * (U32 * (64 + many / 256) + torch.finfo(x.dtype).eps) + (2.0 ** -133 if kind == "bf16" else 0.0)
        within(grad[r], want, bound, "grad")
    assert abs(float(loss[rows - 1])) <= 8 * U32 * 2.0 ** 127.6 and torch.all(grad[rows - 1] == 0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(13, 7), (13, 300), (131, 3000), (131, 9000), (131, 33001), (131, 131089), (13, 40000)])
def test_softmax_loss_of_one_huge_value(ctx, kind, rows, cols):
    """rows whose logits are all the same (every class masked by the same finite value): an even distribution at any magnitude"""
    values = [-1e4, 1e6, -1e9, 1.07e9, -1.08e9, 1e10, -1e10, 1e15, -1e20, 1e30, -8.4e37, 8.6e37, -3e38]
    x = torch.tensor([values[r % 13] for r in range(rows)], device="cuda").to(TYPES[kind])[:, None].expand(rows, cols).contiguous()
    labels = torch.arange(rows, device="cuda") % cols
    loss, lse, grad = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x)
    ctx.softmax_loss(x, labels, loss, grad=grad, lse=lse)
    U32 = torch.finfo(torch.float32).eps / 2
    # a power's exponent is at most 64, rounded by 2^-24 of that, and the same for all; a rounding per addition
    sums = U32 * (64 + cols / 256)
    within(loss, torch.full((rows,), math.log(cols), dtype=torch.float64, device="cuda"), sums + U32 * (4 * 64 + 8), "loss")
    within(lse, x[:, 0].double() + math.log(cols), sums + U32 * (4 * x[:, 0].double().abs() + 8 * math.log(cols) + 64), "lse")
    want = torch.full((rows, cols), 1.0 / cols, dtype=torch.float64, device="cuda")
    want[torch.arange(rows, device="cuda"), labels] -= 1
    within(grad, want, want.abs() * (4 * U32 + torch.finfo(x.dtype).eps / 2 * 1.01) + (sums + 4 * U32) / cols, "grad")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,pad,shift", [(9, 30, 3, 1), (9, 64, 64, 0), (5, 1001, 0, 5), (4, 6000, 8, 2), (3, 40001, 1, 3)])
def test_softmax_loss_strides_and_in_place(ctx, kind, rows, cols, pad, shift):
    g = rng(10, rows, cols)
    labels = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    x, mem = strided(rows, cols, TYPES[kind], pad, shift, g, 2.0)
    check_softmax(ctx, x, labels)  # the gradient's rows are aligned otherwise
    to, mem2 = strided(rows, cols, TYPES[kind], pad, shift, g)
    check_softmax(ctx, x, labels, grad=to)
    inside = slice(shift, shift + rows * (cols + pad))
    if pad:
        assert torch.all(mem2[inside].view(rows, cols + pad)[:, cols:] == 7.0)
    assert torch.all(mem2[:shift] == 7.0) and torch.all(mem2[inside.stop:] == 7.0)
    check_softmax(ctx, x, labels, grad=x)  # written over the logits
    if pad:
        assert torch.all(mem[inside].view(rows, cols + pad)[:, cols:] == 7.0)
    assert torch.all(mem[:shift] == 7.0) and torch.all(mem[inside.stop:] == 7.0)


def test_softmax_loss_gradient_against_differences(ctx):
    g = rng(11, 1)
    x = make_logits(6, 50, "f32", g, 1.0)
    labels = torch.randint(0, 50, (6,), generator=g, device="cuda")
    grad, loss = torch.empty_like(x), torch.empty(6, device="cuda")
    ctx.softmax_loss(x, labels, loss, grad=grad)
    d = torch.randn(6, 50, generator=g, device="cuda")
    h = 2.0 ** -6
    two = [torch.empty(6, device="cuda") for _ in range(2)]
    ctx.softmax_loss(x + h * d, labels, two[0])
    ctx.softmax_loss(x - h * d, labels, two[1])
    slope = (two[0].double() - two[1].double()) / (2 * h)
    # the third derivative along d is below 2 |d|^3 <= 2 * 4.5^3, the losses (below 8) are off by 100 roundings at most
    within(slope, (grad.double() * d.double()).sum(1), h * h / 6 * 2 * 4.5 ** 3 + 8 * 100 * U / h, "slope")


# ---- sampling -----------------------------------------------------------------------------------

def reference_draw(x, u, t, k, p, m):
    """(token, log-probability) of one row from the definition, in 64 bits"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1, -np.inf
    if not t > 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore"):
        y = np.where(x == top, 0.0, np.where(x == -np.inf, -np.inf, (x - top) / t))
    w = np.exp(y)[order]
    count = len(x) if k <= 0 else min(int(k), len(x))
    if p < 1:
        sums = np.cumsum(w[:count])
        count = max(1, int(np.count_nonzero(np.concatenate([[0.0], sums[:-1]]) < p * sums[-1])))
    if m > 0:
        count = max(1, int(np.count_nonzero(w[:count] >= m)))
    kept = np.sort(order[:count])
    mass = np.exp(y[kept])
    sums = np.cumsum(mass)
    if u > 0:
        i = min(int(np.searchsorted(sums, min(u, 1.0) * sums[-1], side="right")), int(np.max(np.nonzero(mass)[0])))
    else:
        i = int(np.nonzero(mass)[0][0])
    return int(kept[i]), float(y[kept[i]] - np.log(sums[-1]))


def check_sample(ctx, x, u, t=None, k=None, p=None, m=None):
    rows = x.shape[0]

    def dev(v, dtype):
        return None if v is None else torch.as_tensor(np.asarray(v), dtype=dtype, device="cuda").expand(rows).contiguous()
    u, t, k, p, m = dev(u, torch.float32), dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(m, torch.float32)
    token = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    logprob = torch.full((rows,), 7.0, device="cuda")
    ctx.sample(x, u, token, logprob=logprob, temperature=t, top_k=k, top_p=p, min_p=m)
    one = torch.empty_like(token)
    ctx.sample(x, u, one, temperature=t, top_k=k, top_p=p, min_p=m)
    assert torch.equal(one, token)
    host = lambda v, other: np.full(rows, other) if v is None else v.cpu().numpy()  # noqa: E731
    xs, hu, ht, hk, hp, hm = x.float().cpu().numpy(), host(u, 0), host(t, 1.0), host(k, 0), host(p, 1.0), host(m, 0.0)
    for r in range(rows):
        want, lp = reference_draw(xs[r], float(hu[r]), float(ht[r]), int(hk[r]), float(hp[r]), float(hm[r]))
        what = (r, x.shape, x.dtype, hu[r], ht[r], hk[r], hp[r], hm[r])
        assert int(token[r]) == want, (int(token[r]), want, what)
        got = float(logprob[r])
        assert got == lp or abs(got - lp) <= abs(lp) * U + 1e-9, (got, lp, what)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (40, 2), (40, 3), (30, 17), (30, 255), (20, 1000), (10, 4099), (6, 20000), (3, 70001)])
def test_sample(ctx, kind, rows, cols):
    g = rng(12, rows, cols)
    rs = np.random.RandomState(rows * 31 + cols)
    for spread in (0.5, 4.0):
        x = make_logits(rows, cols, kind, g, spread)
        u, t = rs.rand(rows).astype(np.float32), rs.uniform(0.3, 1.7, rows)
        k, p, m = rs.randint(1, min(cols, 200) + 1, rows), rs.uniform(0.05, 0.99, rows), rs.uniform(0.001, 0.5, rows)
        check_sample(ctx, x, u)
        check_sample(ctx, x, u, t)
        check_sample(ctx, x, u, t, k=k)
        check_sample(ctx, x, u, t, p=p)
        check_sample(ctx, x, u, t, m=m)
        check_sample(ctx, x, u, t, k=k, p=p, m=m)
        some = rs.rand(rows) < 0.5
        check_sample(ctx, x, u, np.where(some, 0, t), k=np.where(rs.rand(rows) < 0.5, 0, k), p=np.where(some, 1.5, p), m=np.where(rs.rand(rows) < 0.3, 0, m))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols", [15, 16, 64, 65, 128, 129, 256, 257, 512, 513, 1024, 1025])
def test_sample_where_the_form_changes(ctx, kind, cols):
    """numbers of classes around those where a row takes more lanes, or more registers, or another kernel"""
    g, rows = rng(19, cols), 37
    rs = np.random.RandomState(cols)
    x = make_logits(rows, cols, kind, g, 2.0)
    x[1] = x[1, 0]
    x[2, ::2] = -math.inf
    x[3, cols // 3:] = math.nan
    x[4, [cols // 2, cols - 1]] = math.inf
    x[5] = -math.inf
    u = rs.rand(rows).astype(np.float32)
    u[6:9] = [0.0, -1.0, 1.0]
    for i in range(4):
        pick = lambda v, off: np.where(rs.rand(rows) < 0.5, off, v)  # noqa: E731
        t, k = pick(rs.uniform(0.3, 2, rows), 1.0), pick(rs.randint(1, cols + 1, rows), 0)
        p, m = pick(rs.uniform(0.05, 1, rows), 1.0), pick(rs.uniform(0.001, 0.9, rows), 0.0)
        t[rs.rand(rows) < 0.1] = 0
        check_sample(ctx, x, u, t, k=k, p=p, m=m)
    check_sample(ctx, x, u)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(511, 513), (512, 513), (512, 1024), (530, 777)])
def test_sample_of_many_short_rows(ctx, kind, rows, cols):
    """rows enough that each is sorted by one wave, with every filter"""
    g = rng(23, rows, cols)
    rs = np.random.RandomState(rows + cols)
    x = make_logits(rows, cols, kind, g, 2.0)
    x[1] = x[1, 0]
    x[2, ::2] = -math.inf
    x[3, cols // 3:] = math.nan
    x[4, [cols // 2, cols - 1]] = math.inf
    x[5] = -math.inf
    u = rs.rand(rows).astype(np.float32)
    u[6:9] = [0.0, -1.0, 1.0]
    pick = lambda v, off: np.where(rs.rand(rows) < 0.5, off, v)  # noqa: E731
    t, k = pick(rs.uniform(0.3, 2, rows), 1.0), pick(rs.randint(1, cols + 1, rows), 0)
    p, m = pick(rs.uniform(0.05, 1, rows), 1.0), pick(rs.uniform(0.001, 0.9, rows), 0.0)
    t[rs.rand(rows) < 0.1] = 0
    check_sample(ctx, x, u, t, k=k, p=p, m=m)
    check_sample(ctx, x, u, t, k=k)
    check_sample(ctx, x, u, t, p=p)
    check_sample(ctx, x, u, m=m)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [3000, 50000])
def test_sample_of_many_candidates(ctx, kind, cols):
    """a k beyond what fits LDS, nuclei of most of the classes, flat rows, classes that tie by the thousand"""
    g, rows = rng(20, cols), 12
    rs = np.random.RandomState(cols)
    u, t = rs.rand(rows).astype(np.float32), rs.uniform(0.5, 2, rows)
    for spread in (0.0, 0.01, 1.0):
        x = make_logits(rows, cols, kind, g, spread)
        check_sample(ctx, x, u, t, k=rs.randint(cols // 20, cols, rows))
        check_sample(ctx, x, u, t, p=rs.uniform(0.9, 0.9999, rows))
        check_sample(ctx, x, u, t, k=rs.randint(100, 500, rows), p=rs.uniform(0.5, 0.99, rows))
        check_sample(ctx, x, u, t, p=rs.uniform(0.5, 0.99, rows), m=rs.uniform(0.01, 0.9, rows))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sample_ties_and_borders(ctx, kind):
    """equal logits: weights of exactly one, so the numbers of classes and the draws fall on exact borders"""
    for cols in (8, 64, 1024, 40000):
        x = torch.zeros(8, cols, device="cuda", dtype=TYPES[kind])
        u = np.arange(8) / 8
        check_sample(ctx, x, u)                    # class u * cols exactly
        check_sample(ctx, x, u, k=[1, 2, 3, 4, 5, 6, 7, 8])
        check_sample(ctx, x, u, p=0.5)             # the first half, by index
        check_sample(ctx, x, u, k=cols // 2, p=0.25, m=1.0)
        x[:, ::2] = -0.0                           # a tie with 0
        check_sample(ctx, x, u, k=3)
        x[:, 1::2] = -1.0
        check_sample(ctx, x, u, k=cols // 2 + 1)
        check_sample(ctx, x, u, p=0.75, m=0.3)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols", [7, 300, 30000])
def test_sample_odd_logits_and_parameters(ctx, kind, cols):
    g = rng(13, cols)
    x = make_logits(12, cols, kind, g)
    lowest = torch.finfo(x.dtype).min
    x[0] = -math.inf                 # nothing left: token -1
    x[1] = math.nan
    x[2, : cols // 2] = -math.inf
    x[3, cols // 2] = math.inf       # all the mass
    x[4, [1, cols - 1]] = math.inf   # shared
    x[5] = lowest                    # a mask of the type's lowest value everywhere
    x[6, : cols - 1] = lowest
    x[7] = math.nan
    x[7, 3] = -5.0
    x[8, :] = -math.inf
    x[8, cols - 1] = lowest
    u = np.linspace(0, 0.99, 12).astype(np.float32)
    for kw in ({}, {"k": 5}, {"p": 0.6}, {"m": 0.1}, {"k": 50, "p": 0.9, "m": 0.01}, {"t": 0.0}, {"t": 1e-30}, {"t": 1e30}):
        check_sample(ctx, x, u, **kw)
    one = x[9:10].expand(8, cols).contiguous()
    # 0 and beyond the ends; parameters that are no numbers or filter nothing
    check_sample(ctx, one, [0.0, -1.0, 1.0, 2.0, np.nan, 0.5, 0.5, np.float32(1 - 2 ** -24)])
    check_sample(ctx, one, 0.3, t=[np.nan, -1.0, np.inf, 1.0, 1.0, 1.0, 1.0, 1.0], k=[0, 0, 0, -3, cols, cols + 1, 2 ** 31 - 1, 0],
                 p=[1, 1, 1, 1, 1, 0.0, -1.0, np.nan], m=[0, 0, 0, 0, 1.0, 2.0, -1.0, np.nan])


@pytest.mark.parametrize("offset,spread,t", [(0.0, 1.0, 1.0), (1e3, 1.0, 0.7), (-1e3, 1.0, 0.7), (1e5, 1.0, 0.01), (-3e38, 1e36, 1e36),
                                             (3e37, 3e36, 1e36), (0.0, 1e-37, 1e-37), (1e-36, 1e-38, 1e-38), (0.0, 1e-3, 1e30)])
def test_sample_top_p_at_any_scale(ctx, offset, spread, t):
    """the kept classes' border far from zero, close to it and at scales where a logit's step is a large part of a bucket"""
    g = rng(31, 7)
    for rows, cols in ((12, 1500), (4, 30000)):
        x = (torch.randn(rows, cols, generator=g, dtype=torch.float64, device="cuda") * spread * 2 + offset).float()
        x[0, 1::2] = -math.inf
        u = np.linspace(0.03, 0.97, rows).astype(np.float32)
        for p in (0.02, 0.5, 0.93, 0.9999):
            check_sample(ctx, x, u, t, p=p)


def test_sample_does_not_depend_on_the_batch(ctx):
    """a row's token and log-probability are the same alone, in a batch, and at other strides and alignments"""
    g = rng(14, 1)
    for kind in ("f32", "bf16"):
        for cols in (5000, 70001):
            x, _ = strided(300, cols, TYPES[kind], 3, 1, g, 3.0)
            u = torch.rand(300, generator=g, device="cuda")
            p = torch.full((300,), 0.9, device="cuda")
            token, lp = torch.empty(300, dtype=torch.int32, device="cuda"), torch.empty(300, device="cuda")
            ctx.sample(x, u, token, logprob=lp, top_p=p)
            for r in (0, 7, 299):
                t1, l1 = torch.empty(1, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda")
                ctx.sample(x[r:r + 1].contiguous(), u[r:r + 1], t1, logprob=l1, top_p=p[:1])
                assert int(t1) == int(token[r]) and float(l1) == float(lp[r])


def test_sample_follows_the_distribution(ctx):
    """the share of u in [0, 1) that gives a class is its probability, class after class"""
    x = torch.tensor([[0.0, 1.0, -1.0, 2.0]], device="cuda").expand(4096, 4).contiguous()
    u = (torch.arange(4096, device="cuda") + 0.5) / 4096
    token = torch.empty(4096, dtype=torch.int32, device="cuda")
    ctx.sample(x, u, token)
    share = torch.bincount(token.long(), minlength=4).double() / 4096
    assert float((share - torch.softmax(x[0].double(), 0)).abs().max()) <= 1 / 4096
    assert torch.all(token[1:] >= token[:-1])


# ---- streams, graphs, sample sets ---------------------------------------------------------------

def steps(ctx, s, out):
    """lookup, loss with gradient, gradient of the table, a draw"""
    bags = ctx.bags(s["ids"], s["rowptr"], s["val"])
    ctx.embed(bags, s["table"], out["logits"])
    ctx.softmax_loss(out["logits"], s["labels"], out["loss"], grad=out["dlogits"], grad_scale=1.0 / out["loss"].numel(), workspace=out["ws"])
    ctx.embed_order(bags, s["table"].shape[0], out["order"])
    ctx.embed_grad(bags, out["order"], out["dlogits"], out["grad"], workspace=out["ws"])
    ctx.sample(out["logits"], s["u"], out["token"], logprob=out["logprob"], top_p=s["p"], workspace=out["ws"])


def make_steps(ctx, rows, vocab, classes, g):
    ids, rowptr, val, _ = make_bags(torch.randint(0, 60, (rows,), generator=g, device="cuda"), vocab, g)
    s = {"ids": ids, "rowptr": rowptr, "val": val, "table": torch.randn(vocab, classes, generator=g, device="cuda"),
         "labels": torch.randint(0, classes, (rows,), generator=g, device="cuda"), "u": torch.rand(rows, generator=g, device="cuda"),
         "p": torch.full((rows,), 0.8, device="cuda")}
    bags = ctx.bags(ids, rowptr, val)

    def buffers():
        return {"logits": torch.empty(rows, classes, device="cuda"), "dlogits": torch.empty(rows, classes, device="cuda"),
                "loss": torch.empty(rows, device="cuda"), "grad": torch.empty(vocab, classes, device="cuda"),
                "order": torch.empty(ctx.embed_order_bytes(bags, vocab), dtype=torch.uint8, device="cuda"),
                "ws": torch.empty(64 << 20, dtype=torch.uint8, device="cuda"),
                "token": torch.empty(rows, dtype=torch.int32, device="cuda"), "logprob": torch.empty(rows, device="cuda")}
    return s, buffers


KEYS = ("logits", "dlogits", "loss", "grad", "token", "logprob")


@pytest.mark.parametrize("rows,vocab,classes", [(100, 500, 16), (1500, 3000, 40), (3, 50, 9000)])
def test_graphs_of_the_four_together(ctx, rows, vocab, classes):
    """two captured graphs with workspaces of their own, replayed between eager work on changing inputs"""
    from admm_amd import capi
    g = rng(15, rows)
    s, buffers = make_steps(ctx, rows, vocab, classes, g)
    side = torch.cuda.Stream()
    other = capi.Context(0, stream=side.cuda_stream)
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):
        out = buffers()
        with torch.cuda.stream(side):
            steps(other, s, out)  # once outside
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            steps(other, s, out)
        graphs.append((graph, out))
    for turn in range(4):
        s["table"].copy_(torch.randn(vocab, classes, generator=g, device="cuda"))
        s["ids"].copy_(s["ids"][torch.randperm(s["ids"].numel(), generator=g, device="cuda")])
        s["u"].copy_(torch.rand(rows, generator=g, device="cuda"))
        torch.cuda.synchronize()
        for graph, out in graphs:
            for k in KEYS:
                out[k].fill_(5)
            graph.replay()
        eager = buffers()
        steps(ctx, s, eager)
        torch.cuda.synchronize()
        for _, out in graphs:
            for k in KEYS:
                assert torch.equal(out[k], eager[k]), (turn, k)
    del graphs
    other.close()


def test_streams_of_their_own(ctx):
    """contexts on two streams at once, each with its own buffers, against the default stream's results"""
    from admm_amd import capi
    g = rng(16, 1)
    s, buffers = make_steps(ctx, 800, 2000, 64, g)
    want = buffers()
    steps(ctx, s, want)
    torch.cuda.synchronize()
    pairs = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        pairs.append((capi.Context(0, stream=stream.cuda_stream), buffers()))
    torch.cuda.synchronize()
    for _ in range(5):
        for c, out in pairs:
            steps(c, s, out)
    for c, out in pairs:
        c.sync()
        for k in KEYS:
            assert torch.equal(out[k], want[k]), k
        c.close()


def test_the_context_keeps_a_workspace(ctx):
    """calls without a workspace: the context's own grows, and results stay what they are"""
    g = rng(17, 1)
    for rows in (100, 5000, 700):
        ids = make_bags([rows], 50, g, torch.int64)[0]
        check_grad(ctx, ids, None, None, torch.arange(rows, device="cuda"), rows, 50, 64, "f32", "f32", False, g)


def test_a_workspace_does_not_grow_under_capture(ctx):
    """a call that needs a larger workspace than its context has is refused while its stream is captured, and captured once
    the context has it"""
    from admm_amd import capi
    side = torch.cuda.Stream()
    other = capi.Context(0, stream=side.cuda_stream)
    g = rng(21, 1)
    x, u = make_logits(3, 5000, "f32", g), torch.rand(3, generator=g, device="cuda")
    want, token = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    ctx.sample(x, u, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        token.zero_()
        with pytest.raises(capi.AdmmError, match="captured"):
            other.sample(x, u, token)
    with torch.cuda.stream(side):
        other.sample(x, u, token)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.sample(x, u, token)
    for _ in range(3):
        token.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, want)
    del graph
    other.close()


def test_nothing_to_do(ctx):
    """shapes without elements"""
    f = lambda *shape, **kw: torch.zeros(*shape, device="cuda", **kw)  # noqa: E731
    none = ctx.bags(f(0, dtype=torch.int64))
    ctx.embed(none, f(5, 3), f(0, 3))
    ctx.embed(ctx.bags(f(4, dtype=torch.int64)), f(5, 0), f(4, 0))
    out, grad = torch.ones(4, 3, device="cuda"), torch.ones(5, 3, device="cuda")
    ctx.embed(none, f(5, 3), out)
    assert torch.all(out == 1)
    order = ctx.embed_order(none, 5)
    ctx.embed_grad(none, order, f(0, 3), grad, accumulate=True)
    assert torch.all(grad == 1)
    ctx.embed_grad(none, order, f(0, 3), grad)
    assert torch.all(grad == 0)
    ctx.softmax_loss(f(0, 3), f(0, dtype=torch.int64), f(0))
    ctx.sample(f(0, 3), f(0), f(0, dtype=torch.int32))
    empty_rows = ctx.bags(f(0, dtype=torch.int32), f(4, dtype=torch.int64))
    out = torch.ones(3, 3, device="cuda")
    ctx.embed(empty_rows, f(5, 3), out)
    assert torch.all(out == 0)


def test_entries_without_any_row(ctx):
    """row pointers of no row: the gradient is zero, or left as it was, and nothing of grad_out is read (it has no memory)"""
    for n in (5, 100, 20000):
        bags = ctx.bags(torch.randint(0, 50, (n,), device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"))
        order = ctx.embed_order(bags, 50)
        grad = torch.full((50, 8), 3.0, device="cuda")
        ctx.embed_grad(bags, order, torch.empty(0, 8, device="cuda"), grad, accumulate=True)
        assert torch.all(grad == 3.0)
        ctx.embed_grad(bags, order, torch.empty(0, 8, device="cuda"), grad)
        assert torch.all(grad == 0.0)
        ctx.embed(bags, torch.ones(50, 8, device="cuda"), torch.empty(0, 8, device="cuda"))


def test_more_elements_than_32_bits_count(ctx):
    """a table and logits of more than 2^32 elements: rows at both ends"""
    vocab, cols = 1 << 20, 4104
    table = torch.zeros(vocab, cols, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([0, 1, vocab - 1, vocab - 2, vocab // 2], device="cuda")
    g = rng(22, 1)
    rows = torch.randn(5, cols, generator=g, device="cuda").bfloat16()
    table[ids] = rows
    out = torch.empty(5, cols, dtype=torch.bfloat16, device="cuda")
    bags = ctx.bags(ids)
    ctx.embed(bags, table, out)
    assert torch.equal(out, rows)
    ctx.embed_grad(bags, ctx.embed_order(bags, vocab), rows, table, scale=-1.0, accumulate=True)
    assert not table.any()
    table.fill_(1)
    ctx.embed_grad(bags, ctx.embed_order(bags, vocab), rows, table, scale=2.0)
    assert torch.equal(table[ids], rows * 2)
    table[ids] = 0
    assert not table.any()
    del table
    x = torch.zeros(33000, 130200, dtype=torch.bfloat16, device="cuda")
    peak = torch.arange(33000, device="cuda") % 130200
    x[torch.arange(33000, device="cuda"), peak] = 30.0
    token = torch.empty(33000, dtype=torch.int32, device="cuda")
    u = torch.full((33000,), 0.5, device="cuda")
    ctx.sample(x, u, token, top_p=u)
    assert torch.equal(token.long(), peak)
    ctx.sample(x, u, token, top_k=torch.full((33000,), 5, dtype=torch.int32, device="cuda"))
    assert torch.equal(token.long(), peak)
    loss = torch.empty(33000, device="cuda")
    ctx.softmax_loss(x, peak, loss, grad=x)
    assert float(loss.abs().max()) < 1e-7  # 130199 e^-30 = 1.2e-8
    for r in (0, 16500, 32999):
        p = math.exp(-30) / (1 + 130199 * math.exp(-30))
        want = torch.full((130200,), p, dtype=torch.float64, device="cuda")
        want[int(peak[r])] = -130199 * p
        within(x[r], want, want.abs() * (2.0 ** -8 + 1e-4) + 2.0 ** -23, "grad")


def test_python_refusals(ctx):
    from admm_amd import capi
    f = lambda *shape, **kw: torch.zeros(*shape, device="cuda", **kw)  # noqa: E731
    ids = f(4, dtype=torch.int64)
    with pytest.raises(capi.AdmmError, match="is on cpu"):
        ctx.embed(ctx.bags(ids.cpu()), f(5, 3), f(4, 3))
    with pytest.raises(capi.AdmmError, match="adjacent"):
        ctx.embed(ctx.bags(ids), f(3, 5).t(), f(4, 3))
    with pytest.raises(capi.AdmmError, match="float32"):
        ctx.embed(ctx.bags(ids), f(5, 3, dtype=torch.float64), f(4, 3))
    with pytest.raises(capi.AdmmError, match="type"):
        ctx.bags(f(4))
    with pytest.raises(capi.AdmmError, match="adjacent elements"):
        ctx.bags(f(8, dtype=torch.int64)[::2])
    with pytest.raises(capi.AdmmError, match="apart"):
        ctx.embed(ctx.bags(ids), f(1, 3).expand(5, 3), f(4, 3))
    with pytest.raises(capi.AdmmError, match="4 adjacent"):
        ctx.softmax_loss(f(4, 3), f(3, dtype=torch.int64), f(4))
    with pytest.raises(capi.AdmmError, match="type"):
        ctx.sample(f(4, 3), f(4), f(4, dtype=torch.int64))
    with pytest.raises(capi.AdmmError, match="overlaps"):
        x = f(6, 3)
        ctx.embed(ctx.bags(ids), x[:4], x[2:])
    with pytest.raises(capi.AdmmError, match="too large|GPU|is on"):
        ctx.sample(torch.zeros(4, 3), f(4), f(4, dtype=torch.int32))


def test_many_class_regression_on_a_sample_set(ctx):
    """gradient steps of a softmax regression on a resident sample set, against the same steps in 64 bits, then a draw"""
    from conftest import make_synth_csr
    dim, classes, steps_n = 600, 5, 4
    raw = make_synth_csr(400, dim, 12, seed=21, binary=False)
    label = np.random.RandomState(3).randint(0, classes, 400).astype(np.float32)
    csr = ctx.csr_upload(raw.rowptr, raw.col, raw.val, label, dim)
    rowptr, col, val, _ = csr.download()
    X = np.zeros((400, dim))
    for r in range(400):
        for e in range(int(rowptr[r]), int(rowptr[r + 1])):
            X[r, int(col[e])] += float(val[e])
    bags = csr.bags()
    labels = torch.empty(400, device="cuda")
    csr.copy_labels(capi_vec(ctx, labels))
    W = torch.zeros(dim, classes, device="cuda")
    logits, loss, grad = torch.empty(400, classes, device="cuda"), torch.empty(400, device="cuda"), torch.empty(dim, classes, device="cuda")
    order = ctx.embed_order(bags, dim)
    want = np.zeros((dim, classes))
    for _ in range(steps_n):
        ctx.embed(bags, W, logits)
        ctx.softmax_loss(logits, labels, loss, grad=logits, grad_scale=1.0 / 400)
        ctx.embed_grad(bags, order, logits, grad)
        W -= 0.5 * grad
        z = X @ want
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        ref_loss = -np.log(p[np.arange(400), label.astype(int)])
        p[np.arange(400), label.astype(int)] -= 1
        want -= 0.5 / 400 * X.T @ p
    # a coordinate's sum has up to 400 terms, a step moves it by at most 0.5 max|x| and carries the errors of the last
    bound = steps_n * 0.5 * np.abs(X).max() * 500 * U * np.abs(X).sum(1).max()
    within(W.cpu(), torch.from_numpy(want), bound, "weights")
    within(loss.cpu(), torch.from_numpy(ref_loss), bound * np.abs(X).sum(1).max() + 100 * U, "loss")
    token = torch.empty(400, dtype=torch.int32, device="cuda")
    ctx.embed(bags, W, logits)
    ctx.sample(logits, torch.zeros(400, device="cuda"), token, temperature=torch.zeros(400, device="cuda"))
    assert torch.equal(token.long(), logits.argmax(1))
    csr.relabel_by_frequency()
    from admm_amd import capi
    with pytest.raises(capi.AdmmError, match="relabelled"):
        csr.bags()
    order.free()
    csr.destroy()


def capi_vec(ctx, t):
    from admm_amd import capi
    return capi.DeviceVec.from_ptr(ctx, t.data_ptr(), t.numel())
