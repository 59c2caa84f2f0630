"""The many-class operators of the library and their plain forms, case by case.

A model with many classes (or tokens) does four things that the two-class sweeps do for one weight per feature: it
looks rows of a weight matrix up and sums them (`embed`), turns the logits and the labels into a loss and its
gradient (`softmax_loss`), sums the gradient's rows per feature or token (`embed_grad`), and answers with a class
drawn from the distribution (`sample`).

`own` False: elementary torch operations.  `own` True: the library's entry points.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a serving step of a small batch: the tokens that eight sequences have just chosen
        {"name": "embed-8-tokens", "op": "embed", "type": "bf16", "out": "bf16", "rows": 8, "entries": 1, "vocab": 32000, "cols": 1024, "ids": "i64"},
        # a batch of prompts in training or prefill
        {"name": "embed-16384-tokens", "op": "embed", "type": "bf16", "out": "bf16", "rows": 16384, "entries": 1, "vocab": 128000, "cols": 4096, "ids": "i64"},
        # a mini-batch of sparse rows (2^20 features, 40 entries a row, stored values) times the weights of 16 classes
        {"name": "embed-65536-bags", "op": "embed", "type": "f32", "out": "f32", "rows": 65536, "entries": 40, "vocab": 1 << 20, "cols": 16, "ids": "i32"},
        # the gradient of a small vocabulary's table, an odd count of tokens, written whole
        {"name": "embed_grad-4001-tokens", "op": "embed_grad", "type": "bf16", "out": "bf16", "rows": 4001, "entries": 1, "vocab": 32000, "cols": 1024, "ids": "i64", "accumulate": False},
        # the gradient of a large table, added to the float sums of earlier micro-batches
        {"name": "embed_grad-16384-accumulate", "op": "embed_grad", "type": "bf16", "out": "f32", "rows": 16384, "entries": 1, "vocab": 128000, "cols": 2048, "ids": "i64", "accumulate": True},
        # the gradient of the mini-batch of sparse rows
        {"name": "embed_grad-65536-bags", "op": "embed_grad", "type": "f32", "out": "f32", "rows": 65536, "entries": 40, "vocab": 1 << 20, "cols": 16, "ids": "i32", "accumulate": False},
        # loss and gradient of that mini-batch: many short rows
        {"name": "softmax_loss-65536x16", "op": "softmax_loss", "type": "f32", "rows": 65536, "cols": 16, "masked": 0.0, "ignored": 0.0},
        # loss and gradient over a vocabulary, some rows not trained on (prompts, padding)
        {"name": "softmax_loss-8192x32000", "op": "softmax_loss", "type": "bf16", "rows": 8192, "cols": 32000, "masked": 0.0, "ignored": 0.1},
        # odd numbers of rows and classes (no row but the first begins on 16 bytes), a tenth of the classes masked out
        {"name": "softmax_loss-1001x100003", "op": "softmax_loss", "type": "f16", "rows": 1001, "cols": 100003, "masked": 0.1, "ignored": 0.1},
        # one sequence's next token
        {"name": "sample-1x128000", "op": "sample", "type": "bf16", "rows": 1, "cols": 128000, "spread": 3.0, "filters": "both"},
        # a batch whose requests all ask for something else, an odd vocabulary, logits in 32 bits
        {"name": "sample-64x50001", "op": "sample", "type": "f32", "rows": 64, "cols": 50001, "spread": 2.5, "filters": "mixed"},
        # a large batch in nucleus sampling
        {"name": "sample-512x128000", "op": "sample", "type": "bf16", "rows": 512, "cols": 128000, "spread": 3.5, "filters": "top_p"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "softmax_loss", "sample"])
    if op in ("embed", "embed_grad"):
        bags = rng.random() < 0.4
        kind = rng.choice(["f32", "bf16", "f16"])
        case = {"op": op, "type": kind, "out": rng.choice([kind, "f32"])}
        if bags:
            case |= {"rows": _log_int(rng, 1, 65536), "entries": _log_int(rng, 2, 40), "vocab": _log_int(rng, 100, 1 << 20),
                     "cols": _log_int(rng, 1, 16), "ids": "i32"}
        else:
            case |= {"rows": _log_int(rng, 1, 16384), "entries": 1, "vocab": _log_int(rng, 100, 128000),
                     "cols": rng.choice([_log_int(rng, 16, 2048), 8 * _log_int(rng, 2, 256)]), "ids": rng.choice(["i32", "i64"])}
        if op == "embed_grad":
            case["accumulate"] = rng.random() < 0.5
        return case
    if op == "softmax_loss":
        cols = _log_int(rng, 2, 128000)
        return {"op": op, "type": rng.choice(["f32", "bf16", "f16"]), "rows": _log_int(rng, 1, max(1, min(65536, (1 << 27) // cols))),
                "cols": cols, "masked": rng.choice([0.0, 0.3]), "ignored": rng.choice([0.0, 0.2])}
    cols = _log_int(rng, 50, 128000)
    return {"op": op, "type": rng.choice(["f32", "bf16", "f16"]), "rows": _log_int(rng, 1, min(512, max(1, (1 << 25) // cols))),
            "cols": cols, "spread": rng.choice([1.0, 2.5, 4.0]),
            "filters": rng.choice(["none", "top_k", "top_p", "min_p", "both", "mixed"])}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _zipf_ids(g, count, vocab):
    """ids whose frequency falls as 1 / rank, the ranks scattered over the table"""
    u = torch.rand(count, generator=g, device="cuda", dtype=torch.float64)
    rank = torch.clamp((torch.exp(u * math.log(vocab + 1.0)) - 1.0).long(), 0, vocab - 1)
    step = next(s for s in (7919, 104729, 1299709, 1) if math.gcd(s, vocab) == 1)
    return (rank * step + vocab // 3) % vocab


def prepare(case, seed):
    g = _generator(seed)
    rows = case["rows"]
    if case["op"] in ("embed", "embed_grad"):
        kind, vocab, cols = TYPES[case["type"]], case["vocab"], case["cols"]
        s = {"case": case, "scale": float(np.float32(math.sqrt(cols)))}
        if case["entries"] == 1:
            nnz = rows
            ids = _zipf_ids(g, rows, vocab)
            if rows > 16:  # padding
                ids = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.01, torch.full_like(ids, -1), ids)
            s |= {"rowptr": None, "val": None, "row": None}
        else:
            length = torch.poisson(torch.full((rows,), float(case["entries"]), device="cuda"), generator=g).long()
            rowptr = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
            rowptr[1:] = torch.cumsum(length, 0)
            nnz = int(rowptr[-1])
            ids = _zipf_ids(g, nnz, vocab)
            val = torch.rand(nnz, generator=g, device="cuda") * 1.5 + 0.25
            # what a program that has the rows as pairs keeps beside the row pointers
            row = torch.repeat_interleave(torch.arange(rows, device="cuda"), length)
            s |= {"rowptr": rowptr, "val": val, "row": row}
        s["ids"] = ids.to(torch.int32) if case["ids"] == "i32" else ids
        if case["op"] == "embed":
            s["table"] = (torch.randn(vocab, cols, generator=g, device="cuda") * 0.02).to(kind)
        else:
            s["grad_out"] = (torch.randn(rows, cols, generator=g, device="cuda") * 1e-2).to(kind)
            if case["accumulate"]:
                s["grad"] = (torch.randn(vocab, cols, generator=g, device="cuda") * 1e-2).to(TYPES[case["out"]])
        return s
    cols, kind = case["cols"], TYPES[case["type"]]
    if case["op"] == "softmax_loss":
        x = torch.randn(rows, cols, generator=g, device="cuda") * 3.0
        labels = torch.randint(0, cols, (rows,), generator=g, device="cuda")
        # a trained model mostly gives its label one of the largest logits
        x.scatter_add_(1, labels[:, None], torch.rand(rows, 1, generator=g, device="cuda") * 12.0)
        if case["masked"]:
            out = torch.rand(rows, cols, generator=g, device="cuda") < case["masked"]
            out.scatter_(1, labels[:, None], False)
            x.masked_fill_(out, -math.inf)
        if case["ignored"]:
            labels = torch.where(torch.rand(rows, generator=g, device="cuda") < case["ignored"], torch.full_like(labels, -100), labels)
        # the mean over the batch; times a loss scale, as training in 16-bit floats with five exponent bits has one
        scale = (32768.0 if case["type"] == "f16" else 1.0) / rows
        return {"case": case, "logits": x.to(kind), "labels": labels, "grad_scale": float(np.float32(scale))}
    x = torch.randn(rows, cols, generator=g, device="cuda") * case["spread"]
    peak = torch.randint(0, cols, (rows, 4), generator=g, device="cuda")
    x.scatter_add_(1, peak, torch.rand(rows, 4, generator=g, device="cuda") * 8.0)
    r = torch.arange(rows, device="cuda")
    t = torch.rand(rows, generator=g, device="cuda") * 0.6 + 0.6
    k = torch.randint(1, 100, (rows,), generator=g, device="cuda", dtype=torch.int32)
    p = torch.rand(rows, generator=g, device="cuda") * 0.25 + 0.74
    m = torch.rand(rows, generator=g, device="cuda") * 0.1 + 0.01
    f = case["filters"]
    if f == "mixed":  # by row: greedy, temperature alone, top-k, top-p, min-p, all of them
        kinds = r % 6
        t = torch.where(kinds == 0, torch.zeros_like(t), t)
        k = torch.where((kinds == 2) | (kinds == 5), k, torch.zeros_like(k))
        p = torch.where((kinds == 3) | (kinds == 5), p, torch.ones_like(p))
        m = torch.where((kinds == 4) | (kinds == 5), m, torch.zeros_like(m))
    s = {"case": case, "logits": x.to(kind), "temperature": t, "uniform": torch.rand(rows, generator=g, device="cuda")}
    s["top_k"] = k if f in ("top_k", "both", "mixed") else None
    s["top_p"] = p if f in ("top_p", "both", "mixed") else None
    s["min_p"] = m if f in ("min_p", "mixed") else None
    return s


# ---- the library's entry points ---------------------------------------------------------------

_contexts = {}


def _context():
    """one context per device and stream, as a program keeps it"""
    from admm_amd import capi
    stream = torch.cuda.current_stream().cuda_stream
    key = (torch.cuda.current_device(), stream)
    if key not in _contexts:
        _contexts[key] = capi.Context(key[0], stream=stream or capi.DEFAULT_STREAM)
    return _contexts[key]


def _own(s):
    ctx, case = _context(), s["case"]
    if case["op"] == "embed":
        out = torch.empty(case["rows"], case["cols"], dtype=TYPES[case["out"]], device="cuda")
        ctx.embed(ctx.bags(s["ids"], s["rowptr"], s["val"]), s["table"], out, scale=s["scale"])
        return out
    if case["op"] == "embed_grad":
        bags = ctx.bags(s["ids"], s["rowptr"], s["val"])
        grad = s["grad"] if case["accumulate"] else torch.empty(case["vocab"], case["cols"], dtype=TYPES[case["out"]], device="cuda")
        order = torch.empty(ctx.embed_order_bytes(bags, case["vocab"]), dtype=torch.uint8, device="cuda")
        ctx.embed_order(bags, case["vocab"], order)
        ctx.embed_grad(bags, order, s["grad_out"], grad, scale=s["scale"], accumulate=case["accumulate"])
        return grad
    if case["op"] == "softmax_loss":
        grad = torch.empty_like(s["logits"])
        loss = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
        ctx.softmax_loss(s["logits"], s["labels"], loss, grad=grad, grad_scale=s["grad_scale"])
        return {"loss": loss, "grad": grad}
    token = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
    logprob = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
    ctx.sample(s["logits"], s["uniform"], token, logprob=logprob, temperature=s["temperature"], top_k=s["top_k"],
               top_p=s["top_p"], min_p=s["min_p"])
    return {"token": token, "logprob": logprob}


# ---- the plain forms --------------------------------------------------------------------------

def _plain_embed(s):
    case, ids = s["case"], s["ids"].long()
    there = (ids >= 0) & (ids < case["vocab"])
    rows = s["table"][torch.where(there, ids, torch.zeros_like(ids))].float()
    rows = rows * there[:, None]
    if s["val"] is None:
        out = rows * s["scale"]
    else:
        out = torch.zeros(case["rows"], case["cols"], device="cuda").index_add_(0, s["row"], rows * s["val"][:, None]) * s["scale"]
    return out.to(TYPES[case["out"]])


def _plain_embed_grad(s):
    case, ids = s["case"], s["ids"].long()
    there = (ids >= 0) & (ids < case["vocab"])
    rows = s["grad_out"].float() * s["scale"] if s["val"] is None else s["grad_out"].float()[s["row"]] * (s["val"] * s["scale"])[:, None]
    rows = rows * there[:, None]
    ids = torch.where(there, ids, torch.zeros_like(ids))
    if not case["accumulate"]:
        return torch.zeros(case["vocab"], case["cols"], device="cuda").index_add_(0, ids, rows).to(TYPES[case["out"]])
    if case["out"] == "f32":
        return s["grad"].index_add_(0, ids, rows)
    return s["grad"].copy_(s["grad"].float().index_add_(0, ids, rows))


def _plain_softmax_loss(s):
    x, labels = s["logits"].float(), s["labels"]
    on = labels >= 0
    at = torch.where(on, labels, torch.zeros_like(labels))[:, None]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    loss = torch.where(on, (torch.log(total) + top - x.gather(1, at))[:, 0], torch.zeros_like(top[:, 0]))
    grad = e / total
    grad.scatter_add_(1, at, torch.full_like(top, -1.0))
    grad *= (on * s["grad_scale"])[:, None]
    return {"loss": loss, "grad": grad.to(s["logits"].dtype)}


def _plain_sample(s):
    """tokens by value, then by index; top-k, then top-p of what is left, then min-p; drawn in the order of the indexes"""
    x = s["logits"].float()
    rows, cols = x.shape
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    xs, at = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((xs.double() - xs[:, :1].double()) / torch.where(greedy, torch.ones_like(t), t))
    rank = torch.arange(cols, device=x.device)[None, :]
    keep = torch.where(greedy, rank < 1, rank < cols)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = keep & ((k <= 0) | (rank < k))
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        kept = w * keep
        before = torch.cumsum(kept, 1) - kept
        keep = keep & ((p >= 1) | (before < p * kept.sum(1, keepdim=True)) | (rank == 0))
    if s["min_p"] is not None:
        m = s["min_p"].double()[:, None]
        keep = keep & ((m <= 0) | (w >= m) | (rank == 0))
    mass = torch.zeros_like(w).scatter_(1, at, w * keep)  # in the order of the indexes again
    cum = torch.cumsum(mass, 1)
    total = cum[:, -1:]
    token = torch.clamp((cum <= s["uniform"].double()[:, None] * total).sum(1), max=cols - 1)
    logprob = torch.log(mass.gather(1, token[:, None])[:, 0] / total[:, 0])
    return {"token": token.int(), "logprob": logprob.float()}


_PLAIN = {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "softmax_loss": _plain_softmax_loss, "sample": _plain_sample}


def run(s):
    return _own(s) if own else _PLAIN[s["case"]["op"]](s)


# ---- from the definitions, in 64 bits ---------------------------------------------------------

def _pairs(s):
    """(row, id, value) of the stored entries, without padding"""
    ids = s["ids"].long()
    row = torch.arange(ids.numel(), device="cuda") if s["row"] is None else s["row"]
    val = torch.ones(ids.numel(), dtype=torch.float64, device="cuda") if s["val"] is None else s["val"].double()
    there = torch.nonzero((ids >= 0) & (ids < s["case"]["vocab"]))[:, 0]
    return row[there], ids[there], val[there]


def _spread(to, at, source, weight, step=1 << 18):
    """to[at[i]] += weight[i] * source(i), some entries at a time"""
    for b in range(0, at.numel(), step):
        e = slice(b, b + step)
        to.index_put_((at[e],), source(e) * weight[e][:, None], accumulate=True)
    return to


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("embed", "embed_grad"):
        row, ids, val = _pairs(s)
        if case["op"] == "embed":
            out = torch.zeros(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
            return _spread(out, row, lambda e: s["table"][ids[e]].double(), val * s["scale"])
        out = s["grad"].double() if case["accumulate"] else torch.zeros(case["vocab"], case["cols"], dtype=torch.float64, device="cuda")
        return _spread(out, ids, lambda e: s["grad_out"][row[e]].double(), val * s["scale"])
    if case["op"] == "softmax_loss":
        rows, cols = s["logits"].shape
        loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
        grad = torch.zeros(rows, cols, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 26) // cols)
        for b in range(0, rows, step):
            x, label = s["logits"][b:b + step].double(), s["labels"][b:b + step]
            on = torch.nonzero(label >= 0)[:, 0]
            if on.numel():
                lse = torch.logsumexp(x[on], 1)
                loss[b + on] = lse - x[on, label[on]]
                p = torch.exp(x[on] - lse[:, None])
                p[torch.arange(on.numel(), device="cuda"), label[on]] -= 1.0
                grad[b + on] = p * s["grad_scale"]
        return {"loss": loss, "grad": grad}
    x = s["logits"].double().cpu().numpy()
    one = {k: (None if s[k] is None else s[k].double().cpu().numpy()) for k in ("temperature", "top_k", "top_p", "min_p", "uniform")}
    logprob = np.zeros(x.shape[0])
    for r in range(x.shape[0]):
        t = one["temperature"][r]
        if t <= 0:
            continue
        order = np.argsort(-x[r], kind="stable")
        if one["top_k"] is not None and one["top_k"][r] > 0:
            order = order[:int(one["top_k"][r])]
        w = np.exp((x[r][order] - x[r][order[0]]) / t)
        count = order.size
        if one["top_p"] is not None and one["top_p"][r] < 1:
            ends = np.cumsum(w)
            count = min(count, 1 + int(np.searchsorted(ends, one["top_p"][r] * ends[-1], side="left")))
        if one["min_p"] is not None and one["min_p"][r] > 0:
            count = min(count, max(1, int(np.count_nonzero(w >= one["min_p"][r]))))
        back = np.argsort(order[:count])
        ends = np.cumsum(w[:count][back])
        j = min(int(np.searchsorted(ends, one["uniform"][r] * ends[-1], side="right")), count - 1)
        logprob[r] = math.log(w[:count][back][j] / ends[-1])
    return {"token": None, "logprob": torch.from_numpy(logprob)}


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    rows, cols = case["rows"], case["cols"]
    if case["op"] in ("embed", "embed_grad"):
        nnz = rows * case["entries"]
        stored = nnz * (8 if case["ids"] == "i64" else 4) + (nnz * 4 + rows * 8 if case["entries"] > 1 else 0)
        touched = min(nnz, case["vocab"])
        if case["op"] == "embed":
            moved = touched * cols * size[case["type"]] + rows * cols * size[case["out"]]
        else:
            moved = rows * cols * size[case["type"]] + (2 * touched if case["accumulate"] else case["vocab"]) * cols * size[case["out"]]
        return {"bytes": stored + moved, "flops": 2 * nnz * cols}
    if case["op"] == "softmax_loss":
        return {"bytes": 2 * rows * cols * size[case["type"]] + rows * 12, "flops": 8 * rows * cols}
    return {"bytes": rows * cols * size[case["type"]] + rows * 24, "flops": 6 * rows * cols}
