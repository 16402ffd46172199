"""What is measured of the embedding-head operators, and their plain forms.

A row of the binned matrix is a list of tokens (its global bins). The head sums their embeddings, norms the sum, and
takes the softmax cross entropy over its classes; its gradients are clipped by their global norm. Each case here is one
of those operators at one size: `run` computes it with elementary torch operations in 32 bits, or, where `own` is true,
with the calls of hessboost_b200.head.

Sizes: the tokens are those of the repository's own workloads (28 features of 256 bins; 100 features of 128 bins; 2,000
features of 64 bins at 2% density), the widths, class counts and tensor lists are generic.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
    return [
        # one row of 28 features scored as it arrives: latency
        dict(name="embed row bf16", op="embed", layout="bags", train=False, rows=1, per_row=28, tokens=7168, width=64,
             dtype="bf16"),
        # a batch of the 28-feature matrix, 5% of its cells missing, forward and gradient
        dict(name="embed bins f32", op="embed", layout="bags", train=True, rows=65536, per_row=28, tokens=7168,
             width=64, dtype="f32"),
        # a batch of the sparse matrix (CSR rows of about 40 of 2,000 features, some empty), forward and gradient
        dict(name="embed csr bf16", op="embed", layout="csr", train=True, rows=131072, per_row=40, tokens=128000,
             width=128, dtype="bf16"),
        # one row's norm: latency
        dict(name="norm row f32", op="norm", train=False, rows=1, width=64, dtype="f32", strided=False),
        # the head's own width over a batch, forward and backward
        dict(name="norm head bf16", op="norm", train=True, rows=131072, width=128, dtype="bf16", strided=False),
        # wide rows of an odd length, a column slice of a wider matrix
        dict(name="norm wide f32", op="norm", train=True, rows=8191, width=4097, dtype="f32", strided=True),
        # a handful of rows against a thousand classes, loss alone: latency
        dict(name="xent score bf16", op="xent", train=False, rows=16, width=128, classes=1000, dtype="bf16"),
        # ten classes over a large batch of 100 columns, in 32 bits
        dict(name="xent few classes f32", op="xent", train=True, rows=131072, width=100, classes=10, dtype="f32"),
        # odd sizes in 32 bits
        dict(name="xent odd f32", op="xent", train=True, rows=4099, width=257, classes=12289, dtype="f32"),
        # a large vocabulary: the largest case
        dict(name="xent vocab bf16", op="xent", train=True, rows=8192, width=1024, classes=50021, dtype="bf16"),
        # the gradients of a small head: an embedding table, a norm, a classifier
        dict(name="clip head f32", op="clip", tensors=4, total=524_417, dtype="f32"),
        # the gradients of a large model, many tensors of very different sizes
        dict(name="clip many bf16", op="clip", tensors=120, total=120_000_000, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed", "norm", "xent", "xent", "clip"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "embed":
        layout = rng.choice(["bags", "csr", "lookup"])
        width = _log(rng, 8, 1024)
        per_row = 1 if layout == "lookup" else rng.choice([5, 28, 50, 100]) if layout == "bags" else _log(rng, 2, 100)
        most = (1 << 29) // (width * per_row)
        tokens = min(_log(rng, 40, 200_000), (1 << 28) // width)
        return dict(op=op, layout=layout, train=rng.random() < 0.75, rows=_log(rng, 1, min(400_000, most)),
                    per_row=per_row, tokens=tokens, width=width, dtype=rng.choice(["f32", "bf16", "f16"]))
    if op == "norm":
        width = _log(rng, 4, 16384)
        return dict(op=op, train=rng.random() < 0.75, rows=_log(rng, 1, min(400_000, (1 << 26) // width)), width=width,
                    dtype=rng.choice(["f32", "bf16", "f16"]), strided=rng.random() < 0.3)
    if op == "xent":
        width, classes = _log(rng, 8, 2048), _log(rng, 2, 100_000)
        most = min(200_000, (1 << 38) // (width * classes), (1 << 28) // classes, (1 << 27) // width)
        return dict(op=op, train=rng.random() < 0.75, rows=_log(rng, 1, max(2, most)), width=width, classes=classes,
                    dtype=dtype)
    tensors = _log(rng, 1, 300)
    return dict(op=op, tensors=tensors, total=_log(rng, 100 * tensors, 100_000_000), dtype=dtype)


def _embed_state(case, g, dtype):
    n, k, v, d = case["rows"], case["per_row"], case["tokens"], case["width"]
    ptr = None
    if case["layout"] == "csr":
        # about per_row stored cells a row, spread like a binomial's, ids ascending within a row; some rows are empty
        count = torch.poisson(torch.full((n,), float(k), device="cuda"), generator=g)
        count = torch.where(torch.rand(n, generator=g, device="cuda") < 0.01, 0, count).long()
        ptr = torch.cat([count.new_zeros(1), count.cumsum(0)])
        row = torch.repeat_interleave(torch.arange(n, device="cuda"), count)
        ids = torch.randint(v, (row.numel(),), generator=g, device="cuda")
        tok = (torch.sort(row * v + ids).values % v).int()
    elif case["layout"] == "bags":
        # quantile bins: uniform within each feature's own range of ids; 5% of the cells missing
        per = max(1, v // k)
        tok = torch.randint(per, (n, k), generator=g, device="cuda") + torch.arange(k, device="cuda") * per
        tok = torch.where(torch.rand(n, k, generator=g, device="cuda") < 0.05, -1, tok % v).int()
    else:
        # one id a row, a few ids very frequent: P(id) falls as 1 / (id + 1)
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        tok = (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1)
    state = dict(tok=tok, ptr=ptr, scale=float(k) ** -0.5)
    state["table"] = torch.randn(v, d, generator=g, device="cuda").mul_(0.1).to(dtype)
    if case["train"]:
        state["grad"] = torch.randn(n, d, generator=g, device="cuda").mul_(1e-3).to(dtype)
    return state


def _norm_state(case, g, dtype):
    n, d = case["rows"], case["width"]
    pad = 24 if case["strided"] else 0
    x = torch.randn(n, d + pad, generator=g, device="cuda") * 2 + torch.randn(n, 1, generator=g, device="cuda")
    state = dict(x=x.to(dtype)[:, :d])
    state["weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype)
    state["bias"] = (0.1 * torch.randn(d, generator=g, device="cuda")).to(dtype)
    if case["train"]:
        state["grad"] = torch.randn(n, d, generator=g, device="cuda").mul_(1e-2).to(dtype)
    return state


def _xent_state(case, g, dtype):
    n, d, v = case["rows"], case["width"], case["classes"]
    w = torch.randn(v, d, generator=g, device="cuda").mul_(d**-0.5).to(dtype)
    # one row in 32 has no label; the others lean towards theirs, as a head's do while it trains
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    x = torch.randn(n, d, generator=g, device="cuda")
    x += 3 * torch.rand(n, 1, generator=g, device="cuda") * w[labels].float()
    labels = torch.where(torch.rand(n, generator=g, device="cuda") < 1 / 32, -1, labels)
    state = dict(x=x.to(dtype), w=w, labels=labels)
    if case["train"]:
        # sample weights over the batch's size
        state["dloss"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    return state


def _clip_state(case, g, dtype):
    # sizes spread over orders of magnitude, the last one taking what is left; each tensor with its own spread
    k = case["tensors"]
    share = torch.exp(3 * torch.randn(k, generator=g, device="cuda")).double()
    sizes = (share / share.sum() * (case["total"] - k)).long().add_(1).tolist()
    sizes[-1] += case["total"] - sum(sizes)
    grads = [(torch.randn(m, generator=g, device="cuda") * (10.0 ** -(1 + i % 4))).to(dtype) for i, m in enumerate(sizes)]
    flat = torch.empty(case["total"], dtype=dtype, device="cuda")
    return dict(grads=grads, flat=flat, out=list(flat.split(sizes)), max_norm=1.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"embed": _embed_state, "norm": _norm_state, "xent": _xent_state, "clip": _clip_state}[case["op"]]
    return dict(make(case, g, DTYPES[case["dtype"]]), op=case["op"], train=case.get("train", True))


def _embed_plain(s):
    table, tok, ptr, n_tokens = s["table"], s["tok"], s["ptr"], s["table"].shape[0]
    if ptr is not None:
        rows = ptr.numel() - 1
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), ptr[1:] - ptr[:-1], output_size=tok.numel())
    else:
        rows = tok.shape[0]
        row = torch.arange(rows, device="cuda").repeat_interleave(tok.numel() // rows, output_size=tok.numel())
    ids = tok.reshape(-1).long()
    there = ((ids >= 0) & (ids < n_tokens)).float()[:, None] * s["scale"]
    ids = ids.clamp(0, n_tokens - 1)
    terms = table.float()[ids] * there
    out = dict(out=torch.zeros(rows, table.shape[1], device="cuda").index_add_(0, row, terms).to(table.dtype))
    if s["train"]:
        terms = s["grad"].float()[row] * there
        out["dtable"] = torch.zeros(table.shape, device="cuda").index_add_(0, ids, terms).to(table.dtype)
    return out


def _norm_plain(s):
    x, w = s["x"].float(), s["weight"].float()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + EPS)
    xh = (x - mean) * rstd
    out = dict(y=(xh * w + s["bias"].float()).to(s["x"].dtype))
    if s["train"]:
        dy = s["grad"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        out.update(dx=dx.to(s["x"].dtype), dweight=(dy * xh).sum(0).to(s["weight"].dtype),
                   dbias=dy.sum(0).to(s["bias"].dtype))
    return out


def _xent_plain(s):
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.T
    there = (s["labels"] >= 0) & (s["labels"] < w.shape[0])
    label = s["labels"].clamp(0, w.shape[0] - 1)[:, None]
    most = z.max(1, keepdim=True).values
    at_label = z.gather(1, label)
    e = torch.exp(z - most)
    total = e.sum(1, keepdim=True)
    loss = torch.where(there, (most + torch.log(total) - at_label)[:, 0], 0.0)
    out = dict(loss=loss)
    if s["train"]:
        each = torch.where(there, s["dloss"], 0.0)[:, None]
        e *= each / total
        e.scatter_add_(1, label, -each)
        out.update(dx=(e @ w).to(s["x"].dtype), dw=(e.T @ x).to(s["w"].dtype))
    return out


def _clip_plain(s):
    norm = torch.sqrt(torch.stack([t.float().square().sum() for t in s["grads"]]).sum())
    by = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    torch._foreach_copy_(s["out"], [t.float() * by for t in s["grads"]])
    return dict(norm=norm, grads=s["flat"])


def _embed_own(s):
    from hessboost_b200 import head

    out = dict(out=head.embed_forward(s["tok"], s["table"], row_ptr=s["ptr"], scale=s["scale"]))
    if s["train"]:
        out["dtable"] = head.embed_backward(s["grad"], s["tok"], s["table"].shape[0], row_ptr=s["ptr"],
                                            scale=s["scale"])
    return out


def _norm_own(s):
    from hessboost_b200 import head

    y, mean, rstd = head.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=EPS)
    out = dict(y=y)
    if s["train"]:
        out["dx"], out["dweight"], out["dbias"] = head.layer_norm_backward(s["grad"], s["x"], s["weight"], mean, rstd)
    return out


def _xent_own(s):
    from hessboost_b200 import head

    loss, lse = head.linear_xent_forward(s["x"], s["w"], s["labels"])
    out = dict(loss=loss)
    if s["train"]:
        out["dx"], out["dw"] = head.linear_xent_backward(s["dloss"], s["x"], s["w"], s["labels"], lse)
    return out


def _clip_own(s):
    from hessboost_b200 import head

    return dict(norm=head.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"]), grads=s["flat"])


PLAIN = {"embed": _embed_plain, "norm": _norm_plain, "xent": _xent_plain, "clip": _clip_plain}
OWN = {"embed": _embed_own, "norm": _norm_own, "xent": _xent_own, "clip": _clip_own}


def run(state):
    return (OWN if own else PLAIN)[state["op"]](state)


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "embed":
        n, d, v = case["rows"], case["width"], case["tokens"]
        cells = n * case["per_row"]
        ids = cells * (8 if case["layout"] == "lookup" else 4) + (8 * (n + 1) if case["layout"] == "csr" else 0)
        b, f = ids + (min(v, cells) + n) * d * e, cells * d
        return dict(bytes=b + (n + v) * d * e, flops=2 * f) if case["train"] else dict(bytes=b, flops=f)
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        if case["train"]:
            return dict(bytes=4 * n * d * e + 4 * d * e, flops=20 * n * d)
        return dict(bytes=2 * n * d * e + 2 * d * e, flops=8 * n * d)
    if case["op"] == "xent":
        n, d, v = case["rows"], case["width"], case["classes"]
        b, f = (n + v) * d * e + n * 12, 2 * n * d * v
        return dict(bytes=2 * (n + v) * d * e + n * 16, flops=3 * f) if case["train"] else dict(bytes=b, flops=f)
    return dict(bytes=2 * case["total"] * e + 4, flops=3 * case["total"])


def exact(case, seed):
    """The same outputs in 64 bits, from torch's own definitions and their automatic gradients."""
    s = prepare(case, seed)
    fn = torch.nn.functional
    leaf = lambda t: t.double().requires_grad_(s["train"])  # noqa: E731
    if case["op"] == "embed":
        # bags without the ids outside the table
        tok = s["tok"].reshape(-1).long()
        rows = case["rows"]
        if s["ptr"] is None:
            ends = torch.arange(1, rows + 1, device="cuda") * (tok.numel() // rows)
        else:
            ends = s["ptr"][1:]
        there = (tok >= 0) & (tok < case["tokens"])
        kept = torch.cat([there.new_zeros(1, dtype=torch.long), there.long().cumsum(0)])
        starts = torch.cat([ends.new_zeros(1), ends[:-1]])
        table = leaf(s["table"])
        y = fn.embedding_bag(tok[there], table, kept[starts], mode="sum") * s["scale"]
        out = dict(out=y.detach())
        if s["train"]:
            out["dtable"] = torch.autograd.grad(y, table, s["grad"].double())[0]
        return out
    if case["op"] == "norm":
        x, w, b = leaf(s["x"]), leaf(s["weight"]), leaf(s["bias"])
        y = fn.layer_norm(x, (case["width"],), w, b, EPS)
        out = dict(y=y.detach())
        if s["train"]:
            out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (x, w, b), s["grad"].double())
        return out
    if case["op"] == "xent":
        x, w = leaf(s["x"]), leaf(s["w"])
        loss = fn.cross_entropy(fn.linear(x, w), s["labels"], ignore_index=-1, reduction="none")
        out = dict(loss=loss.detach())
        if s["train"]:
            out["dx"], out["dw"] = torch.autograd.grad(loss, (x, w), s["dloss"].double())
        return out
    every = torch.cat([t.double() for t in s["grads"]])
    norm = torch.linalg.vector_norm(every)
    return dict(norm=norm, grads=every * min(1.0, s["max_norm"] / (float(norm) + 1e-6)))
