"""What the token operators cost, and what they have to give: the loss head (softmax cross entropy over a large vocabulary, taken
in pieces of the vocabulary without keeping the logits, with its gradients) and the token embedding (scaled lookup, and its
gradient summed over sorted tokens). The two stand at the ends of a model between the loader's batch and the optimizer step.

`own` False: the plain forms, elementary torch operations in 32 bits. `own` True: the framework's operators, called as a
training program calls them: on device addresses, with a handle made once for the largest batch.
"""
import math

import torch

own = False

DEV = "cuda:0"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _case(name, kind, rows, hidden, vocab, dtype, masked=0.0, scale=1.0, micro=1):
    """rows: tokens of one call. masked: share of rows that the loss mask leaves out (0: no mask is given). scale: the loss scale,
    or the factor of the embedding. micro: micro-batches whose gradients one pass sums into the same buffer."""
    return dict(name=name, kind=kind, rows=rows, hidden=hidden, vocab=vocab, dtype=dtype, masked=masked, scale=scale, micro=micro)


def listed():
    return [
        # a held-out pass over two rows of 2048 tokens of the 1.24 B-parameter model: losses only
        _case("loss-heldout-bf16", "loss", 4096, 2048, 128256, "bf16"),
        # the loss of one token of the f32 model with the odd vocabulary: latency, and one stream of the weights
        _case("loss-one-row-f32", "loss", 1, 512, 100315, "f32"),
        # a training micro-batch of the 1.24 B-parameter model
        _case("train-8k-bf16", "train", 8192, 2048, 128256, "bf16"),
        # an f16 run with a loss scale, half of its positions a prompt that is not scored
        _case("train-masked-f16", "train", 4096, 2048, 151936, "f16", masked=0.5, scale=65536.0),
        # the all-f32 configuration: two rows of 512 tokens
        _case("train-f32", "train", 1024, 512, 100315, "f32"),
        # a narrow hybrid model, the last token of the batch cut off: an odd count of rows
        _case("train-narrow-bf16", "train", 8191, 384, 32000, "bf16"),
        # a handful of tokens through a training step (a debugging run, a short document)
        _case("train-16-rows-bf16", "train", 16, 1024, 32000, "bf16", masked=0.1),
        # the lookup that feeds the first layer, and the same for a few tokens
        _case("lookup-8k-bf16", "lookup", 8192, 2048, 128256, "bf16", scale=45.25),
        _case("lookup-17-f32", "lookup", 17, 512, 100315, "f32"),
        # the gradient of the lookup into an untied table: every row is written
        _case("embed-grads-bf16", "embed", 8192, 2048, 128256, "bf16", scale=45.25),
        # two micro-batches of a narrow f32 model summed into one table
        _case("embed-grads-micro-f32", "embed", 1000, 384, 32000, "f32", micro=2),
        # tied weights: the head's gradient, then the lookup's added to the same tensor
        _case("tied-2k-bf16", "tied", 2048, 2048, 128256, "bf16", scale=45.25),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("loss", "train", "train", "lookup", "embed", "tied"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    hidden = _log(rng, 64, 2048)
    if rng.random() < 0.5:
        hidden = (hidden + 63) // 64 * 64  # what models have; the other half are odd ones
    vocab, rows = _log(rng, 1000, 152000), _log(rng, 1, 8192)
    if dtype == "f32":
        rows = min(rows, 2048)
    masked = rng.choice((0.0, 0.0, round(rng.uniform(0.05, 0.95), 2))) if kind in ("loss", "train", "tied") else 0.0
    scale = rng.choice((1024.0, 65536.0)) if dtype == "f16" and kind == "train" else 1.0 if kind in ("loss", "train") else round(rng.uniform(0.5, 46.0), 2)
    return dict(kind=kind, rows=rows, hidden=hidden, vocab=vocab, dtype=dtype, masked=masked, scale=scale,
                micro=rng.choice((1, 2)) if kind == "embed" else 1)


def _tokens(gen, n, vocab):
    """Ids as text has them: the k-th commonest about 1/k as often as the commonest, spread over the vocabulary."""
    u = torch.rand(n, generator=gen, device=DEV, dtype=torch.float64)
    rank = torch.exp(u * math.log(vocab)).long().clamp_(1, vocab) - 1
    return rank * 7919 % vocab if vocab % 7919 else rank


def _inputs(c, seed):
    """What a program has in hand: weights ~N(0, 0.02), hidden states ~N(0, 1) that lean towards their target's row by a share of
    their own (from rows that know nothing to rows that are sure), the loader's ids, targets and mask."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    n, h, v, t = c["rows"], c["hidden"], c["vocab"], TORCH[c["dtype"]]
    s = {"ids": [_tokens(gen, n, v) for _ in range(c["micro"])]}
    if c["kind"] != "embed":
        s["weight"] = torch.empty(v, h, device=DEV, dtype=torch.float32).normal_(0.0, 0.02, generator=gen).to(t)
    if c["kind"] in ("embed", "tied"):
        s["d_out"] = [torch.empty(n, h, device=DEV).normal_(0.0, 1e-2, generator=gen).to(t) for _ in range(c["micro"])]
    if c["kind"] in ("loss", "train", "tied"):
        s["targets"] = _tokens(gen, n, v)
        lean = torch.rand(n, 1, generator=gen, device=DEV)
        s["hidden"] = (torch.empty(n, h, device=DEV).normal_(0.0, 1.0, generator=gen) + 25.0 * lean * s["weight"][s["targets"]].float()).to(t)
        s["mask"] = (torch.rand(n, generator=gen, device=DEV) >= c["masked"]).float() if c["masked"] else None
    return s


def _grad_scale(c):
    return (c["scale"] if c["kind"] == "train" else 1.0) / c["rows"]


def prepare(case, seed):
    s = _inputs(case, seed)
    n, h, v, t = case["rows"], case["hidden"], case["vocab"], TORCH[case["dtype"]]
    s["case"] = case
    if own:
        import oxidizr_b200 as ox
        code = {"f32": ox.F32, "bf16": ox.BF16, "f16": ox.F16}[case["dtype"]]
        new = lambda *shape, dtype=torch.float32: torch.empty(*shape, device=DEV, dtype=dtype)  # noqa: E731
        s["stream"] = torch.cuda.current_stream().cuda_stream
        if case["kind"] in ("loss", "train", "tied"):
            s["head"] = ox.LossHead(v, h, n, dtype=code)
            s["row_loss"], s["totals"], s["row_stats"] = new(n), new(2), new(n, 2)
        if case["kind"] in ("train", "tied"):
            s["d_hidden"] = new(n, h, dtype=t)
        if case["kind"] in ("train", "tied", "embed"):
            s["d_weight"] = new(v, h, dtype=t)
        if case["kind"] in ("lookup", "embed", "tied"):
            s["embed"] = ox.TokenEmbedding(v, h, n, dtype=code, scale=case["scale"])
            s["out"] = new(n, h, dtype=t)
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_loss(s):
    """loss_i = log sum_v exp(l_iv - m_i) - (l_it - m_i) of the scored rows; sum_i w_i loss_i and sum_i w_i."""
    logits = s["hidden"].float() @ s["weight"].float().T
    w = s["mask"] if s["mask"] is not None else torch.ones_like(logits[:, 0])
    m = logits.max(1, keepdim=True).values
    at = s["targets"][:, None]
    lt = logits.gather(1, at) - m
    e = torch.exp(logits - m)
    z = e.sum(1, keepdim=True)
    loss = torch.where(w != 0, (torch.log(z) - lt)[:, 0], 0.0)
    totals = torch.stack(((loss.double() * w.double()).sum(), w.double().sum())).float()
    return loss, totals, e, z, lt, w


def _plain_train(s):
    c = s["case"]
    loss, totals, e, z, lt, w = _plain_loss(s)
    at = s["targets"][:, None]
    # p - 1 at the target from the sum without it, so that a sure row keeps its digits
    other = e.scatter(1, at, 0.0).sum(1, keepdim=True)
    d = e.div_(z).scatter_(1, at, -other / z)
    d *= w[:, None]
    d_hidden = (d @ s["weight"].float()) * _grad_scale(c)
    d_weight = (d.T @ s["hidden"].float()) * _grad_scale(c)
    t = TORCH[c["dtype"]]
    return loss, totals, d_hidden.to(t), d_weight.to(t)


def _plain_embed(s, table):
    """table += scale * the sum of each token's rows, each micro-batch rounded to the table's type."""
    c = s["case"]
    for ids, d_out in zip(s["ids"], s["d_out"]):
        g = torch.zeros(c["vocab"], c["hidden"], device=DEV).index_add_(0, ids, d_out.float()) * c["scale"]
        table = g.to(TORCH[c["dtype"]]) if table is None else (table.float() + g).to(TORCH[c["dtype"]])
    return table


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        if kind == "loss":
            return dict(zip(("loss", "totals"), _plain_loss(s)))
        if kind == "train":
            return dict(zip(("loss", "totals", "d_hidden", "d_weight"), _plain_train(s)))
        if kind == "lookup":
            return {"out": (s["weight"][s["ids"][0]].float() * c["scale"]).to(TORCH[c["dtype"]])}
        if kind == "embed":
            return {"d_weight": _plain_embed(s, None)}
        loss, totals, d_hidden, d_weight = _plain_train(s)
        out = (s["weight"][s["ids"][0]].float() * c["scale"]).to(TORCH[c["dtype"]])
        return {"out": out, "loss": loss, "totals": totals, "d_hidden": d_hidden, "d_weight": _plain_embed(s, d_weight)}

    n, st = c["rows"], s["stream"]
    got = {}
    if kind in ("lookup", "tied"):
        s["embed"].lookup(s["ids"][0].data_ptr(), n, s["weight"].data_ptr(), s["out"].data_ptr(), stream=st)
        got["out"] = s["out"]
    if kind in ("loss", "train", "tied"):
        batch = dict(rows=n, hidden=s["hidden"].data_ptr(), weight=s["weight"].data_ptr(), targets=s["targets"].data_ptr(),
                     loss_mask=s["mask"].data_ptr() if s["mask"] is not None else None, row_loss=s["row_loss"].data_ptr(),
                     totals=s["totals"].data_ptr(), stream=st)
        got.update(loss=s["row_loss"], totals=s["totals"])
        if kind == "loss":
            s["head"].loss(**batch)
        else:
            s["head"].loss_and_grads(**batch, row_stats=s["row_stats"].data_ptr(), d_hidden=s["d_hidden"].data_ptr(),
                                     d_weight=s["d_weight"].data_ptr(), grad_scale=_grad_scale(c))
            got.update(d_hidden=s["d_hidden"], d_weight=s["d_weight"])
    if kind in ("embed", "tied"):
        for k, (ids, d_out) in enumerate(zip(s["ids"], s["d_out"])):
            s["embed"].grads(ids.data_ptr(), n, d_out.data_ptr(), s["d_weight"].data_ptr(), accumulate=kind == "tied" or k > 0, stream=st)
        got["d_weight"] = s["d_weight"]
    return got


def work(case):
    c = case
    n, h, v, es = c["rows"], c["hidden"], c["vocab"], SIZE[c["dtype"]]
    scored = max(1.0, n * (1.0 - c["masked"]))
    nbytes = flops = 0.0
    if c["kind"] in ("loss", "train", "tied"):
        nbytes += v * h * es + scored * h * es + n * (8 + 4 + (4 if c["masked"] else 0))
        flops += 2.0 * scored * v * h + 4.0 * scored * v
    if c["kind"] in ("train", "tied"):
        nbytes += v * h * es + n * h * es
        flops += 4.0 * scored * v * h
    if c["kind"] in ("lookup", "tied"):
        nbytes += n * (8 + 2.0 * h * es)
        flops += float(n * h)
    if c["kind"] in ("embed", "tied"):
        first = v * h * es if c["kind"] == "embed" else 0  # a table that starts from nothing is written whole
        more = c["micro"] - 1 if c["kind"] == "embed" else 1
        nbytes += first + more * 2 * min(n, v) * h * es + c["micro"] * n * (8 + h * es)
        flops += 2.0 * c["micro"] * n * h
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    n, h, v = c["rows"], c["hidden"], c["vocab"]
    f64 = torch.float64
    got = {}
    if c["kind"] in ("lookup", "tied"):
        got["out"] = torch.index_select(s["weight"].to(f64), 0, s["ids"][0]).mul_(c["scale"])
    d_weight = torch.zeros(v, h, device=DEV, dtype=f64) if c["kind"] in ("train", "embed", "tied") else None
    if c["kind"] in ("loss", "train", "tied"):
        big = s["weight"].to(f64)
        w = s["mask"].to(f64) if s["mask"] is not None else torch.ones(n, device=DEV, dtype=f64)
        losses, d_hidden = torch.zeros(n, device=DEV, dtype=f64), torch.zeros(n, h, device=DEV, dtype=f64)
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            hid, at = s["hidden"][a:b].to(f64), s["targets"][a:b]
            logits = hid.matmul(big.t())
            lse = torch.logsumexp(logits, dim=1)
            here = torch.arange(b - a, device=DEV)
            losses[a:b] = torch.where(w[a:b] != 0, lse - logits[here, at], torch.zeros_like(lse))
            if c["kind"] != "loss":
                p = logits.sub_(lse[:, None]).exp_()
                p[here, at] -= 1.0
                p.mul_(w[a:b, None] * _grad_scale(c))
                d_hidden[a:b] = p.matmul(big)
                d_weight.addmm_(p.t(), hid)
        got["loss"], got["totals"] = losses, torch.stack([losses.dot(w), w.sum()])
        if c["kind"] != "loss":
            got["d_hidden"] = d_hidden
    if c["kind"] in ("embed", "tied"):
        for ids, d_out in zip(s["ids"], s["d_out"]):
            d_weight.index_add_(0, ids, d_out.to(f64), alpha=c["scale"])
    if d_weight is not None:
        got["d_weight"] = d_weight
    return got
