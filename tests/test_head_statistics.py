"""The loss head's statistics where they are most easily lost: rows that are sure of their target, under large logits.

Each row of the hidden states has one element, so that every logit is a single product and exact in f32. What is left of the
tolerance, with u = 2^-24, s the sum of exp(logit - largest) and o = s - 1 what the other words bring to it:
  the largest word's own term is exp(0) = 1, without an error;
  the others' terms are off by 2^-22 for the exponential and by 2 u |x| log2 e for its argument x = logit - largest, at most 58 of
  log2 e here: 4 u + 2 * 58 u of o, with 12 u for expf where parts of the vocabulary are joined;
  s is rounded by u at each addition on its way: 16 + 3 within half a tile, at most 13 joins of parts;
  the logarithm is off by 2 u of itself and log s <= o.
A loss below zero, or a sum below one, is wrong whatever its size.
"""
import numpy as np
import pytest

import oxidizr_b200 as ox

gpu = pytest.mark.gpu
NAMES = {"f32": ox.F32, "bf16": ox.BF16, "f16": ox.F16}
U = 2.0 ** -24


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [16, 40, 300])  # the path for a handful of rows, and two sizes of the tiles'
@pytest.mark.parametrize("gap", [8.0, 20.0])  # of the target's logit to the next
def test_losses_of_sure_rows(dtype, rows, gap):
    import torch
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    hidden, vocab = 64, 3000
    rng = np.random.default_rng(rows + int(gap))
    top = np.linspace(50.0, 200.0, hidden)  # the largest logit of the rows that look at this column
    w = top - gap - rng.random((vocab, hidden)) * (40.0 - gap)
    targets_of = rng.choice(vocab, hidden, replace=False)
    w[targets_of, np.arange(hidden)] = top
    d_w = torch.from_numpy(w).cuda().to(t)
    column = np.arange(rows) % hidden
    x = np.zeros((rows, hidden))
    x[np.arange(rows), column] = rng.choice([0.75, 1.0, 1.25], rows)
    d_x = torch.from_numpy(x).cuda().to(t)
    targets = targets_of[column]
    d_t = torch.from_numpy(targets).cuda()
    logits = d_x.double().cpu().numpy()[np.arange(rows), column][:, None] * d_w.double().cpu().numpy()[:, column].T
    if dtype == "f32":  # three parts of eight bits each: products of up to 26 bits are rounded once
        logits = logits.astype(np.float32).astype(np.float64)
    assert np.array_equal(logits, logits.astype(np.float32))
    m = logits.max(1)
    assert np.array_equal(logits.argmax(1), targets)
    others = np.exp(logits - m[:, None])
    others[np.arange(rows), targets] = 0.0
    o = others.sum(1)
    tol = U * (32 * (1 + o) + (4 + 2 * 58 + 12 + 2) * o)
    if dtype == "f32":  # the six products that make a logit leave 2^-22 of it
        tol = tol + 4 * U * m
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype])
    loss, stats, totals = torch.empty(rows, device="cuda"), torch.empty(rows, 2, device="cuda"), torch.empty(2, device="cuda")
    torch.cuda.synchronize()
    h.loss(rows, d_x.data_ptr(), d_w.data_ptr(), d_t.data_ptr(), row_loss=loss.data_ptr(), row_stats=stats.data_ptr(), totals=totals.data_ptr())
    torch.cuda.synchronize()
    got, st = loss.double().cpu().numpy(), stats.double().cpu().numpy()
    assert np.all(st[:, 1] >= 1.0), st[:, 1].min()
    assert np.all(got >= 0.0), got.min()
    if dtype != "f32":
        assert np.array_equal(st[:, 0], m)
    bad = ~(np.abs(st[:, 1] - (1.0 + o)) <= tol)
    assert not bad.any(), (int(bad.sum()), (np.abs(st[:, 1] - (1.0 + o)) / tol).max())
    bad = ~(np.abs(got - np.log1p(o)) <= tol)
    assert not bad.any(), (int(bad.sum()), (np.abs(got - np.log1p(o)) / tol).max())
    assert abs(float(totals[0]) - np.log1p(o).sum()) <= tol.sum() + U * rows
    h.destroy()


def cut_steps(X, W, t, run):
    """What an accumulator of f32 that is cut, not rounded, at each 16 of K may lose of every row's logit of its target, the sums begun
    anew each `run` steps of 64: (at most, on the mean) - a whole and a half step of the accumulator after each addition."""
    most = np.zeros(len(X))
    at = np.zeros(len(X))
    for k in range(0, X.shape[1], 16):
        if k % (64 * run) == 0:
            at = np.zeros(len(X))
        at = at + (X[:, k:k + 16] * W[t, k:k + 16]).sum(1)
        most += np.exp2(np.floor(np.log2(np.abs(at))) - 23)
    return most, most / 2


@gpu
@pytest.mark.parametrize("dtype, run", [("bf16", 4), ("f16", 4), ("f32", 2)])
@pytest.mark.parametrize("hidden", [512, 2048])
def test_long_sums_keep_their_digits(dtype, run, hidden):
    """Logits near 40 whose products are all positive, beside a word whose logit, 46, is a single product: the loss is the
    difference, and takes over whole what the sum of the products loses. 512 of K stay in one accumulator of 16-bit operands."""
    import torch
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    rows, vocab, words = 512, 1000, 50
    rng = np.random.default_rng(hidden)
    x = rng.uniform(0.5, 1.5, (rows, hidden))
    w = rng.uniform(-0.01, 0.01, (vocab, hidden))
    w[:words] = rng.uniform(0.0, 80.0 / hidden, (words, hidden))
    w[:, 0] = 0.0
    w[words] = 0.0
    x[:, 0], w[words, 0] = 1.0, 46.0
    d_x, d_w = torch.from_numpy(x).cuda().to(t), torch.from_numpy(w).cuda().to(t)
    targets = rng.integers(0, words, rows)
    d_t = torch.from_numpy(targets).cuda()
    X, W = d_x.double().cpu().numpy(), d_w.double().cpu().numpy()
    logits = X @ W.T
    m = logits.max(1)
    want = np.log(np.exp(logits - m[:, None]).sum(1)) + m - logits[np.arange(rows), targets]
    assert np.all(m == 46.0) and want.min() > 1.0
    if dtype != "f32" and hidden <= 512:
        run = 8
    most, mean = cut_steps(X, W, targets, run)
    if dtype == "f32":
        # five more products of the parts stand in a run before the largest: below 2^-6 of it together, cut at the same places, and
        # what the six products leave out is below 3 * 2^-24 of the sum
        most, mean = most * (1 + 2.0 ** -6) + 3 * U * 60, mean * (1 + 2.0 ** -6) + 3 * U * 60
    # runs are joined by rounded additions, U each of a sum below 64; the other terms of the loss as above
    joins = hidden // 64 // run
    if dtype == "f16":
        # a product of two f16 has 22 bits (of two bf16 16). Here it is below 1.5 * 80 / hidden < 2^-2 (hidden 512) and its last bit
        # 2^-21 of its first, while the sum's step is 2^-23 of a sum that passes 1 after a few instructions: bits of every product lie below
        # the step, and each of an instruction's 16 products may be cut by up to a step as the accumulator is: 17 steps at most,
        # half of them on the mean
        most, mean = 17 * most, 17 * mean
    most, rest = most + joins * 64 * U, 48 * U
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype])
    loss, totals = torch.empty(rows, device="cuda"), torch.empty(2, device="cuda")
    torch.cuda.synchronize()
    h.loss(rows, d_x.data_ptr(), d_w.data_ptr(), d_t.data_ptr(), row_loss=loss.data_ptr(), totals=totals.data_ptr())
    torch.cuda.synchronize()
    off = loss.double().cpu().numpy() - want
    assert np.all(np.abs(off) <= most + rest), (np.abs(off) / (most + rest)).max()
    # the cuts are spread evenly over a step: of 512 rows the mean is known to a few hundredths; 1.3 leaves room and is well below the
    # 2 of runs twice as long
    assert abs(off.mean()) <= 1.3 * mean.mean() + 8 * U, (off.mean(), mean.mean())
    assert abs(float(totals[0]) - want.sum()) <= rows * (1.3 * mean.mean() + 8 * U) + U * want.sum()
    h.destroy()
