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
