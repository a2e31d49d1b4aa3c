"""Forms of the loss head that only certain sizes reach: logits kept because the mask leaves few enough rows, in several pieces;
d_hidden's tiles in whole rounds of all pairs of SMs with a rest that is cut; the widest rows of the path for up to 16 rows and the
first that go by tiles; two threads with a handle each. Tolerances: those of the loss head's other tests."""
import threading

import numpy as np
import pytest

import oxidizr_b200 as ox
from tests.test_head import NAMES, U, HALF_STEP, TINY, Problem, ptrs

gpu = pytest.mark.gpu


def mask_rows(pr, rows):
    """Scores the first `rows` rows that a shuffle of the batch puts first; the others hold NaN and take no part."""
    import torch
    order = np.random.default_rng(rows).permutation(pr.N)
    pr.mask = np.zeros(pr.N, np.float32)
    pr.mask[order[:rows]] = 1.0
    pr.w_row = pr.mask.astype(np.float64)
    pr.scored = pr.w_row != 0
    pr.d_x[torch.from_numpy(~pr.scored).cuda()] = float("nan")
    pr.d_m = torch.from_numpy(pr.mask).cuda()
    return pr


@gpu
@pytest.mark.parametrize("dtype, grad", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32")])
def test_the_mask_decides_whether_the_logits_are_kept(dtype, grad):
    """600 rows of 2560 logits are more than two thirds of 4 MiB hold in f32 (699050); 273 rows fit, 274 do not. One handle
    takes them in turn; at least three pieces of the vocabulary."""
    import torch
    rows, hidden, vocab, budget = 600, 1040, 2500, 4 << 20
    kept_rows = budget // 3 * 2 // 4 // 2560
    assert kept_rows == 273
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype], grad_dtype=NAMES[grad], piece_bytes=budget)
    for scored in (150, kept_rows, kept_rows + 1, 1, kept_rows, rows, 0, 64):
        pr = mask_rows(Problem(dtype, rows, hidden, vocab, None, seed=4, grad=grad), scored).solve(scale=0.5)
        o = pr.outputs()
        h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.5)
        torch.cuda.synchronize()
        pr.check(o, o)
        q = pr.outputs()  # the logits formed again give the same bits
        h.loss(**pr.batch(), row_loss=q["row_loss"].data_ptr(), row_stats=q["row_stats"].data_ptr(), totals=q["totals"].data_ptr())
        h.grads(**pr.batch(), row_stats=q["row_stats"].data_ptr(), d_hidden=q["d_hidden"].data_ptr(), d_weight=q["d_weight"].data_ptr(), grad_scale=0.5)
        torch.cuda.synchronize()
        for k in o:
            assert torch.equal(o[k], q[k]), (scored, k)
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype, grad", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("rows, hidden, vocab, piece_bytes", [(5120, 1024, 600, 0), (5120, 1024, 600, 1), (4700, 1030, 300, 0), (18944, 72, 260, 0)])
def test_whole_rounds_of_d_hidden_and_a_rest(dtype, grad, rows, hidden, vocab, piece_bytes):
    """80 tiles of d_hidden, 95, and 74: with 74 pairs of SMs a whole round and a rest of 6, of 21, and none."""
    import torch
    pr = Problem(dtype, rows, hidden, vocab, None, seed=5, grad=grad).solve(scale=0.5)
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype], grad_dtype=NAMES[grad], piece_bytes=piece_bytes)
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.5)
    torch.cuda.synchronize()
    pr.check(o, o)
    h.destroy()


def fine_tolerance(pr, scale):
    """The gradients' tolerances where G keeps twice the type's digits or more."""
    fine = {"bf16": 2.0 ** -16, "f16": 2.0 ** -21, "f32": 2 * U}[pr.dtype]
    half, tiny = HALF_STEP[pr.dtype], TINY[pr.dtype]
    X, W = np.where(pr.scored[:, None], pr.X, 0.0), pr.W
    l = X @ W.T
    e = np.exp(l - l.max(1, keepdims=True))
    s = e.sum(1, keepdims=True)
    p = e / s
    y = np.zeros_like(p)
    y[np.arange(pr.N), np.where(pr.scored, pr.targets, 0)] = 1.0
    g = np.where(pr.scored[:, None], pr.w_row[:, None] * (p - y), 0.0)
    E = (pr.H + 8) * 2 * U * (np.abs(X) @ np.abs(W).T).max(1, keepdims=True)
    low = {"f16": 2.0 ** -38, "bf16": 2.0 ** -126, "f32": 2.0 ** -133}[pr.dtype] * np.abs(pr.w_row).max()
    dg = np.abs(pr.w_row[:, None]) * (p * (2 * E + 1040 * 2 * U + 8 * U) + 4 * U * y) + fine * np.abs(g) + low
    c = abs(scale)
    dh = c * (dg @ np.abs(W) + (pr.V + 64) * 2 * U * (np.abs(g) @ np.abs(W))) + tiny
    dh += half * (np.abs(pr.d_hidden) + dh)
    dw = c * (dg.T @ np.abs(X) + (pr.N + 64) * 2 * U * (np.abs(g).T @ np.abs(X))) + tiny
    dw += half * (np.abs(pr.d_weight) + dw)
    return dh, dw


# (rows, the widest hidden that goes by streams of the weight, the next): 16-bit rows on 16 bytes, f32 ones, and rows off 16 bytes
BOUNDS = [("bf16", 8, 5760, 5768), ("f16", 16, 2816, 2824), ("bf16", 16, 2816, 2824), ("f32", 4, 5760, 5764), ("f32", 8, 3840, 3844), ("f32", 16, 2432, 2436),
          ("bf16", 4, 14015, 14017), ("f16", 8, 7007, 7009), ("bf16", 16, 3487, 3489), ("f32", 3, 14015, 14017)]


@gpu
@pytest.mark.parametrize("dtype, rows, last, first", BOUNDS)
@pytest.mark.parametrize("over", [False, True])
def test_the_widest_rows_of_a_handful(dtype, rows, last, first, over):
    import torch
    hidden, vocab = first if over else last, 90
    pr = Problem(dtype, rows, hidden, vocab, "weights" if rows > 4 else None, seed=6).solve(scale=0.5)
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype])
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.5)
    torch.cuda.synchronize()
    pr.check(o, o)
    if rows <= 8 and not over:
        dh, dw = fine_tolerance(pr, 0.5)
        assert np.all(np.abs(o["d_hidden"].double().cpu().numpy() - pr.d_hidden)[pr.scored] <= dh[pr.scored])
        assert np.all(np.abs(o["d_weight"].double().cpu().numpy() - pr.d_weight) <= dw)
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows, hidden, vocab, gap", [(9, 1024, 2000, 0), (16, 1024, 2000, 8), (16, 64, 3000, 0), (12, 128, 3000, 0), (8, 512, 2000, 0), (1, 256, 2000, 0),
                                                      (16, 100, 900, 3), (7, 33, 900, 0)])
def test_a_handful_of_rows_keeps_twice_the_digits_of_g(dtype, rows, hidden, vocab, gap):
    import torch
    pr = Problem(dtype, rows, hidden, vocab, "weights" if rows > 1 else None, seed=8, gap=gap).solve(scale=0.5)
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype])
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.5)
    torch.cuda.synchronize()
    pr.check(o, o)
    dh, dw = fine_tolerance(pr, 0.5)
    off = np.abs(o["d_hidden"].double().cpu().numpy() - pr.d_hidden)[pr.scored] / dh[pr.scored]
    assert np.all(off <= 1), off.max()
    off = np.abs(o["d_weight"].double().cpu().numpy() - pr.d_weight) / dw
    assert np.all(off <= 1), off.max()
    h.destroy()


@gpu
@pytest.mark.parametrize("rows", [12, 200])
def test_two_threads_with_a_handle_each(rows):
    import torch
    hidden, vocab = 128, 3000
    problems = [Problem("bf16", rows, hidden, vocab, "half", seed=20 + k) for k in range(2)]
    want, got, errors = [], [None, None], []
    for pr in problems:
        h = ox.LossHead(vocab, hidden, rows)
        o = pr.outputs()
        h.loss_and_grads(**pr.batch(), **ptrs(o))
        torch.cuda.synchronize()
        want.append(o)
        h.destroy()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [pr.outputs() for pr in problems]
    meet = threading.Barrier(2)

    def body(k):
        try:
            torch.cuda.set_device(0)
            meet.wait(timeout=60)
            h = ox.LossHead(vocab, hidden, rows)  # made side by side as well
            for _ in range(20):
                h.loss_and_grads(**problems[k].batch(), **ptrs(outs[k]), stream=streams[k].cuda_stream)
            streams[k].synchronize()
            h.destroy()
            got[k] = outs[k]
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=body, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=120)
    assert not errors, errors
    for w, g in zip(want, got):
        assert all(torch.equal(w[k], g[k]) for k in w)
