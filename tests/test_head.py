"""The loss head - softmax cross entropy over a vocabulary taken in pieces, with its gradients - against the definition in 64 bits.

Tolerances, with u = 2^-24 and sums of f32 products held to one step of f32 (2u) per addition, as a matrix unit may cut where an
adder rounds:
  logits    |dl| <= E = (H + 8) 2u max_v sum_h |x||w|          (the products themselves: exact, or within 3 x 2u)
  sums      s is off by r = E + (1024 + 16) 2u relatively: exponentials of arguments off by E, at most 256 + vocab / 64 / 32 + 5
            additions in a chain (the cases have vocab below 60000) and a few roundings of exp
  loss      |d loss| <= 2E + r + 4u (|m| + |l_t| + |log s|)
  g         |dg| <= |w| p (E + r + 8u) + |w| 4u [v = t]  and one rounding to the type: half a step of |g|; f16 is scaled so that the
            largest weight times one stays normal, and loses 2^-25 2^-13 max|w| at most below its normal range. The exponential that
        16-bit operands use flushes results below 2^-126, the smallest normal f32, to zero: 2^-126 |w| (s is one or more)
  d_hidden  scale (sum_v |dg||W| + (V + 64) 2u sum_v |g||W|) and half a step of the result
  d_weight  scale (sum_i |dg||X| + (N + 64) 2u sum_i |g||X|) and half a step of the result; g is not rounded to 16 bits when
            d_weight is f32 (three pieces of 8 bits or more: 2u)
Half a step is eps / 2 of the type relative to the value.
"""
import math

import numpy as np
import pytest

import oxidizr_b200 as ox

gpu = pytest.mark.gpu
NAMES = {"f32": ox.F32, "bf16": ox.BF16, "f16": ox.F16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -140, "bf16": 2.0 ** -125, "f16": 2.0 ** -24}
U = 2.0 ** -24


def torch_type(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


# ------------------------------------------------------------------ refusals, without a GPU
@pytest.mark.parametrize("kw, text", [
    (dict(max_rows=0), "max_rows 0 is outside"), (dict(max_rows=1 << 31), "max_rows 2147483648 is outside"),
    (dict(vocab=0), "vocab 0 is outside"), (dict(vocab=1 << 31), "vocab 2147483648 is outside"),
    (dict(hidden=0), "hidden 0 is outside"), (dict(hidden=(1 << 20) + 1), "hidden 1048577 is outside"),
    (dict(dtype=5, grad_dtype=5), "dtype 5 is none of"), (dict(dtype=ox.BF16, grad_dtype=ox.F16), "grad_dtype 2 is neither"),
    (dict(dtype=ox.F32, grad_dtype=ox.BF16), "grad_dtype 1 is neither"), (dict(device=-1), "device -1"),
])
def test_descriptions_that_cannot_work_are_refused(kw, text):
    with pytest.raises(ox.OxzError, match="OXZ_ERR_INVALID") as e:
        ox.LossHead(**{**dict(vocab=10, hidden=8, max_rows=4, allocate=False), **kw})
    assert text in e.value.message


def test_calls_are_refused_before_they_reach_the_device():
    h = ox.LossHead(10, 8, 4, dtype=ox.BF16, allocate=False)
    p = 1 << 20  # an address that is only looked at
    ok = dict(rows=2, hidden=p, weight=p, targets=p)
    grads = dict(ok, d_hidden=p, d_weight=p)
    for call, text in (
            (lambda: h.loss(**dict(ok, hidden=None)), "null argument"), (lambda: h.loss(**dict(ok, weight=None)), "null argument"),
            (lambda: h.loss(**dict(ok, targets=None)), "null argument"), (lambda: h.loss(**dict(ok, rows=5)), "5 rows, the handle was made for 4"),
            (lambda: h.loss(**ok, hidden_stride=7), "strides 7"), (lambda: h.loss(**dict(ok, hidden=p + 1)), "not aligned to its element"),
            (lambda: h.loss(**dict(ok, targets=p + 4)), "not aligned to its element"), (lambda: h.loss(**ok, loss_mask=p + 2), "not aligned to its element"),
            (lambda: h.loss(**ok, row_loss=p + 2), "not aligned to its element"), (lambda: h.loss(**ok, row_stats=p + 4), "not aligned to its element"),
            (lambda: h.loss(**ok, totals=p + 1), "not aligned to its element"), (lambda: h.loss(**dict(ok, weight=p + 8)), "aligned to 16 bytes"),
            (lambda: h.loss_and_grads(**ok), "neither d_hidden nor d_weight"), (lambda: h.loss_and_grads(**dict(grads, d_weight=p + 8)), "aligned to 16 bytes"),
            (lambda: h.loss_and_grads(**dict(grads, d_hidden=p + 1)), "not aligned to its element"), (lambda: h.loss_and_grads(**grads, d_hidden_stride=3), "strides"),
            (lambda: h.loss_and_grads(**grads, grad_scale=float("inf")), "grad_scale inf"), (lambda: h.loss_and_grads(**grads, grad_scale=1e39), "not a finite f32"),
            (lambda: h.grads(**grads, row_stats=None), "need the rows' statistics")):
        with pytest.raises(ox.OxzError, match="OXZ_ERR_INVALID") as err:
            call()
        assert text in err.value.message, err.value.message
    with pytest.raises(ox.OxzError, match="OXZ_ERR_STATE"):
        h.loss(**ok)
    import torch
    if not torch.cuda.is_available():
        with pytest.raises(ox.OxzError, match="OXZ_ERR_CUDA"):
            h.alloc()
    h.destroy()


# ------------------------------------------------------------------ on the GPU
class Problem:
    """Inputs of one batch on the GPU and the results in 64 bits with their tolerances."""

    def __init__(self, dtype, rows, hidden, vocab, mask=None, seed=0, grad=None, gap=0, sure=True, logit=1.0):
        import torch
        self.dtype, self.grad, self.N, self.H, self.V = dtype, grad or dtype, rows, hidden, vocab
        rng = np.random.default_rng(seed + 1000 * rows + vocab)
        t = torch_type(dtype)
        self.targets = rng.integers(0, vocab, rows)
        w = rng.standard_normal((vocab, hidden)) * 0.05 * logit
        x = rng.standard_normal((rows, hidden))
        if sure and rows:  # some rows know their target
            lean = rng.random((rows, 1)) * 20.0 / max(1.0, 0.05 * math.sqrt(hidden))
            x = x + lean * w[self.targets] / logit
        if mask in ("outside", "both"):
            bad = rng.random(rows) < 0.3
            self.targets[bad] = rng.choice([-1, -100, vocab, vocab + 3, 2 ** 40], int(bad.sum()))
        self.mask = None
        if mask in ("half", "both"):
            self.mask = (rng.random(rows) < 0.5).astype(np.float32)
        elif mask == "none":
            self.mask = np.zeros(rows, np.float32)
        elif mask == "last":
            self.mask = np.zeros(rows, np.float32)
            self.mask[-1] = 1.0
        elif mask == "weights":
            self.mask = (rng.random(rows) * 3.0 * (rng.random(rows) < 0.8)).astype(np.float32)
        self.w_row = np.where((self.targets >= 0) & (self.targets < vocab), 1.0 if self.mask is None else self.mask.astype(np.float64), 0.0)
        self.scored = self.w_row != 0
        self.stride = hidden + gap
        wide = torch.full((rows, self.stride), float("nan"), device="cuda", dtype=t)
        wide[:, :hidden] = torch.from_numpy(x).cuda().to(t)
        self.X = wide[:, :hidden].double().cpu().numpy()
        wide[torch.from_numpy(~self.scored).cuda()] = float("nan")  # rows that take no part may hold anything
        self.d_x = wide
        self.d_w = torch.from_numpy(w).cuda().to(t)
        self.W = self.d_w.double().cpu().numpy()
        self.d_t = torch.from_numpy(self.targets).cuda()
        self.d_m = torch.from_numpy(self.mask).cuda() if self.mask is not None else None

    def solve(self, scale=1.0, before=None):
        X, W, w, on = self.X, self.W, self.w_row[:, None], self.scored
        N, H, V = self.N, self.H, self.V
        t = np.where(on, self.targets, 0)
        l = X @ W.T
        mags = np.abs(X) @ np.abs(W).T
        E = (H + 8) * 2 * U * mags.max(1, initial=0.0)
        m = l.max(1, initial=-np.inf) if N else np.zeros(0)
        e = np.exp(l - m[:, None])
        s = e.sum(1)
        lt = l[np.arange(N), t]
        r = E + 1040 * 2 * U
        self.loss = np.where(on, np.log(s) - (lt - m), 0.0)
        self.loss_tol = np.where(on, 2 * E + r + 4 * U * (np.abs(m) + np.abs(lt) + np.abs(np.log(s))), 0.0)
        self.stats = np.where(on[:, None], np.stack([m, s], 1), 0.0)
        self.stats_tol = np.where(on[:, None], np.stack([E + U * np.abs(m), s * (r + E)], 1), 0.0)
        self.totals = np.array([np.sum(self.loss * self.w_row), np.sum(self.w_row)])
        self.totals_tol = np.array([np.sum(self.loss_tol * np.abs(self.w_row)), 0.0]) + 2 * U * np.abs(self.totals)
        p = e / s[:, None]
        y = np.zeros_like(p)
        y[np.arange(N), t] = 1.0
        g = np.where(on[:, None], w * (p - y), 0.0)
        dg = np.where(on[:, None], np.abs(w) * (p * (E + r + 8 * U)[:, None] + 4 * U * y), 0.0)
        top = np.abs(self.w_row).max(initial=0.0)
        low = {"f16": 2.0 ** -38 * top, "bf16": 2.0 ** -126 * top, "f32": 2.0 ** -133}[self.dtype]
        dg_t = dg + HALF_STEP[self.dtype] * np.abs(g) + low * on[:, None]
        dg_w = dg + 2 * U * np.abs(g) + low * on[:, None] if self.grad == "f32" else dg_t
        c = abs(scale)
        Xs = np.where(on[:, None], X, 0.0)
        self.d_hidden = scale * (g @ W)
        self.d_hidden_tol = c * (dg_t @ np.abs(W) + (V + 64) * 2 * U * (np.abs(g) @ np.abs(W))) * (1 + 4 * U) + TINY[self.dtype]
        self.d_hidden_tol += HALF_STEP[self.dtype] * (np.abs(self.d_hidden) + self.d_hidden_tol)
        self.d_hidden_tol[~on] = 0.0
        self.d_weight = scale * (g.T @ Xs) + (0.0 if before is None else before)
        mag = c * (np.abs(g).T @ np.abs(Xs))
        self.d_weight_tol = c * (dg_w.T @ np.abs(Xs)) + (N + 64) * 2 * U * mag + 4 * U * (mag + (0.0 if before is None else np.abs(before))) + TINY[self.grad]
        self.d_weight_tol += HALF_STEP[self.grad] * (np.abs(self.d_weight) + self.d_weight_tol)
        return self

    def batch(self):
        return dict(rows=self.N, hidden=self.d_x.data_ptr() or 16, hidden_stride=self.stride, weight=self.d_w.data_ptr(),
                    targets=self.d_t.data_ptr() or 16, loss_mask=self.d_m.data_ptr() if self.d_m is not None and self.N else None)

    def outputs(self, gap=0, before=None):
        import torch
        o = dict(row_loss=torch.full((self.N,), 7.0, device="cuda"), row_stats=torch.full((self.N, 2), 7.0, device="cuda"),
                 totals=torch.full((2,), 7.0, device="cuda"),
                 d_hidden=torch.full((self.N, self.H + gap), 7.0, device="cuda", dtype=torch_type(self.dtype)),
                 d_weight=torch.full((self.V, self.H), float("nan"), device="cuda", dtype=torch_type(self.grad)))
        if before is not None:
            o["d_weight"].copy_(before)
        torch.cuda.synchronize()
        return o

    def check(self, o, names):
        for n in names:
            got = o[n].double().cpu().numpy()
            if n == "d_hidden":
                assert np.all(got[:, self.H:] == 7.0), "the elements between rows are not the operator's"
                got = got[:, :self.H]
            want, tol = {"row_loss": (self.loss, self.loss_tol), "row_stats": (self.stats, self.stats_tol), "totals": (self.totals, self.totals_tol),
                         "d_hidden": (self.d_hidden, self.d_hidden_tol), "d_weight": (self.d_weight, self.d_weight_tol)}[n]
            bad = ~(np.abs(got - want) <= tol)
            assert not bad.any(), (n, int(bad.sum()), got.shape, np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4], np.broadcast_to(tol, got.shape)[bad][:4])


def ptrs(o):
    return {k: v.data_ptr() or None for k, v in o.items()}


SHAPES = [(1, 8, 1), (1, 1, 2), (3, 7, 5), (17, 64, 100), (64, 33, 257), (130, 72, 1000), (257, 200, 515), (128, 256, 256), (300, 512, 2053), (512, 64, 4096)]


@gpu
@pytest.mark.parametrize("dtype, grad", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rows, hidden, vocab", SHAPES)
@pytest.mark.parametrize("mask", [None, "both"])
def test_loss_and_gradients(dtype, grad, rows, hidden, vocab, mask):
    import torch
    pr = Problem(dtype, rows, hidden, vocab, mask, grad=grad, gap=0 if mask is None else 3).solve(scale=0.125)
    h = ox.LossHead(vocab, hidden, rows + 3, dtype=NAMES[dtype], grad_dtype=NAMES[grad])
    gap = 0 if mask is None else 5
    o = pr.outputs(gap)
    h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.125, d_hidden_stride=hidden + gap)
    torch.cuda.synchronize()
    pr.check(o, ("row_loss", "row_stats", "totals", "d_hidden", "d_weight"))
    # the same again on another stream gives the same bits; so do the two calls, and one gradient without the other
    side = torch.cuda.Stream().cuda_stream
    for how in ("again", "apart", "hidden", "weight"):
        q = pr.outputs(gap)
        wanted = {k: v for k, v in ptrs(q).items() if not (how == "hidden" and k == "d_weight") and not (how == "weight" and k == "d_hidden")}
        if how == "apart":
            h.loss(**pr.batch(), row_loss=wanted["row_loss"], row_stats=wanted["row_stats"], totals=wanted["totals"], stream=side)
            h.grads(**pr.batch(), row_stats=wanted["row_stats"], d_hidden=wanted["d_hidden"], d_weight=wanted["d_weight"], grad_scale=0.125,
                    d_hidden_stride=hidden + gap, stream=side)
        else:
            h.loss_and_grads(**pr.batch(), **wanted, grad_scale=0.125, d_hidden_stride=hidden + gap, stream=side)
        torch.cuda.synchronize()
        for k in o:
            if k in wanted:
                assert torch.equal(o[k], q[k]), (how, k)
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("mask", ["half", "none", "last", "weights", "outside"])
def test_masks(dtype, mask):
    import torch
    pr = Problem(dtype, 200, 96, 700, mask, seed=3).solve(scale=2.0)
    h = ox.LossHead(700, 96, 200, dtype=NAMES[dtype])
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=2.0)
    torch.cuda.synchronize()
    pr.check(o, o)
    if mask == "none":
        assert not o["d_weight"].any() and not o["d_hidden"].any() and not o["totals"].any()
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype, grad", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("rows, hidden, vocab, pieces", [(150, 72, 1500, 3), (40, 200, 1029, 5), (700, 64, 1024, 2), (9, 8, 60000, 1)])
def test_pieces_and_accumulation(dtype, grad, rows, hidden, vocab, pieces):
    import torch
    rng = np.random.default_rng(8)
    before = torch.from_numpy(rng.standard_normal((vocab, hidden)) * 0.01).cuda().to(torch_type(grad))
    pr = Problem(dtype, rows, hidden, vocab, "half", seed=1, grad=grad).solve(scale=1.0, before=before.double().cpu().numpy())
    size = 4 if dtype == "f32" else 2
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype], grad_dtype=NAMES[grad], piece_bytes=max(1, rows * size * vocab // pieces))
    o = pr.outputs(before=before)
    h.loss_and_grads(**pr.batch(), **ptrs(o), accumulate=True)
    torch.cuda.synchronize()
    pr.check(o, o)
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_rows(dtype):
    import torch
    pr = Problem(dtype, 0, 40, 300)
    h = ox.LossHead(300, 40, 5, dtype=NAMES[dtype])
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o))
    torch.cuda.synchronize()
    assert not o["d_weight"].any() and not o["totals"].any()
    kept = torch.randn(300, 40, device="cuda").to(torch_type(dtype))
    o["d_weight"].copy_(kept)
    torch.cuda.synchronize()
    h.loss_and_grads(**pr.batch(), **ptrs(o), accumulate=True)
    torch.cuda.synchronize()
    assert torch.equal(o["d_weight"], kept)
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_large_logits_and_words_that_cannot_be(dtype):
    """Logits of thousands overflow no exponential; a word whose logit is -inf everywhere takes no part in the loss; a NaN stays in its row."""
    import torch
    pr = Problem(dtype, 33, 64, 500, logit=200.0, sure=False, seed=5).solve()
    h = ox.LossHead(500, 64, 33, dtype=NAMES[dtype])
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o))
    torch.cuda.synchronize()
    assert np.abs(pr.stats[:, 0]).max() > 100
    pr.check(o, o)
    # hidden states above zero, and a word with weights of -inf: its logits are -inf, and the loss is that of the other words
    pr = Problem(dtype, 20, 64, 500, seed=6, sure=False)
    pr.d_x.abs_().add_(0.01)
    pr.X = pr.d_x.double().cpu().numpy()
    pr.targets[:] = np.where(pr.targets == 77, 78, pr.targets)
    pr.d_t.copy_(torch.from_numpy(pr.targets))
    pr.W[77] = 0.0
    keep = np.arange(500) != 77
    l = pr.X @ pr.W.T
    lse = np.log(np.exp(l[:, keep]).sum(1))
    pr.solve()
    pr.d_w[77] = float("-inf")
    o = pr.outputs()
    h.loss(**pr.batch(), **{k: v for k, v in ptrs(o).items() if k in ("row_loss", "row_stats", "totals")})
    torch.cuda.synchronize()
    got = o["row_loss"].double().cpu().numpy()
    assert np.all(np.abs(got - (lse - l[np.arange(20), pr.targets])) <= pr.loss_tol)
    # a NaN in a scored row makes that row's loss NaN and nobody else's
    pr = Problem(dtype, 20, 64, 500, seed=7).solve()
    pr.d_x[4, 3] = float("nan")
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o))
    torch.cuda.synchronize()
    others = np.arange(20) != 4
    assert math.isnan(float(o["row_loss"][4])) and math.isnan(float(o["totals"][0])) and bool(torch.isnan(o["d_hidden"][4]).all())
    assert np.all(np.abs(o["row_loss"].double().cpu().numpy() - pr.loss)[others] <= pr.loss_tol[others])
    assert np.all(np.abs(o["d_hidden"].double().cpu().numpy() - pr.d_hidden)[others] <= pr.d_hidden_tol[others])
    h.destroy()


@gpu
def test_gradients_agree_with_differences():
    import torch
    N, H, V = 7, 24, 90
    pr = Problem("f32", N, H, V, "weights", seed=11).solve()
    h = ox.LossHead(V, H, N, dtype=ox.F32)
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o))
    torch.cuda.synchronize()

    def value(x, w):  # sum of mask * loss over the rows, added in 64 bits
        rl = torch.empty(N, device="cuda")
        torch.cuda.synchronize()
        h.loss(**dict(pr.batch(), hidden=x.data_ptr(), hidden_stride=H, weight=w.data_ptr()), row_loss=rl.data_ptr())
        torch.cuda.synchronize()
        return float((rl.double().cpu() * torch.from_numpy(pr.w_row)).sum())
    step = 2.0 ** -5
    x0, w0 = pr.d_x.clone(), pr.d_w.clone()
    x0[torch.from_numpy(~pr.scored).cuda()] = 0.0
    # a difference is off by the losses' tolerance over the step, and by step^2 / 6 times the third derivative: for a softmax below
    # 2 |a|^3 with a the change of the logits per unit
    noise = 2 * float(pr.totals_tol[0] + np.sum(pr.loss_tol * np.abs(pr.w_row))) / (2 * step)
    third = lambda a: step ** 2 / 6 * 2 * np.sum(np.abs(pr.w_row)) * np.abs(a).max() ** 3  # noqa: E731
    for v, k in ((0, 0), (int(pr.targets[0]), 5), (V - 1, H - 1), (int(pr.targets[3]), 17)):
        up, down = w0.clone(), w0.clone()
        up[v, k] += step
        down[v, k] -= step
        d = (value(x0, up) - value(x0, down)) / (2 * step)
        assert abs(d - float(o["d_weight"][v, k])) <= noise + third(pr.X[:, k]) + 1e-5
    for i in np.where(pr.scored)[0][:4]:
        up, down = x0.clone(), x0.clone()
        up[i, 3] += step
        down[i, 3] -= step
        d = (value(up, w0) - value(down, w0)) / (2 * step)
        assert abs(d - float(o["d_hidden"][i, 3])) <= noise + third(pr.W[:, 3]) + 1e-5
    h.destroy()


@gpu
def test_captured_calls_replay_on_new_values():
    import torch
    h = ox.LossHead(900, 128, 260, dtype=ox.BF16)
    pr = Problem("bf16", 260, 128, 900, "half", seed=20)
    o = pr.outputs()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.5, stream=s.cuda_stream)
    for seed in (21, 22):
        new = Problem("bf16", 260, 128, 900, "half", seed=seed).solve(scale=0.5)
        for to, src in ((pr.d_x, new.d_x), (pr.d_w, new.d_w), (pr.d_t, new.d_t), (pr.d_m, new.d_m)):
            to.copy_(src)
        g.replay()
        torch.cuda.synchronize()
        new.check(o, o)
    del g
    h.destroy()


@gpu
def test_one_handle_serves_batches_of_every_size():
    """What an earlier, larger batch left in the workspace is not seen by a smaller one."""
    import torch
    h = ox.LossHead(650, 72, 400, dtype=ox.BF16)
    for rows, mask in ((400, None), (1, None), (129, "half"), (400, "none"), (37, None), (256, "last"), (399, "both")):
        pr = Problem("bf16", rows, 72, 650, mask, seed=rows).solve()
        o = pr.outputs()
        h.loss_and_grads(**pr.batch(), **ptrs(o))
        torch.cuda.synchronize()
        pr.check(o, o)
        bad = Problem("bf16", 400, 72, 650, seed=9)  # and a batch of NaN in between leaves none behind
        bad.d_x.fill_(float("nan"))
        q = bad.outputs()
        h.loss_and_grads(**bad.batch(), **ptrs(q))
        torch.cuda.synchronize()
        assert bool(torch.isnan(q["d_weight"]).all())
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype, grad", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rows, hidden, vocab, mask, gap", [
    (1, 2056, 700, None, 0), (4, 64, 3000, None, 0), (5, 130, 1111, "half", 6), (8, 128, 257, "weights", 8), (9, 96, 5000, "both", 0), (13, 1500, 900, None, 0),
    (16, 1024, 2100, "half", 16), (16, 40, 33, None, 0), (16, 16, 1, None, 0), (12, 3, 4100, "weights", 1), (16, 2048, 3, None, 0)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_a_handful_of_rows(dtype, grad, rows, hidden, vocab, mask, gap, accumulate):
    """Up to 16 rows, on and off 16-byte bounds, short rows that several threads share, one word, more rows than words."""
    import torch
    rng = np.random.default_rng(8)
    before = torch.from_numpy(rng.standard_normal((vocab, hidden)) * 0.01).cuda().to(torch_type(grad)) if accumulate else None
    pr = Problem(dtype, rows, hidden, vocab, mask, seed=rows, grad=grad, gap=gap).solve(scale=0.5, before=before.double().cpu().numpy() if accumulate else None)
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype], grad_dtype=NAMES[grad])
    o = pr.outputs(before=before)
    h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.5, accumulate=accumulate)
    torch.cuda.synchronize()
    pr.check(o, o)
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype, grad", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("rows, hidden, vocab", [(8, 345, 4000), (9, 345, 4000), (16, 345, 4000), (9, 345, 3000), (16, 517, 2500)])
def test_a_handful_of_odd_rows_over_a_larger_weight(dtype, grad, rows, hidden, vocab):
    """Rows off 16-byte bounds on both sides of what goes by streams of the weight and by tiles; losses alone, then their gradients."""
    import torch
    pr = Problem(dtype, rows, hidden, vocab, "weights", seed=rows, grad=grad).solve(scale=0.5)
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype], grad_dtype=NAMES[grad])
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.5)
    torch.cuda.synchronize()
    pr.check(o, o)
    q = pr.outputs()
    h.loss(**pr.batch(), row_loss=q["row_loss"].data_ptr(), row_stats=q["row_stats"].data_ptr(), totals=q["totals"].data_ptr())
    h.grads(**pr.batch(), row_stats=q["row_stats"].data_ptr(), d_hidden=q["d_hidden"].data_ptr(), d_weight=q["d_weight"].data_ptr(), grad_scale=0.5)
    torch.cuda.synchronize()
    for k in o:
        assert torch.equal(o[k], q[k]), k
    h.destroy()


@gpu
@pytest.mark.parametrize("dtype, grad", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rows, hidden, vocab, piece_bytes", [(40, 1024, 1500, 0), (600, 1040, 2500, 0), (600, 1040, 2500, 4 << 20), (1300, 264, 3000, 5 << 20),
                                                             (2100, 72, 5000, 0), (1025, 512, 700, 1)])
def test_many_tiles(dtype, grad, rows, hidden, vocab, piece_bytes):
    """Several tiles each way: kept logits and logits formed again, d_hidden cut in shares and not, more rows than one block lists."""
    import torch
    pr = Problem(dtype, rows, hidden, vocab, "half", seed=rows, grad=grad).solve(scale=0.5)
    h = ox.LossHead(vocab, hidden, rows, dtype=NAMES[dtype], grad_dtype=NAMES[grad], piece_bytes=piece_bytes)
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o), grad_scale=0.5)
    torch.cuda.synchronize()
    pr.check(o, o)
    q = pr.outputs()
    h.loss(**pr.batch(), row_loss=q["row_loss"].data_ptr(), row_stats=q["row_stats"].data_ptr(), totals=q["totals"].data_ptr())
    h.grads(**pr.batch(), row_stats=q["row_stats"].data_ptr(), d_hidden=q["d_hidden"].data_ptr(), d_weight=q["d_weight"].data_ptr(), grad_scale=0.5)
    torch.cuda.synchronize()
    for k in o:
        assert torch.equal(o[k], q[k]), k
    h.destroy()


@gpu
@pytest.mark.parametrize("rows", [7, 300])
def test_d_hidden_in_place_of_hidden(rows):
    import torch
    pr = Problem("bf16", rows, 136, 500, "half", seed=2).solve()
    h = ox.LossHead(500, 136, rows, dtype=ox.BF16)
    o = pr.outputs()
    h.loss_and_grads(**pr.batch(), **ptrs(o))
    torch.cuda.synchronize()
    x = pr.d_x.clone()
    q = pr.outputs()
    torch.cuda.synchronize()
    h.loss_and_grads(**dict(pr.batch(), hidden=x.data_ptr()), **dict(ptrs(q), d_hidden=x.data_ptr()))
    torch.cuda.synchronize()
    assert torch.equal(x, o["d_hidden"]) and torch.equal(q["d_weight"], o["d_weight"])
    h.destroy()
