"""The token embedding: a scaled lookup and its gradient by sorted tokens, against the definition in 64 bits.

Tolerances: the lookup is one product in f32 and one rounding: half a step of the type, plus 2^-24 for the product. A gradient
element is a sum of k terms in f32 (at most k additions, the factor, the addition to what was there), each off by at most 2^-24
of the sum of magnitudes, and one rounding: half a step of the type of the result.
"""
import math

import numpy as np
import pytest

import oxidizr_b200 as ox

gpu = pytest.mark.gpu
NAMES = {"f32": ox.F32, "bf16": ox.BF16, "f16": ox.F16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -9 * 2, "f16": 2.0 ** -12 * 2}  # torch.finfo(t).eps / 2
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}  # the smallest step


def torch_type(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


# ------------------------------------------------------------------ refusals, without a GPU
@pytest.mark.parametrize("kw, text", [
    (dict(max_tokens=0), "max_tokens 0 is outside"), (dict(max_tokens=1 << 31), "max_tokens 2147483648 is outside"),
    (dict(vocab=0), "vocab 0 is outside"), (dict(vocab=1 << 31), "vocab 2147483648 is outside"),
    (dict(hidden=0), "hidden 0 is outside"), (dict(hidden=(1 << 20) + 1), "hidden 1048577 is outside"),
    (dict(dtype=7, grad_dtype=7), "dtype 7 is none of"), (dict(dtype=ox.BF16, grad_dtype=ox.F16), "grad_dtype 2 is neither"),
    (dict(dtype=ox.F32, grad_dtype=ox.BF16), "grad_dtype 1 is neither"), (dict(scale=float("nan")), "not a finite f32"),
    (dict(scale=1e39), "not a finite f32"), (dict(device=-1), "device -1"),
])
def test_descriptions_that_cannot_work_are_refused(kw, text):
    with pytest.raises(ox.OxzError, match="OXZ_ERR_INVALID") as e:
        ox.TokenEmbedding(**{**dict(vocab=10, hidden=8, max_tokens=4, allocate=False), **kw})
    assert text in e.value.message


def test_calls_are_refused_before_they_reach_the_device():
    e = ox.TokenEmbedding(10, 8, 4, dtype=ox.BF16, allocate=False)
    p = 1 << 20  # an address that is only looked at
    for call, text in (
            (lambda: e.lookup(0, 2, p, p), "null argument"), (lambda: e.lookup(p, 2, 0, p), "null argument"),
            (lambda: e.lookup(p, 2, p, 0), "null argument"), (lambda: e.lookup(p, 5, p, p), "5 tokens, the handle was made for 4"),
            (lambda: e.lookup(p, 2, p, p, out_stride=7), "out_stride 7"), (lambda: e.lookup(p + 4, 2, p, p), "not aligned"),
            (lambda: e.lookup(p, 2, p + 1, p), "not aligned"), (lambda: e.lookup(p, 2, p, p + 1), "not aligned"),
            (lambda: e.grads(0, 2, p, p), "null argument"), (lambda: e.grads(p, 2, 0, p), "null argument"),
            (lambda: e.grads(p, 2, p, 0), "null argument"), (lambda: e.grads(p, 5, p, p), "5 tokens"),
            (lambda: e.grads(p, 2, p, p, d_out_stride=7), "d_out_stride 7"), (lambda: e.grads(p, 2, p + 1, p), "not aligned"),
            (lambda: e.grads(p, 2, p, p + 1), "not aligned")):
        with pytest.raises(ox.OxzError, match="OXZ_ERR_INVALID") as err:
            call()
        assert text in err.value.message
    with pytest.raises(ox.OxzError, match="OXZ_ERR_STATE"):
        e.grads(p, 2, p, p)
    e.lookup(0, 0, 0, 0)  # no tokens: nothing to do, nothing looked at
    e.destroy()
    import torch
    if not torch.cuda.is_available():
        e = ox.TokenEmbedding(10, 8, 4, allocate=False)
        for call in (e.alloc, lambda: e.lookup(p, 2, p, p)):
            with pytest.raises(ox.OxzError, match="OXZ_ERR_CUDA"):
                call()
        e.destroy()


# ------------------------------------------------------------------ on the GPU
def make_ids(kind, n, vocab, rng):
    if kind == "uniform":
        return rng.integers(0, vocab, n)
    if kind == "same":
        return np.full(n, vocab - 1)
    if kind == "zipf":
        return np.minimum(np.floor(np.exp(rng.random(n) * math.log(vocab))).astype(np.int64) - 1, vocab - 1)
    if kind == "two":  # runs that end on and next to the bounds of a warp's chunk
        return np.where(np.arange(n) % 33 < 16, 0, vocab // 2)
    if kind == "outside":
        ids = rng.integers(0, vocab, n)
        ids[::3] = rng.choice([-1, -100, vocab, vocab + 7, 2 ** 40, -2 ** 63], len(ids[::3]))
        return ids
    raise ValueError(kind)


def expected_grads(ids, d_out, vocab, scale):
    """(the sum, the sum of magnitudes, the count of terms) of every element, in 64 bits."""
    H = d_out.shape[1]
    total, mags, count = np.zeros((vocab, H)), np.zeros((vocab, H)), np.zeros((vocab, 1))
    ok = (ids >= 0) & (ids < vocab)
    np.add.at(total, ids[ok], d_out[ok] * scale)
    np.add.at(mags, ids[ok], np.abs(d_out[ok] * scale))
    np.add.at(count, ids[ok], 1)
    return total, mags, count


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n, hidden, vocab, stride", [(1, 8, 1, 0), (1, 1, 5, 0), (17, 512, 1000, 0), (300, 384, 777, 400), (33, 129, 50, 131),
                                                      (5, 2056, 9, 0), (70, 64, 300, 65)])
def test_lookup(dtype, n, hidden, vocab, stride):
    import torch
    rng = np.random.default_rng(n * 7 + hidden)
    scale = 1.0 if n == 1 else 5.65625
    ids = make_ids("outside" if n > 4 else "uniform", n, vocab, rng)
    t = torch_type(dtype)
    table = torch.from_numpy(rng.standard_normal((vocab, hidden)).astype(np.float32)).cuda().to(t)
    out = torch.full((n, stride or hidden), 7.0, device="cuda", dtype=t)
    emb = ox.TokenEmbedding(vocab, hidden, n, dtype=NAMES[dtype], scale=scale, allocate=False)
    d_ids = torch.from_numpy(ids.astype(np.int64)).cuda()
    torch.cuda.synchronize()
    emb.lookup(d_ids.data_ptr(), n, table.data_ptr(), out.data_ptr(), out_stride=stride)
    torch.cuda.synchronize()
    ok = (ids >= 0) & (ids < vocab)
    want = np.where(ok[:, None], table.double().cpu().numpy()[np.where(ok, ids, 0)] * scale, 0.0)
    got = out.double().cpu().numpy()
    assert np.all(np.abs(got[:, :hidden] - want) <= (HALF_STEP[dtype] + 2.0 ** -24) * np.abs(want) + TINY[dtype])
    if scale == 1.0:
        assert np.array_equal(got[:, :hidden], want)  # a factor of one copies
    assert np.all(got[:, hidden:] == 7.0), "the elements between rows are not the operator's"
    emb.destroy()


CASES = [("uniform", 1, 8, 3), ("uniform", 31, 64, 500), ("same", 16, 8, 4), ("same", 17, 8, 4), ("same", 1000, 384, 7), ("two", 700, 136, 40),
         ("zipf", 2049, 384, 5000), ("zipf", 9000, 72, 1000), ("outside", 333, 129, 60), ("outside", 16, 1, 2), ("uniform", 1024, 33, 512),
         ("zipf", 40000, 16, 300000), ("uniform", 5000, 8, 513), ("same", 20000, 40, 1)]


@gpu
@pytest.mark.parametrize("dtype, grad", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("kind, n, hidden, vocab", CASES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_is_the_sum_over_equal_tokens(dtype, grad, kind, n, hidden, vocab, accumulate):
    import torch
    rng = np.random.default_rng(n + 31 * hidden)
    ids = make_ids(kind, n, vocab, rng)
    scale = 0.37
    d_out = torch.from_numpy(rng.standard_normal((n, hidden)).astype(np.float32)).cuda().to(torch_type(dtype))
    old = torch.from_numpy(rng.standard_normal((vocab, hidden)).astype(np.float32)).cuda().to(torch_type(grad))
    table = old.clone() if accumulate else torch.full_like(old, float("nan"))
    emb = ox.TokenEmbedding(vocab, hidden, n + 5, dtype=NAMES[dtype], grad_dtype=NAMES[grad], scale=scale)
    d_ids = torch.from_numpy(ids.astype(np.int64)).cuda()
    torch.cuda.synchronize()
    emb.grads(d_ids.data_ptr(), n, d_out.data_ptr(), table.data_ptr(), accumulate=accumulate)
    torch.cuda.synchronize()
    got = table.double().cpu().numpy()
    total, mags, count = expected_grads(ids, d_out.double().cpu().numpy(), vocab, np.float64(np.float32(scale)))
    before = old.double().cpu().numpy() if accumulate else np.zeros_like(total)
    want = before + total
    err = HALF_STEP[grad] * np.abs(want) + (count + 3) * 2.0 ** -24 * 1.01 * (mags + np.abs(before)) + TINY[grad]
    assert np.all(np.abs(got - want) <= err), np.max(np.abs(got - want) / err)
    none = np.where(count[:, 0] == 0)[0]
    assert np.array_equal(got[none], before[none]), "rows without a token"
    # the same again, on another stream, gives the same bits
    again = old.clone() if accumulate else torch.full_like(old, 3.0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    emb.grads(d_ids.data_ptr(), n, d_out.data_ptr(), again.data_ptr(), accumulate=accumulate, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(again, table)
    emb.destroy()


@gpu
@pytest.mark.parametrize("n", [1024, 1025, 2113, 4736, 4737, 8129, 8191, 8192, 8193])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_at_the_bounds_of_each_way_to_order_the_tokens(n, accumulate):
    """Whole numbers, whose sums are exact: every token has to reach its row once, at the last count of each sort and the first of the
    next, and where the tokens do not divide evenly among the blocks."""
    import torch
    hidden, vocab = 24, 2500
    rng = np.random.default_rng(n)
    ids = torch.from_numpy(make_ids("uniform", n, vocab, rng).astype(np.int64)).cuda()
    d_out = torch.from_numpy(rng.integers(-4, 5, (n, hidden)).astype(np.float32)).cuda()
    old = torch.from_numpy(rng.integers(-4, 5, (vocab, hidden)).astype(np.float32)).cuda()
    table = old.clone() if accumulate else torch.full_like(old, float("nan"))
    emb = ox.TokenEmbedding(vocab, hidden, n, dtype=ox.F32)
    torch.cuda.synchronize()
    emb.grads(ids.data_ptr(), n, d_out.data_ptr(), table.data_ptr(), accumulate=accumulate)
    torch.cuda.synchronize()
    want = torch.zeros_like(old).index_add_(0, ids, d_out) + (old if accumulate else 0)
    assert torch.equal(table, want)
    emb.destroy()


@gpu
def test_gradient_of_strided_rows_and_of_no_tokens():
    import torch
    n, hidden, vocab = 50, 24, 11
    rng = np.random.default_rng(5)
    ids = rng.integers(0, vocab, n)
    wide = torch.from_numpy(rng.standard_normal((n, 40)).astype(np.float32)).cuda()
    table = torch.full((vocab + 1, hidden), 9.0, device="cuda")
    emb = ox.TokenEmbedding(vocab, hidden, n, dtype=ox.F32)
    d_ids = torch.from_numpy(ids).cuda()
    for first in (0, 1, 4):  # whole 16-byte rows, rows that start between two of them, an offset of one piece
        torch.cuda.synchronize()
        emb.grads(d_ids.data_ptr(), n, wide.data_ptr() + 4 * first, table.data_ptr(), d_out_stride=40)
        torch.cuda.synchronize()
        total, mags, count = expected_grads(ids, wide.double().cpu().numpy()[:, first:first + hidden], vocab, 1.0)
        assert np.all(np.abs(table[:vocab].double().cpu().numpy() - total) <= (count + 4) * 2.0 ** -24 * mags)
    assert torch.all(table[vocab] == 9.0), "the row behind the table"
    kept = table.clone()
    emb.grads(0, 0, 0, table.data_ptr(), accumulate=True)
    torch.cuda.synchronize()
    assert torch.equal(kept, table)
    emb.grads(0, 0, 0, table.data_ptr(), accumulate=False)
    torch.cuda.synchronize()
    assert torch.all(table[:vocab] == 0) and torch.all(table[vocab] == 9.0)
    emb.destroy()


@gpu
def test_gradient_agrees_with_differences():
    import torch
    n, hidden, vocab, scale = 12, 16, 5, 3.0
    rng = np.random.default_rng(9)
    ids = torch.from_numpy(rng.integers(0, vocab, n)).cuda()
    table, c = torch.randn(vocab, hidden, device="cuda"), torch.randn(n, hidden, device="cuda")
    emb = ox.TokenEmbedding(vocab, hidden, n, dtype=ox.F32, scale=scale)
    out, grad = torch.empty(n, hidden, device="cuda"), torch.empty_like(table)

    def value(tab):  # sum of c * lookup(tab), the sum in 64 bits
        torch.cuda.synchronize()
        emb.lookup(ids.data_ptr(), n, tab.data_ptr(), out.data_ptr())
        torch.cuda.synchronize()
        return float((out.double() * c.double()).sum())
    torch.cuda.synchronize()
    emb.grads(ids.data_ptr(), n, c.data_ptr(), grad.data_ptr())
    torch.cuda.synchronize()
    for v, h in ((0, 0), (1, 5), (4, 15), (2, 7)):
        up, down = table.clone(), table.clone()
        up[v, h] += 0.25  # the operator is linear: any step will do
        down[v, h] -= 0.25
        step = float(up[v, h].double() - down[v, h].double())
        # each of at most n terms of `value` is rounded by 2^-24 of itself, twice (product, and the two tables)
        tol = 4 * n * 2.0 ** -24 * scale * float((c.abs().double().max() * (table.abs().double().max() + 1))) / step + 2.0 ** -20
        assert abs((value(up) - value(down)) / step - float(grad[v, h])) <= tol
    emb.destroy()


@gpu
def test_captured_calls_replay_on_new_values():
    import torch
    n, hidden, vocab = 600, 128, 200
    rng = np.random.default_rng(2)
    ids = torch.from_numpy(rng.integers(0, vocab, n)).cuda()
    d_out, table = torch.randn(n, hidden, device="cuda"), torch.randn(vocab, hidden, device="cuda")
    out, grad = torch.zeros(n, hidden, device="cuda"), torch.zeros(vocab, hidden, device="cuda")
    emb = ox.TokenEmbedding(vocab, hidden, n, dtype=ox.F32, scale=2.0)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        emb.lookup(ids.data_ptr(), n, table.data_ptr(), out.data_ptr(), stream=s.cuda_stream)
        emb.grads(ids.data_ptr(), n, d_out.data_ptr(), grad.data_ptr(), stream=s.cuda_stream)
    for seed in (3, 4):
        ids.copy_(torch.from_numpy(np.random.default_rng(seed).integers(0, vocab, n)))
        d_out.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, table[ids] * 2.0)
        total, mags, count = expected_grads(ids.cpu().numpy(), d_out.double().cpu().numpy(), vocab, 2.0)
        assert np.all(np.abs(grad.double().cpu().numpy() - total) <= (count + 4) * 2.0 ** -24 * mags)
    del g
    emb.destroy()


@gpu
def test_the_current_device_is_left_as_it_was():
    import torch
    before = torch.cuda.current_device()
    emb = ox.TokenEmbedding(10, 8, 4)
    emb.destroy()
    assert torch.cuda.current_device() == before
    count = torch.cuda.device_count()
    with pytest.raises(ox.OxzError, match="OXZ_ERR_CUDA"):
        ox.TokenEmbedding(10, 8, 4, device=count + 3)
    assert torch.cuda.current_device() == before
