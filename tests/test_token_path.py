"""The token operators as a training run uses them: loader -> lookup -> a stand-in for the layers -> losses and gradients -> lookup's
gradient into the same tied tensor -> the trainer's half of the step, over the optimizer's own buffers.

The layers between are the identity times two, so the whole gradient of the tied tensor is known: that of the losses by the weight
plus twice that of the losses by the hidden states, scattered to the inputs. Tolerances (u = 2^-24, half a step of bf16 h = 2^-8):
the hidden states are inputs of the losses as they were rounded; an element of the head's gradient is off by h of the sum of magnitudes
for the rounding of G (and 1e-4 of it for logits, exponentials and sums, whose bounds are below that at these sizes), and by h of itself
for its rounding; an element of d_hidden the same, which the lookup's gradient passes on; the sum is rounded once more.
"""
import math

import numpy as np
import pytest

import oxidizr_b200 as ox
from oxidizr_b200 import ffi

gpu = pytest.mark.gpu


def test_the_weight_of_a_micro_batch():
    trainer = ox.LitTrainerStep(ox.TrainerConfig(), ox.DpOptimizer([8], allocate=False))
    assert trainer.loss_weight(64, 4) == 1.0 / 256 and trainer.loss_weight(64, 4, 100) == 0.01
    assert trainer.loss_weight(0, 4) == 0.0 and trainer.loss_weight(64, 4, 0) == 0.0


@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("loss_scale", [None, 1024.0])
def test_a_tied_model_steps_from_the_loaders_tokens(tmp_path, masked, loss_scale):
    import torch
    from oxidizr_b200.interop import device_view, state_views
    vocab, hidden, batch, seq, micro = 300, 64, 2, 40, 2
    rows = batch * seq
    rng = np.random.default_rng(4)
    tokens = rng.integers(0, vocab, size=(batch * micro * 3 + 1) * (seq + 1), dtype=np.uint32)
    path = str(tmp_path / "tokens.bin")
    tokens.astype("<u4").tofile(path)
    loader = ox.LitDataLoader(path, batch, seq)
    if masked:
        loader.with_document_mask(7).with_target_mask(20, [3])
    opt = ox.DpOptimizer([vocab * hidden, 5], [False, True], ox.BF16, ox.BF16)
    weight0 = (rng.standard_normal(vocab * hidden) * 0.3).astype(np.float32)
    opt.import_tensor(ffi.STATE_MASTER, 0, weight0)
    opt.import_tensor(ffi.STATE_WORK, 0, torch.from_numpy(weight0).bfloat16().view(torch.int16).numpy().view(np.uint16))
    stream = torch.cuda.Stream()
    opt.set_stream(stream.cuda_stream)
    scaler = ox.LossScaleConfig(initial=loss_scale) if loss_scale else None
    trainer = ox.LitTrainerStep(ox.TrainerConfig(learning_rate=1e-2, weight_decay=0.0, max_grad_norm=1e9, loss_scale=scaler), opt)
    scale = 8.0
    emb = ox.TokenEmbedding(vocab, hidden, rows, scale=scale)
    head = ox.LossHead(vocab, hidden, rows)
    x = torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16)
    dx, totals = torch.empty_like(x), [torch.empty(2, device="cuda") for _ in range(micro)]
    views = state_views(opt)
    before_work = None
    for step in range(3):
        held = []
        with torch.cuda.stream(stream):
            views["grads"][:vocab * hidden].fill_(float("nan"))  # the step's first micro-batch writes every element of the tensor
            work = views["work"][:vocab * hidden].double().view(vocab, hidden).cpu().numpy()
            scored = None
            if masked:  # the step's scored tokens are known before its first backward: the loader's counts of its micro-batches
                pos = loader.position()
                scored = 0
                for _ in range(micro):
                    loader.next_batch(stream.cuda_stream)
                    stream.synchronize()
                    scored += loader.batch_masks()["scored"]()
                loader.seek(pos)
            weights = []
            for k in range(micro):
                i_ptr, t_ptr, _ = loader.next_batch(stream.cuda_stream)
                mask = loader.batch_masks()["loss_mask"] if masked else None
                trainer.embed(emb, 0, i_ptr, rows, x.data_ptr(), stream=stream.cuda_stream)
                x.mul_(2.0)
                weights.append(trainer.loss_and_grads(head, 0, rows, x.data_ptr(), t_ptr, totals[k].data_ptr(), dx.data_ptr(), micro_batches=micro,
                                                      scored=scored, loss_mask=mask, accumulate=k > 0, stream=stream.cuda_stream))
                dx.mul_(2.0)
                trainer.embed_grads(emb, 0, i_ptr, rows, dx.data_ptr(), accumulate=True, stream=stream.cuda_stream)
                stream.synchronize()
                held.append((device_view(i_ptr, rows * 8, torch.int64).cpu().numpy(), device_view(t_ptr, rows * 8, torch.int64).cpu().numpy(),
                             device_view(mask, rows * 4, torch.float32).double().cpu().numpy() if masked else np.ones(rows), x.double().cpu().numpy()))
            grad = views["grads"][:vocab * hidden].double().view(vocab, hidden).cpu().numpy()
        # the definition in 64 bits
        want, tol, loss = np.zeros((vocab, hidden)), np.zeros((vocab, hidden)), 0.0
        h, ls = 2.0 ** -8, loss_scale or 1.0
        for (ids, targets, w, X), weight in zip(held, weights):
            assert weight == (1.0 / scored if masked else 1.0 / (rows * micro))
            logits = X @ work.T
            m = logits.max(1, keepdims=True)
            e = np.exp(logits - m)
            p = e / e.sum(1, keepdims=True)
            loss += weight * float(np.sum(w * (np.log(e.sum(1)) + m[:, 0] - logits[np.arange(rows), targets])))
            p[np.arange(rows), targets] -= 1.0
            g = p * w[:, None] * weight * ls
            head_grad, head_mag = g.T @ X, np.abs(g).T @ np.abs(X)
            dh, dh_mag = 2 * g @ work, 2 * np.abs(g) @ np.abs(work)
            scatter, scatter_tol = np.zeros_like(want), np.zeros_like(want)
            np.add.at(scatter, ids, dh * scale)
            np.add.at(scatter_tol, ids, ((h + 1e-4) * dh_mag + h * np.abs(dh)) * scale * (1 + h))
            # the four roundings of this micro-batch's way into the buffer: head, head's sum, lookup's sum
            tol += (h + 1e-4) * head_mag + scatter_tol
            for add in (head_grad, scatter):
                want += add
                tol += h * (np.abs(want) + tol) + 2.0 ** -24 * np.abs(add)
        assert np.all(np.abs(grad - want) <= tol), np.max(np.abs(grad - want) / tol)
        got_loss = sum(w * float(t[0]) for w, t in zip(weights, totals))
        assert abs(got_loss - loss) <= 1e-4 * (1 + abs(loss))
        assert sum(float(t[1]) for t in totals) == (scored if masked else rows * micro)
        before_work = views["work"].clone()
        returned, norm = trainer.training_step(got_loss)
        assert returned == got_loss and abs(norm - math.sqrt(float(np.sum(grad ** 2))) / ls) <= 1e-5 * norm
        torch.cuda.synchronize()
        assert not torch.equal(before_work[:vocab * hidden], views["work"][:vocab * hidden])
    assert trainer.optimizer_timestep() == 3
    for o in (emb, head, opt):
        o.destroy()
    loader.close()


@gpu
def test_two_handles_on_two_streams_and_two_graphs_of_one():
    """Two handles at once do not disturb each other; two graphs of one handle replay in turn."""
    import torch
    vocab, hidden, rows = 2000, 128, 300
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(vocab, hidden, device="cuda", generator=gen).mul_(0.1).bfloat16()
    jobs = []
    for k in range(2):
        x = torch.randn(rows, hidden, device="cuda", generator=gen).bfloat16()
        t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        jobs.append(dict(x=x, t=t, head=ox.LossHead(vocab, hidden, rows), dx=torch.empty_like(x), dw=torch.empty_like(w), loss=torch.empty(rows, device="cuda"),
                         stream=torch.cuda.Stream()))

    def run(job, head, dx, dw, loss, stream):
        head.loss_and_grads(rows, job["x"].data_ptr(), w.data_ptr(), job["t"].data_ptr(), row_loss=loss.data_ptr(), d_hidden=dx.data_ptr(),
                            d_weight=dw.data_ptr(), stream=stream)
    torch.cuda.synchronize()
    want = []
    for job in jobs:
        run(job, job["head"], job["dx"], job["dw"], job["loss"], 0)
        torch.cuda.synchronize()
        want.append([job[k].clone() for k in ("dx", "dw", "loss")])
        for k in ("dx", "dw", "loss"):
            job[k].zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for job in jobs:
            run(job, job["head"], job["dx"], job["dw"], job["loss"], job["stream"].cuda_stream)
    torch.cuda.synchronize()
    for job, res in zip(jobs, want):
        assert all(torch.equal(job[k], r) for k, r in zip(("dx", "dw", "loss"), res))
    # one handle, its two calls captured apart and replayed one after the other on one stream
    head, graphs, s = jobs[0]["head"], [], torch.cuda.Stream()
    for job in jobs:
        for k in ("dx", "dw", "loss"):
            job[k].zero_()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            run(job, head, job["dx"], job["dw"], job["loss"], s.cuda_stream)
        graphs.append(g)
    with torch.cuda.stream(s):
        for _ in range(2):
            for g in graphs:
                g.replay()
    torch.cuda.synchronize()
    for job, res in zip(jobs, want):
        assert all(torch.equal(job[k], r) for k, r in zip(("dx", "dw", "loss"), res))
    del graphs, g
    for job in jobs:
        job["head"].destroy()


@pytest.mark.parametrize("kw, text", [
    (dict(vocab=31), "31 x 8 elements do not fit tensor 0, which has 240"), (dict(dtype=ox.F16, grad_dtype=ox.F16), "works in dtype 2, the optimizer's weights have 1"),
    (dict(grad_dtype=ox.F32), "writes gradients of dtype 0, the optimizer's have 1"), (dict(device=1), "is on device 1, the optimizer on 0"),
])
@pytest.mark.parametrize("operator", ["embedding", "head"])
def test_operators_that_do_not_fit_the_optimizers_buffers_are_refused(kw, text, operator):
    """Before anything is enqueued: types and sizes that differ would be read and written as if they did not."""
    trainer = ox.LitTrainerStep(ox.TrainerConfig(), ox.DpOptimizer([240, 8], allocate=False))
    p = 1 << 20  # an address that is only looked at
    given = {**dict(vocab=30, hidden=8, dtype=ox.BF16, allocate=False), **kw}
    if operator == "embedding":
        op = ox.TokenEmbedding(max_tokens=4, **given)
        # the lookup reads the weights, its gradient does not
        calls = [] if "dtype" in kw else [lambda: trainer.embed_grads(op, 0, p, 2, p, accumulate=False)]
        if kw != dict(grad_dtype=ox.F32):
            calls.append(lambda: trainer.embed(op, 0, p, 2, p))
    else:
        op = ox.LossHead(max_rows=4, **given)
        calls = [lambda: trainer.loss_and_grads(op, 0, 2, p, p, p, p)]
    for call in calls:
        with pytest.raises(ValueError) as e:
            call()
        assert text in str(e.value)
    op.destroy()
