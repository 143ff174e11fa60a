"""Calls of the training operators at the edges of what their documentation allows."""
import ctypes

import numpy as np
import pytest

import mimir_hip as M
from _serving import Graph, Hip, bf16_value
from _training import U, Mat, held
from test_gpu_gated_linear import hold as hold_gated, make as make_gated, run as run_gated
from test_gpu_linear_ce import hold as hold_ce, make as make_ce, run as run_ce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1), (8, 8)])
@pytest.mark.parametrize("dtype,dim", [("f32", 3), ("f32", 8), ("bf16", 8), ("bf16", 9)])
def test_no_tokens_no_inputs(ctx, dtype, dim, pad, offset):
    """Without tokens no input is there to be read: weights' gradients are zeros, or what they were."""
    v = 300
    kw = dict(dtype=dtype, ld_x=dim + pad, ld_w=dim + pad)
    mean = ctx.to_device(np.full(2, 5, np.float32))
    ctx.linear_cross_entropy(None, None, None, 0, dim, v, None, None, mean, **kw)
    assert (mean.numpy() == 0).all()
    ctx.linear_cross_entropy(None, None, None, 0, dim, v, None, None, None, **kw)
    for accumulate in (True, False):
        DW, DX = Mat(ctx, np.full((v, dim), 3.0), dtype, pad, offset), Mat(ctx, np.full((2, dim), 3.0), dtype, pad, offset)
        ctx.linear_cross_entropy_bwd(None, None, None, None, None, mean, DX.ptr, DW.ptr, 0, dim, v, ld_dx=DX.ld, ld_dw=DW.ld,
                                     accumulate_w=accumulate, **kw)
        assert (DW.get() == (3 if accumulate else 0)).all() and (DX.get() == 3).all()
        ctx.linear_cross_entropy_bwd(None, None, None, None, None, None, DX.ptr, None, 0, dim, v, ld_dx=DX.ld, **kw)
        assert (DX.get() == 3).all()
        A, B = (Mat(ctx, np.full((v, dim), 3.0), dtype, pad, offset) for _ in range(2))
        ctx.gated_linear_bwd(None, None, None, None, None, DX.ptr, A.ptr, B.ptr, 0, v, dim, dtype=dtype, ld_x=v, ld_w=dim + pad,
                             ld_dx=v, ld_dw=A.ld, accumulate_w=accumulate)
        assert (A.get() == (3 if accumulate else 0)).all() and (B.get() == A.get()).all() and (DX.get() == 3).all()


@pytest.fixture(scope="module", params=["", "matbig=1,matpiece=264", "matbig=0,matpiece=136"], ids=["default", "big", "small"])
def tuned(request):
    """A context of its own: the shapes and pieces by rule, or forced."""
    with pytest.MonkeyPatch.context() as mp:
        mp.setenv("MIMIR_TUNE", request.param)
        c = M.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,vocab", [(20, 700), (32, 64), (33, 500), (150, 900), (400, 5000)])
def test_dominant_logits(tuned, tokens, vocab, dtype):
    """Tokens are unit vectors, so logits are the weights' own values, exactly.  One of each token's is far above the
    others: the sum is 1 plus what counts, the loss of that target is never below 0, and nothing but 0 where the others'
    exponentials leave fp32; likewise the gradients."""
    rng = np.random.default_rng(tokens)
    dim = tokens
    x = np.eye(tokens, dtype=np.float32)
    top = held(rng.uniform(5, 3000, tokens) * np.where(rng.random(tokens) < 0.3, -1, 1), dtype)
    # Half of the tokens' other logits are out of reach (exp of -150 is below 2^-149), half some tens below.
    far = np.arange(tokens) % 2 == 0
    gap = np.where(far, rng.uniform(160, 400, (vocab, tokens)), rng.uniform(2, 60, (vocab, tokens)))
    w = held(top - gap, dtype)
    target = rng.integers(0, vocab, tokens).astype(np.int32)
    w[target, np.arange(tokens)] = top
    assert (np.delete(w, 0, 0) <= top).all()
    X, W, t = Mat(tuned, x, dtype), Mat(tuned, w, dtype), tuned.to_device(target)
    loss, lse, mean = (tuned.empty(n) for n in (tokens, tokens, 2))
    DX, DW = Mat(tuned, x, dtype), Mat(tuned, np.full(w.shape, 9.0), dtype)
    tuned.linear_cross_entropy(X.ptr, W.ptr, t, tokens, dim, vocab, loss, lse, mean, dtype=dtype)
    tuned.linear_cross_entropy_bwd(X.ptr, W.ptr, t, lse, None, None, DX.ptr, DW.ptr, tokens, dim, vocab, dtype=dtype)
    loss, lse = loss.numpy(), lse.numpy()
    assert (loss >= 0).all() and (lse >= top).all()
    assert (loss[far] == 0).all() and (lse[far] == top[far]).all()
    assert (DX.get()[far] == 0).all() and (DW.get()[:, far] == 0).all()
    # The others: the exponentials' arguments are off by 3 U of a difference of at most 64 (with exp(-d) at most 1 / (e d)
    # of it, so by 1.2 U), the function by a last place, sums by the number of their terms; lse rounds once.
    z = w.astype(np.float64)
    want = top + np.log(np.exp(z - top).sum(0))
    assert (np.abs(lse - want) <= (5 + 140 + 4 * (vocab / 128 + 1) + 1.01 * np.abs(want)) * U).all()


def plain_cross_entropy(x, w, target):
    """(loss, lse) in float64, and which tokens count."""
    ok = (target >= 0) & (target < len(w))
    z = x.astype(np.float64) @ w.astype(np.float64).T
    top = z.max(1)
    lse = np.log(np.exp(z - top[:, None]).sum(1)) + top
    return np.where(ok, lse - z[np.arange(len(z)), np.where(ok, target, 0)], 0), np.where(ok, lse, 0), ok


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [8191, 8192, 8193, 16385, 70001])
def test_many_tokens_gathered(ctx, tokens, dtype):
    """Blocks of 8192 targets: all, none, some of them counting, the ends of blocks and of the batch."""
    rng = np.random.default_rng(tokens)
    dim, vocab = 8, 24
    x, w = held(rng.standard_normal((tokens, dim)), dtype), held(rng.standard_normal((vocab, dim)), dtype)
    target = rng.integers(0, vocab, tokens).astype(np.int32)
    part = np.arange(tokens) // 4096
    target[(part % 4 == 1) | ((part % 4 == 2) & (rng.random(tokens) < 0.5))] = -1
    want, lses, ok = plain_cross_entropy(x, w, target)
    x[~ok] = np.nan
    X, W, t = Mat(ctx, x, dtype), Mat(ctx, w, dtype), ctx.to_device(target)
    loss, lse, mean = (ctx.to_device(np.full(n, 5, np.float32)) for n in (tokens, tokens, 2))
    ctx.linear_cross_entropy(X.ptr, W.ptr, t, tokens, dim, vocab, loss, lse, mean, dtype=dtype)
    # |z| up to 20: sums of 8 products, exponentials and the sum of 24 of them are off by fewer than 100 U.
    assert (np.abs(loss.numpy() - want) <= 100 * U * (1 + np.abs(lses))).all()
    m = mean.numpy()
    assert m[1] == ok.sum() and abs(m[0] - want.sum() / ok.sum()) <= 200 * U * (1 + want.sum() / ok.sum())
    DX = Mat(ctx, np.full(x.shape, 9.0), dtype)
    ctx.linear_cross_entropy_bwd(X.ptr, W.ptr, t, lse, None, mean, DX.ptr, None, tokens, dim, vocab, dtype=dtype)
    prob = np.exp(np.where(ok[:, None], x, 0).astype(np.float64) @ w.astype(np.float64).T - lses[:, None])
    g = prob.copy()
    g[np.arange(tokens)[ok], target[ok]] -= 1
    g, prob = (np.where(ok[:, None], v, 0) / ok.sum() for v in (g, prob))
    # The exponentials are off by their arguments' errors (|z| up to 20), fewer than 150 U in all; G and the result round
    # once each.
    bound = (prob * 150 * U + np.abs(g) * (2 * 2.0 ** -8 if dtype == "bf16" else 20 * U)) @ np.abs(w.astype(np.float64)) * 1.1
    assert (np.abs(DX.get() - g @ w.astype(np.float64)) <= bound).all() and (DX.get()[~ok] == 0).all()


def test_time_is_linear_in_tokens(ctx):
    """Eight times the tokens may take some eight times as long, not sixty."""
    dim, vocab, most = 8, 16, 1 << 22
    x, w, t = ctx.empty((most, dim)), ctx.empty((vocab, dim)), ctx.empty(most, np.int32)
    loss, lse, mean, dx = ctx.empty(most), ctx.empty(most), ctx.empty(2), ctx.empty((most, dim))
    ctx.fill(x, 0.5)
    ctx.fill(w, 0.25)
    ctx.upload(t, (np.arange(most) % 17 - 1).astype(np.int32))

    def timed(n):
        best = 1e9
        for _ in range(4):
            a, b = M.Event(ctx), M.Event(ctx)
            a.record()
            ctx.linear_cross_entropy(x, w, t, n, dim, vocab, loss, lse, mean)
            ctx.linear_cross_entropy_bwd(x, w, t, lse, None, mean, dx, None, n, dim, vocab)
            b.record()
            ctx.sync()
            best = min(best, a.elapsed_ms(b))
        return best

    small, large = timed(most // 8), timed(most)
    count = (most - 1) // 17 * 16 + (most - 1) % 17  # every 17th token has no target, the first among them
    assert mean.numpy()[1] == np.float32(count)
    assert np.allclose(loss.numpy()[1:17], np.log(vocab), rtol=1e-6)
    assert large < 24 * small, (small, large)


@pytest.mark.parametrize("beside", [False, True])
def test_clipping_of_thousands_of_tensors(ctx, beside):
    """More launches than the clipping adds up the sums of by itself: 4000 tensors of one to some hundred elements."""
    rng = np.random.default_rng(5)
    sizes = rng.integers(0, 300, 4000)
    start = np.concatenate([[0], np.cumsum(sizes)])
    v = (rng.standard_normal(start[-1]) * np.repeat(10.0 ** rng.uniform(-2, 2, 4000), sizes)).astype(np.float32)
    d = ctx.to_device(v)
    out = ctx.to_device(np.zeros_like(v)) if beside else d
    tensors = M.TensorList([(d.ptr + 4 * int(a), int(n), "f32", out.ptr + 4 * int(a)) for a, n in zip(start, sizes)])
    norm = ctx.empty(2)
    ctx.grad_norm(tensors, norm)
    ctx.grad_clip(tensors, 2.5, norm.offset(1))
    want = np.sqrt((v.astype(np.float64) ** 2).sum())
    n = norm.numpy()
    assert n[0] == n[1] and abs(n[0] - want) <= 1.01 * U * want
    clipped = v * (2.5 / (want + 1e-6))
    assert (np.abs(out.numpy() - clipped) <= 3.1 * U * np.abs(clipped)).all()


def test_time_is_linear_in_tensors(ctx):
    """Five times the tensors may take some five times as long, not fifteen."""
    d, norm = ctx.empty(64 * 100000), ctx.empty(1)
    ctx.fill(d, 0.5)

    def timed(count):
        tensors = M.TensorList([(d.ptr + 256 * i, 64, "f32") for i in range(count)])
        best = 1e9
        for _ in range(3):
            a, b = M.Event(ctx), M.Event(ctx)
            a.record()
            ctx.grad_clip(tensors, 1e9, norm)
            b.record()
            ctx.sync()
            best = min(best, a.elapsed_ms(b))
        return best

    small, large = timed(20000), timed(100000)
    assert abs(norm.numpy()[0] - 0.5 * np.sqrt(64 * 100000)) < 1e-3
    assert large < 9 * small, (small, large)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("most,scale", [(1e-30, 1e38), (1e-38, 3e38), (1e-45, 3e38), (1e-20, 1e37), (3e-8, 1e30), (1e-38, 1e-37), (0.0, 1e38)])
def test_clipping_by_tiny_factors(ctx, most, scale, kind):
    """Factors far below fp32's range, of elements near its largest: the products are in it."""
    rng = np.random.default_rng(6)
    most = float(np.float32(most))
    v = held((rng.uniform(0.3, 1, 5003) * scale * rng.choice([-1, 1], 5003)).astype(np.float32), kind)
    m = Mat(ctx, v[None], kind)
    ctx.grad_clip(M.TensorList([(m.ptr, v.size, kind)]), most)
    norm = np.sqrt((v.astype(np.float64) ** 2).sum())
    want = v.astype(np.float64) * (most / (norm + 1e-6))
    # One rounding of the factor and one of the product; bf16 one more, and its subnormals' half step.
    half = U * 2.01 + (1.001 * 2.0 ** -8 if kind == "bf16" else 0)
    tiny = 2.0 ** -134 + 2.0 ** -150 if kind == "bf16" else 2.0 ** -150
    assert (np.abs(m.get()[0] - want) <= half * np.abs(want) + tiny).all()


@pytest.mark.parametrize("beside", [False, True])
def test_infinite_bound_clips_nothing(ctx, beside):
    for bad in (None, np.inf, -np.inf, np.nan):
        v = np.linspace(-3, 5, 9000).astype(np.float32)
        if bad is not None:
            v[77] = bad
        d = ctx.to_device(v)
        out = ctx.to_device(np.zeros_like(v)) if beside else d
        norm = ctx.empty(1)
        ctx.grad_clip(M.TensorList([(d, v.size, "f32", out)]), np.inf, norm)
        got = out.numpy()
        assert np.isnan(got).all() if bad is np.nan else np.array_equal(got, v)


def test_scratch_after_a_capture_is_bounded():
    """A captured call keeps the scratch that its graph holds; eager calls of more and more tokens after it leave no more
    than that and their own behind, and the graph goes on giving its results."""
    rng = np.random.default_rng(8)
    dim, vocab, n, step = 64, 40, 50, 60000
    with M.Context(0) as c:
        hip = Hip(c)

        def free_bytes():
            c.sync()
            free, total = ctypes.c_size_t(), ctypes.c_size_t()
            hip("hipMemGetInfo", ctypes.byref(free), ctypes.byref(total))
            return free.value

        most = 20 * step
        x, w = c.empty((most, dim)), c.to_device(rng.standard_normal((vocab, dim)).astype(np.float32))
        c.fill(x, 0.125)
        t = c.to_device((np.arange(most) % vocab).astype(np.int32))
        loss, lse, mean = c.empty(most), c.empty(most), c.empty(2)
        small = [c.to_device(rng.standard_normal((n, dim)).astype(np.float32)), c.empty(n), c.empty(n), c.empty(2)]
        call = lambda: c.linear_cross_entropy(small[0], w, t, n, dim, vocab, *small[1:])  # noqa: E731
        graphs = [Graph(c, call)]
        graphs[0].launch()
        want = small[1].numpy()
        before, sizes = free_bytes(), []
        for i in range(1, 21):
            c.linear_cross_entropy(x, w, t, i * step, dim, vocab, loss, lse, mean)
            assert mean.numpy()[1] == i * step
            if i == 10:
                graphs.append(Graph(c, call))
            sizes.append(before - free_bytes())
        # The rows' three planes alone, 6 bytes an element; the scratch of the second capture's time stays beside the
        # last one, which is larger by half than it needs at most.  A buffer for each call would be ten times the last.
        last = 6 * dim * most
        assert last < sizes[-1] < 2.5 * last, sizes
        for g in graphs * 2:
            small[1].upload(np.zeros(n, np.float32))
            g.launch()
            c.linear_cross_entropy(x, w, t, 1000, dim, vocab, loss, lse, mean)
            assert np.array_equal(small[1].numpy(), want)
        for g in graphs:
            g.close()


def test_captures_that_grow(ctx):
    """Captures of larger and larger calls, each the first of its size, replayed in any order."""
    rng = np.random.default_rng(9)
    dim, vocab = 72, 300
    with M.Context(0) as c:
        w = c.to_device((rng.standard_normal((vocab, dim)) / 8).astype(np.float32))
        calls, graphs, wants = [], [], []
        for n in (40, 700, 9000, 30000):
            x, t = c.to_device(rng.standard_normal((n, dim)).astype(np.float32)), c.to_device(rng.integers(-1, vocab, n).astype(np.int32))
            loss, lse, mean = c.empty(n), c.empty(n), c.empty(2)
            calls.append((x, t, n, loss, lse, mean))
            graphs.append(Graph(c, lambda: c.linear_cross_entropy(x, w, t, n, dim, vocab, loss, lse, mean)))
        for x, t, n, loss, lse, mean in calls:
            c.linear_cross_entropy(x, w, t, n, dim, vocab, loss, lse, mean)
            wants.append(loss.numpy())
        for i in (3, 0, 2, 1, 0, 3):
            calls[i][3].upload(np.full(calls[i][2], 7, np.float32))
            graphs[i].launch()
            assert np.array_equal(calls[i][3].numpy(), wants[i]), i
        for g in graphs:
            g.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("tokens,masked", [(1, 1.0), (7, 0.5), (17, 1.0), (32, 0.4)])
def test_few_tokens_without_target(tuned, tokens, masked, bad, dtype):
    """As many tokens as take no gathering in the forward: rows that hold anything, targets outside the vocabulary."""
    x, w, t = make_ce(tokens, tokens, 40, 300, dtype, masked)
    t[0] = -1
    none = t < 0
    t[none] = np.resize(np.array([-1, -100, 300, 2 ** 31 - 1, -2 ** 31], np.int64), none.sum()).astype(np.int32)
    x2 = x.copy()
    x2[none] = bad
    for kw in (dict(), dict(use_mean=False, weight=np.linspace(-1, 2, tokens), scale=0.5)):
        hold_ce(run_ce(tuned, x2, w, t, dtype, **kw), x, w, t, dtype, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [5, 40])
def test_rows_far_apart(ctx, tokens, dtype):
    """Row strides of 2^20 elements and more, which tiles do not take as they are."""
    x, w, t = make_ce(tokens, tokens, 24, 70, dtype, 0.2)
    hold_ce(run_ce(ctx, x, w, t, dtype, pad=(1 << 20) - 24 + 8 * (tokens == 5)), x, w, t, dtype)
    a = make_gated(tokens, tokens, 24, 40, dtype)
    hold_gated(run_gated(ctx, *a, "silu", dtype, pad=(1 << 20) - 24), *a, "silu", dtype)


class AmongNans(Mat):
    """A matrix whose buffer holds NaN around and between its rows."""

    FILL = np.float32(np.nan)

    def get(self):
        b = self.dev.numpy()
        b = bf16_value(b) if self.dtype == "bf16" else b
        rows, cols = self.shape
        n = self.at + rows * self.ld
        body = b[self.at:n].reshape(rows, self.ld)
        assert np.isnan(b[:self.at]).all() and np.isnan(b[n:]).all() and np.isnan(body[:, cols:]).all()
        return body[:, :cols].copy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,offset", [(0, 3), (8, 8), (5, 1), (1, 0)])
@pytest.mark.parametrize("tokens,dim,vocab", [(5, 6, 70), (31, 37, 130), (17, 64, 257), (3, 1003, 65), (40, 48, 333), (150, 129, 300)])
def test_nans_between_the_rows(tuned, monkeypatch, tokens, dim, vocab, pad, offset, dtype):
    """Nothing around the rows is looked at: a product with a NaN would show, also one with 0."""
    import test_gpu_gated_linear
    import test_gpu_linear_ce
    monkeypatch.setattr(test_gpu_linear_ce, "Mat", AmongNans)
    monkeypatch.setattr(test_gpu_gated_linear, "Mat", AmongNans)
    x, w, t = make_ce(tokens + dim, tokens, dim, vocab, dtype, 0.2)
    hold_ce(run_ce(tuned, x, w, t, dtype, pad=pad, offset=offset), x, w, t, dtype)
    a = make_gated(tokens + dim, tokens, dim, vocab, dtype)
    hold_gated(run_gated(tuned, *a, "gelu", dtype, pad=pad, offset=offset), *a, "gelu", dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,dim,vocab,masked", [(7, 24, 70, 0.5), (32, 1003, 335, 0.3), (2, 5, 100, 0.0), (20, 64, 3, 0.2), (45, 41, 333, 0.6), (130, 100, 513, 0.3), (300, 40, 777, 0.9)])
def test_scratch_full_of_nans(tuned, tokens, dim, vocab, masked, dtype):
    """What calls of NaN left in the scratch, in planes, sums, statistics and gradients, reaches no later call."""
    for kind in ("f32", "bf16"):
        nan = [np.full(s, np.nan, np.float32) for s in ((400, 1100), (900, 1100))]
        X, W = Mat(tuned, nan[0], kind), Mat(tuned, nan[1], kind)
        t, out = tuned.to_device(np.zeros(400, np.int32)), [tuned.empty(400), tuned.empty(400), tuned.empty(2)]
        DX, DW = Mat(tuned, nan[0], kind), Mat(tuned, nan[1], kind)
        tuned.linear_cross_entropy(X.ptr, W.ptr, t, 400, 1100, 900, *out, dtype=kind)
        tuned.linear_cross_entropy_bwd(X.ptr, W.ptr, t, out[1], None, out[2], DX.ptr, DW.ptr, 400, 1100, 900, dtype=kind)
        assert np.isnan(DX.get()).all()
    x, w, t = make_ce(tokens + dim, tokens, dim, vocab, dtype, masked)
    hold_ce(run_ce(tuned, x, w, t, dtype, pad=3), x, w, t, dtype)
    a = make_gated(tokens + dim, tokens, dim, vocab, dtype)
    hold_gated(run_gated(tuned, *a, "silu", dtype), *a, "silu", dtype)
