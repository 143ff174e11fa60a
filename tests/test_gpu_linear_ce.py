"""Cross entropy of a linear layer against float64: both types, both tile shapes,
the vocabulary in one piece and in several, odd sizes and strides, tokens without a
target (whatever stands in them), gradients written and added to, replays."""
import numpy as np
import pytest

import mimir_hip as M
from _training import Mat, cross_entropy64, cross_entropy_bwd64, held, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["", "matbig=1,matpiece=264", "matbig=0,matpiece=136"], ids=["default", "big", "small"])
def tuned(request):
    """A context of its own: the shapes and pieces by rule, or forced."""
    with pytest.MonkeyPatch.context() as mp:
        mp.setenv("MIMIR_TUNE", request.param)
        c = M.Context(0)
    yield c
    c.close()


def make(seed, tokens, dim, vocab, dtype, masked, spread=2.0):
    rng = np.random.default_rng(seed)
    x = held(rng.standard_normal((tokens, dim)), dtype)
    w = held(rng.standard_normal((vocab, dim)) * spread / np.sqrt(dim), dtype)
    target = rng.integers(0, vocab, tokens).astype(np.int32)
    target[rng.random(tokens) < masked] = -1
    return x, w, target


def run(ctx, x, w, target, dtype, back=True, pad=0, offset=0, weight=None, use_mean=True, scale=1.0, start=None):
    """loss, lse, mean, dx, dw; `start`: (dx, dw) that the gradients are added to."""
    tokens, dim = x.shape
    vocab = len(w)
    X, W = Mat(ctx, x, dtype, pad, offset), Mat(ctx, w, dtype, pad, offset)
    t = ctx.to_device(target)
    loss, lse, mean = (ctx.to_device(np.full(n, 5.0, np.float32)) for n in (max(tokens, 1), max(tokens, 1), 2))
    kw = dict(dtype=dtype, ld_x=X.ld, ld_w=W.ld)
    ctx.linear_cross_entropy(X.ptr, W.ptr, t, tokens, dim, vocab, loss, lse, mean, **kw)
    out = [loss.numpy()[:tokens], lse.numpy()[:tokens], mean.numpy()]
    if back:
        s = start if start is not None else (np.full(x.shape, 9.0), np.full(w.shape, 9.0))
        DX, DW = Mat(ctx, s[0], dtype, pad, offset), Mat(ctx, s[1], dtype, pad, offset)
        g = ctx.to_device(weight.astype(np.float32)) if weight is not None else None
        ctx.linear_cross_entropy_bwd(X.ptr, W.ptr, t, lse, g, mean if use_mean else None, DX.ptr, DW.ptr, tokens, dim, vocab,
                                     scale=scale, ld_dx=DX.ld, ld_dw=DW.ld, accumulate_x=start is not None,
                                     accumulate_w=start is not None, **kw)
        out += [DX.get(), DW.get()]
    assert np.array_equal(X.get(), x, equal_nan=True) and (W.get() == w).all()
    return out


def hold(got, x, w, target, dtype, weight=None, use_mean=True, scale=1.0, start=None):
    c = cross_entropy64(x, w, target)
    loss, lse, mean = got[:3]
    near(lse, c["lse"], c["e_lse"], "lse")
    near(loss, c["loss"], c["e_loss"], "loss")
    assert (loss[~c["ok"]] == 0).all() and (lse[~c["ok"]] == 0).all()
    count = int(c["ok"].sum())
    assert mean[1] == count
    want = c["loss"].sum() / max(1, count)
    assert abs(mean[0] - want) <= c["e_loss"].sum() / max(1, count) + 2.0 ** -23 * abs(want)
    if len(got) == 3:
        return
    factor = scale / (max(1, count) if use_mean else 1)
    g = np.ones(len(x)) if weight is None else weight.astype(np.float64)
    dx, edx, dw, edw = cross_entropy_bwd64(x, w, target, c, g, dtype, factor)
    if start is not None:
        half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
        a, b = held(start[0], dtype), held(start[1], dtype)
        dx, dw = dx + a * c["ok"][:, None] + a * ~c["ok"][:, None], dw + b
        edx, edw = edx + 1.1 * half * np.abs(a), edw + 1.1 * half * np.abs(b)
    near(got[3], dx, edx, "dx")
    near(got[4], dw, edw, "dw")
    if start is None:
        assert (got[3][~c["ok"]] == 0).all()


# tokens, dim, vocab
SIZES = [(1, 1, 1), (1, 8, 2), (7, 24, 70), (32, 296, 1000), (17, 1024, 333), (5, 2048, 64), (20, 8, 3), (9, 37, 71), (32, 1003, 335), (16, 30, 34), (4, 6, 5), (2, 5, 100), (3, 64, 257), (31, 33, 129), (32, 64, 128), (33, 65, 300), (65, 136, 1000),
         (129, 100, 513), (300, 40, 777), (130, 1000, 264)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,dim,vocab", SIZES)
def test_sizes(tuned, tokens, dim, vocab, dtype):
    x, w, t = make(tokens * 7 + dim, tokens, dim, vocab, dtype, 0.0)
    hold(run(tuned, x, w, t, dtype), x, w, t, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,offset", [(0, 3), (8, 0), (5, 1), (24, 8)])
def test_strides_and_alignment(tuned, pad, offset, dtype):
    x, w, t = make(pad + offset, 45, 48, 333, dtype, 0.2)
    hold(run(tuned, x, w, t, dtype, pad=pad, offset=offset), x, w, t, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("masked", [0.5, 1.0])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_tokens_without_target(tuned, masked, bad, dtype):
    """Their rows may hold anything; targets outside the vocabulary are none."""
    x, w, t = make(5, 70, 40, 300, dtype, masked)
    none = t < 0
    t[none] = np.resize(np.array([-1, -100, 300, 2 ** 31 - 1, -2 ** 31], np.int64), none.sum()).astype(np.int32)
    x2 = x.copy()
    x2[none] = bad
    got = run(tuned, x2, w, t, dtype)
    hold(got, x, w, t, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_weights_scale_and_sums(tuned, dtype):
    x, w, t = make(8, 90, 56, 400, dtype, 0.3)
    rng = np.random.default_rng(9)
    weight = rng.standard_normal(90)
    weight[3] = 0
    start = (rng.standard_normal(x.shape), rng.standard_normal(w.shape))
    for kw in (dict(weight=weight, use_mean=False), dict(weight=weight, scale=-3.0), dict(scale=0.125, start=start),
               dict(use_mean=False, weight=weight, start=start)):
        hold(run(tuned, x, w, t, dtype, **kw), x, w, t, dtype, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_logits(tuned, dtype):
    """Logits of some hundreds: the exponentials of all but a few vanish."""
    x, w, t = make(11, 40, 64, 500, dtype, 0.0, spread=100.0)
    hold(run(tuned, x, w, t, dtype), x, w, t, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,dim,vocab", [(2000, 72, 8200), (1300, 520, 1000)])
def test_many_tiles(ctx, tokens, dim, vocab, dtype):
    """The larger tiles by rule, on all XCDs."""
    x, w, t = make(tokens, tokens, dim, vocab, dtype, 0.1)
    hold(run(ctx, x, w, t, dtype), x, w, t, dtype)


def test_no_tokens(ctx):
    w = np.ones((7, 8), np.float32)
    for dtype in ("f32", "bf16"):
        W, DW, mean = Mat(ctx, w, dtype), Mat(ctx, 3 * w, dtype), ctx.to_device(np.full(2, 5, np.float32))
        ctx.linear_cross_entropy(None, W.ptr, None, 0, 8, 7, None, None, mean, dtype=dtype)
        assert (mean.numpy() == 0).all()
        ctx.linear_cross_entropy_bwd(None, W.ptr, None, None, None, None, None, DW.ptr, 0, 8, 7, dtype=dtype, accumulate_w=True)
        assert (DW.get() == 3).all()
        ctx.linear_cross_entropy_bwd(None, W.ptr, None, None, None, mean, None, DW.ptr, 0, 8, 7, dtype=dtype)
        assert (DW.get() == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_gradient_alone_and_in_place(ctx, dtype):
    x, w, t = make(21, 50, 64, 200, dtype, 0.3)
    both = run(ctx, x, w, t, dtype)
    X, W, td = Mat(ctx, x, dtype), Mat(ctx, w, dtype), ctx.to_device(t)
    loss, lse, mean = (ctx.empty(n) for n in (50, 50, 2))
    ctx.linear_cross_entropy(X.ptr, W.ptr, td, 50, 64, 200, loss, lse, mean, dtype=dtype)
    DW = Mat(ctx, np.zeros_like(w), dtype)
    ctx.linear_cross_entropy_bwd(X.ptr, W.ptr, td, lse, None, mean, None, DW.ptr, 50, 64, 200, dtype=dtype)
    assert (DW.get() == both[4]).all()
    ctx.linear_cross_entropy_bwd(X.ptr, W.ptr, td, lse, None, mean, X.ptr, None, 50, 64, 200, dtype=dtype)
    assert (X.get() == both[3]).all()


def test_gradient_against_differences(ctx):
    """dx and dw against central differences of the mean loss in float64."""
    x, w, t = make(33, 6, 9, 11, "f32", 0.2)
    t[0] = 4
    got = run(ctx, x, w, t, "f32")
    h = 1e-4

    def mean(x, w):
        c = cross_entropy64(x, w, t)
        return c["loss"].sum() / c["ok"].sum()

    for which, g in ((0, got[3]), (1, got[4])):
        for at in np.ndindex(*g.shape):
            a = [x.astype(np.float64), w.astype(np.float64)]
            b = [v.copy() for v in a]
            a[which][at] += h
            b[which][at] -= h
            assert abs((mean(*a) - mean(*b)) / (2 * h) - g[at]) < 1e-6  # the differences' own error is h^2 times a third derivative below 10


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_same_bits_again(ctx, dtype):
    x, w, t = make(41, 260, 72, 1000, dtype, 0.3)
    a, b = run(ctx, x, w, t, dtype), run(ctx, x, w, t, dtype)
    for u, v in zip(a, b):
        assert np.array_equal(u, v)
