"""The training operators as a program runs them: a step of a feed-forward block,
the loss of the layer behind it, both backward and the gradients clipped; captured
steps replayed while their inputs change and larger calls run between; other streams,
contexts and threads beside."""
import ctypes
import threading

import numpy as np
import pytest

import mimir_hip as M
from _serving import Graph, Hip, bf16_bits, bf16_value
from _training import activation64, held

pytestmark = pytest.mark.gpu


class Step:
    """x -> act(x Wg) * (x Wu) -> cross entropy over V; the device side of a program that keeps its buffers."""

    def __init__(self, ctx, dtype, tokens, dim, hidden, vocab, act="silu", most=0.05):
        self.ctx, self.dtype, self.sizes, self.act, self.most = ctx, dtype, (tokens, dim, hidden, vocab), act, most
        kind = np.float32 if dtype == "f32" else np.uint16
        e = lambda *s, t=kind: ctx.empty(s, t)  # noqa: E731
        self.x, self.wg, self.wu, self.w = e(tokens, dim), e(dim, hidden), e(dim, hidden), e(vocab, hidden)
        self.y, self.dy, self.dx = e(tokens, hidden), e(tokens, hidden), e(tokens, dim)
        self.gu = ctx.empty((tokens, 2 * hidden))
        self.grads = [e(dim, hidden), e(dim, hidden), e(vocab, hidden)]
        self.target = ctx.empty(tokens, np.int32)
        self.loss, self.lse, self.mean, self.norm = (ctx.empty(n) for n in (tokens, tokens, 2, 1))
        self.list = M.TensorList([(g, g.size, dtype) for g in self.grads])

    def set(self, seed):
        t, d, h, v = self.sizes
        rng = np.random.default_rng(seed)
        self.host = [held(a, self.dtype) for a in (rng.standard_normal((t, d)), rng.standard_normal((d, h)) / np.sqrt(d),
                                                   rng.standard_normal((d, h)) / np.sqrt(d), rng.standard_normal((v, h)))]
        self.at = rng.integers(0, v, t).astype(np.int32)
        self.at[rng.random(t) < 0.25] = -1
        for dev, a in zip((self.x, self.wg, self.wu, self.w), self.host):
            self.ctx.upload(dev, bf16_bits(a) if self.dtype == "bf16" else a)
        self.ctx.upload(self.target, self.at)

    def run(self):
        c, (t, d, h, v), k = self.ctx, self.sizes, dict(dtype=self.dtype)
        c.gated_linear(self.x, self.wg, self.wu, self.y, t, d, h, act=self.act, gate_up=self.gu, **k)
        c.linear_cross_entropy(self.y, self.w, self.target, t, h, v, self.loss, self.lse, self.mean, **k)
        c.linear_cross_entropy_bwd(self.y, self.w, self.target, self.lse, None, self.mean, self.dy, self.grads[2], t, h, v, **k)
        c.gated_linear_bwd(self.x, self.wg, self.wu, self.gu, self.dy, self.dx, self.grads[0], self.grads[1], t, d, h,
                           act=self.act, **k)
        c.grad_clip(self.list, self.most, self.norm)

    def read(self):
        out = [self.mean.numpy(), self.norm.numpy(), self.loss.numpy()]
        for a in (self.dx, *self.grads):
            b = a.numpy()
            out.append(bf16_value(b) if self.dtype == "bf16" else b)
        return out

    def want(self):
        """The same in float64, from the inputs to the clipped gradients."""
        x, wg, wu, w = (a.astype(np.float64) for a in self.host)
        gate, up = x @ wg, x @ wu
        a, slope, _ = activation64(self.act, gate)
        y = a * up
        ok = self.at >= 0
        z = y @ w.T
        top = z.max(1, keepdims=True)
        e = np.exp(z - top)
        lse = np.log(e.sum(1)) + top[:, 0]
        loss = np.where(ok, lse - z[np.arange(len(z)), np.maximum(self.at, 0)], 0)
        g = e / e.sum(1, keepdims=True)
        g[np.arange(len(z)), np.maximum(self.at, 0)] -= 1
        g = np.where(ok[:, None], g / max(1, ok.sum()), 0)
        dy = g @ w
        du, dg = dy * a, dy * up * slope
        grads = [x.T @ dg, x.T @ du, g.T @ y]
        norm = np.sqrt(sum((v ** 2).sum() for v in grads))
        by = min(1.0, self.most / (norm + 1e-6))
        return [np.array([loss.sum() / max(1, ok.sum()), ok.sum()]), np.array([norm]), loss, dg @ wg.T + du @ wu.T] + [v * by for v in grads]


def near(got, want, dtype):
    """Normwise: four products follow one another, each off by some roundings of its type (fp32: 2e-7 of the sums'
    norm each; bf16: 2^-9 on the mean of a rounding, two for each product)."""
    tol = 5e-6 if dtype == "f32" else 2e-2
    for i, (g, w) in enumerate(zip(got, want)):
        assert g.shape == w.shape and np.isfinite(g).all()
        assert np.linalg.norm(g - w) <= tol * np.linalg.norm(w) + 1e-12, i


SIZES = [(5, 64, 96, 200), (70, 136, 200, 333), (300, 256, 520, 1000)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("sizes", SIZES)
def test_a_step(ctx, sizes, act, dtype):
    s = Step(ctx, dtype, *sizes, act=act)
    for seed in (1, 2):
        s.set(seed)
        s.run()
        near(s.read(), s.want(), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", SIZES)
def test_captured_and_replayed(sizes, dtype):
    """The first call of a context is the captured one; between replays the inputs change, and eager calls that need more
    scratch run."""
    with M.Context(0) as c:
        s = Step(c, dtype, *sizes)
        more = Step(c, dtype, 2 * sizes[0] + 700, sizes[1] + 900, sizes[2] + 300, 2 * sizes[3] + 3000)
        s.set(1)
        graph = Graph(c, s.run)
        more.set(3)
        for seed in (1, 4, 5, 1):
            s.set(seed)
            graph.launch()
            c.sync()
            got = s.read()
            if seed == 4:
                more.run()
                near(more.read(), more.want(), dtype)
            s.run()
            for a, b in zip(got, s.read()):
                assert np.array_equal(a, b)
        graph.close()


def test_two_graphs_one_after_the_other():
    with M.Context(0) as c:
        a, b = Step(c, "f32", 40, 64, 96, 200), Step(c, "bf16", 150, 96, 160, 700)
        a.set(1)
        b.set(2)
        ga, gb = Graph(c, a.run), Graph(c, b.run)
        for seed in (5, 6):
            a.set(seed)
            b.set(seed + 10)
            for g in (ga, gb, ga, gb):
                g.launch()
            c.sync()
            near(a.read(), a.want(), "f32")
            near(b.read(), b.want(), "bf16")
        ga.close()
        gb.close()


def test_another_stream(ctx):
    """A stream of the program's own, and back."""
    hip, stream = Hip(ctx), ctypes.c_void_p()
    hip("hipStreamCreateWithFlags", ctypes.byref(stream), 1)
    s = Step(ctx, "bf16", 64, 96, 128, 300)
    s.set(7)
    ctx.check(ctx.lib.mimir_ctx_set_stream(ctx.handle, stream))
    try:
        s.run()
        hip("hipStreamSynchronize", stream)
        near(s.read(), s.want(), "bf16")
    finally:
        ctx.check(ctx.lib.mimir_ctx_set_stream(ctx.handle, None))
    hip("hipStreamDestroy", stream)
    s.set(8)
    s.run()
    near(s.read(), s.want(), "bf16")


def test_contexts_in_threads():
    """Contexts on one GPU share no scratch."""
    errors = []

    def work(i):
        try:
            with M.Context(0) as c:
                s = Step(c, ("f32", "bf16")[i % 2], 100 + 60 * i, 128, 200, 500)
                for seed in range(4):
                    s.set(seed + 10 * i)
                    s.run()
                    near(s.read(), s.want(), s.dtype)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_microbatches_add_up(ctx):
    """Two halves of a batch, gradients added with weights 1/2, against the whole (the same count in each)."""
    rng = np.random.default_rng(3)
    t, d, v = 128, 64, 300
    x, w = rng.standard_normal((t, d)).astype(np.float32), (rng.standard_normal((v, d)) / 8).astype(np.float32)
    at = rng.integers(0, v, t).astype(np.int32)
    X, W, T = ctx.to_device(x), ctx.to_device(w), ctx.to_device(at)
    dx, dw, dw2 = ctx.empty((t, d)), ctx.empty((v, d)), ctx.empty((v, d))
    loss, lse, mean = ctx.empty(t), ctx.empty(t), ctx.empty(2)
    ctx.linear_cross_entropy(X, W, T, t, d, v, loss, lse, mean)
    ctx.linear_cross_entropy_bwd(X, W, T, lse, None, mean, dx, dw, t, d, v)
    ctx.fill(dw2, 0.0)
    h = t // 2
    for i in (0, 1):
        xs, ts, ls = X.offset(i * h * d), T.offset(i * h), lse.offset(i * h)
        ctx.linear_cross_entropy(xs, W, ts, h, d, v, loss.offset(i * h), ls, mean)
        ctx.linear_cross_entropy_bwd(xs, W, ts, ls, None, mean, None, dw2, h, d, v, scale=0.5, accumulate_w=True)
    a, b = dw.numpy(), dw2.numpy()
    assert np.linalg.norm(a - b) <= 2e-6 * np.linalg.norm(a)
