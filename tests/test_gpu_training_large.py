"""Training operators on matrices of more than 2^31 elements, gradients among them,
against float64 in the rows where an offset of 32 bits would go wrong: the last ones,
and the first."""
import numpy as np
import pytest

from _serving import bf16_bits, bf16_value
from _training import U, UB, activation64, held, steps

pytestmark = pytest.mark.gpu
KIND = {"f32": np.float32, "bf16": np.uint16}


def stored(a, dtype):
    return bf16_bits(a) if dtype == "bf16" else np.asarray(a, np.float32)


def read(buf, first, shape, dtype):
    a = buf.offset(first, shape).numpy()
    return bf16_value(a) if dtype == "bf16" else a


def constant(ctx, buf, value, dtype):
    """A whole buffer of one value (bf16: pairs of them as one float's bits)."""
    if dtype == "bf16":
        bits = int(bf16_bits(np.float32([value]))[0])
        pair = np.array([bits | bits << 16], np.uint32).view(np.float32)[0]
        ctx.check(ctx.lib.mimir_fill_f32(ctx.handle, buf.ptr, buf.size // 2, pair))
    else:
        ctx.fill(buf, value)


@pytest.mark.parametrize("dtype,dim", [("f32", 4099), ("bf16", 4104)])
def test_cross_entropy_of_a_large_vocabulary(ctx, dtype, dim):
    """w and dw of 2.2 G elements.  All rows of w but the last ones are zeros, so their logits are 0 and their rows of dw
    are all -- but for targets -- the same sum of x."""
    tokens, vocab, last = 40, 530000, 50
    rng = np.random.default_rng(1)
    x = held(rng.standard_normal((tokens, dim)), dtype)
    tail = held(rng.standard_normal((last, dim)) * (3 / np.sqrt(dim)), dtype)
    target = rng.integers(0, vocab, tokens).astype(np.int32)
    target[:8] = vocab - 1 - np.arange(8)
    target[8], target[9] = -1, 0
    w, dw, dx = ctx.empty(vocab * dim, KIND[dtype]), ctx.empty(vocab * dim, KIND[dtype]), ctx.empty((tokens, dim), KIND[dtype])
    constant(ctx, w, 0.0, dtype)
    w.offset((vocab - last) * dim, (last, dim)).upload(stored(tail, dtype))
    X, T = ctx.to_device(stored(x, dtype)), ctx.to_device(target)
    loss, lse = ctx.empty(tokens), ctx.empty(tokens)
    ctx.linear_cross_entropy(X, w, T, tokens, dim, vocab, loss, lse, dtype=dtype)
    ctx.linear_cross_entropy_bwd(X, w, T, lse, None, None, dx, dw, tokens, dim, vocab, dtype=dtype)
    ok = target >= 0
    z = x.astype(np.float64) @ tail.astype(np.float64).T
    ez = np.abs(x.astype(np.float64)) @ np.abs(tail.astype(np.float64)).T * steps(dim) * U
    want = np.where(ok, np.log(vocab - last + np.exp(z).sum(1)), 0)
    in_tail = np.where(ok & (target >= vocab - last), z[np.arange(tokens), np.maximum(target - vocab + last, 0)], 0)
    # Sums of ones in tiles of 64 to 256 rows, joined over some thousand tiles; logits up to 12.
    e_lse = ez.max(1) + (140 + 4 * vocab / 64 / 32 + 40) * U + 2 * U * want
    assert (np.abs(lse.numpy() - want) <= e_lse).all()
    assert (np.abs(loss.numpy() - np.where(ok, want - in_tail, 0)) <= e_lse + ez.max(1) + U * want).all()
    half = UB if dtype == "bf16" else U
    rel = UB * UB if dtype == "bf16" else 0  # G in two terms

    def g_of(rows, logits, e_logits):
        p = np.exp(logits - want[:, None])
        g = np.where(ok[:, None], p - (target[:, None] == rows[None, :]), 0)
        e = np.where(ok[:, None], p * (e_logits + e_lse[:, None] + (3 * np.abs(logits - want[:, None]) + 4) * U), 0)
        return g, e + np.abs(g) * (rel + 3 * U)

    ax = np.abs(x.astype(np.float64))
    for first, logits, e in ((vocab - last, z, ez), (vocab - 2 * last, np.zeros_like(z), 0 * ez), (0, np.zeros_like(z), 0 * ez)):
        g, eg = g_of(first + np.arange(last), logits, e)
        rows = g.T @ x.astype(np.float64)
        bound = eg.T @ ax + (np.abs(g) + eg).T @ ax * steps(tokens) * U + 1.1 * half * np.abs(rows)
        assert (np.abs(read(dw, first * dim, (last, dim), dtype) - rows) <= 1.05 * bound + 2.0 ** -120).all(), first
    g, eg = g_of(vocab - last + np.arange(last), z, ez)
    at = np.abs(tail.astype(np.float64))
    rows = g @ tail.astype(np.float64)
    bound = eg @ at + (np.abs(g) + eg) @ at * (steps(vocab) + 100) * U + 1.1 * half * np.abs(rows)
    got = read(dx, 0, (tokens, dim), dtype)
    assert (np.abs(got - rows) <= 1.05 * bound + 2.0 ** -120).all() and (got[~ok] == 0).all()
    for b in (w, dw, dx):
        b.free()


@pytest.mark.parametrize("dtype,dim", [("f32", 4099), ("bf16", 4104)])
def test_cross_entropy_of_many_tokens(ctx, dtype, dim):
    """x and dx of 2.2 G elements: all tokens but the last are alike."""
    tokens, vocab, last = 530000, 20, 50
    rng = np.random.default_rng(2)
    w = held(rng.standard_normal((vocab, dim)) * (2 / np.sqrt(dim)), dtype)
    tail = held(rng.standard_normal((last, dim)), dtype)
    x, dx = ctx.empty(tokens * dim, KIND[dtype]), ctx.empty(tokens * dim, KIND[dtype])
    constant(ctx, x, 0.25, dtype)
    x.offset((tokens - last) * dim, (last, dim)).upload(stored(tail, dtype))
    target = rng.integers(-1, vocab, tokens).astype(np.int32)
    W, T = ctx.to_device(stored(w, dtype)), ctx.to_device(target)
    dw = ctx.empty((vocab, dim), KIND[dtype])
    loss, lse = ctx.empty(tokens), ctx.empty(tokens)
    ctx.linear_cross_entropy(x, W, T, tokens, dim, vocab, loss, lse, dtype=dtype)
    ctx.linear_cross_entropy_bwd(x, W, T, lse, None, None, dx, dw, tokens, dim, vocab, dtype=dtype)
    half = UB if dtype == "bf16" else U
    w64, got_lse, got_loss = w.astype(np.float64), lse.numpy(), loss.numpy()
    for first, rows in ((tokens - last, tail), (0, np.full((last, dim), 0.25, np.float32))):
        rows = rows.astype(np.float64)
        t = target[first:first + last]
        ok = t >= 0
        z = rows @ w64.T
        ez = (np.abs(rows) @ np.abs(w64).T * steps(dim) * U).max(1)
        want = np.where(ok, np.log(np.exp(z).sum(1)), 0)
        e_lse = ez + 200 * U + 2 * U * np.abs(want)
        assert (np.abs(got_lse[first:first + last] - want) <= e_lse).all()
        assert (np.abs(got_loss[first:first + last] - np.where(ok, want - z[np.arange(last), np.maximum(t, 0)], 0)) <= 2 * e_lse + 10 * U).all()
        p = np.where(ok[:, None], np.exp(z - want[:, None]), 0)
        g = p.copy()
        g[np.arange(last)[ok], t[ok]] -= 1
        eg = p * ((ez + e_lse)[:, None] + (3 * np.abs(z - want[:, None]) + 4) * U) + np.abs(g) * (half + 3 * U)
        d = g @ w64
        bound = eg @ np.abs(w64) + (np.abs(g) + eg) @ np.abs(w64) * 20 * U + 1.1 * half * np.abs(d)
        got = read(dx, first * dim, (last, dim), dtype)
        assert (np.abs(got - d) <= 1.05 * bound + 2.0 ** -120).all() and (got[~ok] == 0).all()
    for b in (x, dx):
        b.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gated_gradients_of_many_tokens(ctx, dtype):
    """gate_up of 2.3 G values, dy of 1.15 G: the last rows of dx, the first and last columns of both weights' gradients."""
    tokens, dim, hidden, last, c = 70001, 8, 16384, 3, 0.5
    rng = np.random.default_rng(3)
    x = held(rng.standard_normal((tokens, dim)), dtype)
    wg, wu = (held(rng.standard_normal((dim, hidden)) / np.sqrt(dim), dtype) for _ in range(2))
    X, G, W = (ctx.to_device(stored(a, dtype)) for a in (x, wg, wu))
    y, dy, gu = ctx.empty(tokens * hidden, KIND[dtype]), ctx.empty(tokens * hidden, KIND[dtype]), ctx.empty(tokens * 2 * hidden)
    dx, dg, du = ctx.empty((tokens, dim), KIND[dtype]), ctx.empty((dim, hidden), KIND[dtype]), ctx.empty((dim, hidden), KIND[dtype])
    constant(ctx, dy, c, dtype)
    if tokens * hidden % 2 and dtype == "bf16":
        dy.offset(tokens * hidden - 1, (1,)).upload(stored(np.float32([c]), dtype))
    ctx.gated_linear(X, G, W, y, tokens, dim, hidden, gate_up=gu, dtype=dtype)
    ctx.gated_linear_bwd(X, G, W, gu, dy, dx, dg, du, tokens, dim, hidden, dtype=dtype)
    half, rel = (UB, UB) if dtype == "bf16" else (U, 0)

    def parts(xs, g, u):
        """dg, du and what they may be off by (gates below 20)."""
        xs, g, u = (v.astype(np.float64) for v in (xs, g, u))
        gate, up = xs @ g, xs @ u
        eg, eu = (np.abs(xs) @ np.abs(v) * steps(dim) * U for v in (g, u))
        a, slope, v = activation64("silu", gate)
        ea, es = 1.2 * eg + np.abs(a) * (10 + 6 * np.abs(v)) * U, 1.7 * eg + (12 + 6 * np.abs(v)) * 2 * U
        d_gate, d_up = c * up * slope, c * a
        return ((d_gate, c * (eu * (np.abs(slope) + es) + np.abs(up) * es) + np.abs(d_gate) * (rel + 3 * U)),
                (d_up, c * ea + np.abs(d_up) * (rel + 3 * U)))

    (a, ea), (b, eb) = parts(x[-last:], wg, wu)
    wg64, wu64 = wg.astype(np.float64), wu.astype(np.float64)
    want = a @ wg64.T + b @ wu64.T
    bound = ea @ np.abs(wg64).T + eb @ np.abs(wu64).T + ((np.abs(a) + ea) @ np.abs(wg64).T + (np.abs(b) + eb) @ np.abs(wu64).T) * (
        steps(2 * hidden) + 100) * U + 1.1 * half * np.abs(want)
    assert (np.abs(read(dx, (tokens - last) * dim, (last, dim), dtype) - want) <= 1.05 * bound).all()
    got_g, got_u = read(dg, 0, (dim, hidden), dtype), read(du, 0, (dim, hidden), dtype)
    x64 = x.astype(np.float64)
    for cols in (slice(0, 3), slice(hidden - 3, hidden)):
        for got, (d, e) in zip((got_g, got_u), parts(x, wg[:, cols], wu[:, cols])):
            want = x64.T @ d
            bound = np.abs(x64).T @ e + np.abs(x64).T @ (np.abs(d) + e) * (steps(tokens) + 100) * U + 1.1 * half * np.abs(want)
            assert (np.abs(got[:, cols] - want) <= 1.05 * bound).all()
    for v in (y, dy, gu):
        v.free()
