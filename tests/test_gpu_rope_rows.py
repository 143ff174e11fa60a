"""Rotary positions per token against float64, bit for bit: pairs half the rotated
part apart and side by side, part of the head, strides, odd sizes, positions
outside the tables; the gradient against differences and the transposed formula."""
import numpy as np
import pytest

import mimir_hip as M
from _serving import rotate

pytestmark = pytest.mark.gpu


def tables(rows, rot, **kw):
    return M.rope_table_scaled(rows, rot, **kw)


def run(ctx, q, k, pos, rot, interleaved, cos_t, sin_t, back=False, ld_extra=0, offset=0, acc=None, in_place=False):
    """(q_out, k_out) of the device for q / k [tokens, heads, d]."""
    t, d = q.shape[0], q.shape[2]
    outs, args = [], []
    for x in (q, k):
        w = x.shape[1] * d
        ld = w + ld_extra
        buf = np.full(offset + max(t, 1) * ld + 4, 7.5, np.float32)
        rows = buf[offset:offset + t * ld].reshape(t, ld)
        rows[:, :w] = x.reshape(t, w)
        dev = ctx.to_device(buf)
        if in_place:
            out = dev
        else:
            o = np.full_like(buf, -3.25)
            if acc is not None:
                o[:] = acc
            out = ctx.to_device(o)
        args.append((dev, out, ld))
    rope = M.Rope(ctx.to_device(cos_t), ctx.to_device(sin_t), cos_t.shape[0], rot, interleaved)
    dpos = ctx.to_device(np.asarray(pos, np.int32)) if t else ctx.empty(1, np.int32)
    call = ctx.rope_rows_bwd if back else ctx.rope_rows
    extra = {"accumulate": acc is not None} if back else {}
    (dq, oq, lq), (dk, ok, lk) = args
    call(dq.offset(offset), oq.offset(offset), q.shape[1], dk.offset(offset), ok.offset(offset), k.shape[1], t, d, dpos, rope,
         ld_q=lq, ld_k=lk, ld_q_out=lq, ld_k_out=lk, **extra)
    for x, (dev, out, ld) in zip((q, k), args):
        w = x.shape[1] * d
        got = out.numpy()
        rows = got[offset:offset + t * ld].reshape(t, ld)
        # What is not a head stays as it was.
        keep = 7.5 if in_place else (acc if acc is not None else -3.25)
        assert (got[:offset] == keep).all() and (got[offset + t * ld:] == keep).all() and (rows[:, w:] == keep).all()
        outs.append(rows[:, :w].reshape(x.shape).copy())
    return outs


def rand(seed, t, hq, hk, d):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((t, hq, d)).astype(np.float32), rng.standard_normal((t, hk, d)).astype(np.float32),
            rng.integers(0, 40, t))


# tokens, q heads, k heads, head_dim, rot_dim: vector rows, rows of odd vectors,
# scalar rows (odd heads, rotated parts that are no multiple of 8), more slots than
# a workgroup's, no tokens.
CASES = [(1, 1, 1, 8, 8), (7, 32, 8, 128, 128), (5, 4, 2, 128, 64), (3, 2, 2, 80, 32), (9, 3, 1, 36, 16), (33, 5, 5, 12, 8),
         (4, 2, 1, 7, 6), (6, 3, 2, 10, 2), (2, 1, 1, 2, 2), (3, 2, 2, 66, 60), (300, 8, 8, 64, 64), (0, 2, 2, 16, 16),
         (11, 2, 1, 320, 128), (5, 1, 3, 4, 4)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hk,d,rot", CASES)
def test_forward_bits(ctx, t, hq, hk, d, rot, interleaved):
    q, k, pos = rand(t + d, t, hq, hk, d)
    c, s = tables(40, rot)
    for back in (False, True):
        got = run(ctx, q, k, pos, rot, interleaved, c, s, back=back)
        for x, y in zip((q, k), got):
            np.testing.assert_array_equal(y, rotate(x, pos, c, s, rot, interleaved, back))


@pytest.mark.parametrize("ld_extra,offset", [(0, 1), (3, 0), (4, 4), (17, 2)])
def test_strides_and_alignment(ctx, ld_extra, offset):
    q, k, pos = rand(1, 13, 3, 2, 24)
    c, s = tables(40, 16)
    got = run(ctx, q, k, pos, 16, False, c, s, ld_extra=ld_extra, offset=offset)
    for x, y in zip((q, k), got):
        np.testing.assert_array_equal(y, rotate(x, pos, c, s, 16, False))


@pytest.mark.parametrize("d,rot,interleaved", [(32, 32, False), (32, 16, True), (9, 6, False)])
def test_in_place(ctx, d, rot, interleaved):
    q, k, pos = rand(2, 21, 4, 2, d)
    c, s = tables(40, rot)
    got = run(ctx, q, k, pos, rot, interleaved, c, s, in_place=True)
    for x, y in zip((q, k), got):
        np.testing.assert_array_equal(y, rotate(x, pos, c, s, rot, interleaved))


@pytest.mark.parametrize("d,rot", [(32, 32), (10, 6)])
def test_positions_outside_the_table_give_zeros(ctx, d, rot):
    q, k, _ = rand(3, 6, 2, 1, d)
    pos = np.array([-1, 0, 39, 40, 2 ** 31 - 1, -2 ** 31])
    c, s = tables(40, rot)
    got = run(ctx, q, k, pos, rot, False, c, s)
    for x, y in zip((q, k), got):
        np.testing.assert_array_equal(y, rotate(x, pos, c, s, rot, False))
        assert not y[[0, 3, 4, 5]].any()
    # A gradient that accumulates gets nothing there.
    got = run(ctx, q, k, pos, rot, False, c, s, back=True, acc=2.0)
    for x, y in zip((q, k), got):
        np.testing.assert_array_equal(y, np.float32(2) + rotate(x, pos, c, s, rot, False, back=True))


@pytest.mark.parametrize("d,rot,interleaved", [(64, 64, False), (64, 32, True), (6, 4, True)])
def test_accumulate(ctx, d, rot, interleaved):
    q, k, pos = rand(4, 19, 3, 2, d)
    c, s = tables(40, rot)
    got = run(ctx, q, k, pos, rot, interleaved, c, s, back=True, acc=0.75)
    for x, y in zip((q, k), got):
        np.testing.assert_array_equal(y, np.float32(0.75) + rotate(x, pos, c, s, rot, interleaved, back=True))


def test_gradient_against_differences(ctx):
    """<dy, R(x + h) - R(x - h)> / 2h is dx: the rotation is linear, so a step of 1
    is exact up to the roundings of its two values: 2 heads of 8 dimensions, each
    value below 2^3, off by half a step 2^-22 at most, twice."""
    q, k, pos = rand(5, 2, 1, 1, 8)
    c, s = tables(40, 6, magnitude=1.25)
    dy, _, _ = rand(6, 2, 1, 1, 8)
    dx = run(ctx, dy, dy, pos, 6, True, c, s, back=True)[0]
    for t in range(2):
        for i in range(8):
            up, down = q.copy(), q.copy()
            up[t, 0, i] += 1
            down[t, 0, i] -= 1
            yu = run(ctx, up, k, pos, 6, True, c, s)[0].astype(np.float64)
            yd = run(ctx, down, k, pos, 6, True, c, s)[0].astype(np.float64)
            step = float(up[t, 0, i]) - float(down[t, 0, i])
            want = ((yu - yd) * dy).sum() / step
            assert abs(want - dx[t, 0, i]) <= 8 * 2.0 ** -22 * np.abs(dy).max() + 2.0 ** -22


def test_one_side_only(ctx):
    q, k, pos = rand(7, 5, 3, 2, 16)
    c, s = tables(40, 16)
    rope = M.Rope(ctx.to_device(c), ctx.to_device(s), 40, 16)
    dp = ctx.to_device(pos.astype(np.int32))
    for x in (q, k):
        h = x.shape[1]
        dx, out = ctx.to_device(x), ctx.empty(x.shape)
        ctx.rope_rows(None, None, 0, dx, out, h, 5, 16, dp, rope)
        np.testing.assert_array_equal(out.numpy(), rotate(x, pos, c, s, 16, False))
        ctx.rope_rows(dx, out, h, None, None, 0, 5, 16, dp, rope)
        np.testing.assert_array_equal(out.numpy(), rotate(x, pos, c, s, 16, False))


def test_agrees_with_rope_at_consecutive_positions(ctx):
    """mimir_rope_fwd takes fp32 products: one rounding of each and of their sum."""
    rng = np.random.default_rng(8)
    q, k = (rng.standard_normal((1, 50, 4, 64)).astype(np.float32) for _ in range(2))
    c, s = M.rope_table(60, 64)
    dc, ds = ctx.to_device(c), ctx.to_device(s)
    dq, dk, oq, ok = ctx.to_device(q), ctx.to_device(k), ctx.empty(q.shape), ctx.empty(k.shape)
    ctx.rope(dq, oq, 4, dk, ok, 4, 1, 50, 64, 5, dc, ds, 60)
    ours = run(ctx, q[0], k[0], np.arange(5, 55), 64, False, c, s)
    for a, b, x in zip((oq, ok), ours, (q[0], k[0])):
        size = np.abs(x).reshape(50, 4, 2, 32).sum(2)  # |x0| + |x1| bounds both products
        bound = 2.0 * 2.0 ** -24 * np.concatenate((size, size), -1)
        assert (np.abs(a.numpy()[0] - b) <= bound).all()


def test_kept_outputs_have_the_same_bits(ctx):
    q, k, pos = rand(9, 40, 4, 2, 64)
    c, s = tables(40, 64)
    a = run(ctx, q, k, pos, 64, False, c, s)
    ctx.set_output_caching(True)
    try:
        b = run(ctx, q, k, pos, 64, False, c, s)
    finally:
        ctx.set_output_caching(False)
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x, y)
