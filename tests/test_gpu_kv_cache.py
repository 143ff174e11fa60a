"""The paged cache written and read back, bit for bit against numpy: every type,
page size and head width, single tokens and prompts, rotation on the way, rows that
no sequence has, pages that the cache does not have, rows of zeros, NaN and
infinities, and the border between two 8-bit codes."""
import numpy as np
import pytest

import mimir_hip as M
from _serving import Paged, bf16_bits, held, i8_rows, rotate

pytestmark = pytest.mark.gpu
TYPES = ["f32", "bf16", "i8"]


def append(ctx, p, k, v, q=None, rope=None, tables=None, ld_extra=0, offset=0):
    """kv_append of packed rows (k, v, q [tokens, heads, d]); (cache, batch, q_out)."""
    cache, batch = p.device()
    t, d = k.shape[0], p.d

    def rows(x, ld):
        buf = np.full(offset + t * ld, 99.0, np.float32)
        buf[offset:].reshape(t, ld)[:, :x.shape[1] * d] = x.reshape(t, -1)
        return ctx.to_device(buf).offset(offset)

    ld = p.kv_heads * d + ld_extra
    out, ld_q, heads = None, None, 0
    if q is not None:
        heads = q.shape[1]
        ld_q = heads * d + ld_extra
        out = ctx.to_device(np.full((t, ld_q), -5.0, np.float32))
    ctx.kv_append(cache, batch, rows(k, ld), rows(v, ld), ld_kv=ld, rope=rope, q=rows(q, ld_q) if q is not None else None,
                  q_out=out, heads=heads, ld_q=ld_q, ld_q_out=ld_q)
    got = None
    if q is not None:
        o = out.numpy()
        assert (o[:, heads * d:] == -5).all()
        got = o[:, :heads * d].reshape(q.shape)
    return cache, batch, got


def expected(p, k, v):
    """The cache's host arrays after the batch's rows went in."""
    import copy
    e = copy.copy(p)
    e.host = {n: a.copy() for n, a in p.host.items()}
    e.scale = {n: a.copy() for n, a in p.scale.items()}
    for s, (n, m) in enumerate(p.lens):
        for i in range(n):
            pos = m - n + i
            if pos < 0:
                continue
            page, at = p.slot(s, pos)
            if not 0 <= page < p.pages:
                continue
            for name, x in (("k", k), ("v", v)):
                x = x[p.start[s] + i]
                row = e.host[name][page, :, at]
                row[:] = 0
                if p.dtype == "f32":
                    row[:, :p.d] = x
                elif p.dtype == "bf16":
                    row[:, :p.d] = bf16_bits(x)
                else:
                    row[:, :p.d], e.scale[name][page, :, at] = i8_rows(x)
    return e


def assert_cache(p, cache, e):
    for name, dev in (("k", cache.k), ("v", cache.v)):
        got, want = dev.numpy(), e.host[name]
        if p.dtype == "f32":  # NaN slots stay NaN
            got, want = got.view(np.uint32), want.view(np.uint32)
        np.testing.assert_array_equal(got, want, err_msg=name)
    if p.dtype == "i8":
        for name, dev in (("k", cache.k_scale), ("v", cache.v_scale)):
            np.testing.assert_array_equal(dev.numpy().view(np.uint32) & 0x7FFFFFFF, e.scale[name].view(np.uint32) & 0x7FFFFFFF)


def rand_rows(seed, *shapes):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal(s).astype(np.float32) for s in shapes]


# lens, kv heads, head_dim, page: one token, pages that a prompt ends in the middle
# of or fills, sequences without new tokens, every lane width (8, 16, 32), heads
# that are no multiple of 4 or 16, an empty first and last sequence.
BATCHES = [([(1, 1)], 1, 64, 16), ([(1, 17), (1, 16), (1, 33)], 2, 128, 16), ([(16, 16), (5, 40)], 3, 80, 16),
           ([(0, 20), (3, 3), (0, 0), (50, 70)], 2, 32, 32), ([(7, 100)], 1, 256, 48), ([(4, 5), (2, 9)], 2, 7, 16),
           ([(3, 30)], 5, 100, 64), ([(2, 2), (9, 200)], 1, 1, 16), ([(70, 70)], 2, 130, 80), ([(1, 3)] * 70, 1, 16, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,kh,d,page", BATCHES)
def test_append_and_read(ctx, dtype, lens, kh, d, page):
    p = Paged(ctx, dtype, lens, kh, d, page, seed=d)
    k, v = rand_rows(d, (p.tokens, kh, d), (p.tokens, kh, d))
    cache, batch, _ = append(ctx, p, k, v)
    assert_cache(p, cache, expected(p, k, v))
    ko, vo = ctx.empty((p.tokens, kh, d)), ctx.empty((p.tokens, kh, d))
    ctx.kv_read(cache, batch, ko, vo)
    np.testing.assert_array_equal(ko.numpy(), held(k, dtype))
    np.testing.assert_array_equal(vo.numpy(), held(v, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,kh,ld_extra", [(32, 3, 2, 0), (128, 4, 1, 0), (7, 2, 2, 1)])
def test_many_tokens(ctx, dtype, d, heads, kh, ld_extra):
    """Enough for several a workgroup, whose last one is not full; sequences that end
    inside one, some without new tokens."""
    lens = [(4000, 4000), (1, 9), (0, 0), (1, 1), (1, 1), (0, 5), (4998, 5010)]
    p = Paged(ctx, dtype, lens, kh, d, 64, seed=d)
    k, v, q = rand_rows(d + 1, (p.tokens, kh, d), (p.tokens, kh, d), (p.tokens, heads, d))
    rot = d // 2 * 2
    c, s = M.rope_table_scaled(5010, rot)
    rope = M.Rope(ctx.to_device(c), ctx.to_device(s), 5010, rot, False)
    pos = np.concatenate([np.arange(m - n, m) for n, m in lens])
    cache, batch, got = append(ctx, p, k, v, q, rope, ld_extra=ld_extra)
    np.testing.assert_array_equal(got, rotate(q, pos, c, s, rot, False))
    turned = rotate(k, pos, c, s, rot, False)
    assert_cache(p, cache, expected(p, turned, v))
    ld = kh * d + ld_extra
    ko, vo = (ctx.to_device(np.full((p.tokens, ld), -4.0, np.float32)) for _ in range(2))
    ctx.kv_read(cache, batch, ko, vo, ld_out=ld)
    for out, x in ((ko, turned), (vo, v)):
        o = out.numpy()
        np.testing.assert_array_equal(o[:, :kh * d].reshape(x.shape), held(x, dtype))
        assert (o[:, kh * d:] == -4).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_kept_outputs_have_the_same_bits(ctx, dtype):
    """Queries and rows read back written with plain stores."""
    lens, d = [(30, 40), (1, 2)], 64
    p = Paged(ctx, dtype, lens, 2, d, 16)
    k, v, q = rand_rows(8, (31, 2, d), (31, 2, d), (31, 4, d))
    c, s = M.rope_table_scaled(40, d)
    rope = M.Rope(ctx.to_device(c), ctx.to_device(s), 40, d, False)
    pos = np.concatenate([np.arange(m - n, m) for n, m in lens])
    ctx.set_output_caching(True)
    try:
        cache, batch, got = append(ctx, p, k, v, q, rope)
        ko = ctx.empty((31, 2, d))
        ctx.kv_read(cache, batch, ko, None)
        ko = ko.numpy()
    finally:
        ctx.set_output_caching(False)
    np.testing.assert_array_equal(got, rotate(q, pos, c, s, d, False))
    np.testing.assert_array_equal(ko, held(rotate(k, pos, c, s, d, False), dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot,interleaved", [(128, 128, False), (64, 32, True), (80, 16, False), (256, 256, True), (10, 6, False),
                                               (6, 6, True), (37, 20, True), (48, 4, False)])
def test_append_rotated(ctx, dtype, d, rot, interleaved):
    lens, kh, heads = [(3, 20), (1, 1), (11, 50)], 2, 6
    p = Paged(ctx, dtype, lens, kh, d, 16, seed=1)
    k, v, q = rand_rows(2 + d, (15, kh, d), (15, kh, d), (15, heads, d))
    c, s = M.rope_table_scaled(50, rot)
    rope = M.Rope(ctx.to_device(c), ctx.to_device(s), 50, rot, interleaved)
    pos = np.concatenate([np.arange(m - n, m) for n, m in lens])
    cache, _, got = append(ctx, p, k, v, q, rope)
    assert_cache(p, cache, expected(p, rotate(k, pos, c, s, rot, interleaved), v))
    np.testing.assert_array_equal(got, rotate(q, pos, c, s, rot, interleaved))
    # Keys alone.
    cache, _, _ = append(ctx, p, k, v, None, rope)
    assert_cache(p, cache, expected(p, rotate(k, pos, c, s, rot, interleaved), v))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ld_extra,offset", [(4, 0), (3, 0), (0, 1), (8, 4)])
def test_strides_and_alignment(ctx, dtype, ld_extra, offset):
    p = Paged(ctx, dtype, [(5, 9), (4, 30)], 2, 24, 16)
    k, v, q = rand_rows(3, (9, 2, 24), (9, 2, 24), (9, 4, 24))
    c, s = M.rope_table_scaled(30, 8)
    rope = M.Rope(ctx.to_device(c), ctx.to_device(s), 30, 8)
    pos = np.concatenate([np.arange(4, 9), np.arange(26, 30)])
    cache, batch, got = append(ctx, p, k, v, q, rope, ld_extra=ld_extra, offset=offset)
    kr = rotate(k, pos, c, s, 8, False)
    assert_cache(p, cache, expected(p, kr, v))
    np.testing.assert_array_equal(got, rotate(q, pos, c, s, 8, False))
    ld = 48 + ld_extra
    out = ctx.to_device(np.full(offset + 9 * ld, -5.0, np.float32))
    ctx.kv_read(cache, batch, None, out.offset(offset), ld_out=ld)
    o = out.numpy()[offset:].reshape(9, ld)
    np.testing.assert_array_equal(o[:, :48].reshape(9, 2, 24), held(v, dtype))
    assert (o[:, 48:] == -5).all() and (out.numpy()[:offset] == -5).all()


def test_query_in_place(ctx):
    p = Paged(ctx, "bf16", [(6, 6)], 1, 32, 16)
    k, v, q = rand_rows(4, (6, 1, 32), (6, 1, 32), (6, 2, 32))
    c, s = M.rope_table_scaled(6, 32)
    rope = M.Rope(ctx.to_device(c), ctx.to_device(s), 6, 32)
    cache, batch = p.device()
    dq = ctx.to_device(q)
    ctx.kv_append(cache, batch, ctx.to_device(k), ctx.to_device(v), rope=rope, q=dq, q_out=dq, heads=2)
    np.testing.assert_array_equal(dq.numpy(), rotate(q, np.arange(6), c, s, 32, False))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_behind_the_last_sequence_and_pages_that_are_none(ctx, dtype):
    """Rows that no sequence has are left as they are; pages outside the cache and
    positions below 0 hold nothing and read as zeros."""
    lens = [(3, 3), (5, 2), (20, 40), (1, 1)]  # the second has more new tokens than cached ones
    p = Paged(ctx, dtype, lens, 2, 20, 16, tokens=35)
    p.table[2, 1] = p.pages  # positions 16 .. 31 of the third
    p.table[3, 0] = -1
    k, v, q = rand_rows(5, (35, 2, 20), (35, 2, 20), (35, 2, 20))
    c, s = M.rope_table_scaled(40, 16)
    rope = M.Rope(ctx.to_device(c), ctx.to_device(s), 40, 16)
    pos = np.concatenate([np.arange(m - n, m) for n, m in lens])
    kr = k.copy()
    kr[:29] = rotate(k[:29], pos, c, s, 16, False)
    cache, batch, got = append(ctx, p, k, v, q, rope)
    e = expected(p, kr, v)
    assert_cache(p, cache, e)
    np.testing.assert_array_equal(got[:29], rotate(q[:29], pos, c, s, 16, False))
    assert (got[29:] == -5).all() and not got[3:6].any()
    out = ctx.to_device(np.full((35, 2, 20), -5.0, np.float32))
    ctx.kv_read(cache, batch, out, None)
    want = held(kr, dtype)
    want[29:] = -5
    want[3:6] = 0            # positions -3 .. -1
    third = np.arange(20, 40)
    want[8:28][third < 32] = 0
    want[28] = 0
    np.testing.assert_array_equal(out.numpy(), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_bounds_hold_whatever_the_arrays_say(ctx, dtype):
    """Starts and lengths past the host's bounds: nothing outside the buffers is
    read or written, and a sequence within them is served."""
    p = Paged(ctx, dtype, [(4, 20), (3, 10)], 1, 16, 16, spare_pages=3)
    k, v = rand_rows(6, (7, 1, 16), (7, 1, 16))
    both, p.lens = p.lens, [(4, 20)]
    want = expected(p, k, v)
    p.lens = both
    p.start = np.array([0, 4, 1 << 30], np.int32)
    p.kv_len = np.array([20, 1 << 30], np.int32)  # held to 20 keys, 4 new tokens
    cache, _, _ = append(ctx, p, k, v)
    mine = [p.table[0, 0], p.table[0, 1]]
    got = cache.k.numpy()
    w = want.host["k"]
    if dtype == "f32":
        got, w = got.view(np.uint32), w.view(np.uint32)
    np.testing.assert_array_equal(got[mine], w[mine])


def test_eight_bit_special_rows(ctx):
    p = Paged(ctx, "i8", [(9, 9)], 1, 20, 16)
    k, v = rand_rows(7, (9, 1, 20), (9, 1, 20))
    k[0] = 0
    k[1, 0, 3] = np.nan
    k[2, 0, 19] = -np.inf
    k[3] *= np.float32(1e-38)            # a scale below the normal floats
    k[4] = np.float32(3e38) * np.sign(k[4])
    k[5] = 0
    k[5, 0, 7] = np.float32(1e-45)       # the smallest subnormal
    k[6, 0] = np.float32(2.0) * np.arange(-10, 10)
    k[7, 0, 1:] = 0
    k[8] = -0.0
    cache, batch, _ = append(ctx, p, k, v)
    assert_cache(p, cache, expected(p, k, v))
    out = ctx.empty((9, 1, 20))
    ctx.kv_read(cache, batch, out, None)
    got = out.numpy()
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all() and not got[0].any() and not got[8].any()
    np.testing.assert_array_equal(got[[3, 4, 5, 6, 7]], held(k, "i8")[[3, 4, 5, 6, 7]])


def test_bf16_special_values(ctx):
    p = Paged(ctx, "bf16", [(1, 1)], 1, 16, 16)
    k = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 3.4e38, 1e-40, 1.00390625, 1.01171875, -1.00390625, 65535.9, 2.0 ** -133,
                  2.0 ** -134, 1.5, -7.0, 1e30], np.float32).reshape(1, 1, 16)
    cache, batch, _ = append(ctx, p, k, k)
    page, at = p.slot(0, 0)
    got = bf16_bits(k[0, 0])
    dev = cache.k.numpy()[page, 0, at]
    assert (dev[0] & 0x7F80) == 0x7F80 and (dev[0] & 0x7F)  # some NaN
    np.testing.assert_array_equal(dev[1:], got[1:])


def test_eight_bit_codes_next_to_their_borders(ctx):
    """Quotients x * 127 / max at and one step around k + 1/2, for many maxima."""
    rng = np.random.default_rng(8)
    d, n = 256, 400
    k = np.zeros((n, 1, d), np.float32)
    for t in range(n):
        m = np.float32(rng.uniform(0.5, 4) * 2.0 ** rng.integers(-60, 60)) if t % 4 else np.float32(127.0 * 2.0 ** rng.integers(-9, 9))
        half = rng.integers(-126, 126, d - 1) + 0.5
        x = (half * float(m) / 127.0).astype(np.float32)
        step = rng.integers(-1, 2, d - 1)
        x = np.where(step > 0, np.nextafter(x, np.float32(np.inf)), np.where(step < 0, np.nextafter(x, np.float32(-np.inf)), x))
        k[t, 0, 1:] = x
        k[t, 0, 0] = m
    p = Paged(ctx, "i8", [(n, n)], 1, d, 16)
    cache, _, _ = append(ctx, p, k, k)
    assert_cache(p, cache, expected(p, k, k))


@pytest.mark.parametrize("dtype", TYPES)
def test_whole_sequences_read_back(ctx, dtype):
    """Appended in steps, read at once: a batch whose new tokens are all cached ones."""
    kh, d = 2, 40
    total = [23, 50]
    p = Paged(ctx, dtype, [(t, t) for t in total], kh, d, 16)
    k, v = rand_rows(9, (73, kh, d), (73, kh, d))
    cache, whole = p.device()
    done = [0, 0]
    for step in ([10, 1], [1, 30], [12, 19]):
        rows = np.concatenate([np.arange(done[0], done[0] + step[0]), 23 + np.arange(done[1], done[1] + step[1])])
        done = [done[s] + step[s] for s in range(2)]
        b = M.KVBatch(ctx.to_device(np.array([0, step[0], sum(step)], np.int32)), ctx.to_device(np.array(done, np.int32)),
                      ctx.to_device(p.table), 2, sum(step), p.ld, max(step), 50)
        ctx.kv_append(cache, b, ctx.to_device(k[rows]), ctx.to_device(v[rows]))
    ko, vo = ctx.empty(k.shape), ctx.empty(v.shape)
    ctx.kv_read(cache, whole, ko, vo)
    np.testing.assert_array_equal(ko.numpy(), held(k, dtype))
    np.testing.assert_array_equal(vo.numpy(), held(v, dtype))


def test_cache_of_its_own_buffers(ctx):
    cache = M.KVCache(ctx, "i8", 3, 16, 2, 20)
    assert cache.k.shape == (3, 2, 16, 32) and cache.k_scale.shape == (3, 2, 16) and cache.k.dtype == np.int8
    cache.close()
    with pytest.raises(M.MimirError):
        M.KVCache(ctx, "f32", 3, 17, 2, 20)
