"""Attention of new tokens over a paged cache against float64: every cache type,
single tokens and chunks, shared heads, page sizes, odd lengths and head widths;
NaN and infinities in keys that a token does not see; rows without keys, rows
behind the last sequence, pages that are none; splits of the keys; graphs."""
import numpy as np
import pytest

import mimir_hip as M
from _serving import Paged, attention64, held

pytestmark = pytest.mark.gpu
TYPES = ["f32", "bf16", "i8"]
SENTINEL = -77.0


def case(seed, dtype, lens, kh, heads, d, amp=1.0):
    """(q [tokens, heads, d], per sequence the k and v that the cache holds)."""
    rng = np.random.default_rng(seed)
    tokens = sum(n for n, _ in lens)
    q = (amp * rng.standard_normal((max(tokens, 1), heads, d))).astype(np.float32)
    kv = [tuple(rng.standard_normal((m, kh, d)).astype(np.float32) for _ in range(2)) for _, m in lens]
    return q, kv


def fill(p, kv):
    for s, (k, v) in enumerate(kv):
        p.fill("k", s, k)
        p.fill("v", s, v)


def attend(ctx, p, q, causal=True, scale=None, ld_extra=0, offset=0, out_fill=SENTINEL):
    cache, batch = p.device()
    heads = q.shape[1]
    w = heads * p.d
    ld = w + ld_extra
    buf = np.zeros(offset + q.shape[0] * ld, np.float32)
    buf[offset:].reshape(-1, ld)[:, :w] = q.reshape(q.shape[0], w)
    dq = ctx.to_device(buf)
    out = ctx.to_device(np.full_like(buf, out_fill))
    ctx.attention_paged(cache, batch, dq.offset(offset), out.offset(offset), heads, causal=causal, scale=scale, ld_q=ld, ld_out=ld)
    o = out.numpy()
    assert (o[:offset] == out_fill).all() and (o[offset:].reshape(-1, ld)[:, w:] == out_fill).all()
    return o[offset:].reshape(-1, ld)[:, :w].reshape(q.shape)


def check(got, p, q, kv, causal=True, scale=None):
    sc = float(np.float32(1.0) / np.sqrt(np.float32(p.d))) if scale is None else scale
    for s, (n, m) in enumerate(p.lens):
        rows = slice(p.start[s], p.start[s] + n)
        k, v = (held(x, p.dtype) for x in kv[s])
        want, tol = attention64(q[rows], k, v, m - n, causal, sc)
        err = np.abs(got[rows] - want)
        assert np.isfinite(got[rows]).all(), f"sequence {s}"
        worst = np.unravel_index(np.argmax(err - tol), err.shape) if err.size else None
        assert (err <= tol).all(), f"sequence {s} (n={n}, m={m}): {err[worst]:.3g} > {tol[worst]:.3g} at {worst}"


# lens, kv heads, heads, head_dim, page
SHAPES = [
    ([(1, 1)], 1, 1, 16, 16),
    ([(1, 100), (1, 7)], 8, 8, 64, 16),
    ([(1, 31), (1, 32), (1, 33), (1, 64), (1, 65)], 2, 8, 128, 16),
    ([(1, 1000)], 2, 2, 128, 64),
    ([(1, 4100)], 1, 4, 64, 32),
    ([(1, 257)] * 9, 4, 4, 80, 48),
    ([(2, 300), (1, 299), (4, 301)], 2, 10, 128, 16),
    ([(1, 500)], 1, 16, 32, 16),
    ([(1, 500)], 1, 17, 128, 16),
    ([(1, 90)], 1, 40, 96, 16),
    ([(3, 150)], 1, 64, 64, 64),
    ([(1, 200), (1, 3)], 2, 4, 256, 32),
    ([(1, 130)], 1, 3, 200, 16),
    ([(1, 77)], 3, 3, 1, 16),
    ([(5, 61)], 2, 4, 7, 16),
    ([(1, 140)], 1, 2, 130, 16),
    ([(33, 33)], 1, 1, 128, 16),
    ([(64, 64), (100, 100), (1, 1)], 2, 2, 64, 16),
    ([(130, 400)], 2, 8, 128, 64),
    ([(257, 257)], 1, 4, 80, 48),
    ([(40, 1111)], 1, 1, 128, 80),
    ([(96, 97), (31, 500), (1, 300), (0, 40), (2, 2)], 2, 6, 64, 16),
    ([(70, 70)], 2, 2, 256, 16),
    ([(50, 90)], 1, 3, 100, 16),
    ([(45, 60)], 2, 2, 20, 32),
    ([(300, 700), (1, 900)], 4, 4, 112, 256),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,kh,heads,d,page", SHAPES)
def test_causal(ctx, dtype, lens, kh, heads, d, page):
    q, kv = case(d + heads, dtype, lens, kh, heads, d)
    p = Paged(ctx, dtype, lens, kh, d, page, seed=page)
    fill(p, kv)
    check(attend(ctx, p, q), p, q, kv)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,kh,heads,d,page", [SHAPES[i] for i in (1, 6, 17, 21, 23)])
def test_all_keys(ctx, dtype, lens, kh, heads, d, page):
    q, kv = case(3, dtype, lens, kh, heads, d)
    p = Paged(ctx, dtype, lens, kh, d, page)
    fill(p, kv)
    check(attend(ctx, p, q, causal=False), p, q, kv, causal=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("amp", [0.0, 12.0, 60.0])
def test_peaked_and_flat_scores(ctx, dtype, amp):
    """One key takes nearly all the weight, or all keys share it; the maximum moves
    late (a growing ramp of scores) or comes first."""
    lens = [(1, 700), (40, 333)]
    q, kv = case(5, dtype, lens, 1, 4, 64, amp)
    for k, _ in kv:
        k[:, :, 0] += np.linspace(-3, 3, k.shape[0])[:, None]
    q[:, :2, 0] += 10
    q[:, 2:, 0] -= 10
    p = Paged(ctx, dtype, lens, 1, 64, 16)
    fill(p, kv)
    check(attend(ctx, p, q), p, q, kv)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 1e-20])
def test_scale(ctx, scale):
    lens = [(1, 50), (35, 80)]
    q, kv = case(6, "bf16", lens, 2, 4, 32)
    p = Paged(ctx, "bf16", lens, 2, 32, 16)
    fill(p, kv)
    check(attend(ctx, p, q, scale=scale), p, q, kv, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ld_extra,offset", [(1, 0), (0, 3), (4, 4), (5, 1)])
def test_strides_and_alignment(ctx, dtype, ld_extra, offset):
    lens = [(1, 45), (37, 37)]
    q, kv = case(7, dtype, lens, 2, 4, 36)
    p = Paged(ctx, dtype, lens, 2, 36, 16)
    fill(p, kv)
    check(attend(ctx, p, q, ld_extra=ld_extra, offset=offset), p, q, kv)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_rows_without_keys_and_behind_the_last_sequence(ctx, dtype, causal):
    # More new tokens than cached ones: the first stand below position 0.
    lens = [(5, 2), (0, 30), (3, 0), (40, 33), (1, 1)]
    q, kv = case(8, dtype, lens, 1, 2, 32)
    q = np.concatenate([q, q[:6]])
    p = Paged(ctx, dtype, lens, 1, 32, 16, tokens=q.shape[0])
    fill(p, kv)
    got = attend(ctx, p, q, causal=causal)
    check(got, p, q, kv, causal=causal)
    assert (got[p.new_tokens:] == SENTINEL).all()
    assert not got[5:8].any()
    if causal:
        assert not got[:3].any() and not got[8:15].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_pages_that_are_none(ctx, dtype):
    """Their keys are left out."""
    lens, d = [(1, 100), (50, 100)], 64
    q, kv = case(9, dtype, lens, 1, 2, d)
    p = Paged(ctx, dtype, lens, 1, d, 16)
    fill(p, kv)
    p.table[0, 2], p.table[1, 0], p.table[1, 3] = -1, p.pages, 2 ** 31 - 1
    got = attend(ctx, p, q, causal=False)
    for s, gone in ((0, [2]), (1, [0, 3])):
        keep = np.array([j for j in range(100) if j // 16 not in gone])
        k, v = (held(x, dtype)[keep] for x in kv[s])
        rows = slice(p.start[s], p.start[s + 1])
        want, tol = attention64(q[rows], k, v, 0, False, float(np.float32(1.0) / np.sqrt(np.float32(d))))
        assert (np.abs(got[rows] - want) <= tol).all()
    p.table[:] = -1
    assert not attend(ctx, p, q).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("lens", [[(4, 40)], [(60, 200)]])
def test_what_a_token_does_not_see_does_not_reach_it(ctx, dtype, bad, lens):
    """NaN and infinities in the keys and values of later tokens, as they stand
    after the last token too (slots that no token has are NaN in every test)."""
    (n, m), d = lens[0], 64
    q, kv = case(10, dtype, lens, 1, 4, d)
    k, v = kv[0]
    p = Paged(ctx, dtype, lens, 1, d, 16)
    clean = m - 3
    k[clean:], v[clean + 1:] = bad, bad
    fill(p, kv)
    got = attend(ctx, p, q)
    sees = np.arange(m - n, m) < clean
    want, tol = attention64(q[sees], held(k[:clean], dtype), held(v[:clean], dtype), m - n, True,
                            float(np.float32(1.0) / np.sqrt(np.float32(d))))
    assert (np.abs(got[sees] - want) <= tol).all()
    if np.isnan(bad):
        assert np.isnan(got[~sees]).all()


def test_eight_bit_rows_of_nan_that_a_token_does_not_see(ctx):
    lens, d = [(60, 200)], 64
    q, kv = case(11, "i8", lens, 1, 4, d)
    k, v = kv[0]
    k[190, 0, 3], v[195, 0, 0] = np.nan, np.inf
    p = Paged(ctx, "i8", lens, 1, d, 16)
    fill(p, kv)
    got = attend(ctx, p, q)
    want, tol = attention64(q[:50], held(k[:190], "i8"), held(v[:190], "i8"), 140, True,
                            float(np.float32(1.0) / np.sqrt(np.float32(d))))
    assert (np.abs(got[:50] - want) <= tol).all()
    assert np.isnan(got[50:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[(1, 200)], [(60, 200)]])
def test_infinite_queries_and_values_that_are_seen(ctx, dtype, lens):
    """Rows with an infinite query element are NaN or as fp32 gives them; the others
    are not touched.  A value of infinity in one dimension reaches that dimension."""
    d = 64
    (n, m), = lens
    q, kv = case(12, dtype, lens, 1, 4, d)
    k, v = kv[0]
    q[0, 1, 5] = np.inf
    if dtype != "i8":
        v[7, 0, 9] = np.inf
    p = Paged(ctx, dtype, lens, 1, d, 16)
    fill(p, kv)
    got = attend(ctx, p, q)
    sc = float(np.float32(1.0) / np.sqrt(np.float32(d)))
    vz = v.copy()
    if dtype != "i8":
        vz[7, 0, 9] = 0
    q0 = q.copy()
    q0[0, 1, 5] = 0
    want, tol = attention64(q0, held(k, dtype), held(vz, dtype), m - n, True, sc)
    ok = np.ones(got.shape, bool)
    ok[0, 1] = False
    if dtype != "i8":
        ok[:, :, 9] = False
        others = np.delete(got[:, :, 9].reshape(-1), 1)
        assert np.isposinf(others).all()
    assert (np.abs(got - want) <= tol)[ok].all()
    assert not np.isfinite(got[0, 1]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_values(ctx, dtype):
    """Keys, queries and values far from 1, which fp32 holds."""
    lens, d = [(1, 150), (40, 150)], 64
    for qa, ka, va in ((1e-18, 1e18, 1e30), (1e15, 1e-15, 1e-30), (1e-3, 1e3, 3e36)):
        q, kv = case(13, dtype, lens, 2, 4, d, qa)
        kv = [((k * ka).astype(np.float32), (v * va).astype(np.float32)) for k, v in kv]
        p = Paged(ctx, dtype, lens, 2, d, 16)
        fill(p, kv)
        check(attend(ctx, p, q), p, q, kv)


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_twice_and_in_any_company(ctx, dtype):
    """The same call gives the same bits, whatever ran between."""
    lens, d = [(1, 3000), (2, 900), (40, 640)], 128
    q, kv = case(14, dtype, lens, 2, 8, d)
    p = Paged(ctx, dtype, lens, 2, d, 64)
    fill(p, kv)
    a = attend(ctx, p, q)
    other = Paged(ctx, dtype, [(3, 50)], 1, 32, 16)
    qo, kvo = case(15, dtype, [(3, 50)], 1, 2, 32)
    fill(other, kvo)
    attend(ctx, other, qo)
    np.testing.assert_array_equal(a, attend(ctx, p, q))


@pytest.mark.parametrize("dtype", TYPES)
def test_bounds_larger_than_the_batch(ctx, dtype):
    """max_new and max_len may be larger than what the arrays say."""
    lens, d = [(1, 60), (20, 45)], 64
    q, kv = case(16, dtype, lens, 2, 4, d)
    p = Paged(ctx, dtype, lens, 2, d, 16, spare_entries=300, max_new=500, max_len=4000)
    fill(p, kv)
    check(attend(ctx, p, q), p, q, kv)


def test_arrays_past_their_bounds(ctx):
    """Lengths and starts past the host's bounds are held to them."""
    lens, d = [(2, 60), (4, 45)], 32
    q, kv = case(17, "f32", lens, 1, 2, d)
    p = Paged(ctx, "f32", lens, 1, d, 16)
    fill(p, kv)
    p.start = np.array([0, 2, 1 << 30], np.int32)
    got = attend(ctx, p, q)
    check(got, p, q, kv)
    p.start = np.array([0, 2, 6], np.int32)
    p.kv_len = np.array([60, -5], np.int32)
    got = attend(ctx, p, q)
    assert not got[2:].any()


def test_agrees_with_the_whole_sequence_core(ctx):
    """mimir_attention_fwd over the same keys and values, each side within its bound."""
    n, heads, d = 200, 4, 64
    q, kv = case(18, "f32", [(n, n)], heads, heads, d)
    k, v = kv[0]
    p = Paged(ctx, "f32", [(n, n)], heads, d, 16)
    fill(p, kv)
    got = attend(ctx, p, q)
    out = ctx.empty((n, heads * d))
    ctx.attention(ctx.to_device(q.reshape(n, -1)), ctx.to_device(k.reshape(n, -1)), ctx.to_device(v.reshape(n, -1)), out, 1, n, n,
                  heads, d, True)
    _, tol = attention64(q, k, v, 0, True, float(np.float32(1.0) / np.sqrt(np.float32(d))))
    assert (np.abs(got - out.numpy().reshape(got.shape)) <= 2 * tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[(1, 1500)], [(60, 1500)]])
def test_nan_in_some_dimensions_and_late_keys(ctx, dtype, lens):
    """A value that is NaN in one dimension reaches that dimension alone, a key's NaN
    all of the rows that see it; wherever the rows' keys are cut."""
    d = 64
    (n, m), = lens
    q, kv = case(19, dtype, lens, 1, 4, d)
    k, v = kv[0]
    if dtype != "i8":
        v[300, 0, 9] = np.nan
    p = Paged(ctx, dtype, lens, 1, d, 16)
    fill(p, kv)
    sc = float(np.float32(1.0) / np.sqrt(np.float32(d)))
    vz = v.copy()
    vz[300, 0, 9] = 0 if dtype != "i8" else vz[300, 0, 9]
    want, tol = attention64(q, held(k, dtype), held(vz, dtype), m - n, True, sc)
    got = attend(ctx, p, q)
    ok = np.ones(got.shape, bool)
    if dtype != "i8":
        ok[:, :, 9] = False
        assert np.isnan(got[:, :, 9]).all()
    assert (np.abs(got - want) <= tol)[ok].all()
    k[m - 1, 0, 3] = np.nan
    fill(p, kv)
    got = attend(ctx, p, q)
    ok[n - 1] = False
    assert (np.abs(got - want) <= tol)[ok].all()
    assert np.isnan(got[n - 1]).all()
