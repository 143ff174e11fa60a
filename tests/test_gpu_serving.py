"""The serving operators as a program runs them: prompts in chunks and single
steps over one cache, captured steps that are replayed while their lengths change,
other streams and contexts beside; and attention over batches that are dealt to the
workgroups in every way (many sequences, few, two tiles of rows, cut anywhere),
caches past 2^32 bytes and the longest context that a call may have."""
import ctypes
import os
import shutil
import subprocess
import threading

import numpy as np
import pytest

import mimir_hip as M
from _serving import Graph, Hip, Paged, U, attention64, held, rotate, stride_of, tuned_context
from test_gpu_attention_paged import attend, case, check, fill

pytestmark = pytest.mark.gpu
TYPES = ["f32", "bf16", "i8"]
THETA = 10000.0


def scale_of(d):
    return float(np.float32(1.0) / np.sqrt(np.float32(d)))


class Layer:
    """One layer's rope, cache and attention over packed rows; the device side of a
    program that keeps its buffers."""

    def __init__(self, ctx, dtype, sequences, longest, heads, kv_heads, d, rot, page, most_tokens, seed):
        self.ctx, self.heads, self.kv_heads, self.d = ctx, heads, kv_heads, d
        self.cos, self.sin = M.rope_table_scaled(longest, rot, THETA)
        self.rot = rot
        self.rope = M.Rope(ctx.to_device(self.cos), ctx.to_device(self.sin), longest, rot, False)
        per = -(-longest // page)
        self.cache = M.KVCache(ctx, dtype, sequences * per, page, kv_heads, d)
        table = np.random.default_rng(seed).permutation(sequences * per).astype(np.int32).reshape(sequences, per)
        self.table, self.per, self.sequences, self.longest = ctx.to_device(table), per, sequences, longest
        self.start, self.len = ctx.to_device(np.zeros(sequences + 1, np.int32)), ctx.to_device(np.zeros(sequences, np.int32))
        w = (heads + 2 * kv_heads) * d
        self.qkv, self.q = ctx.empty((most_tokens, w)), ctx.empty((most_tokens, heads * d))
        self.most = most_tokens

    def set(self, news, lens, qkv):
        self.ctx.upload(self.start, np.concatenate([[0], np.cumsum(news)]).astype(np.int32))
        self.ctx.upload(self.len, np.asarray(lens, np.int32))
        self.ctx.upload(self.qkv.offset(0, qkv.shape), np.ascontiguousarray(qkv))

    def run(self, out, tokens, max_new):
        h, kh, d = self.heads, self.kv_heads, self.d
        batch = M.KVBatch(self.start, self.len, self.table, self.sequences, tokens, self.per, max_new, self.longest)
        w = (h + 2 * kh) * d
        self.ctx.kv_append(self.cache, batch, self.qkv.offset(h * d), self.qkv.offset((h + kh) * d), ld_kv=w, rope=self.rope,
                           q=self.qkv, q_out=self.q, heads=h, ld_q=w)
        self.ctx.attention_paged(self.cache, batch, self.q, out, h, causal=True)


def wanted(x, dtype, heads, kv_heads, d, layer):
    """What a whole sequence of rows x [m, (heads + 2 kv_heads) d] gives, and how far
    off it may be: rotated rows are the same bits, so attention's bound is all."""
    m = x.shape[0]
    at = np.arange(m)
    q = rotate(x[:, :heads * d].reshape(m, heads, d), at, layer.cos, layer.sin, layer.rot, False)
    k = rotate(x[:, heads * d:(heads + kv_heads) * d].reshape(m, kv_heads, d), at, layer.cos, layer.sin, layer.rot, False)
    v = x[:, (heads + kv_heads) * d:].reshape(m, kv_heads, d)
    return attention64(q, held(k, dtype), held(v, dtype), 0, True, scale_of(d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kh,d,rot,page", [(8, 2, 64, 64, 16), (3, 3, 80, 32, 48), (4, 1, 256, 128, 64)])
def test_prompts_chunks_and_steps(ctx, dtype, heads, kh, d, rot, page):
    """Three sequences that begin at different times, their prompts in chunks of any
    size, then step by step in one batch: every token as over its whole sequence."""
    total = [150, 61, 97]
    w = (heads + 2 * kh) * d
    rng = np.random.default_rng(heads)
    x = [rng.standard_normal((n, w)).astype(np.float32) for n in total]
    layer = Layer(ctx, dtype, 3, 160, heads, kh, d, rot, page, 160, seed=2)
    got = [np.zeros((n, heads * d), np.float32) for n in total]
    plan = [(100, 0, 5), (30, 16, 1), (0, 30, 64), (1, 1, 1), (2, 0, 3)]
    done = [0, 0, 0]
    out = ctx.empty((160, heads * d))
    while any(a < b for a, b in zip(done, total)):
        news = plan.pop(0) if plan else (1, 1, 1)
        news = [min(n, b - a) for n, a, b in zip(news, done, total)]
        rows = np.concatenate([x[s][done[s]:done[s] + n] for s, n in enumerate(news)])
        done = [a + n for a, n in zip(done, news)]
        layer.set(news, done, rows)
        layer.run(out, rows.shape[0], max(news))
        o, at = out.numpy(), 0
        for s, n in enumerate(news):
            got[s][done[s] - n:done[s]] = o[at:at + n]
            at += n
    for s in range(3):
        want, tol = wanted(x[s], dtype, heads, kh, d, layer)
        assert (np.abs(got[s].reshape(want.shape) - want) <= tol).all(), f"sequence {s}"


# News per step; the graph's bounds are the largest of all: single tokens (streams,
# cut and whole), several (two tiles of rows), chunks beside steps (both kernels).
PLANS = [
    (2000, [(1, 1, 1), (1, 0, 1), (1, 1, 1)], [(900, 30, 1990), (5, 0, 17), (1999, 1000, 1)]),
    (400, [(3, 1, 2), (3, 3, 3), (1, 0, 0)], [(90, 30, 395), (5, 3, 17), (400, 0, 1)]),
    (2000, [(70, 1, 3), (0, 64, 1), (40, 33, 1)], [(900, 30, 1990), (5, 64, 17), (1999, 1000, 1)]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("longest,news,lens", PLANS)
def test_captured_and_replayed_with_other_lengths(dtype, longest, news, lens):
    """A context's first calls are captured (its workspace is made then); replays see
    the lengths, pages and rows of their time, with eager work between, and give the
    bits of the eager calls."""
    heads, kh, d = 8, 1, 64
    w = (heads + 2 * kh) * d
    tokens, most = max(sum(n) for n in news), max(max(n) for n in news)
    ctx, other = M.Context(0), M.Context(0)
    try:
        a = Layer(ctx, dtype, 3, longest, heads, kh, d, d, 16, tokens, seed=3)
        b = Layer(other, dtype, 3, longest, heads, kh, d, d, 16, tokens, seed=3)
        out_a, out_b = ctx.empty((tokens, heads * d)), other.empty((tokens, heads * d))
        junk = ctx.empty((tokens, heads * d))
        rng = np.random.default_rng(4)
        whole = [rng.standard_normal((longest, w)).astype(np.float32) for _ in range(3)]
        fillers = [c.to_device(np.concatenate(whole)) for c in (ctx, other)]

        def whole_sequences(pages):
            """In both caches, in these pages."""
            for layer, filler in zip((a, b), fillers):
                layer.ctx.upload(layer.table, pages)
                layer.ctx.upload(layer.start, (np.arange(4) * longest).astype(np.int32))
                layer.ctx.upload(layer.len, np.full(3, longest, np.int32))
                batch = M.KVBatch(layer.start, layer.len, layer.table, 3, 3 * longest, layer.per, longest, longest)
                layer.ctx.kv_append(layer.cache, batch, filler.offset(heads * d), filler.offset((heads + kh) * d), ld_kv=w)

        graph = Graph(ctx, lambda: a.run(out_a, tokens, most))
        try:
            for turn, (n, m) in enumerate(zip(news * 2, lens * 2)):
                rows = rng.standard_normal((tokens, w)).astype(np.float32)
                whole_sequences(rng.permutation(3 * a.per).astype(np.int32).reshape(3, a.per))
                for layer, out in ((a, out_a), (b, out_b)):
                    layer.set(n, m, rows)
                    layer.ctx.fill(out, -3.0)
                ctx.sync()
                graph.launch()
                ctx.sync()
                b.run(out_b, tokens, most)
                got, want = out_a.numpy(), out_b.numpy()
                np.testing.assert_array_equal(got, want, err_msg=f"replay {turn}")
                assert (got[sum(n):] == -3).all()
                a.run(junk, tokens, most)  # eager work of the same context, the same rows again
                np.testing.assert_array_equal(junk.numpy()[:sum(n)], want[:sum(n)])
        finally:
            graph.close()
    finally:
        ctx.close()
        other.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_on_a_stream_of_the_program(dtype):
    c = M.Context(0)
    hip = Hip(c)
    stream = ctypes.c_void_p()
    hip("hipStreamCreate", ctypes.byref(stream))
    try:
        lens = [(1, 700), (1, 40), (90, 300)]
        q, kv = case(1, dtype, lens, 2, 8, 64)
        p = Paged(c, dtype, lens, 2, 64, 16)
        fill(p, kv)
        first = attend(c, p, q)
        c.check(c.lib.mimir_ctx_set_stream(c.handle, stream))
        on = attend(c, p, q)
        c.check(c.lib.mimir_ctx_set_stream(c.handle, None))
        check(on, p, q, kv)
        np.testing.assert_array_equal(first, on)
    finally:
        c.close()
        hip("hipStreamDestroy", stream)


@pytest.mark.parametrize("dtype", TYPES)
def test_two_contexts_at_once(dtype):
    """Threads with a context each: neither sees the other's workspace."""
    lens = [[(1, 3000), (1, 2999)], [(80, 900), (1, 5), (33, 700)]]
    cs = [M.Context(0), M.Context(0)]
    got = [[], []]

    def work(i):
        q, kv = case(20 + i, dtype, lens[i], 2, 8, 64)
        p = Paged(cs[i], dtype, lens[i], 2, 64, 16)
        fill(p, kv)
        for _ in range(10):
            got[i].append(attend(cs[i], p, q))
        got[i].append((p, q, kv))

    try:
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for outs in got:
            p, q, kv = outs.pop()
            assert len(outs) == 10
            check(outs[0], p, q, kv)
            for o in outs[1:]:
                np.testing.assert_array_equal(o, outs[0])
    finally:
        for c in cs:
            c.close()


def many(seed, count, new, most):
    rng = np.random.default_rng(seed)
    out = []
    for _ in range(count):
        n = int(rng.integers(0, new + 1))
        out.append((n, n + int(rng.integers(0, most))))
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,new,most,kh,heads,d", [
    (150, 1, 40, 1, 2, 32),      # nothing is cut, short
    (131, 1, 1300, 1, 4, 64),    # more sequences than a wave's lanes, dealt in runs
    (64, 2, 1100, 2, 4, 32),
    (65, 2, 1100, 1, 16, 48),    # up to 32 rows
    (200, 3, 1030, 3, 3, 16),
    (70, 40, 60, 1, 4, 64),      # both kernels
    (129, 70, 30, 2, 2, 16),
])
def test_many_sequences(ctx, dtype, count, new, most, kh, heads, d):
    lens = many(count, count, new, most)
    q, kv = case(count, dtype, lens, kh, heads, d)
    p = Paged(ctx, dtype, lens, kh, d, 16, max_len=max(1100, most + new))
    p.table = np.pad(p.table, ((0, 0), (0, 100)), constant_values=-1)
    p.ld = p.table.shape[1]
    fill(p, kv)
    check(attend(ctx, p, q), p, q, kv)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,kh,heads,d", [
    ([(2, 1200), (2, 30), (2, 1029)], 1, 10, 64),          # 20 rows: a tile and a part of one
    ([(3, 1500), (1, 1499), (2, 3)], 2, 16, 128),          # 8, 16 and 24
    ([(4, 2000)], 4, 32, 128),                             # 32
    ([(4, 1111), (4, 1111)], 1, 8, 256),
    ([(11, 1300), (5, 1200)], 1, 3, 80),                   # 33: two tiles and one row
    ([(64, 1100)], 2, 2, 96),                              # 64, of one head
    ([(16, 16), (16, 1040)], 1, 4, 112),
    ([(17, 1500)], 1, 2, 20),
])
def test_two_tiles_of_rows(ctx, dtype, lens, kh, heads, d):
    q, kv = case(d, dtype, lens, kh, heads, d)
    p = Paged(ctx, dtype, lens, kh, d, 32)
    fill(p, kv)
    check(attend(ctx, p, q), p, q, kv)
    check(attend(ctx, p, q, causal=False), p, q, kv, causal=False)


@pytest.mark.parametrize("tune", ["paged=1", "paged=3", "paged=61", "paged=300", "paged=100000", "paged=5,attnwaves=4",
                                  "paged=40,attnwaves=8", "attnwaves=4", "attnwaves=8"])
def test_dealt_to_any_number_of_workgroups(tune):
    """Blocks cut anywhere, several to a workgroup, or one each."""
    c = tuned_context(tune)
    try:
        for dtype in TYPES:
            for lens, kh, heads, d in (([(1, 1500), (0, 9), (1, 64), (1, 1300)], 2, 8, 64), ([(3, 1400), (2, 1301)], 1, 8, 128),
                                       ([(40, 1100), (1, 1500), (130, 131)], 1, 4, 64), ([(300, 900)], 2, 2, 96),
                                       ([(70, 1200)], 1, 2, 256)):
                for causal in (True, False):
                    q, kv = case(len(tune), dtype, lens, kh, heads, d)
                    p = Paged(c, dtype, lens, kh, d, 48)
                    fill(p, kv)
                    check(attend(c, p, q, causal=causal), p, q, kv, causal=causal)
    finally:
        c.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 5, 80])
def test_cache_past_2_32_bytes(ctx, dtype, n):
    """Pages at both ends of a cache whose keys take more than 2^32 bytes: written, read
    back and attended."""
    d, kh, page, heads, m = 128, 2, 256, 4, 700
    row = stride_of(d) * {"f32": 4, "bf16": 2, "i8": 1}[dtype]
    pages = (1 << 32) // (kh * page * row) + 3
    cache = M.KVCache(ctx, dtype, pages, page, kh, d)
    try:
        rng = np.random.default_rng(n)
        q = rng.standard_normal((n, heads * d)).astype(np.float32)
        k, v = (rng.standard_normal((m, kh * d)).astype(np.float32) for _ in range(2))
        table = np.array([[pages - 1, 0, pages - 2]], np.int32)
        up = ctx.to_device
        whole = M.KVBatch(up(np.array([0, m], np.int32)), up(np.array([m], np.int32)), up(table), 1, m, 3, m, m)
        ctx.kv_append(cache, whole, up(k), up(v))
        k2, v2 = ctx.empty((m, kh * d)), ctx.empty((m, kh * d))
        ctx.kv_read(cache, whole, k2, v2)
        kh_, vh_ = (held(a.reshape(m, kh, d), dtype) for a in (k, v))
        np.testing.assert_array_equal(k2.numpy().reshape(m, kh, d), kh_)
        np.testing.assert_array_equal(v2.numpy().reshape(m, kh, d), vh_)
        last = M.KVBatch(up(np.array([0, n], np.int32)), up(np.array([m], np.int32)), up(table), 1, n, 3, n, m)
        out = ctx.empty((n, heads * d))
        ctx.attention_paged(cache, last, up(q), out, heads, causal=True)
        want, tol = attention64(q.reshape(n, heads, d), kh_, vh_, m - n, True, scale_of(d))
        assert (np.abs(out.numpy().reshape(want.shape) - want) <= tol).all()
    finally:
        cache.close()


@pytest.mark.parametrize("dtype", ["bf16", "i8"])
def test_the_longest_context(ctx, dtype):
    """2^30 - 16 keys, one page over and over, so that the softmax is that of the
    page's keys.  Sums over equal addends may drift by half a step each time: a run of
    2^21 keys is 2^14 steps of a wave, so weights and sums are off by 2^15 U each at
    most, besides what attention64 allows a page."""
    page, d, heads = 1 << 13, 16, 4
    m = (1 << 30) - 16
    entries = -(-m // page)
    q, kv = case(30, dtype, [(1, page)], 1, heads, d)
    p = Paged(ctx, dtype, [(1, page)], 1, d, page, spare_pages=0, spare_entries=0)
    fill(p, kv)
    cache, _ = p.device()
    up = ctx.to_device
    batch = M.KVBatch(up(np.array([0, 1], np.int32)), up(np.array([m], np.int32)), up(np.zeros((1, entries), np.int32)), 1, 1,
                      entries, 1, m)
    out = ctx.empty((1, heads * d))
    ctx.attention_paged(cache, batch, up(q), out, heads, causal=True)
    k, v = (held(x, dtype) for x in kv[0])
    want, tol = attention64(q, k, v, page - 1, True, scale_of(d))
    # The last page lacks 16 of its keys: of 2^17 pages' weight.
    s = np.einsum("hd,kd->hk", q[0].astype(np.float64), k[:, 0].astype(np.float64)) * scale_of(d)
    e = np.exp(s - s.max())
    part = e.copy()
    part[:, -16:] = 0
    weight = e * (entries - 1) + part
    want = (weight @ v[:, 0].astype(np.float64) / weight.sum(1, keepdims=True))[None]
    mag = (weight @ np.abs(v[:, 0].astype(np.float64)) / weight.sum(1, keepdims=True))[None]
    tol = tol + 2 * (1 << 15) * U * mag
    assert (np.abs(out.numpy().reshape(want.shape) - want) <= tol).all()


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_cpp_adapter(tmp_path):
    here, lib = os.path.dirname(os.path.abspath(__file__)), os.path.dirname(M.LIB_PATH)
    exe = tmp_path / "test_serving_device"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-pthread", f"-I{here}/../include", "-o", str(exe),
                    os.path.join(here, "cpp", "test_serving_device.cpp"), f"-L{lib}", "-lmimir_hip", f"-Wl,-rpath,{lib}"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "0 failures", r.stdout + r.stderr


@pytest.mark.parametrize("seed,count", [(0, 64), (1, 65), (2, 4095), (3, 4096), (4, 4200), (5, 9000)])
def test_tokens_of_thousands_of_sequences(ctx, seed, count):
    """Which sequence a token is of, by what is written and read back: runs of sequences
    without new tokens, several tokens, rows behind the last one."""
    rng = np.random.default_rng(seed)
    n = rng.choice([0, 1, 1, 2, 5], size=count)
    hole = int(rng.integers(0, max(1, count - 200)))
    n[hole:hole + 150] = 0
    kh, d, page = 1, 4, 16
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    tokens = int(start[-1]) + 3
    table = rng.permutation(count).astype(np.int32)
    up = ctx.to_device
    cache = M.KVCache(ctx, "f32", count, page, kh, d)
    try:
        x = np.arange(tokens * d, dtype=np.float32).reshape(tokens, d)
        kv_len = np.maximum(n, rng.integers(0, 17, count)).astype(np.int32)
        batch = M.KVBatch(up(start), up(kv_len), up(table), count, tokens, 1, 5, page)
        ctx.kv_append(cache, batch, up(x), up(-x))
        k = cache.k.numpy().reshape(count, page, stride_of(d))
        for s in range(count):
            got = k[table[s], kv_len[s] - n[s]:kv_len[s], :d]
            np.testing.assert_array_equal(got, x[start[s]:start[s + 1]])
        ko, vo = (up(np.full((tokens, d), -9.0, np.float32)) for _ in range(2))
        ctx.kv_read(cache, batch, ko, vo)
        np.testing.assert_array_equal(ko.numpy()[:-3], x[:-3])
        np.testing.assert_array_equal(vo.numpy()[:-3], -x[:-3])
        assert (ko.numpy()[-3:] == -9).all() and (vo.numpy()[-3:] == -9).all()
    finally:
        cache.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_runs_over_thousands_of_sequences(ctx, dtype):
    """Most without new tokens, in stretches; lengths from 1 to 1400."""
    rng = np.random.default_rng(40)
    count, d = 4500, 16
    n = np.zeros(count, int)
    n[rng.choice(count, 300, replace=False)] = rng.integers(1, 3, 300)
    n[1000:1130] = 1
    lens = [(int(x), int(x + rng.integers(0, 1400 if i % 7 == 0 else 30))) if x else (0, 5) for i, x in enumerate(n)]
    q, kv = case(41, dtype, lens, 1, 2, d)
    p = Paged(ctx, dtype, lens, 1, d, 16, max_len=1500)
    p.table = np.pad(p.table, ((0, 0), (0, 10)), constant_values=-1)
    p.ld = p.table.shape[1]
    fill(p, kv)
    check(attend(ctx, p, q), p, q, kv)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,kh,heads,d,page", [
    ([(65, 65)], 1, 1, 256, 16),
    ([(128, 300)], 2, 2, 256, 48),
    ([(129, 129), (1, 700), (33, 1200), (0, 9)], 1, 2, 256, 16),
    ([(200, 1500), (70, 70)], 1, 3, 192, 32),
    ([(90, 91)], 2, 4, 144, 16),
    ([(100, 160)], 1, 1, 130, 16),
    ([(67, 900)], 1, 2, 201, 64),
    ([(80, 20), (300, 300)], 1, 1, 250, 16),
])
def test_wide_heads_of_many_rows(ctx, dtype, lens, kh, heads, d, page):
    q, kv = case(d + page, dtype, lens, kh, heads, d)
    p = Paged(ctx, dtype, lens, kh, d, page)
    fill(p, kv)
    check(attend(ctx, p, q), p, q, kv)
    check(attend(ctx, p, q, causal=False, ld_extra=1, offset=3), p, q, kv, causal=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tune", ["paged=1", "paged=7", "paged=256"])
def test_wide_heads_dealt_to_any_number_of_workgroups(dtype, tune):
    c = tuned_context(tune)
    try:
        lens = [(150, 700), (70, 640), (1, 1300)]
        q, kv = case(50, dtype, lens, 1, 2, 256)
        p = Paged(c, dtype, lens, 1, 256, 16)
        fill(p, kv)
        check(attend(c, p, q), p, q, kv)
    finally:
        c.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_wide_heads_holes_and_nan(ctx, dtype):
    """Pages that are none, a NaN in one dimension, in a key that some rows see, and in
    what no row sees (slots without tokens are NaN in every test)."""
    lens, d, m = [(100, 500)], 256, 500
    q, kv = case(51, dtype, lens, 1, 1, d)
    k, v = kv[0]
    p = Paged(ctx, dtype, lens, 1, d, 16)
    fill(p, kv)
    p.table[0, 3] = -1
    keep = np.array([j for j in range(m) if j // 16 != 3])
    got = attend(ctx, p, q, causal=False)
    want, tol = attention64(q, held(k, dtype)[keep], held(v, dtype)[keep], 0, False, scale_of(d))
    assert (np.abs(got - want) <= tol).all()
    p = Paged(ctx, dtype, lens, 1, d, 16)
    if dtype != "i8":
        v[100, 0, 200] = np.nan
    k[450, 0, 7] = np.nan
    fill(p, kv)
    got = attend(ctx, p, q)
    vz = v.copy()
    vz[100, 0, 200] = 0 if dtype != "i8" else vz[100, 0, 200]
    want, tol = attention64(q[:50], held(k, dtype)[:450], held(vz, dtype)[:450], 400, True, scale_of(d))
    ok = np.ones(want.shape, bool)
    if dtype != "i8":
        ok[:, :, 200] = False
        assert np.isnan(got[:, :, 200]).all()
    assert (np.abs(got[:50] - want) <= tol)[ok].all()
    assert np.isnan(got[50:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(3, 64), (100, 64), (100, 256)])
@pytest.mark.parametrize("pages", [0, 2])
def test_no_keys_at_all(ctx, dtype, n, d, pages):
    """A cache without pages, or a call whose bound is no keys: rows of zeros, nothing
    written, rows read back as zeros."""
    cache = M.KVCache(ctx, dtype, pages, 16, 1, d)
    up = ctx.to_device
    batch = M.KVBatch(up(np.array([0, n], np.int32)), up(np.array([n], np.int32)), None, 1, n, 0, n, 0)
    try:
        x = up(np.ones((n, d), np.float32))
        out = up(np.full((n, 2 * d), 5.0, np.float32))
        ctx.kv_append(cache, batch, x, x)
        ctx.attention_paged(cache, batch, up(np.ones((n, 2 * d), np.float32)), out, 2)
        assert not out.numpy().any()
        back = up(np.full((n, d), 5.0, np.float32))
        ctx.kv_read(cache, batch, back, None)
        assert not back.numpy().any()
    finally:
        cache.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,max_new", [(3, 1 << 29), (3000, 3000), (3000, (1 << 30) - 1)])
def test_bounds_far_above_what_sequences_have(ctx, dtype, count, max_new):
    """A bound of new tokens that no launch of a workgroup per block would hold: single
    tokens of a key each, whose rows are that key's value.  Its weight is 1 and the sum's
    reciprocal too; the value is put together from up to three terms and scaled once, half
    a step of fp32 each."""
    kh, group, d, page = 16, 16, 16, 16
    rng = np.random.default_rng(count)
    v = rng.standard_normal((count, kh, d)).astype(np.float32)
    cache = M.KVCache(ctx, dtype, count, page, kh, d)
    try:
        up = ctx.to_device
        table = rng.permutation(count).astype(np.int32)
        batch = M.KVBatch(up(np.arange(count + 1, dtype=np.int32)), up(np.ones(count, np.int32)), up(table), count, count, 1,
                          max_new, page)
        dv = up(v)
        ctx.kv_append(cache, batch, dv, dv)
        out = up(np.full((count, kh, group, d), 5.0, np.float32))
        ctx.attention_paged(cache, batch, up(rng.standard_normal((count, kh * group * d)).astype(np.float32)), out, kh * group)
        want = held(v, dtype)[:, :, None, :].astype(np.float64)
        assert (np.abs(out.numpy() - want) <= 4 * U * np.abs(want)).all()
    finally:
        cache.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 250])
@pytest.mark.parametrize("waves", [4, 8])
@pytest.mark.parametrize("lens", [[(140, 1300), (70, 900), (1, 300)], [(200, 250), (70, 90), (3, 3)]])
def test_every_width_of_the_kernel_of_many_rows(dtype, d, waves, lens):
    """Cut and joined, and whole: some of these hold a few registers in memory."""
    c = tuned_context(f"attnwaves={waves}")
    try:
        q, kv = case(d + waves, dtype, lens, 1, 2, d)
        p = Paged(c, dtype, lens, 1, d, 16)
        fill(p, kv)
        check(attend(c, p, q), p, q, kv)
        check(attend(c, p, q, causal=False), p, q, kv, causal=False)
    finally:
        c.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("waves", [4, 8])
@pytest.mark.parametrize("pages", [0, 2])
def test_no_keys_and_no_page_table_by_waves(dtype, d, waves, pages):
    """As above by each width of the kernel of many rows: eight waves take one turn more
    than there are tiles, of which there are none."""
    c = tuned_context(f"attnwaves={waves}")
    try:
        n, count = 140, 3
        cache = M.KVCache(c, dtype, pages, 16, 1, d)
        up = c.to_device
        batch = M.KVBatch(up((np.arange(count + 1) * n).astype(np.int32)), up(np.zeros(count, np.int32)), None, count, count * n,
                          0, n, 0)
        out = up(np.full((count * n, d), 5.0, np.float32))
        c.attention_paged(cache, batch, up(np.ones((count * n, d), np.float32)), out, 1)
        assert not out.numpy().any()
        cache.close()
    finally:
        c.close()


@pytest.mark.parametrize("d", [100, 128])
def test_no_keys_and_no_page_table_in_more_blocks_than_workgroups(ctx, d):
    """fp32 heads of 97 to 128, more blocks of 128 rows than the GPU has compute units:
    eight waves by the rule of sizes alone."""
    n, count = 129, 150  # two blocks of 128 rows a sequence, 300 in all
    cache = M.KVCache(ctx, "f32", 2, 16, 1, d)
    try:
        up = ctx.to_device
        batch = M.KVBatch(up((np.arange(count + 1) * n).astype(np.int32)), up(np.zeros(count, np.int32)), None, count, count * n,
                          0, n, 0)
        out = up(np.full((count * n, d), 5.0, np.float32))
        ctx.attention_paged(cache, batch, up(np.ones((count * n, d), np.float32)), out, 1)
        assert not out.numpy().any()
    finally:
        cache.close()


def test_pages_that_two_sequences_share(ctx):
    """A prefix that is in the cache once."""
    d, page, m = 32, 16, 40000
    q, kv = case(60, "bf16", [(1, m)], 1, 4, d)
    p = Paged(ctx, "bf16", [(1, m), (1, 0)], 1, d, page)
    fill(p, [kv[0], (kv[0][0][:0], kv[0][1][:0])])
    p.table[1, :] = p.table[0, :]
    p.kv_len = np.array([m, 1000], np.int32)
    p.lens = [(1, m), (1, 1000)]
    q2 = np.concatenate([q, q])
    got = attend(ctx, p, q2)
    check(got, p, q2, [kv[0], (kv[0][0][:1000], kv[0][1][:1000])])
