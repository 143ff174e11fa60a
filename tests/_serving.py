"""Plain 64-bit forms of the serving operators (rotary positions per token, the
paged key/value cache, attention over it) and the batches their tests use."""
import ctypes

import numpy as np

import mimir_hip as M

U = 2.0 ** -24  # half a step of fp32, relative


def stride_of(d):
    return (d + 15) // 16 * 16


# --- rotary positions --------------------------------------------------------

def rotate(x, positions, cos_t, sin_t, rot, interleaved, back=False):
    """x [tokens, heads, d] rotated in float64 and rounded once to fp32; rows at
    positions outside the tables are zeros."""
    x = np.asarray(x, np.float64)
    y = x.copy()
    pos = np.asarray(positions)
    ok = (pos >= 0) & (pos < cos_t.shape[0])
    at = np.where(ok, pos, 0)
    c = cos_t[at].astype(np.float64)[:, None, :]
    s = sin_t[at].astype(np.float64)[:, None, :] * (-1.0 if back else 1.0)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    y[~ok] = 0
    return y.astype(np.float32)


# --- the cache ---------------------------------------------------------------

def bf16_bits(x):
    """fp32 to bf16, nearest even; NaN stays NaN."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    nan = (b & 0x7FFFFFFF) > 0x7F800000
    r[nan] = 0x7FC0
    return r


def bf16_value(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def i8_rows(x):
    """codes and scales of rows of fp32 (last axis)."""
    a = np.abs(x).max(-1).astype(np.float64)
    finite = np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        code = np.rint(x.astype(np.float64) * 127.0 / a[..., None])
        scale = (a.astype(np.float32) / np.float32(127)).astype(np.float32)
    code[~finite | (a == 0)] = 0
    return code.astype(np.int8), np.where(finite, scale, np.float32(np.nan)).astype(np.float32)


def held(x, dtype):
    """The values that a cache of `dtype` holds of rows x, as fp32."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "bf16":
        return bf16_value(bf16_bits(x))
    code, scale = i8_rows(x)
    with np.errstate(all="ignore"):
        return (code.astype(np.float32) * scale[..., None]).astype(np.float32)


class Paged:
    """Sequences with (new, cached) lengths `lens` in a shuffled paged cache on the
    device.  Slots that no token has are NaN."""

    def __init__(self, ctx, dtype, lens, kv_heads, d, page, seed=0, spare_pages=2, spare_entries=1, tokens=None, max_new=None,
                 max_len=None):
        self.ctx, self.dtype, self.lens, self.kv_heads, self.d, self.page = ctx, dtype, lens, kv_heads, d, page
        rng = np.random.default_rng(seed)
        used = [-(-m // page) for _, m in lens]
        self.pages = sum(used) + spare_pages
        self.ld = max(used, default=0) + spare_entries
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(lens), max(self.ld, 1)), -7, np.int32)
        at = 0
        for s, n in enumerate(used):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.kv_len = np.array([m for _, m in lens], np.int32)
        self.new_tokens = int(self.start[-1])
        self.tokens = self.new_tokens if tokens is None else tokens
        self.max_new = max((n for n, _ in lens), default=0) if max_new is None else max_new
        self.max_len = max((m for _, m in lens), default=0) if max_len is None else max_len
        shape = (self.pages, kv_heads, page, stride_of(d))
        np_type = {"f32": np.float32, "bf16": np.uint16, "i8": np.int8}[dtype]
        self.host = {n: np.full(shape, {"f32": np.nan, "bf16": 0x7FC0, "i8": 127}[dtype], np_type) for n in ("k", "v")}
        self.scale = {n: np.full(shape[:3], np.nan, np.float32) for n in ("k", "v")}

    def slot(self, s, p):
        return int(self.table[s, p // self.page]), p % self.page

    def fill(self, name, s, x):
        """Rows x [m, kv_heads, d] of sequence s, as the cache would hold them."""
        x = np.asarray(x, np.float32)
        if self.dtype == "i8":
            code, scale = i8_rows(x)
        for p in range(x.shape[0]):
            page, at = self.slot(s, p)
            row = self.host[name][page, :, at]
            row[:] = 0
            if self.dtype == "f32":
                row[:, :self.d] = x[p]
            elif self.dtype == "bf16":
                row[:, :self.d] = bf16_bits(x[p])
            else:
                row[:, :self.d] = code[p]
                self.scale[name][page, :, at] = scale[p]

    def device(self):
        """(KVCache, KVBatch) on the device, from the host state."""
        up = self.ctx.to_device
        scales = [up(self.scale[n]) for n in ("k", "v")] if self.dtype == "i8" else [None, None]
        self.cache = M.KVCache(self.ctx, self.dtype, self.pages, self.page, self.kv_heads, self.d, up(self.host["k"]),
                               up(self.host["v"]), *scales)
        self.batch = M.KVBatch(up(self.start), up(self.kv_len), up(self.table), len(self.lens), self.tokens, self.ld,
                               self.max_new, self.max_len)
        return self.cache, self.batch


# --- attention ---------------------------------------------------------------

def attention64(q, k, v, first, causal, scale):
    """q [n, heads, d] at positions first .., k / v [m, kv_heads, d]: the core in
    float64 and how far an fp32 evaluation may be from it.

    With u = 2^-24: a score is a sum of d products and a few roundings of its
    operands, each off by at most u relative to sum |q_i k_i| scale; the error of a
    sum of n rounded terms grows like sqrt(n) u (4 standard deviations).  A change e
    of all scores changes a normalised weight by at most 2 e, and the weighted sum by
    2 e sum p |v|; exp and the two sums over the keys add theirs."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    q64, k64, v64 = (np.asarray(x, np.float64) for x in (q, k, v))
    out, tol = np.zeros((n, heads, d)), np.zeros((n, heads, d))
    for h in range(heads):
        g = h // group
        s = q64[:, h] @ k64[:, g].T * scale
        sa = np.abs(q64[:, h]) @ np.abs(k64[:, g]).T * abs(scale)
        for i in range(n):
            m = min(max(first + i + 1, 0), k.shape[0]) if causal else k.shape[0]
            if m == 0:
                continue
            e = np.exp(s[i, :m] - max(s[i, :m].max(), -1e30))
            p = e / (e.sum() + 1e-9)
            out[i, h] = p @ v64[:m, g]
            mag = p @ np.abs(v64[:m, g])
            score = (4 * np.sqrt(d) + 8) * sa[i, :m].max()
            tol[i, h] = U * mag * (2 * score + 8 + 2 * (4 * np.sqrt(m) + 8)) + 1e-37
    return out, tol


# --- contexts and graphs -----------------------------------------------------

def tuned_context(tune):
    """A context of its own with MIMIR_TUNE set."""
    import os
    old = os.environ.get("MIMIR_TUNE")
    os.environ["MIMIR_TUNE"] = tune
    try:
        return M.Context(0)
    finally:
        if old is None:
            del os.environ["MIMIR_TUNE"]
        else:
            os.environ["MIMIR_TUNE"] = old


class Hip:
    """The runtime's own stream and graph calls, through the library that links it."""

    def __init__(self, ctx):
        self.lib = ctypes.CDLL(M._lib.LIB_PATH)

    def __call__(self, name, *args):
        st = getattr(self.lib, name)(*args)
        assert st == 0, f"{name}: {st}"


class Graph:
    """What `calls` enqueues on the context's stream, captured."""

    def __init__(self, ctx, calls):
        self.ctx, self.hip = ctx, Hip(ctx)
        ctx.lib.mimir_ctx_stream.restype = ctypes.c_void_p
        self.stream = ctypes.c_void_p(ctx.lib.mimir_ctx_stream(ctx.handle))
        graph, self.exe = ctypes.c_void_p(), ctypes.c_void_p()
        self.hip("hipStreamBeginCapture", self.stream, 1)  # thread local
        try:
            calls()
        finally:
            self.hip("hipStreamEndCapture", self.stream, ctypes.byref(graph))
        self.hip("hipGraphInstantiate", ctypes.byref(self.exe), graph, None, None, ctypes.c_size_t(0))
        self.hip("hipGraphDestroy", graph)

    def launch(self):
        self.hip("hipGraphLaunch", self.exe, self.stream)

    def close(self):
        self.hip("hipGraphExecDestroy", self.exe)
