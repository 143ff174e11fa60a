"""Norm and clipping of many gradients against float64: both types, lists of none
to several hundred tensors, odd sizes and alignments, in place and beside, values
whose squares leave fp32's range, NaN and infinities."""
import math

import numpy as np
import pytest

import mimir_hip as M
from _serving import bf16_bits, bf16_value
from _training import U, held

pytestmark = pytest.mark.gpu


class Tensors:
    """Tensors of (elements, type) in one buffer each, `offset` elements in."""

    def __init__(self, ctx, values, dtypes, offset=0, beside=False):
        self.ctx, self.values, self.dtypes, self.offset = ctx, values, dtypes, offset
        self.bufs, self.outs, items = [], [], []
        for v, t in zip(values, dtypes):
            buf = np.full(offset + len(v) + 16, -77.0, np.float32)
            buf[offset:offset + len(v)] = v
            raw = bf16_bits(buf) if t == "bf16" else buf
            d = ctx.to_device(raw)
            o = ctx.to_device(bf16_bits(np.full_like(buf, -77.0)) if t == "bf16" else np.full_like(buf, -77.0)) if beside else d
            self.bufs.append(d)
            self.outs.append(o)
            size = d.dtype.itemsize
            items.append((d.ptr + offset * size, len(v), t, o.ptr + offset * size))
        self.list = M.TensorList(items)

    def get(self, which):
        out = []
        for d, v, t in zip(which, self.values, self.dtypes):
            b = d.numpy()
            b = bf16_value(b) if t == "bf16" else b
            assert (b[:self.offset] == -77).all() and (b[self.offset + len(v):] == -77).all()
            out.append(b[self.offset:self.offset + len(v)])
        return out


def norm64(values):
    return math.sqrt(math.fsum(float((np.asarray(v, np.float64) ** 2).sum()) for v in values))


def clipped(values, dtypes, most):
    """The formula in float64, and the bound: the factor and the product round once each, the norm's error is far below."""
    by = min(1.0, most / (norm64(values) + 1e-6))
    want = [np.asarray(v, np.float64) * by for v in values]
    half = {"f32": U, "bf16": 2.0 ** -8}
    # bf16's subnormals: half of 2^-133.
    return want, [2.01 * U * np.abs(w) + 1.001 * half[t] * np.abs(w) + (2.0 ** -134 if t == "bf16" else 2.0 ** -150) for w, t in zip(want, dtypes)]


def check(ctx, values, dtypes, most, offset=0, beside=False):
    values = [held(v, t) for v, t in zip(values, dtypes)]
    T = Tensors(ctx, values, dtypes, offset, beside)
    norm = ctx.to_device(np.full(3, 5, np.float32))
    ctx.grad_norm(T.list, norm.offset(1))
    n = norm.numpy()
    want = norm64(values)
    assert n[0] == 5 and n[2] == 5 and abs(n[1] - want) <= 1.01 * U * want
    ctx.grad_clip(T.list, most, norm.offset(2))
    assert norm.numpy()[2] == n[1]
    got = T.get(T.outs)
    for g, w, b in zip(got, *clipped(values, dtypes, most)):
        over = np.abs(g - w) > b
        assert not over.any()
    if beside:
        for a, v in zip(T.get(T.bufs), values):
            assert np.array_equal(a, v)
    return got


SETS = [[1], [0, 5, 0], [1, 2, 3, 4, 7, 8, 9], [8191, 8192, 8193], [100000, 1, 16384, 333], [3] * 97, [50] * 300 + [70000]]


@pytest.mark.parametrize("beside", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "mixed"])
@pytest.mark.parametrize("sizes", SETS, ids=[f"set{i}" for i in range(len(SETS))])
def test_norm_and_clip(ctx, sizes, kind, offset, beside):
    rng = np.random.default_rng(len(sizes))
    values = [rng.standard_normal(n) * 10 ** rng.uniform(-3, 1) for n in sizes]
    dtypes = [kind if kind != "mixed" else ("f32", "bf16")[i % 2] for i in range(len(sizes))]
    check(ctx, values, dtypes, 0.5, offset, beside)


@pytest.mark.parametrize("beside", [False, True])
def test_small_norms_are_left_alone(ctx, beside):
    rng = np.random.default_rng(3)
    values = [rng.standard_normal(n).astype(np.float32) for n in (10, 9000)]
    got = check(ctx, values, ["f32", "bf16"], 1e4, beside=beside)
    assert np.array_equal(got[0], values[0]) and np.array_equal(got[1], held(values[1], "bf16"))


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e25, 1e38])
def test_range(ctx, scale):
    """Squares far outside fp32."""
    rng = np.random.default_rng(4)
    v = [(rng.uniform(0.5, 1.5, n) * scale).astype(np.float32) for n in (1000, 33)]
    T = Tensors(ctx, v, ["f32", "f32"])
    norm = ctx.empty(1)
    ctx.grad_norm(T.list, norm)
    want = norm64(v)
    got = norm.numpy()[0]
    assert np.isinf(got) if want > 3.41e38 else abs(got - want) <= 1.01 * U * want
    ctx.grad_clip(T.list, 1.0)
    for g, w, b in zip(T.get(T.bufs), *clipped(v, ["f32", "f32"], 1.0)):
        over = np.abs(g - w) > b
        assert not over.any()


def test_nan_and_infinity(ctx):
    for bad in (np.nan, np.inf):
        v = [np.ones(100, np.float32), np.ones(9000, np.float32)]
        v[1][77] = bad
        T = Tensors(ctx, v, ["f32", "bf16"], beside=True)
        norm = ctx.empty(1)
        ctx.grad_clip(T.list, 1.0, norm)
        n = norm.numpy()[0]
        assert np.isnan(n) if np.isnan(bad) else np.isinf(n)
        a, b = T.get(T.outs)
        if np.isnan(bad):
            assert np.isnan(a).all() and np.isnan(b).all()
        else:
            assert (a == 0).all() and np.isnan(b[77]) and (np.delete(b, 77) == 0).all()


def test_nothing(ctx):
    norm = ctx.to_device(np.full(1, 5, np.float32))
    for sizes in ([], [0, 0]):
        T = Tensors(ctx, [np.zeros(n, np.float32) for n in sizes], ["f32"] * len(sizes))
        norm.upload(np.full(1, 5, np.float32))
        ctx.grad_norm(T.list, norm)
        assert norm.numpy()[0] == 0
        norm.upload(np.full(1, 5, np.float32))
        ctx.grad_clip(T.list, 1.0, norm)
        assert norm.numpy()[0] == 0
    T = Tensors(ctx, [np.ones(5, np.float32)], ["f32"])
    ctx.grad_clip(T.list, 0.0)
    assert (T.get(T.bufs)[0] == 0).all()


def test_large(ctx):
    """More chunks than the grid has workgroups, in one tensor and over many."""
    rng = np.random.default_rng(6)
    a = rng.standard_normal(40_000_003).astype(np.float32)
    check(ctx, [a[:1000], a, a[:8192 * 3]], ["f32", "f32", "bf16"], 1.0, beside=True)
