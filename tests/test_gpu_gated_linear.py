"""Gated products of a feed-forward block against float64: both types and
activations, both tile shapes, hidden columns in one piece and in several, odd
sizes and strides, gradients written and added to."""
import numpy as np
import pytest

import mimir_hip as M
from _serving import bf16_value
from _training import Mat, UB, U, gated64, gated_bwd64, held, near

pytestmark = pytest.mark.gpu
SENTINEL = np.float32(5.0)


@pytest.fixture(scope="module", params=["", "matbig=1,matpiece=264", "matbig=0,matpiece=136"], ids=["default", "big", "small"])
def tuned(request):
    """A context of its own: the shapes and pieces by rule, or forced."""
    with pytest.MonkeyPatch.context() as mp:
        mp.setenv("MIMIR_TUNE", request.param)
        c = M.Context(0)
    yield c
    c.close()


def make(seed, tokens, dim, hidden, dtype, spread=1.0):
    rng = np.random.default_rng(seed)
    x = held(rng.standard_normal((tokens, dim)), dtype)
    wg, wu = (held(rng.standard_normal((dim, hidden)) * spread / np.sqrt(dim), dtype) for _ in range(2))
    return x, wg, wu, held(rng.standard_normal((tokens, hidden)), dtype)


def run(ctx, x, wg, wu, dy, act, dtype, keep=True, back=True, pad=0, offset=0, start=None, want=("dx", "dw")):
    tokens, dim = x.shape
    hidden = wg.shape[1]
    X, G, W, DY = (Mat(ctx, a, dtype, pad, offset) for a in (x, wg, wu, dy))
    Y = Mat(ctx, np.full(dy.shape, 9.0), dtype, pad, offset)
    gu = ctx.to_device(np.full(max(1, tokens * 2 * hidden) + 8, SENTINEL)) if keep else None
    kw = dict(act=act, dtype=dtype, ld_x=X.ld, ld_w=G.ld)
    ctx.gated_linear(X.ptr, G.ptr, W.ptr, Y.ptr, tokens, dim, hidden, gate_up=gu, ld_y=Y.ld, **kw)
    out = {"y": Y.get()}
    if keep:
        n = gu.numpy()
        assert (n[tokens * 2 * hidden:][-8:] == SENTINEL).all()
        out["gate_up"] = n[:tokens * 2 * hidden].reshape(tokens, 2, hidden)
    if back:
        s = start or [np.full(a.shape, 9.0) for a in (x, wg, wu)]
        DX, DG, DU = (Mat(ctx, a, dtype, pad, offset) for a in s)
        ctx.gated_linear_bwd(X.ptr, G.ptr, W.ptr, gu, DY.ptr, DX.ptr if "dx" in want else None, DG.ptr if "dw" in want else None,
                             DU.ptr if "dw" in want else None, tokens, dim, hidden, ld_dy=DY.ld, ld_dx=DX.ld, ld_dw=DG.ld,
                             accumulate_x=start is not None, accumulate_w=start is not None, **kw)
        out.update(dx=DX.get(), dwg=DG.get(), dwu=DU.get())
    assert (X.get() == x).all() and (G.get() == wg).all() and (W.get() == wu).all()
    return out


def hold(got, x, wg, wu, dy, act, dtype, start=None):
    c = gated64(x, wg, wu, act, dtype)
    near(got["y"], c["y"], c["ey"], "y")
    if "gate_up" in got:
        near(got["gate_up"][:, 0], c["gate"], c["eg"], "gate")
        near(got["gate_up"][:, 1], c["up"], c["eu"], "up")
    if "dx" in got:
        for i, (name, (want, bound)) in enumerate(gated_bwd64(x, wg, wu, dy, c, dtype).items()):
            if start is not None:
                s = held(start[i], dtype)
                want, bound = want + s, bound + 1.1 * (UB if dtype == "bf16" else U) * np.abs(s)
            near(got[name], want, bound, name)


SIZES = [(1, 1, 1), (1, 8, 3), (7, 24, 72), (32, 296, 1000), (17, 1024, 40), (5, 2048, 64), (40, 1100, 70), (70, 2051, 129), (20, 8, 8), (31, 136, 36), (9, 37, 71), (32, 1003, 335), (16, 30, 34), (4, 6, 5), (2, 5, 100), (3, 64, 257), (31, 33, 129), (32, 64, 128), (33, 65, 300), (65, 136, 520),
         (129, 100, 513), (300, 40, 77), (130, 1000, 264), (1000, 16, 24)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("tokens,dim,hidden", SIZES)
def test_sizes(tuned, tokens, dim, hidden, act, dtype):
    a = make(tokens * 7 + dim, tokens, dim, hidden, dtype)
    hold(run(tuned, *a, act, dtype), *a, act, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,offset", [(0, 3), (8, 0), (5, 1), (24, 8)])
def test_strides_and_alignment(tuned, pad, offset, dtype):
    a = make(pad + offset, 45, 48, 328, dtype)
    hold(run(tuned, *a, "silu", dtype, pad=pad, offset=offset), *a, "silu", dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sums_and_parts(tuned, dtype):
    a = make(8, 90, 56, 400, dtype)
    rng = np.random.default_rng(9)
    start = [rng.standard_normal(v.shape) for v in a[:3]]
    hold(run(tuned, *a, "gelu", dtype, start=start), *a, "gelu", dtype, start=start)
    full = run(tuned, *a, "gelu", dtype)
    dx = run(tuned, *a, "gelu", dtype, want=("dx",))
    dw = run(tuned, *a, "gelu", dtype, want=("dw",))
    assert (dx["dx"] == full["dx"]).all() and (dx["dwg"] == 9).all() and (dx["dwu"] == 9).all()
    assert (dw["dwg"] == full["dwg"]).all() and (dw["dwu"] == full["dwu"]).all() and (dw["dx"] == 9).all()
    assert (run(tuned, *a, "gelu", dtype, keep=False, back=False)["y"] == full["y"]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_far_gates(tuned, act, dtype):
    """Gates of some hundreds: an activation is its input or nothing there."""
    a = make(13, 40, 64, 200, dtype, spread=60.0)
    hold(run(tuned, *a, act, dtype), *a, act, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,dim,hidden", [(2050, 72, 3000), (1300, 1500, 520)])
def test_many_tiles(ctx, tokens, dim, hidden, dtype):
    a = make(tokens, tokens, dim, hidden, dtype)
    hold(run(ctx, *a, "silu", dtype), *a, "silu", dtype)


def test_no_tokens(ctx):
    w = np.ones((6, 10), np.float32)
    for dtype in ("f32", "bf16"):
        W, A, B = Mat(ctx, w, dtype), Mat(ctx, 3 * w, dtype), Mat(ctx, 3 * w, dtype)
        ctx.gated_linear(None, W.ptr, W.ptr, None, 0, 6, 10, dtype=dtype)
        ctx.gated_linear_bwd(None, W.ptr, W.ptr, None, None, None, A.ptr, B.ptr, 0, 6, 10, dtype=dtype, accumulate_w=True)
        assert (A.get() == 3).all() and (B.get() == 3).all()
        ctx.gated_linear_bwd(None, W.ptr, W.ptr, None, None, None, A.ptr, B.ptr, 0, 6, 10, dtype=dtype)
        assert (A.get() == 0).all() and (B.get() == 0).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_against_differences(ctx, act):
    x, wg, wu, dy = make(33, 4, 6, 7, "f32")
    got = run(ctx, x, wg, wu, dy, act, "f32")
    h = 1e-4

    def value(*a):
        return (gated64(*a, act, "f32")["y"] * dy).sum()

    for which, name in enumerate(("dx", "dwg", "dwu")):
        for at in np.ndindex(*got[name].shape):
            a = [v.astype(np.float64) for v in (x, wg, wu)]
            b = [v.copy() for v in a]
            a[which][at] += h
            b[which][at] -= h
            # The differences' own error: h^2 / 6 times third derivatives of some tens.
            assert abs((value(*a) - value(*b)) / (2 * h) - got[name][at]) < 5e-6


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_same_bits_again(ctx, dtype):
    a = make(41, 260, 72, 1000, dtype)
    u, v = run(ctx, *a, "silu", dtype), run(ctx, *a, "silu", dtype)
    for name in u:
        assert np.array_equal(u[name], v[name]), name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_past_32_bits(ctx, dtype):
    """gate_up of more than 2^31 values, y of more than 2^32 bytes in fp32: the last rows."""
    tokens, dim, hidden, last = 70001, 8, 16384, 3
    x, wg, wu, _ = make(3, tokens, dim, 1, dtype)
    rng = np.random.default_rng(4)
    wg, wu = (held(rng.standard_normal((dim, hidden)), dtype) for _ in range(2))
    X, G, W = Mat(ctx, x, dtype), Mat(ctx, wg, dtype), Mat(ctx, wu, dtype)
    y = ctx.empty(tokens * hidden, np.float32 if dtype == "f32" else np.uint16)
    gu = ctx.empty(tokens * 2 * hidden)
    ctx.gated_linear(X.ptr, G.ptr, W.ptr, y, tokens, dim, hidden, gate_up=gu, dtype=dtype)
    c = gated64(x[-last:], wg, wu, "silu", dtype)
    got = y.offset((tokens - last) * hidden, (last, hidden)).numpy()
    near(bf16_value(got) if dtype == "bf16" else got, c["y"], c["ey"], "y")
    keep = gu.offset((tokens - last) * 2 * hidden, (last, 2, hidden)).numpy()
    near(keep[:, 0], c["gate"], c["eg"], "gate")
    near(keep[:, 1], c["up"], c["eu"], "up")
    y.free()
    gu.free()
