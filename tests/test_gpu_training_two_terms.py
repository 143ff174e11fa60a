"""Gradients of bf16 matrices held in two terms between the products, with more tokens
than take them by themselves, against float64: off by their own rounding and the second
term's, no more."""
import numpy as np
import pytest

import mimir_hip as M
from _training import UB, Mat, activation64, cross_entropy64, cross_entropy_bwd64, gated64, gated_bwd64, near
from test_gpu_gated_linear import make as make_gated
from test_gpu_linear_ce import make as make_ce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["", "matbig=1,matpiece=264", "matbig=0,matpiece=136"], ids=["default", "big", "small"])
def tuned(request):
    """A context of its own: the shapes and pieces by rule, or forced."""
    with pytest.MonkeyPatch.context() as mp:
        mp.setenv("MIMIR_TUNE", request.param)
        c = M.Context(0)
    yield c
    c.close()


def rounded(want, bound32, terms):
    """fp32's bound, the result's rounding to bf16 and the two terms' 2^-16 of what is summed."""
    return bound32 + 1.02 * UB * np.abs(want) + 1.1 * UB * UB * terms


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("tokens,dim,vocab", [(129, 40, 300), (300, 101, 777), (1100, 72, 2000)])
def test_cross_entropy(tuned, tokens, dim, vocab, accumulate):
    x, w, t = make_ce(tokens, tokens, dim, vocab, "bf16", 0.2)
    X, W, T = Mat(tuned, x, "bf16", 3, 1), Mat(tuned, w, "bf16", 8), tuned.to_device(t)
    loss, lse, mean = (tuned.empty(n) for n in (tokens, tokens, 2))
    kw = dict(dtype="bf16", ld_x=X.ld, ld_w=W.ld)
    tuned.linear_cross_entropy(X.ptr, W.ptr, T, tokens, dim, vocab, loss, lse, mean, **kw)
    c = cross_entropy64(x, w, t)
    factor = 1 / c["ok"].sum()
    dx, edx, dw, edw = cross_entropy_bwd64(x, w, t, c, np.ones(tokens), "f32", factor)
    g = np.exp(c["z"] - c["lse"][:, None])
    g[np.arange(tokens)[c["ok"]], t[c["ok"]]] -= 1
    g = np.abs(np.where(c["ok"][:, None], g, 0)) * factor
    DX, DW = Mat(tuned, np.zeros(x.shape), "bf16"), Mat(tuned, np.zeros(w.shape), "bf16")
    tuned.linear_cross_entropy_bwd(X.ptr, W.ptr, T, lse, None, mean, DX.ptr, DW.ptr, tokens, dim, vocab, two_terms=True,
                                   accumulate_x=accumulate, accumulate_w=accumulate, **kw)
    near(DX.get(), dx, rounded(dx, edx, g @ np.abs(w.astype(np.float64))), "dx")
    near(DW.get(), dw, rounded(dw, edw, g.T @ np.abs(np.where(c["ok"][:, None], x, 0).astype(np.float64))), "dw")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("tokens,dim,hidden", [(129, 40, 300), (300, 101, 777), (1100, 72, 1000)])
def test_gated_products(tuned, tokens, dim, hidden, act):
    x, wg, wu, dy = make_gated(tokens, tokens, dim, hidden, "bf16")
    X, G, W, DY = Mat(tuned, x, "bf16", 3, 1), Mat(tuned, wg, "bf16", 5), Mat(tuned, wu, "bf16", 5), Mat(tuned, dy, "bf16", 1)
    Y, DX, DG, DU = (Mat(tuned, np.full(a.shape, 9.0), "bf16") for a in (dy, x, wg, wu))
    gu = tuned.empty((tokens, 2 * hidden))
    kw = dict(act=act, dtype="bf16", ld_x=X.ld, ld_w=G.ld)
    tuned.gated_linear(X.ptr, G.ptr, W.ptr, Y.ptr, tokens, dim, hidden, gate_up=gu, **kw)
    tuned.gated_linear_bwd(X.ptr, G.ptr, W.ptr, gu, DY.ptr, DX.ptr, DG.ptr, DU.ptr, tokens, dim, hidden, ld_dy=DY.ld, two_terms=True, **kw)
    c = gated64(x, wg, wu, act, "f32")
    ax, a = np.abs(x.astype(np.float64)), [np.abs(v.astype(np.float64)) for v in (wg, wu)]
    act64, slope, _ = activation64(act, c["gate"])
    dg, du = np.abs(dy * c["up"] * slope), np.abs(dy * act64)
    terms = {"dx": dg @ a[0].T + du @ a[1].T, "dwg": ax.T @ dg, "dwu": ax.T @ du}
    got = {"dx": DX.get(), "dwg": DG.get(), "dwu": DU.get()}
    for name, (want, bound) in gated_bwd64(x, wg, wu, dy, c, "f32").items():
        near(got[name], want, rounded(want, bound, terms[name]), name)


def test_errors_by_size(ctx):
    """Normwise: one term is off by about 1.4 times a single rounding, two terms by that rounding."""
    x, wg, wu, dy = make_gated(7, 1000, 64, 512, "bf16")
    X, G, W, DY = (Mat(ctx, a, "bf16") for a in (x, wg, wu, dy))
    Y, DX, DG, DU = (Mat(ctx, np.zeros(a.shape), "bf16") for a in (dy, x, wg, wu))
    gu = ctx.empty((1000, 1024))
    ctx.gated_linear(X.ptr, G.ptr, W.ptr, Y.ptr, 1000, 64, 512, gate_up=gu, dtype="bf16")
    want = gated_bwd64(x, wg, wu, dy, gated64(x, wg, wu, "silu", "f32"), "f32")
    off = {}
    for two in (False, True):
        ctx.gated_linear_bwd(X.ptr, G.ptr, W.ptr, gu, DY.ptr, DX.ptr, DG.ptr, DU.ptr, 1000, 64, 512, dtype="bf16", two_terms=two)
        off[two] = [np.linalg.norm(m.get() - want[n][0]) / np.linalg.norm(want[n][0]) for m, n in ((DX, "dx"), (DG, "dwg"), (DU, "dwu"))]
    # A rounding to bf16 is off by 2^-8 of the binade's bottom at most, evenly spread: 2^-8 / sqrt 3 of it in the mean
    # square, and values spread over the binade are 1.4 to 1.5 times its bottom: 0.0016.
    for one, two in zip(off[False], off[True]):
        assert two < 0.0019 and one > 1.2 * two, off
