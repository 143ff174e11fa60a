"""Plain 64-bit forms of the training operators (cross entropy of a linear layer,
gated products, gradients' norm and clipping) with the bounds that their results
are held to."""
import numpy as np

from _serving import bf16_bits, bf16_value

U = 2.0 ** -24   # half a step of fp32, relative
UB = 2.0 ** -8   # of bf16


def held(x, dtype):
    """fp32 values as a matrix of `dtype` holds them."""
    x = np.asarray(x, np.float32)
    return bf16_value(bf16_bits(x)) if dtype == "bf16" else x


class Mat:
    """A matrix on the device: rows of `ld` elements, `offset` elements into its buffer, `fill` around it."""

    FILL = -77.0

    def __init__(self, ctx, values, dtype, pad=0, offset=0):
        values = np.asarray(values, np.float32)
        rows, cols = values.shape
        self.ctx, self.dtype, self.shape, self.ld, self.at = ctx, dtype, (rows, cols), cols + pad, offset
        buf = np.full(offset + rows * self.ld + 16, self.FILL, np.float32)
        buf[offset:offset + rows * self.ld].reshape(rows, self.ld)[:, :cols] = values
        self.dev = ctx.to_device(bf16_bits(buf) if dtype == "bf16" else buf)
        self.ptr = self.dev.ptr + offset * self.dev.dtype.itemsize

    def get(self):
        """The values; what stands around them is as it was."""
        b = self.dev.numpy()
        b = bf16_value(b) if self.dtype == "bf16" else b
        rows, cols = self.shape
        n = self.at + rows * self.ld
        body = b[self.at:n].reshape(rows, self.ld)
        assert (b[:self.at] == self.FILL).all() and (b[n:] == self.FILL).all() and (body[:, cols:] == self.FILL).all()
        return body[:, :cols].copy()


# --- cross entropy -----------------------------------------------------------

def steps(k):
    """Roundings of an fp32 sum of k products on the matrix cores, sixteen to a rounding, with the dropped
    products of two splits (fp32 operands) and the joining of parts."""
    return k / 16 + 12


def cross_entropy64(x, w, target):
    """{loss, lse, mean, z, p, in} and bounds on loss and lse, in float64."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    vocab = w.shape[0]
    ok = (target >= 0) & (target < vocab)
    xs = np.where(ok[:, None], x, 0.0)
    z = xs @ w.T
    ez = (np.abs(xs) @ np.abs(w).T) * steps(x.shape[1]) * U
    top = z.max(1, keepdims=True)
    e = np.exp(z - top)
    lse = np.log(e.sum(1)) + top[:, 0]
    zt = z[np.arange(len(x)), np.where(ok, target, 0)]
    # Each exponential: its argument's product with log2 e, rounded (|z| + |top|), the function's own last place; a
    # lane's sum of at most 128 of them, the tiles' sums.
    eps = 3 * (np.abs(z).max(1) + np.abs(top[:, 0])) + 140 + 4 * (vocab / 128 + 1)
    elz = ez.max(1) + eps * U
    elses = elz + 4 * U * np.abs(lse)
    eloss = elses + ez[np.arange(len(x)), np.where(ok, target, 0)] + U * np.abs(lse - zt)
    zero = np.zeros(len(x))
    return dict(z=z, ez=ez, ok=ok, lse=np.where(ok, lse, zero), loss=np.where(ok, lse - zt, zero),
                e_lse=np.where(ok, elses, zero), e_loss=np.where(ok, eloss, zero))


def cross_entropy_bwd64(x, w, target, c, g, dtype, factor=1.0):
    """(dx, bound, dw, bound) for g's weight of each token, from cross_entropy64's c; `factor` of all."""
    x, w = np.where(c["ok"][:, None], np.asarray(x, np.float64), 0.0), np.asarray(w, np.float64)
    n, vocab = c["z"].shape
    p = np.exp(c["z"] - c["lse"][:, None])
    hot = np.zeros_like(p)
    hot[np.arange(n)[c["ok"]], target[c["ok"]]] = 1.0
    gs = np.where(c["ok"], g, 0.0)[:, None]
    G = gs * (p - hot)
    # p is off by its argument's error and the exponential's; the difference and the weight round once each.
    rel = c["ez"] + c["e_lse"][:, None] + (3 * (np.abs(c["z"]) + np.abs(c["lse"][:, None])) + 4) * U
    # Exponentials below fp32's least normal value are zeros.
    eG = np.abs(gs) * (p * rel + 2.0 ** -126) + 3 * U * np.abs(G)
    if dtype == "bf16":
        eG += np.abs(G) * (UB * UB if n <= 128 else UB) * 1.01
    half = UB if dtype == "bf16" else U
    aG = np.abs(G) + eG
    dx = (G @ w) * factor
    dw = (G.T @ x) * factor
    edx = (eG @ np.abs(w) + aG @ np.abs(w) * (steps(vocab) + 32) * U) * abs(factor) + 1.01 * half * np.abs(dx) + 4 * U * np.abs(dx)
    edw = (eG.T @ np.abs(x) + aG.T @ np.abs(x) * steps(n) * U) * abs(factor) + 1.01 * half * np.abs(dw) + 4 * U * np.abs(dw)
    return dx, edx * 1.05, dw, edw * 1.05


def near(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.isfinite(got).all(), f"{what}: not finite"
    err = np.abs(got.astype(np.float64) - want)
    over = err - bound
    if err.size and over.max() > 0:
        at = np.unravel_index(np.argmax(over), over.shape)
        raise AssertionError(f"{what}: {err[at]:.3g} off {want[at]:.6g} at {at}, bound {bound[at]:.3g}; {(over > 0).sum()} of {over.size} over")


# --- gated products ----------------------------------------------------------

def activation64(name, x):
    """(act, act', the logistic's argument) in float64."""
    if name == "silu":
        v, dv = x, np.ones_like(x)
    else:
        k = 2 * np.sqrt(2 / np.pi)
        v, dv = k * (x + 0.044715 * x ** 3), k * (1 + 3 * 0.044715 * x ** 2)
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-v))
        one_s = 1 / (1 + np.exp(v))
    return x * s, s + x * s * one_s * dv, v


def gated64(x, wg, wu, act, dtype):
    """{y, bound, gate, up and what their products may be off by}."""
    x, wg, wu = (np.asarray(a, np.float64) for a in (x, wg, wu))
    gate, up = x @ wg, x @ wu
    eg, eu = (np.abs(x) @ np.abs(w) * steps(x.shape[1]) * U for w in (wg, wu))
    a, slope, v = activation64(act, gate)
    # act' is at most 1.13 and act'' 1.6 of either form; the exponential's argument rounds a few times (6 U |v|), the
    # function, the reciprocal and the products a few more.
    ea = 1.2 * eg + np.abs(a) * (10 + 6 * np.abs(v)) * U
    half = UB if dtype == "bf16" else U
    y = a * up
    ey = ea * np.abs(up) + (np.abs(a) + ea) * eu + 2 * U * np.abs(y) + 1.01 * half * np.abs(y) + 2.0 ** -126
    s = np.abs(slope) + np.abs(slope - a / np.where(gate == 0, 1, gate))
    es = 1.7 * eg + s * (12 + 6 * np.abs(v)) * U
    return dict(y=y, ey=ey, gate=gate, up=up, eg=eg, eu=eu, a=a, ea=ea, slope=slope, es=es)


def gated_bwd64(x, wg, wu, dy, c, dtype):
    """{name: (value, bound)} of dx, dwg, dwu from gated64's c."""
    x, wg, wu, dy = (np.asarray(a, np.float64) for a in (x, wg, wu, dy))
    n, d = x.shape
    du, dg = dy * c["a"], dy * c["up"] * c["slope"]
    edu = np.abs(dy) * c["ea"] + 2 * U * np.abs(du)
    edg = np.abs(dy) * (c["eu"] * (np.abs(c["slope"]) + c["es"]) + np.abs(c["up"]) * c["es"]) + 3 * U * np.abs(dg)
    if dtype == "bf16":
        r = 1.01 * (UB * UB if n <= 128 else UB)
        edu, edg = edu + r * np.abs(du), edg + r * np.abs(dg)
    half = UB if dtype == "bf16" else U
    adu, adg = np.abs(du) + edu, np.abs(dg) + edg
    out = {}
    k = steps(2 * wg.shape[1]) + 70
    dx = dg @ wg.T + du @ wu.T
    out["dx"] = dx, 1.05 * (edg @ np.abs(wg).T + edu @ np.abs(wu).T + (adg @ np.abs(wg).T + adu @ np.abs(wu).T) * k * U + 1.01 * half * np.abs(dx)) + 2.0 ** -120
    for name, g, e, a in (("dwg", dg, edg, adg), ("dwu", du, edu, adu)):
        w = x.T @ g
        out[name] = w, 1.05 * (np.abs(x).T @ e + np.abs(x).T @ a * (steps(n) + 70) * U + 1.01 * half * np.abs(w)) + 2.0 ** -120
    return out
