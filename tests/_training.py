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
