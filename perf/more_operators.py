"""Cases of a training step's operators: the cross entropy of a linear output
layer without its logits, the gated products of a feed-forward block, and the
norm and clipping of many gradients.

A case is a dict of plain values.  ``prepare`` makes its inputs on the GPU,
``run`` is one pass (elementary torch where ``own`` is false, the library's
entry points where it is true), ``exact`` the same results in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
F32, F64 = torch.float32, torch.float64
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
_LIB = []


def lib():
    """The package and the one context that a single-threaded program keeps."""
    if not _LIB:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mimir-framework_amd"))
        import mimir_hip

        _LIB.extend([mimir_hip, mimir_hip.Context(0)])
    return _LIB


# --- cases -------------------------------------------------------------------

def listed():
    def loss(name, **c):
        return dict(name=name, op="loss", **{"masked": 0.0, "pad": 0, **c})

    def gated(name, **c):
        return dict(name=name, op="gated", **{"pad": 0, **c})

    def clip(name, **c):
        return dict(name=name, op="clip", **c)

    return [
        # The score of one short text: the smallest call, all latency.
        loss("loss_score_small", type="f32", tokens=17, dim=256, vocab=1000, back=False),
        # A few continuations scored against a whole vocabulary: the weights' bytes.
        loss("loss_score", type="bf16", tokens=32, dim=4096, vocab=32000, back=False),
        # An evaluation batch.
        loss("loss_eval", type="bf16", tokens=2048, dim=4096, vocab=32000, back=False),
        # A small model's training step in full precision; the prompts' tokens have no target.
        loss("loss_train", type="f32", tokens=1024, dim=1024, vocab=32000, back=True, masked=0.4),
        # Odd sizes, rows with a stride.
        loss("loss_train_odd", type="bf16", tokens=777, dim=1001, vocab=50001, back=True, masked=0.1, pad=7),
        # A training step of the widest rows.
        loss("loss_train_wide", type="bf16", tokens=8192, dim=4096, vocab=32000, back=True),
        # One token of seven sequences through a feed-forward block.
        gated("gated_step", type="f32", act="silu", tokens=7, dim=1024, hidden=2752, back=False),
        # A prompt.
        gated("gated_prompt", type="bf16", act="silu", tokens=2048, dim=4096, hidden=11008, back=False),
        # A small model's training step in full precision, an odd number of tokens.
        gated("gated_train", type="f32", act="gelu", tokens=1021, dim=1024, hidden=2752, back=True),
        # A training step of the widest rows.
        gated("gated_train_wide", type="bf16", act="silu", tokens=8192, dim=4096, hidden=11008, back=True),
        # A small model: four layers' gradients.
        clip("clip_small", type="f32", dim=256, hidden=688, layers=4, vocab=1000, most=1.0),
        # A larger one's: matrices in bf16, the norms' gradients in fp32.
        clip("clip_large", type="mixed", dim=2048, hidden=5504, layers=6, vocab=32000, most=1.0),
    ]


def span(rng, lo, hi):
    """A size between lo and hi, even over the logarithm, odd ones among them."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.4 and n >= 64:
        n = n // 32 * 32
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["loss", "loss", "gated", "gated", "clip"])
    if op == "clip":
        c = dict(op=op, type=rng.choice(["f32", "bf16", "mixed"]), dim=span(rng, 16, 2048), layers=span(rng, 1, 40),
                 vocab=span(rng, 100, 32000), most=rng.choice([0.25, 1.0, 1e4]))
        c["hidden"] = span(rng, 16, 4 * c["dim"])
        while work(c)["bytes"] > 1.2e9:
            c["layers"] = max(1, c["layers"] // 2)
            c["vocab"] = max(1, c["vocab"] // 2)
        return c
    c = dict(op=op, type=rng.choice(["f32", "bf16", "bf16"]), back=rng.random() < 0.6, pad=rng.choice([0, 0, 0, 8, 5]),
             tokens=span(rng, 1, 8192), dim=span(rng, 32, 4096))
    if op == "loss":
        c.update(vocab=span(rng, 50, 64000), masked=rng.choice([0.0, 0.0, 0.3, 0.9]))
    else:
        c.update(hidden=span(rng, 32, 16384), act=rng.choice(["silu", "gelu"]))
    # In full precision no more than a tenth of the products of the largest listed cases.
    while work(c)["flops"] > (4.4e12 if c["type"] == "bf16" else 4.4e11):
        c["tokens"] = c["tokens"] // 2
    return c


def clip_shapes(c):
    """[(elements, type)] of a model's gradients: the embedding, each layer's matrices and norms, the last norm."""
    d, f = c["dim"], c["hidden"]
    wide = "f32" if c["type"] == "f32" else "bf16"
    thin = "bf16" if c["type"] == "bf16" else "f32"
    layer = [(3 * d * d, wide), (d * d, wide), (d * f, wide), (d * f, wide), (f * d, wide), (d, thin), (d, thin)]
    return [(c["vocab"] * d, wide)] + layer * c["layers"] + [(d, thin)]


# --- inputs ------------------------------------------------------------------

class Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        return torch.randn(shape, generator=self.g, device=DEV).mul_(scale)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device=DEV)

    def ints(self, n, hi):
        return torch.randint(hi, (n,), generator=self.g, device=DEV)


def matrix(r, rows, cols, pad, dtype, scale=1.0):
    """rows x cols in rows of cols + pad."""
    return r.normal(rows, cols + pad, scale=scale).to(dtype)[:, :cols]


def prepare(case, seed):
    c, r = case, Rand(seed)
    s = {"case": c}
    if c["op"] == "clip":
        # Gradients of different size from tensor to tensor, as layers have them.
        shapes = clip_shapes(c)
        size = r.uniform(len(shapes)).mul_(3).exp_().mul_(1e-3).tolist()
        s["grads"] = [r.normal(n, scale=a).to(TYPES[t]) for (n, t), a in zip(shapes, size)]
        s["out"] = [torch.empty_like(g) for g in s["grads"]]
        s["norm"] = torch.empty(1, device=DEV)
        torch.cuda.synchronize()
        return s
    t, d, pad, kind = c["tokens"], c["dim"], c["pad"], TYPES[c["type"]]
    # Rows as a norm layer leaves them.
    s["x"] = matrix(r, t, d, pad, kind)
    empty = dict(device=DEV, dtype=kind)
    if c["op"] == "loss":
        s["w"] = matrix(r, c["vocab"], d, pad, kind, scale=2 / math.sqrt(d))
        target = r.ints(t, c["vocab"])
        target[r.uniform(t) < c["masked"]] = -1
        s["target"] = target.to(torch.int32)
        s["loss"], s["lse"], s["mean"] = torch.empty(t, device=DEV), torch.empty(t, device=DEV), torch.empty(2, device=DEV)
        if c["back"]:
            s["dx"], s["dw"] = torch.empty(t, d, **empty), torch.empty(c["vocab"], d, **empty)
    else:
        f = c["hidden"]
        s["wg"], s["wu"] = (matrix(r, d, f, pad, kind, scale=1 / math.sqrt(d)) for _ in range(2))
        s["y"] = torch.empty(t, f, **empty)
        if c["back"]:
            s["dy"] = r.normal(t, f, scale=0.1).to(kind)
            s["gate_up"] = torch.empty(t, 2 * f, device=DEV)
            s["dx"], s["dwg"], s["dwu"] = torch.empty(t, d, **empty), torch.empty(d, f, **empty), torch.empty(d, f, **empty)
    # The library works on a stream of its own: the inputs have to be there.
    torch.cuda.synchronize()
    return s


# --- the library's calls -----------------------------------------------------

def run_own(s):
    M, ctx = lib()
    c = s["case"]
    if c["op"] == "clip":
        if "list" not in s:  # which a program keeps
            s["list"] = M.TensorList([(g.data_ptr(), g.numel(), "f32" if g.dtype == F32 else "bf16", o.data_ptr())
                                      for g, o in zip(s["grads"], s["out"])])
        ctx.grad_clip(s["list"], c["most"], s["norm"].data_ptr())
        return {"norm": s["norm"], "grads": s["out"]}
    p = {k: v.data_ptr() for k, v in s.items() if torch.is_tensor(v)}
    t, d, ld_x = c["tokens"], c["dim"], s["x"].stride(0)
    if c["op"] == "loss":
        kw = dict(dtype=c["type"], ld_x=ld_x, ld_w=s["w"].stride(0))
        ctx.linear_cross_entropy(p["x"], p["w"], p["target"], t, d, c["vocab"], p["loss"], p["lse"], p["mean"], **kw)
        out = {"loss": s["loss"], "lse": s["lse"], "mean": s["mean"]}
        if c["back"]:
            ctx.linear_cross_entropy_bwd(p["x"], p["w"], p["target"], p["lse"], None, p["mean"], p["dx"], p["dw"], t, d,
                                         c["vocab"], **kw)
            out.update(dx=s["dx"], dw=s["dw"])
        return out
    f = c["hidden"]
    kw = dict(act=c["act"], dtype=c["type"], ld_x=ld_x, ld_w=s["wg"].stride(0))
    ctx.gated_linear(p["x"], p["wg"], p["wu"], p["y"], t, d, f, gate_up=p.get("gate_up"), **kw)
    if not c["back"]:
        return s["y"]
    ctx.gated_linear_bwd(p["x"], p["wg"], p["wu"], p["gate_up"], p["dy"], p["dx"], p["dwg"], p["dwu"], t, d, f, **kw)
    return {k: s[k] for k in ("y", "dx", "dwg", "dwu")}


# --- plain forms -------------------------------------------------------------

def run_plain(s):
    c = s["case"]
    if c["op"] == "clip":
        total = torch.stack([(g.to(F32) * g.to(F32)).sum(dtype=F64) for g in s["grads"]]).sum()
        norm = total.sqrt()
        by = (c["most"] / (norm + 1e-6)).clamp(max=1.0).to(F32)
        return {"norm": norm.to(F32).reshape(1), "grads": [(g.to(F32) * by).to(g.dtype) for g in s["grads"]]}
    kind = TYPES[c["type"]]
    x = s["x"].to(F32)
    if c["op"] == "loss":
        w = s["w"].to(F32)
        z = x @ w.T
        row = torch.arange(c["tokens"], device=DEV)
        counts = s["target"] >= 0
        at = s["target"].clamp(min=0).long()
        top = z.amax(1, keepdim=True)
        lse = (z - top).exp().sum(1).log() + top[:, 0]
        loss = torch.where(counts, lse - z[row, at], 0.0)
        lse = torch.where(counts, lse, 0.0)
        count = counts.sum().to(F32)
        mean = torch.stack([loss.sum(dtype=F64).to(F32) / count.clamp(min=1), count])
        out = {"loss": loss, "lse": lse, "mean": mean}
        if c["back"]:
            g = (z - lse[:, None]).exp()
            g[row, at] -= 1
            g = torch.where(counts[:, None], g / count.clamp(min=1), 0.0)
            out.update(dx=(g @ w).to(kind), dw=(g.T @ x).to(kind))
        return out
    wg, wu = s["wg"].to(F32), s["wu"].to(F32)
    gate, up = x @ wg, x @ wu
    if c["act"] == "silu":
        sig = 1 / (1 + (-gate).exp())
        act, slope = gate * sig, sig + gate * sig * (1 - sig)
    else:
        k = math.sqrt(2 / math.pi)
        sig = 1 / (1 + (-2 * k * (gate + 0.044715 * gate ** 3)).exp())
        act, slope = gate * sig, sig + gate * sig * (1 - sig) * 2 * k * (1 + 3 * 0.044715 * gate * gate)
    y = (act * up).to(kind)
    if not c["back"]:
        return y
    dy = s["dy"].to(F32)
    du, dg = dy * act, dy * up * slope
    return {"y": y, "dx": (dg @ wg.T + du @ wu.T).to(kind), "dwg": (x.T @ dg).to(kind), "dwu": (x.T @ du).to(kind)}


def run(state):
    return run_own(state) if own else run_plain(state)


# --- the same in 64 bits -----------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "clip":
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.to(F64))) ** 2 for g in s["grads"]))
        by = min(1.0, c["most"] / (norm + 1e-6))
        return {"norm": torch.tensor([norm], device=DEV, dtype=F64), "grads": [g.to(F64) * by for g in s["grads"]]}
    x = s["x"].to(F64).requires_grad_(c["back"])
    if c["op"] == "loss":
        w = s["w"].to(F64).requires_grad_(c["back"])
        has = (s["target"] >= 0).nonzero()[:, 0]
        z = torch.mm(x[has], w.t())
        lse = torch.logsumexp(z, 1)
        loss = lse - z.gather(1, s["target"][has].long()[:, None])[:, 0]
        mean = loss.sum() / max(1, len(has))
        full = torch.zeros(2, c["tokens"], device=DEV, dtype=F64)
        full[0, has], full[1, has] = loss.detach(), lse.detach()
        out = {"loss": full[0], "lse": full[1], "mean": torch.stack([mean.detach(), mean.detach().new_tensor(len(has))])}
        if c["back"]:
            mean.backward()
            out.update(dx=x.grad, dw=w.grad)
        return out
    w = [s[n].to(F64).requires_grad_(c["back"]) for n in ("wg", "wu")]
    gate, up = torch.mm(x, w[0]), torch.mm(x, w[1])
    if c["act"] == "silu":
        act = gate * torch.sigmoid(gate)
    else:
        act = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
    y = act * up
    if not c["back"]:
        return y
    y.backward(s["dy"].to(F64))
    return {"y": y.detach(), "dx": x.grad, "dwg": w[0].grad, "dwu": w[1].grad}


# --- what a pass cannot do without -------------------------------------------

def work(case):
    c = case
    if c["op"] == "clip":
        shapes = clip_shapes(c)
        return {"bytes": sum(2 * n * BYTES[t] for n, t in shapes) + 4, "flops": sum(3 * n for n, _ in shapes)}
    t, d, b = c["tokens"], c["dim"], BYTES[c["type"]]
    if c["op"] == "loss":
        v = c["vocab"]
        # Inputs and gradients; targets, losses and statistics.
        return {"bytes": (t * d + v * d) * b * (2 if c["back"] else 1) + 12 * t + 8, "flops": 2 * t * d * v * (3 if c["back"] else 1)}
    f = c["hidden"]
    once = (t * d + 2 * d * f) * b
    return {"bytes": (2 * once + 2 * t * f * b) if c["back"] else once + t * f * b, "flops": 4 * t * d * f * (3 if c["back"] else 1)}
