"""Cases of the serving operators: rotary positions per token, a cache of keys
and values in pages (written and read back), and attention over that cache.

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
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "i8": 1}
THETA = 10000.0
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
    def rope(name, **c):
        return dict(name=name, op="rope", **c)

    def store(name, **c):
        return dict(name=name, op="store", **c)

    def attend(name, **c):
        return dict(name=name, op="attend", **c)

    return [
        # One decoding step of seven sequences: the smallest call, all latency.
        rope("rope_step", tokens=7, heads=32, kv_heads=8, head_dim=128, rot_dim=128, interleaved=False, far=4000, back=False),
        # A training batch of packed documents, q and k as column blocks of one QKV buffer.
        rope("rope_train", tokens=8192, heads=32, kv_heads=8, head_dim=128, rot_dim=128, interleaved=False, far=0, back=False),
        # The gradient of a layer that rotates half of each head, pairs side by side, an odd number of tokens.
        rope("rope_train_back", tokens=4099, heads=28, kv_heads=4, head_dim=128, rot_dim=64, interleaved=True, far=0, back=True),
        # A decoding step of 48 sequences: q rotated, k and v into a bf16 cache.
        store("store_step", type="bf16", seqs=48, new=1, past=4000, how="even", page=16, heads=32, kv_heads=8, head_dim=128,
              rot_dim=128, interleaved=False),
        # A chunk of prompts after some context, kept in full precision; heads of 80 of which 32 are rotated.
        store("store_chunk", type="f32", seqs=5, new=333, past=700, how="ragged", page=48, heads=16, kv_heads=2, head_dim=80,
              rot_dim=32, interleaved=True),
        # Whole prompts into an 8-bit cache.
        store("store_prompt", type="i8", seqs=3, new=5000, past=0, how="ragged", page=64, heads=32, kv_heads=8, head_dim=128,
              rot_dim=128, interleaved=False),
        # The smallest attention call: two short sequences, every head with its own keys.
        attend("attend_step_small", type="f32", seqs=2, new=1, past=100, how="even", page=16, heads=8, kv_heads=8, head_dim=64),
        # A serving batch: 64 sequences of different lengths, one token each, 8-bit cache.
        attend("attend_step_batch", type="i8", seqs=64, new=1, past=8190, how="ragged", page=64, heads=32, kv_heads=8, head_dim=128),
        # One sequence with a very long context.
        attend("attend_step_long", type="bf16", seqs=1, new=1, past=131001, how="even", page=64, heads=32, kv_heads=8, head_dim=128),
        # A chunk of one long prompt against what is cached already.
        attend("attend_chunk", type="bf16", seqs=1, new=512, past=8300, how="even", page=64, heads=32, kv_heads=8, head_dim=128),
        # Whole prompts of different lengths in full precision.
        attend("attend_prompt", type="f32", seqs=4, new=2048, past=0, how="ragged", page=32, heads=16, kv_heads=16, head_dim=128),
        # Prompt chunks and single tokens in one batch, odd sizes, 8-bit cache.
        attend("attend_mixed", type="i8", seqs=24, new=217, past=3001, how="mixed", page=16, heads=20, kv_heads=4, head_dim=80),
    ]


def span(rng, lo, hi):
    """A size between lo and hi, even over the logarithm, odd ones among them."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.4 and n >= 64:
        n = n // 32 * 32
    return max(lo, min(hi, n))


def _layout(rng):
    kv = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 2, 4, 4, 5, 8])
    return dict(heads=kv * group, kv_heads=kv, head_dim=rng.choice([32, 64, 64, 72, 80, 96, 112, 128, 128, 128, 256]))


def draw(rng):
    op = rng.choice(["rope", "store", "attend", "attend"])
    c = dict(op=op, **_layout(rng))
    rot = c["head_dim"] if rng.random() < 0.5 else c["head_dim"] // rng.choice([2, 4]) // 2 * 2
    width = (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]
    if op == "rope":
        c.update(tokens=span(rng, 1, min(16384, (1 << 25) // width)), rot_dim=rot, interleaved=rng.random() < 0.5,
                 far=rng.choice([0, 0, 5000, 100000]), back=rng.random() < 0.5)
        return c
    c["type"] = rng.choice(["f32", "bf16", "i8"])
    c["page"] = rng.choice([16, 16, 32, 48, 64, 128, 256])
    kind = rng.choice(["step", "step", "chunk", "prompt"])
    c["how"] = "even" if kind == "step" else rng.choice(["even", "ragged", "mixed"])
    if op == "store":
        c["new"] = rng.choice([1, 1, 2]) if kind == "step" else span(rng, 16, 4096)
        most = max(1, (1 << 25) // (c["new"] * width))
        c["seqs"] = span(rng, 1, min(most, 256 if kind == "step" else 16))
        c["past"] = 0 if kind == "prompt" else span(rng, 1, 8192)
        c.update(rot_dim=rot, interleaved=rng.random() < 0.5)
        return c
    if kind == "step":
        c["new"] = rng.choice([1, 1, 1, 2, 4])
        c["past"] = span(rng, 1, 131072)
        if rng.random() < 0.5:
            c["how"] = "ragged"
    else:
        c["new"] = span(rng, 16, 2048)
        c["past"] = 0 if kind == "prompt" else span(rng, 16, 16384)
    c["seqs"] = span(rng, 1, 96)
    # No more bytes or products than the largest listed cases have.
    while (w := work(c))["bytes"] > 570e6 or w["flops"] > 71e9:
        for size in ("seqs", "new", "past"):
            if c[size] > 1:
                c[size] //= 2
                break
    return c


def lengths(c):
    """[(new tokens, tokens cached after them)] of each sequence; the first has the most."""
    out = []
    for s in range(c["seqs"]):
        part = 1.0 if s == 0 else (s * 0.6180339887498949) % 1.0
        new = past = 1.0
        if c["how"] == "ragged":
            new, past = part, part
        elif c["how"] == "mixed":
            new, past = (1.0 if s % 8 == 0 else 0.0), part
        n = max(1, int(round(c["new"] * new)))
        out.append((n, n + int(round(c["past"] * past))))
    return out


# --- inputs ------------------------------------------------------------------

class Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        t = torch.randn(shape, generator=self.g, device=DEV)
        return t.mul_(scale) if scale != 1.0 else t

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device=DEV)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)

    def ints(self, n, hi):
        return torch.randint(hi, (n,), generator=self.g, device=DEV)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def tables(rows, rot_dim):
    """cos and sin of every position and pair, as a program makes them once."""
    f = THETA ** (-torch.arange(0, rot_dim, 2, device=DEV, dtype=F64) / rot_dim)
    a = torch.arange(rows, device=DEV, dtype=F64)[:, None] * f
    return a.cos().to(F32), a.sin().to(F32)


def padded(head_dim):
    return (head_dim + 15) // 16 * 16


def prepare(case, seed):
    c, r = case, Rand(seed)
    h, kh, d = c["heads"], c["kv_heads"], c["head_dim"]
    s = {"case": case}
    if c["op"] == "rope":
        t, ld = c["tokens"], (h + 2 * kh) * d
        s["x"] = r.normal(t, ld)
        # Packed documents of about 1000 tokens that each start again, or
        # single tokens anywhere in their sequences.
        at = torch.arange(t, device=DEV)
        s["pos"] = ((at + r.ints(1, 1000)) % 1000 if not c["far"] else r.ints(t, c["far"])).to(torch.int32)
        s["cos"], s["sin"] = tables(c["far"] or 1000, c["rot_dim"])
        s["q"], s["k"] = torch.empty(t, h * d, device=DEV), torch.empty(t, kh * d, device=DEV)
    else:
        ls = lengths(c)
        t, longest = sum(n for n, _ in ls), max(m for _, m in ls)
        per = -(-longest // c["page"])
        used = [-(-m // c["page"]) for _, m in ls]
        pages = sum(used)
        starts = [0]
        for n, _ in ls:
            starts.append(starts[-1] + n)
        s.update(tokens=t, longest=longest, new=max(n for n, _ in ls), pages=pages)
        s["start"], s["len"] = ints(starts), ints([m for _, m in ls])
        # Each sequence's pages, anywhere in the cache; entries past its end say -1.
        table = torch.full((len(ls), per), -1, dtype=torch.int32, device=DEV)
        table[torch.arange(per, device=DEV)[None, :] < ints(used)[:, None]] = r.perm(pages).to(torch.int32)
        s["table"] = table
        shape = (pages, kh, c["page"], padded(d))
        if c["op"] == "store":
            s["x"] = r.normal(t, (h + 2 * kh) * d)
            s["cos"], s["sin"] = tables(longest, c["rot_dim"])
            for n in ("keys", "values"):
                s[n] = torch.zeros(shape, dtype=TYPES[c["type"]], device=DEV)
                s[n + "_scale"] = torch.zeros(shape[:3], device=DEV)
            s["q"] = torch.empty(t, h * d, device=DEV)
            s["k"], s["v"] = torch.empty(t, kh * d, device=DEV), torch.empty(t, kh * d, device=DEV)
        else:
            s["q"] = r.normal(t, h * d, scale=1.5)
            for n in ("keys", "values"):
                x = r.normal(*shape)
                x[..., d:] = 0
                if c["type"] == "i8":
                    x = x.mul_(45).round_().clamp_(-127, 127)
                s[n] = x.to(TYPES[c["type"]])
                s[n + "_scale"] = r.uniform(*shape[:3]).mul_(0.02).add_(0.01)
                del x
            s["out"] = torch.empty(t, h * d, device=DEV)
    # The library works on a stream of its own: the inputs have to be there.
    torch.cuda.synchronize()
    return s


# --- the library's calls -----------------------------------------------------

def handles(s):
    """The library's descriptions of a state's buffers, which a program keeps."""
    if "lib" not in s:
        M, ctx = lib()
        c = s["case"]
        hs = {"ctx": ctx}
        if "cos" in s:
            hs["rope"] = M.Rope(s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], c["rot_dim"], c["interleaved"])
        if "table" in s:
            hs["cache"] = M.KVCache(ctx, c["type"], s["pages"], c["page"], c["kv_heads"], c["head_dim"],
                                    *(s[n].data_ptr() for n in ("keys", "values", "keys_scale", "values_scale")))
            hs["batch"] = M.KVBatch(s["start"].data_ptr(), s["len"].data_ptr(), s["table"].data_ptr(), c["seqs"], s["tokens"],
                                    s["table"].shape[1], s["new"], s["longest"])
        s["lib"] = hs
    return s["lib"]


def run_own(s):
    c, hs = s["case"], handles(s)
    ctx, h, kh, d = hs["ctx"], c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "rope":
        x, ld = s["x"].data_ptr(), s["x"].shape[1]
        call = ctx.rope_rows_bwd if c["back"] else ctx.rope_rows
        call(x, s["q"].data_ptr(), h, x + 4 * h * d, s["k"].data_ptr(), kh, c["tokens"], d, s["pos"].data_ptr(), hs["rope"],
             ld_q=ld, ld_k=ld)
        return {"q": s["q"], "k": s["k"]}
    if c["op"] == "store":
        x, ld = s["x"].data_ptr(), s["x"].shape[1]
        ctx.kv_append(hs["cache"], hs["batch"], x + 4 * h * d, x + 4 * (h + kh) * d, ld_kv=ld, rope=hs["rope"], q=x,
                      q_out=s["q"].data_ptr(), heads=h, ld_q=ld)
        ctx.kv_read(hs["cache"], hs["batch"], s["k"].data_ptr(), s["v"].data_ptr())
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    ctx.attention_paged(hs["cache"], hs["batch"], s["q"].data_ptr(), s["out"].data_ptr(), h, causal=True)
    return s["out"]


# --- plain forms -------------------------------------------------------------

def rotate(x, cos, sin, interleaved, back=False):
    """x [t, heads, d] by tables [t, pairs]; dimensions past the pairs stay."""
    n = cos.shape[-1]
    x0, x1 = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    cos, sin = cos[:, None], sin[:, None]
    if back:
        sin = -sin
    y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    y = torch.stack((y0, y1), -1).flatten(-2) if interleaved else torch.cat((y0, y1), -1)
    return torch.cat((y, x[..., 2 * n:]), -1)


def rows(s):
    """Of each new token: its sequence, its place among the new ones, its position."""
    t = torch.arange(s["tokens"], device=DEV)
    seq = (t[:, None] >= s["start"][None, :]).sum(1) - 1
    i = t - s["start"][seq]
    return seq, i, s["len"][seq] - (s["start"][seq + 1] - s["start"][seq]) + i


def held(x, kind):
    """What the cache holds of x [t, heads, d]: values, and 8-bit ones' scales."""
    if kind != "i8":
        return x.to(TYPES[kind]), None
    a = x.abs().amax(-1)
    # In 64 bits: values next to the border between two codes.
    code = (x.to(F64) * 127 / a.to(F64)[..., None]).nan_to_num(0.0).round()
    return code.to(torch.int8), a / 127


def run_plain(s):
    c = s["case"]
    h, kh, d = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "rope":
        t, at = c["tokens"], s["pos"].long()
        q, k = s["x"][:, :h * d].reshape(t, h, d), s["x"][:, h * d:(h + kh) * d].reshape(t, kh, d)
        cos, sin = s["cos"][at], s["sin"][at]
        return {"q": rotate(q, cos, sin, c["interleaved"], c["back"]).reshape(t, -1),
                "k": rotate(k, cos, sin, c["interleaved"], c["back"]).reshape(t, -1)}
    seq, i, at = rows(s)
    t = s["tokens"]
    if c["op"] == "store":
        q, k, v = (x.reshape(t, -1, d) for x in s["x"].split((h * d, kh * d, kh * d), 1))
        # In 64 bits: what is held of a rotated key is next to borders too.
        cos, sin = s["cos"][at].to(F64), s["sin"][at].to(F64)
        q, k = (rotate(x.to(F64), cos, sin, c["interleaved"]).to(F32) for x in (q, k))
        page, slot = s["table"][seq, at // c["page"]].long(), at % c["page"]
        out = {"q": q.reshape(t, -1)}
        for name, x in (("keys", k), ("values", v)):
            x, scale = held(x, c["type"])
            s[name][page, :, slot, :d] = x
            if scale is not None:
                s[name + "_scale"][page, :, slot] = scale
            y = s[name][page, :, slot, :d].to(F32)
            if scale is not None:
                y = y * s[name + "_scale"][page, :, slot][..., None]
            out[name[0]] = y.reshape(t, -1)
        return out
    n, new, group = c["seqs"], s["new"], h // kh

    def gathered(name):  # [sequence, head, position, d]
        x = s[name][s["table"].clamp(min=0).long()].to(F32)
        if c["type"] == "i8":
            x = x * s[name + "_scale"][s["table"].clamp(min=0).long()][..., None]
        return x.transpose(1, 2).flatten(2, 3)[..., :d]

    q = s["q"].new_zeros(n, new, kh, group, d)
    q[seq, i] = s["q"].reshape(t, kh, group, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, kh, new * group, d)
    x = torch.matmul(q, gathered("keys").transpose(2, 3).contiguous()) * (1 / math.sqrt(d))
    x = x.reshape(n, kh, new, group, -1)
    count = (s["start"][1:] - s["start"][:-1])
    last = s["len"][:, None] - count[:, None] + torch.arange(new, device=DEV)  # the last key that a token sees
    last = torch.minimum(last, s["len"][:, None] - 1)
    hidden = torch.arange(x.shape[-1], device=DEV) > last[..., None]
    x.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    total = x.sum(-1, keepdim=True) + 1e-9
    y = torch.matmul(x.reshape(n, kh, new * group, -1), gathered("values")).reshape(n, kh, new, group, d) / total
    return y.permute(0, 2, 1, 3, 4)[seq, i].reshape(t, h * d)


def run(state):
    return run_own(state) if own else run_plain(state)


# --- the same in 64 bits -----------------------------------------------------

def turned(x, cos, sin, interleaved):
    """x [t, heads, d] as complex numbers times the tables'."""
    n = cos.shape[-1]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(x[..., a].to(F64), x[..., b].to(F64)) * torch.complex(cos.to(F64), sin.to(F64))[:, None]
    y = x.to(F64).clone()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    h, kh, d = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "rope":
        at = s["pos"].long()
        x = s["x"].view(c["tokens"], -1, d)
        y = turned(x[:, :h + kh], s["cos"][at], -s["sin"][at] if c["back"] else s["sin"][at], c["interleaved"])
        return {"q": y[:, :h].flatten(1), "k": y[:, h:].flatten(1)}
    ls = lengths(c)
    if c["op"] == "store":
        at = torch.cat([torch.arange(m - n, m, device=DEV) for n, m in ls])
        x = s["x"].view(s["tokens"], -1, d)
        y = turned(x[:, :h + kh], s["cos"][at], s["sin"][at], c["interleaved"])
        # A key is rounded to 32 bits once it is rotated; that is what is held.
        out = {"q": y[:, :h].flatten(1), "k": y[:, h:].to(F32).to(F64), "v": x[:, h + kh:].to(F64)}
        for n in ("k", "v"):
            if c["type"] == "i8":
                most = out[n].abs().amax(-1, keepdim=True)
                out[n] = torch.where(most > 0, (out[n] * 127 / most).round() * (most / 127), most)
            elif c["type"] == "bf16":
                out[n] = out[n].to(F32).to(torch.bfloat16).to(F64)
            out[n] = out[n].flatten(1)
        return out
    out, first = torch.empty(s["tokens"], h, d, device=DEV, dtype=F64), 0
    for b, (n, m) in enumerate(ls):
        ids = s["table"][b, :-(-m // c["page"])].long()
        for g in range(kh):
            k, v = (s[name][ids, g].to(F64) * (s[name + "_scale"][ids, g].to(F64)[..., None] if c["type"] == "i8" else 1.0)
                    for name in ("keys", "values"))
            k, v = k.reshape(-1, k.shape[-1])[:m, :d], v.reshape(-1, v.shape[-1])[:m, :d]
            for j in range(g * (h // kh), (g + 1) * (h // kh)):
                q = s["q"][first:first + n].view(n, h, d)[:, j].to(F64)
                p = q @ k.T / math.sqrt(d)
                p = p.masked_fill(torch.ones(n, m, device=DEV, dtype=torch.bool).triu(m - n + 1), -math.inf)
                out[first:first + n, j] = torch.softmax(p, -1) @ v
        first += n
    return out.flatten(1)


# --- what a pass cannot do without -------------------------------------------

def work(case):
    c = case
    h, kh, d = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "rope":
        n = c["tokens"] * (h + kh)
        return {"bytes": 8 * n * d + 4 * c["tokens"] * (1 + c["rot_dim"]), "flops": 3 * n * c["rot_dim"]}
    ls = lengths(c)
    new = sum(n for n, _ in ls)
    held_bytes = d * BYTES[c["type"]] + (4 if c["type"] == "i8" else 0)  # of a token and head, of K or V
    if c["op"] == "store":
        # Written from fp32 and read back to fp32; q rotated.
        one = 2 * kh * (4 * d + 2 * held_bytes + 4 * d)
        return {"bytes": new * (8 * h * d + one + 4 * c["rot_dim"]), "flops": new * (3 * (h + kh) * c["rot_dim"] + 4 * kh * d)}
    cached = sum(m for _, m in ls)
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in ls)
    return {"bytes": 8 * new * h * d + 2 * cached * kh * held_bytes + 4 * cached // c["page"], "flops": 4 * pairs * h * d}
