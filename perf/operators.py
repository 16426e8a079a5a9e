"""The operators of a serving path over a paged cache, as cases to be timed and checked: rotary positions
with the norm of queries and keys, keys and values written into pages and read back, and attention of
chunks and single tokens over the pages.

A case is one program of ``pjrt_amd.graph``, compiled once and launched on device buffers, or, in its plain
form, the same in elementary torch operations.  A batch is described as a serving loop keeps it: rows of new
tokens one sequence after another, the lengths of the sequences with them, and each one's pages.
"""
import math
import os
import sys

import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
_EPS = 1e-6


def listed():
    return [
        # queries and keys of one new token (latency)
        {"name": "rotary_token", "kind": "rotary", "t": 1, "hq": 16, "hkv": 4, "hd": 128, "rot": 128,
         "layout": "half", "norm": True, "dt": "bf16", "start": 1000, "factor": 1.0},
        # a long prompt: the rows of a fused projection, normalised and rotated on the way to the cache
        {"name": "rotary_prompt", "kind": "rotary", "t": 8192, "hq": 32, "hkv": 8, "hd": 128, "rot": 128,
         "layout": "half", "norm": True, "dt": "bf16", "start": 0, "factor": 1.0},
        # part of the head, interleaved, frequencies scaled for a long context, far positions, sizes nobody rounded
        {"name": "rotary_far_f32", "kind": "rotary", "t": 777, "hq": 12, "hkv": 3, "hd": 80, "rot": 32,
         "layout": "interleaved", "norm": False, "dt": "f32", "start": 1000003, "factor": 8.0},
        # the backward direction: a training step's gradients of a layer's queries and of the norm's weight
        {"name": "rotary_grad", "kind": "rotary_grad", "t": 4096, "hq": 32, "hd": 128, "rot": 128,
         "layout": "half", "norm": True, "dt": "bf16", "start": 0, "factor": 1.0},
        # one new token of each of many sequences goes into the cache
        {"name": "append_tokens", "kind": "append", "seqs": 64, "new": 1, "ctx": 500, "hkv": 8, "hd": 128,
         "page": 16, "dt": "bf16", "cache": "bf16", "pad": 0},
        # a prompt goes into a cache of 8 bits and is read back
        {"name": "append_read_i8", "kind": "append_read", "seqs": 3, "new": 1365, "ctx": 1365, "hkv": 8, "hd": 128,
         "page": 64, "dt": "bf16", "cache": "i8", "pad": 1},
        # one token of a small decoder (latency)
        {"name": "attend_token", "kind": "attend", "seqs": 1, "new": 1, "ctx": 1000, "hq": 12, "hkv": 12, "hd": 64,
         "page": 16, "window": 0, "dt": "bf16", "cache": "bf16", "pad": 0, "chunk": 0},
        # a full batch of single tokens, grouped heads, sequences of different lengths
        {"name": "attend_tokens", "kind": "attend", "seqs": 64, "new": 1, "ctx": 4000, "hq": 32, "hkv": 8, "hd": 128,
         "page": 16, "window": 0, "dt": "bf16", "cache": "bf16", "pad": 0, "chunk": 0},
        # the same over 8 bits, longer
        {"name": "attend_tokens_i8", "kind": "attend", "seqs": 48, "new": 1, "ctx": 8000, "hq": 32, "hkv": 8,
         "hd": 128, "page": 64, "window": 0, "dt": "bf16", "cache": "i8", "pad": 0, "chunk": 0},
        # a chunk of a long prompt
        {"name": "attend_chunk", "kind": "attend", "seqs": 1, "new": 2048, "ctx": 8192, "hq": 32, "hkv": 8, "hd": 128,
         "page": 64, "window": 0, "dt": "bf16", "cache": "bf16", "pad": 0, "chunk": 0},
        # chunks and single tokens in one batch, a window, odd pages, rows behind the last sequence
        {"name": "attend_mixed", "kind": "attend", "seqs": 24, "new": 1, "ctx": 1500, "hq": 16, "hkv": 4, "hd": 64,
         "page": 24, "window": 1000, "dt": "f16", "cache": "f16", "pad": 5, "chunk": 509},
        # full precision, small chunks (a speculated continuation), an uncommon head
        {"name": "attend_f32", "kind": "attend", "seqs": 5, "new": 7, "ctx": 700, "hq": 8, "hkv": 4, "hd": 96,
         "page": 16, "window": 0, "dt": "f32", "cache": "f32", "pad": 0, "chunk": 0},
    ]


def _log(rng, lo, hi, of=1):
    """A whole number in [lo, hi], even over its logarithm, a multiple of `of`."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / of)) * of))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "rotary_grad", "append", "append_read", "attend", "attend", "attend"])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    if kind in ("rotary", "rotary_grad"):
        hd = rng.choice([32, 64, 80, 96, 128, 128, 256])
        rot = rng.choice([hd, hd, hd // 2, hd // 4])
        c = {"kind": kind, "t": 1, "hq": hkv * group, "hd": hd, "rot": rot,
             "layout": rng.choice(["half", "interleaved"]), "norm": rng.random() < 0.6,
             "dt": rng.choice(["bf16", "bf16", "f16", "f32"]), "start": _log(rng, 1, 2000000),
             "factor": rng.choice([1.0, 1.0, 4.0, 16.0])}
        if kind == "rotary":
            c["hkv"] = hkv
        else:
            c["norm"] = True
        c["t"] = _log(rng, 1, max(1, min(8192, (1 << 25) // (hkv * (group + 1) * hd))))
        return c
    page = rng.choice([1, 8, 16, 24, 32, 64, 100, 128])
    hd = rng.choice([64, 64, 80, 96, 128, 128])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    cache = rng.choice([dt, dt, "i8"])
    if kind != "attend":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(2048, (1 << 22) // (seqs * hkv * hd))))
        if cache == "i8":
            kind = "append_read"          # eight bits are seen as the values that they are read back as
        return {"kind": kind, "seqs": seqs, "new": new, "ctx": new + _log(rng, 1, 600), "hkv": hkv, "hd": hd,
                "page": page, "dt": dt, "cache": cache, "pad": rng.choice([0, 0, 3])}
    shape = rng.choice(["token", "tokens", "chunk", "mixed"])
    window = rng.choice([0, 0, 0, 128, 777])
    c = {"kind": kind, "seqs": 1, "new": 1, "ctx": 1, "hq": hkv * group, "hkv": hkv, "hd": hd, "page": page,
         "window": window, "dt": dt, "cache": cache, "pad": rng.choice([0, 0, 4]), "chunk": 0}
    if shape == "token":
        c.update(ctx=_log(rng, 1, 20000))
    elif shape == "tokens":
        c.update(seqs=_log(rng, 2, 64), ctx=_log(rng, 16, 4000), new=rng.choice([1, 1, 1, 4]))
    elif shape == "chunk":
        c.update(new=_log(rng, 16, 300 if dt == "f32" else 1500))
        c.update(ctx=c["new"] + _log(rng, 1, 1000 if dt == "f32" else 5000))
    else:
        c.update(seqs=_log(rng, 4, 32), ctx=_log(rng, 64, 2000), chunk=_log(rng, 16, 100 if dt == "f32" else 600))
    c["ctx"] = max(c["ctx"], c["new"])
    return c


# ---- the batch of a case -----------------------------------------------------------------------

def _batch(c):
    """(new tokens, length with them) of each sequence: lengths spread from half to one and a half of `ctx`, as
    requests that began at different times have; with `chunk` the first and the last bring chunks."""
    n, out = c["seqs"], []
    for i in range(n):
        new, ctx = c["new"], c["ctx"]
        if n > 1:
            ctx = ctx // 2 + ctx * ((i * 37 + 11) % n) // n
        if c.get("chunk") and i in (0, n - 1):
            new = c["chunk"] if i == 0 else max(1, c["chunk"] // 4)
        out.append((new, max(ctx, new)))
    return out


def _positions(c):
    """Rows of several sequences: each `start` further on, and within one by one."""
    t = c["t"]
    part = max(1, (t + 2) // 3)
    return [c["start"] + (r // part) * 1000 + r % part for r in range(t)]


def _inv_freq(c):
    """theta^(-2 i / rot); with a factor over 1 the slow ones are divided by it, the fast ones kept and those
    between blended by how many turns they make over the original context of 4096."""
    rot, factor = c["rot"], c["factor"]
    out = []
    for i in range(rot // 2):
        f = 10000.0 ** (-2.0 * i / rot)
        if factor > 1.0:
            turns = 4096 * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            f = f * keep + f / factor * (1.0 - keep)
        out.append(f)
    return out


def _magnitude(c):
    return 0.1 * math.log(c["factor"]) + 1.0 if c["factor"] > 1.0 else 1.0


def _pages_of(c):
    """Pages a sequence's row of the table holds, and pages in the pool (a few more than are in use)."""
    need = [-(-length // c["page"]) for _, length in _batch(c)]
    return max(need), sum(need) + 3


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)

    def normal(shape, std=1.0, dt="f32"):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(_TORCH[dt])

    if c["kind"] in ("rotary", "rotary_grad"):
        s = {"pos": torch.tensor(_positions(c), dtype=torch.int32, device="cuda")}
        if c["norm"]:
            s["wq"] = 1.0 + normal((c["hd"],), 0.1)
        if c["kind"] == "rotary":
            # rows of the fused projection: queries, keys and values of a token side by side
            s["qkv"] = normal((c["t"], (c["hq"] + 2 * c["hkv"]) * c["hd"]), 1.0, c["dt"])
            if c["norm"]:
                s["wk"] = 1.0 + normal((c["hd"],), 0.1)
        else:
            s["x"] = normal((c["t"], c["hq"], c["hd"]), 1.0, c["dt"])
            s["dy"] = normal((c["t"], c["hq"], c["hd"]), 1.0, c["dt"])
        return s
    batch = _batch(c)
    most, pool = _pages_of(c)
    rows = sum(n for n, _ in batch) + c["pad"]
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(batch), most), -1, dtype=torch.int32, device="cuda")   # -1: no page
    at, cu = 0, [0]
    for i, (n, length) in enumerate(batch):
        k = -(-length // c["page"])
        table[i, :k] = order[at:at + k]
        at += k
        cu.append(cu[-1] + n)
    s = {"cu": torch.tensor(cu, dtype=torch.int32, device="cuda"), "table": table,
         "lens": torch.tensor([length for _, length in batch], dtype=torch.int32, device="cuda")}
    shape = (pool, c["hkv"], c["page"], c["hd"])
    for name in ("k", "v"):
        if c["cache"] == "i8":
            s[name + "_pages"] = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
            s[name + "_scale"] = torch.rand(shape[:3], generator=gen, device="cuda") * 0.02 + 0.005
        else:
            s[name + "_pages"] = normal(shape, 1.0, c["cache"])
    if c["kind"] == "attend":
        s["q"] = normal((rows, c["hq"], c["hd"]), 1.5, c["dt"])
    else:
        s["k"] = normal((rows, c["hkv"], c["hd"]), 1.0, c["dt"])
        s["v"] = normal((rows, c["hkv"], c["hd"]), 1.0, c["dt"])
    return s


# ---- the framework's programs ---------------------------------------------------------------------

_RT = []


def _runtime():
    """The process's client: one device, opened once."""
    if not _RT:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pjrt-ocl_amd", "python")
        if path not in sys.path:
            sys.path.insert(0, path)
        from pjrt_amd.runtime import Runtime
        _RT.append(Runtime(device=0))
    return _RT[0]


def _compiled(c, s):
    """The case's program with its inputs in order and its outputs' buffers."""
    rt = _runtime()
    from pjrt_amd import graph
    g = graph.Graph()
    ins, outs, kept = [], [], []

    def take(name, dt):
        ins.append(s[name])
        return g.input(tuple(s[name].shape), dt)

    def give(tensor, dt):
        g.output(tensor)
        outs.append(torch.empty(tensor.shape, dtype=_TORCH[dt], device="cuda"))

    if c["kind"] in ("rotary", "rotary_grad"):
        hd, dt = c["hd"], c["dt"]
        freq = graph.rotary_frequencies(c["rot"], 10000.0, factor=c["factor"], original=4096)
        opts = dict(interleaved=c["layout"] == "interleaved", magnitude=_magnitude(c), eps=_EPS)
        pos = take("pos", "i32")
        wq = take("wq", "f32") if c["norm"] else None
        if c["kind"] == "rotary":
            width = (c["hq"] + 2 * c["hkv"]) * hd
            qkv = take("qkv", dt)
            wk = take("wk", "f32") if c["norm"] else None
            q = g.view(qkv, (c["t"], c["hq"], hd), (width, hd, 1), 0)
            k = g.view(qkv, (c["t"], c["hkv"], hd), (width, hd, 1), c["hq"] * hd)
            give(g.rotary(q, pos, freq, weight=wq, **opts), dt)
            give(g.rotary(k, pos, freq, weight=wk, **opts), dt)
        else:
            dx, dw = g.rotary_grad(take("dy", dt), take("x", dt), pos, freq, weight=wq, **opts)
            give(dx, dt)
            give(dw, "f32")
    else:
        batch = g.paged_batch(seqs=c["seqs"], max_pages=s["table"].shape[1])
        ins += [s["cu"], s["lens"], s["table"]]
        pool = s["k_pages"].shape[0]
        cache = g.paged_cache(pages=pool, heads=c["hkv"], page=c["page"], head_dim=c["hd"], dtype=c["cache"])
        ins += [s["k_pages"], s["v_pages"]] + ([s["k_scale"], s["v_scale"]] if c["cache"] == "i8" else [])
        if c["kind"] == "attend":
            give(g.paged_attention(take("q", c["dt"]), cache, batch, scale=c["hd"] ** -0.5, window=c["window"]),
                 c["dt"])
        else:
            k = take("k", c["dt"])
            g.cache_append(cache, batch, k, take("v", c["dt"]))
            if c["kind"] == "append_read":
                kk, vv = g.cache_read(cache, batch, rows=s["k"].shape[0], dtype="f32")
                give(kk, "f32")
                give(vv, "f32")
            else:
                kept = [s["k_pages"], s["v_pages"]]       # written in place
    return {"program": rt.compile(g.build()), "in": ins, "out": outs, "kept": kept}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["batch"] = _batch(case) if "seqs" in case else None        # the serving loop's own record of it
    if case["kind"] in ("rotary", "rotary_grad"):
        s["freq"] = torch.tensor(_inv_freq(case), dtype=torch.float64, device="cuda")
    if own:
        s.update(_compiled(case, s))
        torch.cuda.synchronize()        # the program runs on the runtime's own stream
    return s


def run(state):
    if own:
        state["program"].enqueue(state["in"], state["out"])
        return state["kept"] or state["out"]
    return _PLAIN[state["case"]["kind"]](state)


# ---- plain forms ---------------------------------------------------------------------------------

def _angles(s):
    """cos and sin of position times frequency, the angle in 64 bits."""
    a = s["pos"].double()[:, None] * s["freq"][None, :]
    return torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]


def _pairs(c, z):
    """The two halves that are rotated against each other, and the rest of the head."""
    rot = c["rot"]
    if c["layout"] == "half":
        return z[..., :rot // 2], z[..., rot // 2:rot], z[..., rot:]
    return z[..., 0:rot:2], z[..., 1:rot:2], z[..., rot:]


def _joined(c, a, b, rest):
    if c["layout"] == "half":
        return torch.cat([a, b, rest], -1)
    return torch.cat([torch.stack([a, b], -1).flatten(-2), rest], -1)


def _plain_rotary(s):
    c = s["case"]
    t, hd = c["t"], c["hd"]
    cos, sin = _angles(s)
    m = _magnitude(c)
    out = []
    for first, heads, w in ((0, c["hq"], "wq"), (c["hq"] * hd, c["hkv"], "wk")):
        z = s["qkv"][:, first:first + heads * hd].float().reshape(t, heads, hd)
        if c["norm"]:
            z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + _EPS) * s[w]
        a, b, rest = _pairs(c, z)
        out.append(_joined(c, (a * cos - b * sin) * m, (b * cos + a * sin) * m, rest).to(_TORCH[c["dt"]]))
    return out


def _plain_rotary_grad(s):
    c = s["case"]
    cos, sin = _angles(s)
    m = _magnitude(c)
    a, b, rest = _pairs(c, s["dy"].float())
    dz = _joined(c, (a * cos + b * sin) * m, (b * cos - a * sin) * m, rest)
    x = s["x"].float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    dw = (dz * x * r).flatten(0, 1).sum(0)
    g = dz * s["wq"]
    dx = r * g - x * (r * r * r) * (x * g).mean(-1, keepdim=True)
    return [dx.to(_TORCH[c["dt"]]), dw]


def _slots(s, i, first, last):
    """(page, slot) of positions first..last - 1 of sequence i."""
    p = torch.arange(first, last, device="cuda")
    page = s["case"]["page"]
    return s["table"][i].long()[p // page], p % page


def _plain_append(s):
    c, row = s["case"], 0
    for i, (n, length) in enumerate(s["batch"]):
        pages, slots = _slots(s, i, length - n, length)
        for name in ("k", "v"):
            x = s[name][row:row + n]
            if c["cache"] == "i8":
                x = x.float()
                scale = x.abs().amax(-1) * (1.0 / 127.0)
                q = torch.round(x / scale[..., None])
                s[name + "_pages"][pages, :, slots] = torch.where(scale[..., None] > 0, q, 0.0).to(torch.int8)
                s[name + "_scale"][pages, :, slots] = scale
            else:
                s[name + "_pages"][pages, :, slots] = x
        row += n
    return [s["k_pages"], s["v_pages"]]


def _gather(s, i, first, last):
    """Keys and values of positions first..last - 1 of sequence i, [positions, heads, head dim] in f32."""
    pages, slots = _slots(s, i, first, last)
    out = []
    for name in ("k", "v"):
        x = s[name + "_pages"][pages, :, slots].float()
        if s["case"]["cache"] == "i8":
            x = x * s[name + "_scale"][pages, :, slots][..., None]
        out.append(x)
    return out


def _plain_append_read(s):
    _plain_append(s)
    out = [torch.zeros(s["k"].shape, device="cuda"), torch.zeros(s["v"].shape, device="cuda")]
    row = 0
    for i, (n, length) in enumerate(s["batch"]):
        for o, x in zip(out, _gather(s, i, length - n, length)):
            o[row:row + n] = x
        row += n
    return out


def _plain_attend(s):
    c, row = s["case"], 0
    hkv, hd, g = c["hkv"], c["hd"], c["hq"] // c["hkv"]
    out = torch.zeros(s["q"].shape, dtype=_TORCH[c["dt"]], device="cuda")
    for i, (n, length) in enumerate(s["batch"]):
        first = max(0, length - n - c["window"] + 1) if c["window"] else 0
        k, v = _gather(s, i, first, length)
        q = s["q"][row:row + n].float().reshape(n, hkv, g, hd).permute(1, 0, 2, 3).reshape(hkv, n * g, hd)
        w = torch.matmul(q, k.permute(1, 2, 0).contiguous()) * hd ** -0.5
        if n > 1 or c["window"]:
            at = torch.arange(length - n, length, device="cuda").repeat_interleave(g)[:, None]
            key = torch.arange(first, length, device="cuda")[None, :]
            hidden = key > at
            if c["window"]:
                hidden = hidden | (key <= at - c["window"])
            w.masked_fill_(hidden, -math.inf)
        w = torch.exp(w - w.amax(-1, keepdim=True))
        o = torch.matmul(w, v.permute(1, 0, 2).contiguous()) / w.sum(-1, keepdim=True)
        out[row:row + n] = o.reshape(hkv, n, g, hd).permute(1, 0, 2, 3).reshape(n, c["hq"], hd).to(out.dtype)
        row += n
    return [out]


_PLAIN = {"rotary": _plain_rotary, "rotary_grad": _plain_rotary_grad, "append": _plain_append,
          "append_read": _plain_append_read, "attend": _plain_attend}


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    c, k = case, case["kind"]
    if k == "rotary":
        n = c["t"] * (c["hq"] + c["hkv"]) * c["hd"]
        return {"bytes": 2 * n * _SIZE[c["dt"]] + 4 * c["t"], "flops": (3 * c["rot"] // c["hd"] + 4 * c["norm"] + 1) * n}
    if k == "rotary_grad":
        n = c["t"] * c["hq"] * c["hd"]
        return {"bytes": 3 * n * _SIZE[c["dt"]] + 8 * c["hd"], "flops": 14 * n}
    rows = sum(n for n, _ in _batch(c))
    per = c["hkv"] * c["hd"] * _SIZE[c["cache"]] + (4 * c["hkv"] if c["cache"] == "i8" else 0)
    if k in ("append", "append_read"):
        new = 2 * rows * c["hkv"] * c["hd"]
        moved = new * _SIZE[c["dt"]] + 2 * rows * per
        return {"bytes": moved + (2 * rows * per + 4 * new if k == "append_read" else 0), "flops": 3 * new}
    pairs = keys = 0
    for n, length in _batch(c):
        first = length - n
        w = c["window"] or length
        pairs += sum(min(p + 1, w) for p in range(first, length))
        keys += length - max(0, first + 1 - w)
    return {"bytes": 2 * rows * c["hq"] * c["hd"] * _SIZE[c["dt"]] + 2 * keys * per,
            "flops": 4 * pairs * c["hq"] * c["hd"]}


# ---- the same in 64 bits ----------------------------------------------------------------------------

def _turned(c, x, pos, sign):
    """Each pair of a head as a complex number, times the unit vector of its angle."""
    rot = c["rot"]
    f = torch.tensor(_inv_freq(c), dtype=torch.float64, device=x.device)
    a = sign * pos.double()[:, None, None] * f
    unit = torch.complex(torch.cos(a), torch.sin(a)) * _magnitude(c)
    y = x.clone()
    if c["layout"] == "half":
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * unit
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * unit
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "rotary":
        heads = s["qkv"].double().reshape(c["t"], -1, c["hd"])
        out = []
        for x, w in ((heads[:, :c["hq"]], "wq"), (heads[:, c["hq"]:c["hq"] + c["hkv"]], "wk")):
            if c["norm"]:
                x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["hd"] + _EPS) * s[w].double()
            out.append(_turned(c, x, s["pos"], 1.0))
        return out
    if c["kind"] == "rotary_grad":
        x, w = s["x"].double(), s["wq"].double()
        dz = _turned(c, s["dy"].double(), s["pos"], -1.0)
        ms = (x ** 2).sum(-1, keepdim=True) / c["hd"] + _EPS
        u = x / torch.sqrt(ms)
        g = dz * w
        return [(g - u * (g * u).sum(-1, keepdim=True) / c["hd"]) / torch.sqrt(ms), (dz * u).sum((0, 1))]
    batch, page = _batch(c), c["page"]
    table = s["table"].long()
    if c["kind"] == "append" and c["cache"] != "i8":
        row, pools = 0, [s["k_pages"].double(), s["v_pages"].double()]
        for i, (n, length) in enumerate(batch):
            for j in range(n):
                p = length - n + j
                for pool, name in zip(pools, ("k", "v")):
                    pool[table[i, p // page], :, p % page] = s[name][row + j].double()
            row += n
            if row > 20000:
                return None
        return pools
    if c["kind"] in ("append", "append_read"):
        return None                       # what eight bits make of a value has no exact value
    hkv, g, hd = c["hkv"], c["hq"] // c["hkv"], c["hd"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for i, (n, length) in enumerate(batch):
        ids = table[i, :-(-length // page)]
        at = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        seen = key <= at
        if c["window"]:
            seen &= key > at - c["window"]
        for h in range(hkv):
            kv = []
            for name in ("k", "v"):
                x = s[name + "_pages"][ids, h].double()
                if c["cache"] == "i8":
                    x = x * s[name + "_scale"][ids, h].double()[..., None]
                kv.append(x.reshape(-1, hd)[:length])
            for j in range(g):
                q = s["q"][row:row + n, h * g + j].double()
                w = (q @ kv[0].t().contiguous() / math.sqrt(hd)).masked_fill(~seen, -math.inf)
                out[row:row + n, h * g + j] = torch.softmax(w, -1) @ kv[1]
        row += n
    return [out]
