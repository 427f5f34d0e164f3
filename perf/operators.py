"""The operators of a transformer denoiser block as measured work: masked attention, rotary positions, gated norms.

``listed()`` and ``draw()`` give cases, ``prepare()`` what a caller has in hand before the call, ``run()`` one pass: in plain
torch operations where ``own`` is false, by the package's kernels where it is true.  ``exact()`` is the definition in 64 bits.
"""
import functools
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


def listed():
    return [
        # one query token over the 432 keys of a level-2 frame: latency is all of it
        dict(name="one token, short keys", op="attn", train=False, type="bf16", nb=1, tq=1, tk=432, heads=20, kv_heads=20,
             d=64, cap=0.0, bias=True, causal=True, prefix=0, ragged=False, docs=""),
        # one new token for each of 16 requests over their caches: the keys' bytes are all of it
        dict(name="one token, long caches", op="attn", train=False, type="bf16", nb=16, tq=1, tk=16384, heads=32,
             kv_heads=8, d=128, cap=50.0, bias=False, causal=True, prefix=0, ragged=True, docs=""),
        # frames of several resolutions packed into one row of tokens, rows left over behind the last
        dict(name="packed frames", op="attn", train=False, type="bf16", nb=1, tq=9001, tk=9001, heads=5, kv_heads=5, d=64,
             cap=0.0, bias=False, causal=False, prefix=0, ragged=False, docs="4608,2592,1151,431,108"),
        # a prompt read in at once: causal behind a prefix seen from everywhere, distance bias, shared heads
        dict(name="prefix and distance", op="attn", train=False, type="fp16", nb=2, tq=2500, tk=2500, heads=16, kv_heads=4,
             d=128, cap=0.0, bias=True, causal=True, prefix=300, ragged=False, docs=""),
        # a few rows of tokens trained with padding behind each: launches count
        dict(name="train, small padded", op="attn", train=True, type="fp16", nb=4, tq=108, tk=108, heads=20, kv_heads=20,
             d=64, cap=0.0, bias=False, causal=False, prefix=0, ragged=False, docs="77"),
        # guidance through packed frames with capped scores
        dict(name="train, packed and capped", op="attn", train=True, type="bf16", nb=1, tq=4700, tk=4700, heads=10,
             kv_heads=10, d=64, cap=30.0, bias=False, causal=False, prefix=0, ragged=False, docs="1728,1728,801,432"),
        # a long causal row with four query heads to a key head
        dict(name="train, long causal", op="attn", train=True, type="bf16", nb=1, tq=4097, tk=4097, heads=32, kv_heads=8,
             d=128, cap=0.0, bias=False, causal=True, prefix=0, ragged=False, docs=""),
        # the new tokens' queries and keys, far along their requests
        dict(name="rotary, new tokens", op="rotary", type="bf16", rows=16, heads=40, d=128, rot=128, off=0,
             interleaved=False, inverse=False, far=1000000, scaled=8.0),
        # the gradient of all queries and keys of a batch of frames, half of each head turned
        dict(name="rotary gradient, frames", op="rotary", type="bf16", rows=27648, heads=40, d=64, rot=32, off=16,
             interleaved=True, inverse=True, far=6912, scaled=1.0),
        # the tokens of one serving step between two blocks
        dict(name="norms, new tokens", op="norms", train=False, type="bf16", rows=16, c=4096, first="rms", second="rms",
             gate=1, a=1.0, s=0.5),
        # a batch of frames at the widest level, conditioned by a gate for each frame
        dict(name="train norms, frames", op="norms", train=True, type="bf16", rows=27648, c=320, first="layer",
             second="layer", gate=4, a=1.0, s=1.0),
        # a large training batch, norms on both sides of the block, one learned gate
        dict(name="train norms, wide", op="norms", train=True, type="bf16", rows=16384, c=4096, first="rms", second="rms",
             gate=1, a=1.0, s=0.7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "rotary", "norms"])
    if op == "rotary":
        d = 8 * rng.randint(2, 16)
        rot = 2 * rng.randint(1, d // 2) if rng.random() < 0.4 else 8 * rng.randint(1, d // 8)
        heads = rng.randint(1, 48)
        rows = _log(rng, 1, max(2, min(60000, 70_000_000 // (heads * d))))
        return dict(op=op, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rows=rows, heads=heads, d=d, rot=rot,
                    off=rng.randint(0, d - rot), interleaved=rng.random() < 0.5, inverse=rng.random() < 0.5,
                    far=_log(rng, 100, 4000000), scaled=rng.choice([1.0, 4.0, 32.0]))
    if op == "norms":
        c = 8 * _log(rng, 4, 1024)
        rows = _log(rng, 1, max(2, min(60000, 60_000_000 // c)))
        gate = rng.choice([0, 1, 1, rows, max(1, min(rows, rng.randint(2, 9)))])
        rows -= rows % max(1, gate)
        return dict(op=op, train=rng.random() < 0.6, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rows=rows, c=c,
                    first=rng.choice(["none", "layer", "rms"]), second=rng.choice(["none", "layer", "rms"]), gate=gate,
                    a=rng.choice([1.0, 0.8]), s=rng.choice([1.0, 0.25]))
    kv_heads = rng.choice([1, 2, 3, 5, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7])
    d = rng.choice([64, 64, 128, 128, 8 * rng.randint(1, 16)])
    cap, bias = rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.35
    form = rng.choice(["token", "self", "self", "tail"])
    c = dict(op=op, type=rng.choice(["bf16", "bf16", "fp16"]), heads=heads, kv_heads=kv_heads, d=d, cap=cap, bias=bias,
             docs="", prefix=0, ragged=False)
    if form == "token":  # a few query rows at the end of caches filled to different lengths
        tk, nb = _log(rng, 1, 16384), rng.randint(1, 16)
        return dict(c, train=False, nb=nb, tq=min(tk, rng.choice([1, 1, 1, 2, 5])), tk=tk, causal=True, ragged=True)
    nb = rng.randint(1, 4)
    t = _log(rng, 8, max(9, min(6000, int(math.sqrt(450_000_000 / (nb * heads))))))
    if form == "tail":  # a later piece of a row: fewer queries than keys
        return dict(c, train=rng.random() < 0.5, nb=nb, tq=max(1, t // rng.randint(2, 9)), tk=t, causal=rng.random() < 0.7)
    causal = rng.random() < 0.5
    docs = ",".join(str(max(1, int(t * f))) for f in ((0.45, 0.3, 0.2) if t > 20 else (0.6,))) if rng.random() < 0.5 else ""
    return dict(c, train=rng.random() < 0.5, nb=nb, tq=t, tk=t, causal=causal, docs=docs,
                prefix=max(1, t // 5) if causal and rng.random() < 0.4 else 0)


def _lengths(case):
    """The filled length of each sequence's keys: all of them, or spread between a sixteenth and the whole."""
    nb, tk, tq = case["nb"], case["tk"], case["tq"]
    if not case["ragged"]:
        return [tk] * nb
    return [max(tq, tk * (1 + (11 * b + 15) % 16) // 16) for b in range(nb)]


def _prefixes(case):
    return [max(1, case["prefix"] - 37 * b) for b in range(case["nb"])]


def _documents(case):
    """One sequence's document numbers, -1 behind the last one."""
    ids = []
    for n, length in enumerate(case["docs"].split(",")):
        ids += [n] * int(length)
    return (ids + [-1] * case["tk"])[:case["tk"]]


def _rows_of(gen, rows, cols, dtype, scale=1.0):
    return (torch.randn(rows, cols, generator=gen, device=DEV) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = TYPES[case["type"]]
    st = {"case": case}
    if case["op"] == "attn":
        nb, tq, tk, h, g, d = (case[k] for k in ("nb", "tq", "tk", "heads", "kv_heads", "d"))
        # capped scores are those of a model whose scores grow: wider queries
        width = 3.0 if case["cap"] else 1.5
        if tq == tk:  # q | k | v of a token in one row, as one projection writes them
            qkv = _rows_of(gen, nb * tk, (h + 2 * g) * d, dt)
            qkv[:, :h * d] *= width
            st["q"], st["k"], st["v"] = qkv[:, :h * d], qkv[:, h * d:(h + g) * d], qkv[:, (h + g) * d:]
        else:
            st["q"] = _rows_of(gen, nb * tq, h * d, dt, width)
            st["k"], st["v"] = _rows_of(gen, nb * tk, g * d, dt), _rows_of(gen, nb * tk, g * d, dt)
        ints = dict(dtype=torch.int32, device=DEV)
        st["kv_len"] = torch.tensor(_lengths(case), **ints) if case["ragged"] else None
        st["prefix"] = torch.tensor(_prefixes(case), **ints) if case["prefix"] else None
        st["docs"] = torch.tensor(_documents(case), **ints).repeat(nb) if case["docs"] else None
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEV) / h) if case["bias"] else None
        st["o"], st["lse"] = torch.empty(nb * tq, h * d, dtype=dt, device=DEV), torch.empty(nb, h, tq, device=DEV)
        if case["train"]:
            st["dout"] = _rows_of(gen, nb * tq, h * d, dt)
            st["dq"] = torch.empty(nb * tq, h * d, dtype=dt, device=DEV)
            st["dk"], st["dv"] = (torch.empty(nb * tk, g * d, dtype=dt, device=DEV) for _ in range(2))
    elif case["op"] == "rotary":
        rows, rot = case["rows"], case["rot"]
        st["x"] = _rows_of(gen, rows, case["heads"] * case["d"], dt)
        st["y"] = torch.empty_like(st["x"])
        st["pos"] = torch.randint(0, case["far"], (rows,), generator=gen, device=DEV, dtype=torch.int32)
        # frequencies of the base 10000, slowed down to reach further
        i = torch.arange(0, rot, 2, device=DEV, dtype=torch.float64)
        st["freqs"] = 10000.0 ** (-i / rot) / case["scaled"]
        st["mag"] = 1.0 + 0.1 * math.log(case["scaled"])
    else:
        rows, c, gate = case["rows"], case["c"], case["gate"]
        st["x"], st["y"] = _rows_of(gen, rows, c, dt, 2.0), _rows_of(gen, rows, c, dt) + 0.25
        st["gate"] = _rows_of(gen, gate, c, dt, 0.5) if gate else None
        for n, kind in (("1", case["first"]), ("2", case["second"])):
            st["w" + n] = torch.randn(c, generator=gen, device=DEV) * 0.2 + 1.0 if kind != "none" else None
            st["b" + n] = torch.randn(c, generator=gen, device=DEV) * 0.2 if kind == "layer" else None
        st["r"], st["h"] = torch.empty_like(st["x"]), torch.empty_like(st["x"]) if case["second"] != "none" else None
        st["stats"] = torch.empty(rows, 4, device=DEV)
        if case["train"]:
            st["dr"] = _rows_of(gen, rows, c, dt)
            st["dh"] = _rows_of(gen, rows, c, dt) if st["h"] is not None else None
            st["dx"], st["dy"] = torch.empty_like(st["x"]), torch.empty_like(st["x"])
            st["dgate"] = torch.empty_like(st["gate"]) if gate else None
            for k in ("w1", "b1", "w2", "b2"):
                st["d" + k] = torch.empty(c, device=DEV) if st[k] is not None else None
    return st


def run(st):
    op = st["case"]["op"]
    if own:
        return {"attn": _attn_own, "rotary": _rotary_own, "norms": _norms_own}[op](st)
    return {"attn": _attn, "rotary": _rotary, "norms": _norms}[op](st)


# ---------------------------------------------------------------- the package's calls
@functools.lru_cache(None)
def _context():
    from depth_completion_amd.ops import Ctx
    return Ctx("cuda:0")


def _attn_own(st):
    from depth_completion_amd import ops
    c = st["case"]
    kw = dict(nb=c["nb"], tq=c["tq"], tk=c["tk"], heads=c["heads"], kv_heads=c["kv_heads"], d=c["d"], softcap=c["cap"],
              slopes=st["slopes"], causal=c["causal"], prefix=st["prefix"], kv_len=st["kv_len"], doc_q=st["docs"],
              doc_k=st["docs"])
    ops.attn_mask_fwd(_context(), st["q"], st["k"], st["v"], st["o"], st["lse"], **kw)
    if not c["train"]:
        return {"o": st["o"], "lse": st["lse"]}
    ops.attn_mask_bwd(_context(), st["q"], st["k"], st["v"], st["o"], st["lse"], st["dout"], st["dq"], st["dk"], st["dv"],
                      **kw)
    return {k: st[k] for k in ("o", "lse", "dq", "dk", "dv")}


def _rotary_own(st):
    from depth_completion_amd import ops
    c = st["case"]
    return ops.rotary(_context(), st["x"], c["rows"], c["heads"], c["d"], st["freqs"], st["y"], pos=st["pos"], off=c["off"],
                      interleaved=c["interleaved"], inverse=c["inverse"], mag=st["mag"])


def _norms_own(st):
    from depth_completion_amd import ops
    c = st["case"]
    kw = dict(first=c["first"], second=c["second"], w1=st["w1"], b1=st["b1"], w2=st["w2"], b2=st["b2"], gate=st["gate"],
              a=c["a"], s=c["s"])
    ops.resnorm_fwd(_context(), st["x"], st["y"], c["rows"], c["c"], st["r"], st["h"], st["stats"], **kw)
    if not c["train"]:
        return {"r": st["r"], "h": st["h"]}
    ops.resnorm_bwd(_context(), st["x"], st["y"], c["rows"], c["c"], st["stats"], st["dr"], st["dh"], st["dx"], st["dy"],
                    dgate=st["dgate"], dw1=st["dw1"], db1=st["db1"], dw2=st["dw2"], db2=st["db2"], **kw)
    return {k: st[k] for k in ("r", "h", "dx", "dy", "dgate", "dw1", "db1", "dw2", "db2")}


# ---------------------------------------------------------------- the plain forms
def _heads(x, nb, t, kv_heads, d):
    """[nb t][heads d] -> [nb][kv_heads][group][t][d] in 32 bits."""
    return x.float().reshape(nb, t, kv_heads, -1, d).permute(0, 2, 3, 1, 4).contiguous()


def _rows(x, dtype):
    nb, g, n, t, d = x.shape
    return x.permute(0, 3, 1, 2, 4).reshape(nb * t, g * n * d).to(dtype)


def _visible(st):
    """[nb][1][1][tq][tk] truth values, and the distances of queries and keys."""
    c = st["case"]
    nb, tq, tk = c["nb"], c["tq"], c["tk"]
    j = torch.arange(tk, device=DEV).view(1, 1, tk)
    length = (st["kv_len"] if st["kv_len"] is not None else torch.full((nb,), tk, device=DEV)).view(nb, 1, 1)
    pos = torch.arange(tq, device=DEV).view(1, tq, 1) + length - tq
    see = (j < length).expand(nb, tq, tk)
    if c["causal"]:
        now = j <= pos
        see = see & (now if st["prefix"] is None else now | (j < st["prefix"].view(nb, 1, 1)))
    if st["docs"] is not None:
        ids = st["docs"].view(nb, tk)
        see = see & (ids.view(nb, tq, 1) == ids.view(nb, 1, tk)) & (ids.view(nb, tq, 1) >= 0)
    return see.view(nb, 1, 1, tq, tk), (pos - j).abs().view(nb, 1, 1, tq, tk)


def _attn(st):
    c = st["case"]
    nb, tq, tk, h, g, d = (c[k] for k in ("nb", "tq", "tk", "heads", "kv_heads", "d"))
    dt = TYPES[c["type"]]
    q, k, v = _heads(st["q"], nb, tq, g, d), _heads(st["k"], nb, tk, g, d), _heads(st["v"], nb, tk, g, d)
    see, far = _visible(st)
    scale = 1.0 / math.sqrt(d)
    raw = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    s = c["cap"] * torch.tanh(raw / c["cap"]) if c["cap"] else raw
    capped = s
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, g, h // g, 1, 1) * far
    s = s.masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).reshape(nb, h, tq)
    o = torch.matmul(p, v)
    if not c["train"]:
        return {"o": _rows(o, dt), "lse": lse}
    do = _heads(st["dout"], nb, tq, g, d)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do).sum(2, keepdim=True)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = p * (dp - (o * do).sum(-1, keepdim=True)) * scale
    if c["cap"]:
        ds = ds * (1.0 - (capped / c["cap"]).square())
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q).sum(2, keepdim=True)
    return {"o": _rows(o, dt), "lse": lse, "dq": _rows(dq, dt), "dk": _rows(dk, dt), "dv": _rows(dv, dt)}


def _rotary(st):
    c = st["case"]
    rows, heads, d, rot, off = (c[k] for k in ("rows", "heads", "d", "rot", "off"))
    y = st["x"].float().reshape(rows, heads, d).clone()
    # far positions turn many times: the angles in 64 bits
    angle = st["pos"].double().view(rows, 1) * st["freqs"].view(1, -1)
    cos, sin = ((f(angle) * st["mag"]).float().view(rows, 1, rot // 2) for f in (torch.cos, torch.sin))
    sin = -sin if c["inverse"] else sin
    part = y[..., off:off + rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if c["interleaved"] else (part[..., :rot // 2], part[..., rot // 2:])
    p, q = a * cos - b * sin, a * sin + b * cos
    y[..., off:off + rot] = torch.stack((p, q), -1).flatten(-2) if c["interleaved"] else torch.cat((p, q), -1)
    return y.reshape(rows, heads * d).to(st["x"].dtype)


EPS = 1e-5


def _norm(v, kind):
    """(normalised rows, 1 / deviation)"""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    k = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    return v * k, k


def _norm_back(dn, n, k, kind):
    dv = dn - n * (dn * n).mean(-1, keepdim=True)
    if kind == "layer":
        dv = dv - dn.mean(-1, keepdim=True)
    return dv * k


def _affine(n, w, b):
    n = n * w
    return n if b is None else n + b


def _norms(st):
    c = st["case"]
    rows, first, second, a, s = c["rows"], c["first"], c["second"], c["a"], c["s"]
    dt = st["x"].dtype
    x, y = st["x"].float(), st["y"].float()
    gate = None if st["gate"] is None else st["gate"].float().repeat_interleave(rows // c["gate"], 0)
    u = y
    if first != "none":
        n1, k1 = _norm(y, first)
        u = _affine(n1, st["w1"], st["b1"])
    r = a * x + s * (u if gate is None else u * gate)
    out = {"r": r.to(dt), "h": None}
    if second != "none":
        n2, k2 = _norm(r, second)
        out["h"] = _affine(n2, st["w2"], st["b2"]).to(dt)
    if not c["train"]:
        return out
    dr = st["dr"].float()
    out.update(dict.fromkeys(("dgate", "dw1", "db1", "dw2", "db2")))
    if second != "none":
        dh = st["dh"].float()
        out["dw2"] = (dh * n2).sum(0)
        out["db2"] = dh.sum(0) if second == "layer" else None
        dr = dr + _norm_back(dh * st["w2"], n2, k2, second)
    out["dx"] = (a * dr).to(dt)
    du = s * dr
    if gate is not None:
        out["dgate"] = (du * u).reshape(c["gate"], -1, c["c"]).sum(1).to(dt)
        du = du * gate
    dy = du
    if first != "none":
        out["dw1"] = (du * n1).sum(0)
        out["db1"] = du.sum(0) if first == "layer" else None
        dy = _norm_back(du * st["w1"], n1, k1, first)
    out["dy"] = dy.to(dt)
    return out


# ---------------------------------------------------------------- what a pass cannot do without
def _pairs(case):
    """Visible pairs of a query and a key over all sequences."""
    tq, tk, n = case["tq"], case["tk"], 0
    if case["docs"]:
        ids = _documents(case)
        at, spans = 0, []
        while at < tk and ids[at] >= 0:
            end = at
            while end < tk and ids[end] == ids[at]:
                end += 1
            spans.append((at, end))
            at = end
    for length, prefix in zip(_lengths(case), _prefixes(case) if case["prefix"] else [0] * case["nb"]):
        for lo, hi in spans if case["docs"] else [(0, length)]:
            rows = range(lo, hi) if case["docs"] else range(length - tq, length)
            if case["causal"]:
                n += sum(max(0, min(hi, max(p + 1, prefix)) - lo) for p in rows)
            else:
                n += len(rows) * (hi - lo)
    return n


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "attn":
        nb, tq, h, g, d = (case[k] for k in ("nb", "tq", "heads", "kv_heads", "d"))
        q, kv = nb * tq * h * d * size, sum(_lengths(case)) * g * d * size
        pairs = _pairs(case) * h
        if case["train"]:  # forward, then the gradients from the inputs, the output and its gradient
            return {"bytes": 6 * q + 6 * kv + 2 * nb * h * tq * 4, "flops": 14 * d * pairs}
        return {"bytes": 2 * q + 2 * kv + nb * h * tq * 4, "flops": 4 * d * pairs}
    if case["op"] == "rotary":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * case["d"] * size + 4 * case["rows"], "flops": 3 * n * case["rot"]}
    n, two = case["rows"] * case["c"], case["second"] != "none"
    forward, backward = 3 + two, 5 + two
    return {"bytes": n * size * (forward + (backward if case["train"] else 0)) + case["gate"] * case["c"] * size * (1 + 2 * case["train"]),
            "flops": n * (12 + 30 * case["train"])}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"attn": _attn_exact, "rotary": _rotary_exact, "norms": _norms_exact}[case["op"]](case, st)


def _attn_exact(case, st):
    nb, tq, tk, h, g, d = (case[k] for k in ("nb", "tq", "tk", "heads", "kv_heads", "d"))
    names = ("o", "lse", "dq", "dk", "dv") if case["train"] else ("o", "lse")
    out = {"o": torch.zeros(nb, tq, h, d), "lse": torch.zeros(nb, h, tq), "dq": torch.zeros(nb, tq, h, d),
           "dk": torch.zeros(nb, tk, g, d), "dv": torch.zeros(nb, tk, g, d)}
    out = {k: out[k].to(DEV, torch.float64) for k in names}
    lengths, prefixes = _lengths(case), _prefixes(case)
    ids = torch.tensor(_documents(case), device=DEV) if case["docs"] else None
    for b in range(nb):
        n = lengths[b]
        at, keys = torch.arange(tq, device=DEV) + n - tq, torch.arange(n, device=DEV)
        hidden = torch.zeros(tq, n, dtype=torch.bool, device=DEV)
        if case["causal"]:
            hidden |= (keys[None, :] > at[:, None]) & (keys[None, :] >= (prefixes[b] if case["prefix"] else 0))
        if ids is not None:
            hidden |= (ids[:tq, None] != ids[None, :n]) | (ids[None, :n] < 0)
        empty = hidden.all(1)
        for head in range(h):
            kv = head * g // h
            q, k, v = (st[x].reshape(nb, -1, st[x].shape[1] // d, d)[b, :m, i].double()
                       for x, m, i in (("q", tq, head), ("k", n, kv), ("v", n, kv)))
            s = q @ k.T / d ** 0.5
            slope = 1.0
            if case["cap"]:
                t = torch.tanh(s / case["cap"])
                s, slope = t * case["cap"], 1 - t * t
            if case["bias"]:
                s = s - st["slopes"][head].double() * (at[:, None] - keys[None, :]).abs()
            s[hidden] = -math.inf
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - torch.where(empty, 0.0, lse)[:, None])
            out["o"][b, :, head], out["lse"][b, head] = p @ v, lse
            if case["train"]:
                do = st["dout"].reshape(nb, tq, h, d)[b, :, head].double()
                dp = do @ v.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * slope / d ** 0.5
                out["dv"][b, :n, kv] += p.T @ do
                out["dk"][b, :n, kv] += ds.T @ q
                out["dq"][b, :, head] = ds @ k
    return {k: x if k == "lse" else x.reshape(x.shape[0] * x.shape[1], -1) for k, x in out.items()}


def _rotary_exact(case, st):
    rows, heads, d, rot, off = (case[k] for k in ("rows", "heads", "d", "rot", "off"))
    x = st["x"].double().reshape(rows, heads, d)
    y = x.clone()
    turn = st["pos"].double()[:, None] * st["freqs"][None, :] * (-1 if case["inverse"] else 1)
    unit = torch.polar(torch.full_like(turn, st["mag"]), turn)[:, None, :]
    i = torch.arange(rot // 2, device=DEV)
    one, two = (off + 2 * i, off + 2 * i + 1) if case["interleaved"] else (off + i, off + i + rot // 2)
    z = torch.complex(x[..., one], x[..., two]) * unit
    y[..., one], y[..., two] = z.real, z.imag
    return y.reshape(rows, heads * d)


def _norms_exact(case, st):
    """The values from the formulas, the gradients by differentiation of them in 64 bits."""
    rows, c = case["rows"], case["c"]
    take = {k: st[k].double().requires_grad_(case["train"]) for k in ("x", "y", "gate", "w1", "b1", "w2", "b2") if st[k] is not None}

    def norm(v, kind, n):
        if kind == "none":
            return v
        centre = v.mean(1, keepdim=True) if kind == "layer" else 0.0
        mean2 = ((v - centre) ** 2).sum(1, keepdim=True) / c
        return (v - centre) / torch.sqrt(mean2 + EPS) * take["w" + n] + take.get("b" + n, 0.0)

    with torch.enable_grad():
        u = norm(take["y"], case["first"], "1")
        if case["gate"]:
            u = (u.view(case["gate"], -1, c) * take["gate"][:, None, :]).view(rows, c)
        r = case["a"] * take["x"] + case["s"] * u
        h = norm(r, case["second"], "2") if case["second"] != "none" else None
    out = {"r": r.detach(), "h": None if h is None else h.detach()}
    if case["train"]:
        loss = (r * st["dr"].double()).sum()
        if h is not None:
            loss = loss + (h * st["dh"].double()).sum()
        grads = torch.autograd.grad(loss, list(take.values()))
        out.update(dict.fromkeys(("dx", "dy", "dgate", "dw1", "db1", "dw2", "db2")))
        out.update({"d" + k: v for k, v in zip(take, grads)})
    return out
