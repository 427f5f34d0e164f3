"""Masked attention (dc_attn_mask_*) against the definition in 64 bits, forward and gradients (GPU).

Tolerances, relative to the 2-norm of the result, u = half a step of the type (bf16 2^-8, fp16 2^-11): the output carries one
rounding of itself and one of the weights P; the gradients carry one of themselves, one of P or dS and, through rowsum(dO o), one
of o.  Each is at most u in the norm, so o is held to 2 u and the gradients to 4 u.  Where a row sees one key alone dP and
rowsum(dO o) cancel: what fp32 sums of d products leave, 2^-18 of the gradients' sum without signs, is allowed beside that.  The
log-sum is computed in fp32 from exact products: 2e-6 of max(1, |lse|), 1e-5 where scores pass tanh, whose fp32 form is off by
2e-7 of the cap.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

dev = torch.device("cuda:0")
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from depth_completion_amd.ops import Ctx
    return Ctx(dev, ws_mb=1)


def definition(q, k, v, c, dout=None):
    """o, lse and gradients in 64 bits on the CPU, a head at a time."""
    nb, tq, tk, h, g, d = (c[x] for x in ("nb", "tq", "tk", "heads", "kv_heads", "d"))
    q, k, v = (x.double().cpu().reshape(nb, -1, n, d) for x, n in ((q, h), (k, g), (v, g)))
    do = None if dout is None else dout.double().cpu().reshape(nb, tq, h, d)
    scale = c.get("scale") or d ** -0.5
    cap, slopes = c.get("softcap", 0.0), c.get("slopes")
    o, lse = torch.zeros(nb, tq, h, d, dtype=torch.float64), torch.zeros(nb, h, tq, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    size = {"dq": 0.0, "dk": 0.0, "dv": 0.0}
    for b in range(nb):
        n = tk if c.get("kv_len") is None else min(max(int(c["kv_len"][b]), 0), tk)
        pos, key = torch.arange(tq) + n - tq, torch.arange(tk)
        see = (key < n)[None].expand(tq, tk)
        if c.get("causal"):
            pre = int(c["prefix"][b]) if c.get("prefix") is not None else 0
            see = see & ((key[None] <= pos[:, None]) | (key[None] < pre))
        if c.get("doc_q") is not None:
            iq, ik = c["doc_q"].cpu().view(nb, tq)[b], c["doc_k"].cpu().view(nb, tk)[b]
            see = see & (iq[:, None] == ik[None]) & (iq[:, None] >= 0)
        for i in range(h):
            j = i * g // h
            # what no pair reaches counts as zero
            kk, vv = (torch.where(see.any(0)[:, None], x[b, :, j], 0.0) for x in (k, v))
            qq = torch.where(see.any(1)[:, None], q[b, :, i], 0.0)
            s = qq @ kk.T * scale
            slope = 1.0
            if cap:
                t = torch.tanh(s / cap)
                s, slope = t * cap, 1 - t * t
            if slopes is not None:
                s = s - float(slopes[i]) * (pos[:, None] - key[None]).abs()
            s = s.masked_fill(~see, -math.inf)
            lse[b, i] = torch.logsumexp(s, 1)
            p = torch.where(see, torch.exp(s - torch.where(see.any(1), lse[b, i], 0.0)[:, None]), 0.0)
            o[b, :, i] = p @ vv
            if do is not None:
                dd = torch.where(see.any(1)[:, None], do[b, :, i], 0.0)
                dp = dd @ vv.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * slope * scale
                dq[b, :, i] = ds @ kk
                whole = p * (dp.abs() + (p * dp).sum(1, keepdim=True).abs()) * scale
                size["dq"] += float((whole @ kk.abs()).norm())
                size["dk"] += float((whole.T @ qq.abs()).norm())
                dk[b, :, j] += ds.T @ qq
                dv[b, :, j] += p.T @ dd
    flat = lambda x: x.reshape(x.shape[0] * x.shape[1], -1)  # noqa: E731
    return flat(o), lse, flat(dq), flat(dk), flat(dv), size


def inputs(c, dtype, seed=0, qscale=1.0, fused=False):
    g = torch.Generator().manual_seed(seed)
    nb, tq, tk, h, kv, d = (c[x] for x in ("nb", "tq", "tk", "heads", "kv_heads", "d"))
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, do = r(nb * tq, h * d) * qscale, r(nb * tk, kv * d), r(nb * tk, kv * d), r(nb * tq, h * d)
    if fused:   # one row holds q | k | v and a margin
        row = torch.cat([q, k, v, torch.full((nb * tq, 24), float("nan"))], 1).to(dtype).to(dev)
        a, b = h * d, kv * d
        return row[:, :a], row[:, a:a + b], row[:, a + b:a + 2 * b], do.to(dtype).to(dev)
    return tuple(x.to(dtype).to(dev) for x in (q, k, v, do))


def rel(a, b):
    return float((a.double().cpu() - b).norm() / b.norm().clamp_min(1e-30))


def check(ctx, c, dtype, train=True, seed=0, qscale=1.0, fused=False, tensors=None):
    from depth_completion_amd import ops
    q, k, v, do = tensors or inputs(c, dtype, seed, qscale, fused)
    nq, nk = c["nb"] * c["tq"], c["nb"] * c["tk"]
    hq, hk = c["heads"] * c["d"], c["kv_heads"] * c["d"]
    pad = 16   # columns behind the last head stay as they were
    o = torch.full((nq + 1, hq + pad), 7.0, dtype=dtype, device=dev)
    lse = torch.full((c["nb"], c["heads"], c["tq"]), 7.0, device=dev)
    kw = {x: y for x, y in c.items()}
    ops.attn_mask_fwd(ctx, q, k, v, o, lse, **kw)
    ro, rl, rq, rk, rv, size = definition(q, k, v, c, do if train else None)
    u = U[dtype]
    assert torch.equal(torch.isinf(lse.cpu()), torch.isinf(rl))
    seen = torch.isfinite(rl)
    tol = 1e-5 if c.get("softcap") else 2e-6
    if seen.any():
        assert float(((lse.cpu().double() - rl)[seen].abs() / rl[seen].abs().clamp_min(1.0)).max()) < tol
    assert rel(o[:nq, :hq], ro) < 2 * u
    assert (o[:nq, hq:] == 7).all() and (o[nq:] == 7).all()
    empty = (~seen).permute(0, 2, 1).reshape(nq, c["heads"], 1).expand(-1, -1, c["d"]).reshape(nq, hq)
    assert (o[:nq, :hq].cpu()[empty] == 0).all()
    if not train:
        return
    dq, dk, dv = (torch.full((n + 1, w + pad), 7.0, dtype=dtype, device=dev) for n, w in ((nq, hq), (nk, hk), (nk, hk)))
    ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, dq, dk, dv, **kw)
    for name, x, r, n, w in (("dq", dq, rq, nq, hq), ("dk", dk, rk, nk, hk), ("dv", dv, rv, nk, hk)):
        assert torch.isfinite(x[:n, :w]).all(), name
        off = float((x[:n, :w].double().cpu() - r).norm())
        assert off <= max(4 * u * float(r.norm()), 2.0 ** -18 * size[name]), (name, off, float(r.norm()), size[name])
        assert (x[:n, w:] == 7).all() and (x[n:] == 7).all(), name


def shape(nb, tq, tk, heads, kv_heads, d, **kw):
    return dict(nb=nb, tq=tq, tk=tk, heads=heads, kv_heads=kv_heads, d=d, **kw)


TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


@TYPES
@pytest.mark.parametrize("nb,tq,tk,heads,kv_heads,d", [
    (1, 1, 1, 1, 1, 64), (1, 1, 432, 20, 20, 64), (3, 1, 700, 8, 2, 128), (2, 5, 1031, 7, 1, 64), (1, 32, 33, 4, 4, 40),
    (1, 33, 1, 2, 2, 8), (2, 64, 64, 4, 2, 64), (1, 129, 257, 3, 1, 128), (1, 300, 1500, 6, 2, 72), (2, 511, 130, 4, 4, 128)])
def test_lengths_and_heads(ctx, nb, tq, tk, heads, kv_heads, d, dtype):
    check(ctx, shape(nb, tq, tk, heads, kv_heads, d), dtype)


@TYPES
@pytest.mark.parametrize("tq,tk,d", [(1, 300, 128), (200, 200, 64), (70, 333, 64), (333, 70, 128), (20, 7, 64)])
@pytest.mark.parametrize("prefix", [False, True])
def test_causal_and_prefix(ctx, tq, tk, d, prefix, dtype):
    c = shape(3, tq, tk, 4, 2, d, causal=True)
    if prefix:
        c["prefix"] = torch.tensor([0, tk // 3, tk + 5], dtype=torch.int32, device=dev)
    check(ctx, c, dtype)


@TYPES
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tq,causal", [(1, True), (4, True), (4, False), (100, True)])
def test_filled_lengths(ctx, tq, causal, d, dtype):
    """Keys behind the filled length may hold anything; no length at all leaves rows empty."""
    lens = [0, 1, 64, 333, 4000, -3]
    c = shape(6, tq, 400, 6, 2, d, causal=causal, kv_len=torch.tensor(lens, dtype=torch.int32, device=dev))
    q, k, v, do = inputs(c, dtype, 3)
    for x in (k, v):
        for b, n in enumerate(lens):
            x.view(6, 400, -1)[b, max(n, 0):] = float("nan")
    check(ctx, c, dtype, tensors=(q, k, v, do))


def documents(kind, t, nb=1):
    g = torch.Generator().manual_seed(t)
    if kind == "packed":      # ragged, the last one ends inside a tile, padding behind it
        cuts = [0, t // 3, t // 3 + 1, t // 2, t - t // 7]
        ids = torch.full((t,), -1)
        for n in range(4):
            ids[cuts[n]:cuts[n + 1]] = n + 5
    elif kind == "mixed":     # any order
        ids = torch.randint(-1, 4, (t,), generator=g)
    elif kind == "one":
        ids = torch.zeros(t, dtype=torch.long)
    else:                     # nothing belongs anywhere
        ids = torch.full((t,), -1)
    return ids.to(torch.int32).repeat(nb).to(dev)


@TYPES
@pytest.mark.parametrize("kind", ["packed", "mixed", "one", "none"])
@pytest.mark.parametrize("t,d", [(20, 64), (300, 64), (517, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_documents(ctx, kind, t, d, causal, dtype):
    """Rows in no document hold NaN and infinities in every operand; they reach nothing."""
    ids = documents(kind, t, 2)
    c = shape(2, t, t, 4, 2, d, doc_q=ids, doc_k=ids, causal=causal)
    q, k, v, do = inputs(c, dtype, 5)
    for n, x in enumerate((q, k, v, do)):
        x[ids < 0] = float("nan") if n % 2 else float("inf")
    check(ctx, c, dtype, tensors=(q, k, v, do))


def runs(lengths, t, start=0):
    """int32 [t]: documents of these lengths from number `start` on, rows in none behind them."""
    ids = torch.full((t,), -1, dtype=torch.int32)
    at = 0
    for n, length in enumerate(lengths):
        ids[at:at + length] = n + start
        at += length
    return ids.to(dev)


@TYPES
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,d,lengths,t", [
    (3, 3, 64, [60, 431, 90, 1000], 1700), (4, 1, 128, [1100, 70, 500], 1700), (1, 1, 64, [5, 2300, 1, 130], 2500),
    (2, 1, 64, [40] * 30, 1201)])
def test_documents_in_parts(ctx, heads, kv_heads, d, lengths, t, causal, dtype):
    """Few blocks whose documents differ in length, so that some of them are split and some are not."""
    ids = runs(lengths, t)
    check(ctx, shape(1, t, t, heads, kv_heads, d, doc_q=ids, doc_k=ids, causal=causal), dtype, seed=21)


@pytest.mark.parametrize("prefix", [False, True])
def test_documents_of_filled_lengths(ctx, prefix):
    """Queries and keys of their own documents and counts, filled keys, a causal mask and a prefix, over two sequences."""
    iq = torch.cat([runs([200, 300, 150], 700, 1), runs([700], 700, 2)])
    ik = torch.cat([runs([100, 600, 500], 1500), runs([33, 67, 1000], 1500)])
    c = shape(2, 700, 1500, 4, 2, 64, doc_q=iq, doc_k=ik, causal=True,
              kv_len=torch.tensor([1400, 640], dtype=torch.int32, device=dev))
    if prefix:
        c["prefix"] = torch.tensor([900, 0], dtype=torch.int32, device=dev)
    check(ctx, c, torch.bfloat16, seed=22)


def test_documents_that_change_between_replays(ctx):
    """A captured call takes its documents from where they lie when it runs."""
    from depth_completion_amd import ops
    t = 1300
    ids = runs([700, 90, 400], t)
    c = shape(1, t, t, 4, 2, 64, doc_q=ids, doc_k=ids)
    q, k, v, do = inputs(c, torch.bfloat16, 23)
    bufs = [torch.empty_like(q), torch.empty(1, 4, t, device=dev), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]

    def step(o, lse, dq, dk, dv):
        ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
        ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, dq, dk, dv, **c)

    step(*bufs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*bufs)
    for lengths in ([700, 90, 400], [30, 1200], [1300], [], [64] * 20):
        ids.copy_(runs(lengths, t))
        graph.replay()
        got = [b.clone() for b in bufs]
        want = [torch.empty_like(b) for b in bufs]
        step(*want)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), lengths


def test_documents_across(ctx):
    """Queries and keys of different counts; a query document without keys and a key document without queries."""
    iq = torch.tensor([0] * 40 + [3] * 30 + [1] * 31, dtype=torch.int32, device=dev)
    ik = torch.tensor([1] * 100 + [0] * 90 + [2] * 60 + [-1] * 5, dtype=torch.int32, device=dev)
    c = shape(1, 101, 255, 2, 1, 64, doc_q=iq, doc_k=ik)
    check(ctx, c, torch.bfloat16)
    # the gradients of rows that see nothing may hold anything
    q, k, v, do = inputs(c, torch.bfloat16, 9)
    do[40:70] = float("nan")
    q[40:70] = float("inf")
    check(ctx, c, torch.bfloat16, tensors=(q, k, v, do))


@TYPES
@pytest.mark.parametrize("tq,tk,d", [(1, 500, 128), (3, 100, 64), (190, 190, 64), (140, 300, 128)])
@pytest.mark.parametrize("cap,bias", [(20.0, False), (0.0, True), (30.0, True)])
def test_shaped_scores(ctx, tq, tk, d, cap, bias, dtype):
    slopes = 2.0 ** -torch.arange(1.0, 7.0, device=dev) if bias else None
    check(ctx, shape(2, tq, tk, 6, 3, d, softcap=cap, slopes=slopes), dtype, qscale=4.0)
    check(ctx, shape(2, tq, tk, 6, 3, d, softcap=cap, slopes=slopes, causal=True, scale=0.3), dtype)


@TYPES
def test_scores_far_apart(ctx, dtype):
    """Scores that rise and fall by hundreds along the keys: the running maximum moves late, early and not at all."""
    c = shape(1, 96, 640, 2, 1, 64, scale=1.0)
    q, k, v, do = inputs(c, dtype, 1)
    ramp = torch.linspace(-6, 6, 640, device=dev)
    for order in (ramp, ramp.flip(0), ramp.abs()):
        kk = (k.float() * 0.1 + order[:, None] * q.float()[0, :64].sign()[None]).to(dtype)
        check(ctx, c, dtype, train=False, tensors=(q, kk, v, do))


def test_views_and_slices(ctx):
    """q | k | v in one row with a margin of NaN, and column slices of row buffers."""
    from depth_completion_amd import ops
    c = shape(2, 150, 150, 4, 2, 64, causal=True)
    check(ctx, c, torch.bfloat16, fused=True)
    q, k, v, _ = inputs(c, torch.bfloat16, 4)
    buf = torch.cat([torch.full((300, 8), float("nan"), device=dev), q.float(), k.float(), v.float()], 1).bfloat16()
    a, b = torch.empty_like(q), torch.empty_like(q)
    lse = torch.empty(2, 4, 150, device=dev)
    ops.attn_mask_fwd(ctx, q, k, v, a, lse, **c)
    ops.attn_mask_fwd(ctx, ops.S(buf, 8), ops.S(buf, 264), ops.S(buf, 392), b, lse, **c)
    assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["dq", "dk"])
def test_small_output_gradients_keep_their_digits(ctx, name):
    """fp16 with dout at the border of its subnormals: dS alone would be a few units of 2^-24.  The other factor is scaled up so
    that the gradient itself has its digits in the type."""
    from depth_completion_amd import ops
    c = shape(1, 300, 300, 2, 1, 64)
    q, k, v, do = inputs(c, torch.float16, 2)
    up = 64.0 if name == "dq" else 1 / 64.0
    q, k, do = (q.float() / up).half(), (k.float() * up).half(), (do.float() * 2.0 ** -14).half()
    o, lse = torch.empty_like(q), torch.empty(1, 2, 300, device=dev)
    ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
    got = dict(zip(("dq", "dk", "dv"), (torch.empty_like(q), torch.empty_like(k), torch.empty_like(v))))
    ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, *got.values(), **c)
    want = dict(zip(("dq", "dk"), definition(q, k, v, c, do)[2:4]))
    assert rel(got[name], want[name]) < 4 * U[torch.float16]


def test_gradients_by_differences(ctx):
    """sum(o w) falls as the gradients say when q, k and v move along a direction (fp32 sum of the forward's fp16 output)."""
    from depth_completion_amd import ops
    c = shape(1, 80, 80, 4, 2, 64, causal=True, softcap=10.0)
    q, k, v, w = inputs(c, torch.float16, 6, qscale=0.5)
    o, lse = torch.empty_like(q), torch.empty(1, 4, 80, device=dev)
    ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.attn_mask_bwd(ctx, q, k, v, o, lse, w, dq, dk, dv, **c)
    for x, g in ((q, dq), (k, dk), (v, dv)):
        step = 2.0 ** -5 * g.float().sign()   # along the gradient's signs: the sum moves by |g|_1 a step
        vals = []
        for sign in (1, -1):
            old = x.clone()
            x += (sign * step).to(x.dtype)
            ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
            vals.append((o.double() * w.double()).sum().item())
            x.copy_(old)
        want = 2 * 2.0 ** -5 * g.double().abs().sum().item()
        # third differences of a step of 2^-5 and the rounding of x: below 3 %
        assert abs(vals[0] - vals[1] - want) < 0.03 * want


def test_far_keys(ctx):
    """A cache whose last rows lie beyond 2^31 elements: the addresses are 64 bits wide."""
    from depth_completion_amd import ops
    tk, g, d, ld = 70000, 1, 64, 32768   # 2.3e9 elements, 4.6 GB each
    k, v = (torch.zeros(tk, ld, dtype=torch.bfloat16, device=dev) for _ in range(2))
    gen = torch.Generator(device=dev).manual_seed(1)
    kk, vv = (torch.randn(tk, d, generator=gen, device=dev).bfloat16() for _ in range(2))
    k[:, :d], v[:, :d] = kk, vv
    for tq in (1, 40):
        q = torch.randn(tq, 2 * d, generator=gen, device=dev).bfloat16()
        c = shape(1, tq, tk, 2, g, d, causal=True)
        a, b = torch.empty_like(q), torch.empty_like(q)
        la, lb = (torch.empty(1, 2, tq, device=dev) for _ in range(2))
        ops.attn_mask_fwd(ctx, q, k, v, a, la, **c)
        ops.attn_mask_fwd(ctx, q, kk, vv, b, lb, **c)
        assert torch.equal(a, b) and torch.equal(la, lb)
        check(ctx, c, torch.bfloat16, train=False, tensors=(q, kk, vv, q))


def test_same_bits_every_time(ctx):
    """No atomics on values: two passes give the same bits, split keys and split sweeps included."""
    from depth_completion_amd import ops
    for c in (shape(1, 1, 5000, 8, 2, 128), shape(1, 200, 1500, 8, 1, 64, causal=True)):
        q, k, v, do = inputs(c, torch.bfloat16, 8)
        got = []
        for _ in range(2):
            o, lse = torch.empty_like(q), torch.empty(1, 8, c["tq"], device=dev)
            ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
            dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
            ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, dq, dk, dv, **c)
            got.append((o, lse, dq, dk, dv))
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_two_graphs_and_a_stream(ctx):
    """Two captured graphs and an eager call on a third stream run beside each other: each has its own scratch."""
    from depth_completion_amd import ops
    cs = [shape(1, 1, 6000, 8, 2, 128, causal=True), shape(1, 260, 260, 4, 2, 64, doc_q=documents("packed", 260),
                                                            doc_k=documents("packed", 260))]
    graphs, outs, want = [], [], []
    side = torch.cuda.Stream()
    for c in cs:
        q, k, v, do = inputs(c, torch.bfloat16, 8)
        bufs = [torch.empty_like(q), torch.empty(1, c["heads"], c["tq"], device=dev), torch.empty_like(q),
                torch.empty_like(k), torch.empty_like(v)]

        def step(c=c, q=q, k=k, v=v, do=do, bufs=bufs):
            o, lse, dq, dk, dv = bufs
            ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
            ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, dq, dk, dv, **c)

        step()
        torch.cuda.synchronize()
        want.append([b.clone() for b in bufs])
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step()
        graphs.append((gr, step))
        outs.append(bufs)
    other = inputs(cs[0], torch.bfloat16, 8)
    o3, l3 = torch.empty_like(other[0]), torch.empty(1, 8, 1, device=dev)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        for bufs in outs:
            for b in bufs:
                b.fill_(3.0)
        o3.fill_(3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0][0].replay()
        with torch.cuda.stream(s2):
            graphs[1][0].replay()
        with torch.cuda.stream(side):
            ops.attn_mask_fwd(ctx, *other[:3], o3, l3, **cs[0])
        torch.cuda.synchronize()
        for bufs, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(bufs, ref))
        assert torch.equal(o3, want[0][0])


@TYPES
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tq,tk,causal", [(130, 200, False), (130, 200, True), (70, 90, False), (5, 300, True), (513, 1100, True)])
def test_bias_that_grows_with_distance(ctx, tq, tk, causal, d, dtype):
    """Slopes of either sign, and row counts that end inside a tile: what lies behind the last row weighs nothing, however far."""
    slopes = torch.tensor([-0.05, 0.05, -2.0, 0.5], device=dev)
    check(ctx, shape(2, tq, tk, 4, 2, d, slopes=slopes, causal=causal), dtype, seed=31)


@TYPES
@pytest.mark.parametrize("tq,d", [(4, 64), (130, 64), (33, 128), (129, 128)])
@pytest.mark.parametrize("cap", [64.0, 65.0, 1e4, 1e6, 1e30])
def test_wide_caps(ctx, cap, tq, d, dtype):
    """A cap far above the scores leaves them as they are, one that they reach bends them."""
    slopes = 2.0 ** -torch.arange(1.0, 3.0, device=dev)
    check(ctx, shape(1, tq, 300, 2, 1, d, softcap=cap, slopes=slopes), dtype, qscale=4.0, seed=32)
    check(ctx, shape(1, tq, 300, 2, 2, d, softcap=cap, scale=0.5, causal=True), dtype, qscale=8.0, seed=33)


@TYPES
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["documents", "causal"])
def test_short_rows_in_long_calls(ctx, kind, d, dtype):
    """Gradients of rows of few keys inside a call of many, each document (or the first rows of a causal call) against its own norm.
    The values share an offset of 16, which P (dP - rowsum) takes out again: rowsum(dO o) from a rounded o is off by up to 2^-8 (fp16
    2^-11) of it, many times the differences' own roundings."""
    from depth_completion_amd import ops
    lengths, t = [12, 500, 30, 300, 400], 1500
    ids = runs(lengths, t) if kind == "documents" else None
    c = shape(1, t, t, 2, 1, d, **(dict(doc_q=ids, doc_k=ids) if ids is not None else dict(causal=True)))
    q, k, v, do = inputs(c, dtype, 41)
    v = (16.0 + 0.25 * v.float()).to(dtype)
    o, lse = torch.empty_like(q), torch.empty(1, 2, t, device=dev)
    ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, dq, dk, dv, **c)
    _, _, rq, rk, _, _ = definition(q, k, v, c, do)
    at = 0
    for n in lengths if ids is not None else [1024]:
        rows = slice(at, at + n)
        assert rel(dq[rows], rq[rows]) < 4 * U[dtype], (at, n)
        assert ids is None or rel(dk[rows], rk[rows]) < 4 * U[dtype], (at, n)
        at += n


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tq,docs,kv_heads", [(4, False, 2), (70, False, 1), (200, True, 2)])
def test_large_values_of_two_keys(ctx, tq, docs, kv_heads, d):
    """fp16 values near the type's largest, weights near a half and a dout with their signs: P (dP - rowsum) passes the type's range,
    the gradients, of small q and k, do not.  (q and k of 2^-10: no gradient is above 1.5 d 60000 2^-10 2 rows.)"""
    ids = (torch.arange(tq, dtype=torch.int32, device=dev) // 2).repeat(2) if docs else None
    c = shape(2, tq, tq if docs else 2, 2, kv_heads, d, **(dict(doc_q=ids, doc_k=ids) if docs else {}))
    q, k, v, do = inputs(c, torch.float16, 51)
    q, k = (q.float() * 2.0 ** -10).half(), (k.float() * 2.0 ** -10).half()
    size = 40000.0 + 20000.0 * torch.rand(v.shape, generator=torch.Generator().manual_seed(1)).to(dev)
    alternate = 1.0 - 2.0 * (torch.arange(v.shape[0], device=dev) % 2)[:, None]
    v = (size * alternate).half()
    do = (do.float() * 0.25 + 1.5).half()
    if not docs:   # (all rows add up in the two keys' gradients)
        do = (do.float() / tq).half()
        q = q * 4
    check(ctx, c, torch.float16, tensors=(q, k, v, do))


@pytest.mark.parametrize("d", [64, 128])
def test_large_values_among_many_keys(ctx, d):
    """The same with two heavy keys among 1100 (more than the rows whose rowsum has a sweep of its own), and four rows whose dout
    is large beside the others'.  The heavy keys are both 50 in each column, to 0.05, so their shares of dQ cancel but for a tenth:
    dS of each is rounded, by u at most, and so is o in rowsum(dO o), by u of sum |dO o|, which is |rowsum| where dO and o have one sign
    each, as in the rows that count.  Both bound dQ's error by u times the norm of P (|dP| + |rowsum|) |K|, `size`, beside its own
    rounding."""
    from depth_completion_amd import ops
    t = 1100
    c = shape(1, t, t, 2, 1, d, scale=0.04 / d)
    q, k, v, do = inputs(c, torch.float16, 52)
    signs = torch.sign(q[:1, :d].float())
    q = (4.0 * signs.repeat(t, 2) + 0.2 * q.float()).half()
    k = 0.05 * k.float()
    k[:2] += 50.0 * signs
    v = v.float()
    v[0], v[1] = 60000.0, -30000.0
    do = 0.01 * do.float()
    do[::300] += 1.5
    k, v, do = k.half(), v.half(), do.half()
    o, lse = torch.empty_like(q), torch.empty(1, 2, t, device=dev)
    ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, dq, dk, dv, **c)
    ro, _, rq, rk, rv, size = definition(q, k, v, c, do)
    u = U[torch.float16]
    assert rel(o, ro) < 2 * u
    for name, x, r in (("dq", dq, rq), ("dk", dk, rk), ("dv", dv, rv)):
        off, norm = float((x.double().cpu() - r).norm()), float(r.norm())
        assert off <= max(4 * u * norm, 2 * u * size[name] + u * norm if name == "dq" else 0.0), (name, off, norm, size[name])


def near(ctx, c, dtype, seed, qscale=1.0):
    """As check(), against what independent roundings leave: one is off by u at most and by u / sqrt(3) in the root mean square, k of
    them by sqrt(k / 3) u.  k: o its own and P's, dV its own and P's, dQ and dK their own, dS's and that of o in rowsum(dO o)."""
    from depth_completion_amd import ops
    q, k, v, do = inputs(c, dtype, seed, qscale)
    o, lse = torch.empty_like(q), torch.empty(c["nb"], c["heads"], c["tq"], device=dev)
    ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, dq, dk, dv, **c)
    ro, rl, rq, rk, rv, _ = definition(q, k, v, c, do)
    seen = torch.isfinite(rl)
    assert torch.equal(torch.isinf(lse.cpu()), ~seen)
    assert float(((lse.cpu().double() - rl)[seen].abs() / rl[seen].abs().clamp_min(1.0)).max()) < (1e-5 if c.get("softcap") else 2e-6)
    for name, x, r, n in (("o", o, ro, 2), ("dv", dv, rv, 2), ("dq", dq, rq, 3), ("dk", dk, rk, 3)):
        assert rel(x, r) < math.sqrt(n / 3) * U[dtype], (name, rel(x, r), U[dtype])


@TYPES
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nb,tq,tk,heads,kv_heads,lengths,kv_len,cap,causal", [
    (1, 1500, 1500, 2, 1, [700, 90, 600], None, 0.0, False),      # a bias inside documents, some blocks split
    (2, 300, 300, 4, 2, [140, 130], None, 25.0, True),            # with a cap, short rows
    (1, 1700, 1700, 2, 2, [1100, 500], None, 25.0, False),
    (3, 200, 900, 4, 1, None, [900, 333, 640], 0.0, True),        # a bias over filled lengths
    (1, 200, 5000, 2, 1, None, None, 0.0, True),                  # split keys, split sweeps
    (1, 200, 5000, 2, 1, None, None, 25.0, False),
    (2, 5, 3000, 4, 2, [1000, 1900], [3000, 2500], 0.0, True)])   # a few rows at the end of two caches
def test_bias_with_other_masks(ctx, nb, tq, tk, heads, kv_heads, lengths, kv_len, cap, causal, d, dtype):
    c = shape(nb, tq, tk, heads, kv_heads, d, softcap=cap, causal=causal,
              slopes=torch.tensor([0.01, -0.002, 0.03, 0.001][:heads], device=dev))
    if lengths:
        ids = runs(lengths, tk)
        c["doc_k"] = ids.repeat(nb)
        c["doc_q"] = c["doc_k"] if tq == tk else ids[sum(lengths) - tq:sum(lengths)].repeat(nb)
    if kv_len:
        c["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device=dev)
    near(ctx, c, dtype, 61)


@TYPES
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tk", [1024, 1025, 1088, 1153])
def test_border_of_short_rows(ctx, tk, d, dtype):
    """16 tiles of keys, where rowsum has a sweep of its own, and 17 and more, where it is taken from o."""
    near(ctx, shape(1, 130, tk, 2, 1, d), dtype, 62)
    near(ctx, shape(1, tk, tk, 2, 2, d, causal=True), dtype, 63)


def test_same_bits_of_other_forms(ctx):
    """As test_same_bits_every_time: listed documents in parts, short rows, fp16 sums that are swept again, wide caps."""
    from depth_completion_amd import ops
    ids = runs([900, 60, 700], 1700)
    for c, dtype, big in ((shape(1, 1700, 1700, 3, 1, 64, doc_q=ids, doc_k=ids, softcap=30.0), torch.bfloat16, 1.0),
                          (shape(2, 300, 300, 4, 2, 128, causal=True), torch.float16, 30000.0),
                          (shape(1, 50, 700, 8, 2, 128, softcap=500.0), torch.float16, 1.0)):
        q, k, v, do = inputs(c, dtype, 71)
        v = (v.float().clamp(-2, 2) * big).to(dtype)
        got = []
        for _ in range(3):
            o, lse = torch.empty_like(q), torch.empty(c["nb"], c["heads"], c["tq"], device=dev)
            ops.attn_mask_fwd(ctx, q, k, v, o, lse, **c)
            dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
            ops.attn_mask_bwd(ctx, q, k, v, o, lse, do, dq, dk, dv, **c)
            got.append((o, lse, dq, dk, dv))
        for other in got[1:]:
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got[0], other))
