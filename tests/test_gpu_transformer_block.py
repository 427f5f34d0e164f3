"""The operators of a transformer block in a row, as a denoiser uses them on packed frames (GPU): projection, rotary positions on q
and k in place, masked attention, projection, the norms with gate and residual scale, and the gradients all the way back, against
the same block differentiated in 64 bits.

Tolerance: a forward value passes 5 roundings to bf16 (qkv, turned q and k, P and o, y, the output) and a gradient as many again on
its way back; each is at most u = 2^-8 of the norm and none is amplified (unit-scale projections, norms), so 6 u and 12 u bound
them.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

dev = torch.device("cuda:0")
U = 2.0 ** -8
T, H, G, D, C = 700, 6, 3, 64, 384
WIDTH = (H + 2 * G) * D


def block(graph):
    """Runs the block forward and back; with ``graph`` captured once and replayed. Returns what it got and its inputs."""
    from depth_completion_amd import ops
    ctx = ops.Ctx(dev)
    g = torch.Generator().manual_seed(3)
    bf = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(torch.bfloat16).to(dev)  # noqa: E731
    x, hin = bf(T, C), bf(T, C)
    wqkv, wo = bf(WIDTH, C, scale=C ** -0.5), bf(C, H * D, scale=(H * D) ** -0.5)
    gate, dr, dh = bf(5, C), bf(T, C), bf(T, C)
    w1, w2 = (1 + 0.1 * torch.randn(C, generator=g).to(dev) for _ in range(2))
    ids = torch.tensor([0] * 250 + [1] * 190 + [2] * 200 + [-1] * 60, dtype=torch.int32, device=dev)
    pos = torch.cat([torch.arange(n) for n in (250, 190, 200, 60)]).to(torch.int32).to(dev)
    freqs, mag = ops.rotary_freqs(32, theta=100.0, device=dev)
    new = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=dev)  # noqa: E731
    b = dict(qkv=new(T, WIDTH), o=new(T, H * D), y=new(T, C), r=new(T, C), h=new(T, C), dx=new(T, C), dy=new(T, C), do=new(T, H * D),
             dqkv=new(T, WIDTH), dhin=new(T, C), dgate=new(5, C), lse=torch.empty(1, H, T, device=dev),
             stats=torch.empty(T, 4, device=dev), dw1=torch.empty(C, device=dev), dw2=torch.empty(C, device=dev))
    wqkv_t, wo_t = wqkv.t().contiguous(), wo.t().contiguous()
    norms = dict(first="rms", second="rms", w1=w1, w2=w2, gate=gate, s=0.5)
    mask = dict(nb=1, tq=T, tk=T, heads=H, kv_heads=G, d=D, softcap=20.0, doc_q=ids, doc_k=ids)

    def step():
        parts = lambda t: (t, ops.S(t, H * D), ops.S(t, (H + G) * D))  # noqa: E731
        ops.linear(ctx, hin, wqkv, T, WIDTH, b["qkv"])
        ops.rotary(ctx, b["qkv"], T, H + G, D, freqs, pos=pos, mag=mag)
        ops.attn_mask_fwd(ctx, *parts(b["qkv"]), b["o"], b["lse"], **mask)
        ops.linear(ctx, b["o"], wo, T, C, b["y"])
        ops.resnorm_fwd(ctx, x, b["y"], T, C, b["r"], b["h"], b["stats"], **norms)
        ops.resnorm_bwd(ctx, x, b["y"], T, C, b["stats"], dr, dh, b["dx"], b["dy"], dgate=b["dgate"], dw1=b["dw1"], dw2=b["dw2"],
                        **norms)
        ops.linear(ctx, b["dy"], wo_t, T, H * D, b["do"])
        ops.attn_mask_bwd(ctx, *parts(b["qkv"]), b["o"], b["lse"], b["do"], *parts(b["dqkv"]), **mask)
        ops.rotary(ctx, b["dqkv"], T, H + G, D, freqs, pos=pos, mag=mag, inverse=True)
        ops.linear(ctx, b["dqkv"], wqkv_t, T, C, b["dhin"])

    step()
    torch.cuda.synchronize()
    if graph:
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            step()
        for _ in range(3):
            for t in b.values():
                t.fill_(5.0)
            cg.replay()
            torch.cuda.synchronize()
    return b, dict(x=x, hin=hin, wqkv=wqkv, wo=wo, gate=gate, w1=w1, w2=w2, dr=dr, dh=dh, ids=ids, pos=pos, freqs=freqs)


def definition(i):
    v = {k: i[k].double().cpu().requires_grad_(True) for k in ("x", "hin", "gate", "w1", "w2")}
    qkv = v["hin"] @ i["wqkv"].double().cpu().T
    q, k, val = (t.reshape(T, -1, D) for t in qkv.split([H * D, G * D, G * D], 1))
    a = i["pos"].double().cpu()[:, None] * i["freqs"].cpu()[None]
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    turn = lambda t: torch.cat([t[..., :16] * c - t[..., 16:32] * s, t[..., :16] * s + t[..., 16:32] * c, t[..., 32:]], -1)  # noqa: E731
    q, k = turn(q), turn(k)
    k, val = k.repeat_interleave(H // G, 1), val.repeat_interleave(H // G, 1)
    ids = i["ids"].cpu()
    see = (ids[:, None] == ids[None]) & (ids[:, None] >= 0)
    sc = 20.0 * torch.tanh(torch.einsum("ihd,jhd->hij", q, k) / 8.0 / 20.0)
    p = torch.where(see, torch.softmax(sc.masked_fill(~see, -1e30), -1), 0.0)
    o = torch.einsum("hij,jhd->ihd", p, val).reshape(T, H * D)
    y = o @ i["wo"].double().cpu().T
    rms = lambda t, w: t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-5) * w  # noqa: E731
    r = v["x"] + 0.5 * v["gate"].repeat_interleave(T // 5, 0) * rms(y, v["w1"])
    h = rms(r, v["w2"])
    loss = (r * i["dr"].double().cpu()).sum() + (h * i["dh"].double().cpu()).sum()
    grads = dict(zip(v, torch.autograd.grad(loss, list(v.values()))))
    return dict(o=o, y=y, r=r, h=h, dx=grads["x"], dhin=grads["hin"], dgate=grads["gate"], dw1=grads["w1"], dw2=grads["w2"])


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_block(graph):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    got, inputs = block(graph)
    for k, want in definition(inputs).items():
        want = want.detach()
        off = float((got[k].double().cpu() - want).norm() / want.norm())
        assert off < (12 if k.startswith("d") else 6) * U, (k, off)
