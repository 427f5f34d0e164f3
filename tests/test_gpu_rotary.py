"""Rotary positions (dc_rotary) against the definition in 64 bits (GPU).

Tolerance: one rounding to the type (half a step u of the element), and the sines' error times the pair's size: the sine unit
is good to 2^-19 of a turn's unit circle, fp32 sines of a turn rounded to fp32 to 2^-21.  |y - want| <= u |want| + e |pair| m.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

dev = torch.device("cuda:0")
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from depth_completion_amd.ops import Ctx
    return Ctx(dev, ws_mb=1)


def definition(x, pos, freqs, heads, d, off, interleaved, inverse, mag):
    y = x.double().cpu().reshape(-1, heads, d).clone()
    rot = 2 * len(freqs)
    a = pos.double().cpu()[:, None] * freqs.double().cpu()[None]
    c, s = torch.cos(a)[:, None] * mag, torch.sin(a)[:, None] * mag * (-1 if inverse else 1)
    i = torch.arange(rot // 2)
    p, q = (off + 2 * i, off + 2 * i + 1) if interleaved else (off + i, off + i + rot // 2)
    e, f = y[..., p].clone(), y[..., q].clone()
    y[..., p], y[..., q] = e * c - f * s, e * s + f * c
    size = torch.zeros_like(y)
    size[..., p] = size[..., q] = torch.sqrt(e * e + f * f) * mag
    return y.reshape(len(x), -1), size.reshape(len(x), -1)


def close(y, want, size):
    u, e = U[y.dtype], 2.0 ** -21 if y.dtype is torch.float32 else 2.0 ** -19
    tiny = 2.0 ** -25 if y.dtype is torch.float16 else 0.0   # half a step of fp16's subnormals
    off = (y.double().cpu() - want).abs() - (u * want.abs() * (1 + 2.0 ** -10) + e * size + tiny)
    assert float(off.max()) <= 0.0, float(off.max())


def freqs_of(rot, theta=10000.0):
    return theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)


@pytest.mark.parametrize("dtype", list(U), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,d,off,rot", [
    (1, 1, 64, 0, 64), (3, 40, 128, 0, 128), (257, 5, 64, 16, 32), (70, 3, 80, 0, 20), (33, 2, 66, 1, 2), (5, 7, 37, 3, 30),
    (2000, 24, 128, 64, 64), (1, 300, 16, 0, 16)])
def test_rotary(ctx, rows, heads, d, off, rot, interleaved, dtype):
    from depth_completion_amd import ops
    g = torch.Generator(device=dev).manual_seed(rows)
    x = torch.randn(rows, heads * d, generator=g, device=dev).to(dtype)
    pos = torch.randint(-5, 4000000, (rows,), generator=g, device=dev, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    f = freqs_of(rot)
    for inverse in (False, True):
        y = torch.full((rows + 1, heads * d + 8), 7.0, dtype=dtype, device=dev)
        ops.rotary(ctx, x, rows, heads, d, f, y, pos=pos, off=off, interleaved=interleaved, inverse=inverse, mag=1.25)
        close(y[:rows, :heads * d], *definition(x, pos, f, heads, d, off, interleaved, inverse, 1.25))
        assert (y[rows:] == 7).all() and (y[:, heads * d:] == 7).all()
        z = torch.cat([x, x], 1)   # in place, in a wider row
        ops.rotary(ctx, z, rows, heads, d, f, pos=pos, off=off, interleaved=interleaved, inverse=inverse, mag=1.25)
        assert torch.equal(z[:, :heads * d], y[:rows, :heads * d]) and torch.equal(z[:, heads * d:], x)


def test_rows_of_sequences(ctx):
    """Without positions row r stands at pos0 + r % t."""
    from depth_completion_amd import ops
    x = torch.randn(3 * 50, 128, device=dev).bfloat16()
    a, b = torch.empty_like(x), torch.empty_like(x)
    pos = (100 + torch.arange(150, device=dev) % 50).int()
    ops.rotary(ctx, x, 150, 2, 64, freqs_of(64), a, pos=pos)
    ops.rotary(ctx, x, 150, 2, 64, freqs_of(64), b, t=50, pos0=100)
    assert torch.equal(a, b)


def test_values_beside_and_slices(ctx):
    """NaN and infinities stay in their pairs; unaligned column offsets take the narrow path with the same result."""
    from depth_completion_amd import ops
    x = torch.randn(64, 4 * 64, device=dev).bfloat16()
    x[3, 5], x[9, 70] = float("nan"), float("inf")
    y = torch.empty_like(x)
    ops.rotary(ctx, x, 64, 4, 64, freqs_of(32), y, t=64, off=8)
    bad = ~torch.isfinite(y)
    assert bad[3].nonzero().flatten().tolist() == [5] and bad[9].nonzero().flatten().tolist() == [70]
    x[9, 80] = float("nan")   # column 16 of head 1: pairs with column 32
    ops.rotary(ctx, x, 64, 4, 64, freqs_of(32), y, t=64, off=8)
    assert (~torch.isfinite(y))[9].nonzero().flatten().tolist() == [70, 80, 96]
    wide = torch.full((64, 300), float("nan"), device=dev).bfloat16()
    wide[:, 3:259] = x
    out = torch.empty(64, 300, device=dev).bfloat16()
    ops.rotary(ctx, ops.S(wide, 3), 64, 4, 64, freqs_of(32), ops.S(out, 3), t=64, off=8)
    assert torch.equal(out[:, 3:259].nan_to_num(), y.nan_to_num())


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(ctx, interleaved):
    """The turn back is the adjoint: <turn(x), w> = <x, turn_back(w)>, and differences of a linear map are exact."""
    from depth_completion_amd import ops
    x, w = (torch.randn(40, 3 * 48, device=dev) for _ in range(2))
    y, g = torch.empty_like(x), torch.empty_like(x)
    kw = dict(t=40, pos0=77, off=8, interleaved=interleaved, mag=0.75)
    ops.rotary(ctx, x, 40, 3, 48, freqs_of(32), y, **kw)
    ops.rotary(ctx, w, 40, 3, 48, freqs_of(32), g, inverse=True, **kw)
    a, b = (y.double() * w.double()).sum(), (x.double() * g.double()).sum()
    assert abs(float(a - b)) < 1e-5 * float(y.norm() * w.norm())
    e = torch.zeros_like(x)
    e[7, 60] = 0.5
    z = torch.empty_like(x)
    ops.rotary(ctx, x + e, 40, 3, 48, freqs_of(32), z, **kw)
    assert abs(float(((z.double() - y.double()) * w.double()).sum()) - 0.5 * float(g[7, 60])) < 1e-4


def test_captured(ctx):
    from depth_completion_amd import ops
    x = torch.randn(33, 4 * 64, device=dev).bfloat16()
    pos = torch.arange(33, device=dev, dtype=torch.int32)
    y, f = torch.empty_like(x), freqs_of(64)
    ops.rotary(ctx, x, 33, 4, 64, f, y, pos=pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary(ctx, x, 33, 4, 64, f, y, pos=pos)
    for k in range(3):   # other positions and values in the same places
        pos.add_(1000 * k)
        x.mul_(-1.5)
        graph.replay()
        want = torch.empty_like(x)
        ops.rotary(ctx, x, 33, 4, 64, f, want, pos=pos)
        assert torch.equal(y, want)


@pytest.mark.parametrize("scaling", ["none", "linear", "base", "parts"])
def test_scaled_frequencies(ctx, scaling):
    from depth_completion_amd import ops
    f, mag = ops.rotary_freqs(128, scaling=scaling, factor=8.0, trained=4096, device=dev)
    x = torch.randn(9, 128, device=dev)
    pos = torch.arange(9, device=dev, dtype=torch.int32) * 4000
    y = torch.empty_like(x)
    ops.rotary(ctx, x, 9, 1, 128, f, y, pos=pos, mag=mag)
    close(y, *definition(x, pos, f, 1, 128, 0, False, False, mag))
    assert math.isclose(mag, 1 + 0.1 * math.log(8) if scaling == "parts" else 1.0, rel_tol=1e-6)
