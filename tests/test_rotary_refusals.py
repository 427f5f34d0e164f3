"""Frequencies of the rotary positions (host), and what the rotary call refuses (CPU: nothing is launched)."""
import ctypes as C
import math

import pytest
import torch

from depth_completion_amd import _lib, ops


def test_frequencies():
    f, mag = ops.rotary_freqs(64)
    want = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert mag == 1.0 and f.dtype is torch.float64 and torch.allclose(f, want, rtol=1e-14, atol=0)
    assert torch.allclose(ops.rotary_freqs(64, scaling="linear", factor=4.0)[0], want / 4, rtol=1e-14, atol=0)
    base = ops.rotary_freqs(64, scaling="base", factor=4.0)[0]
    assert base[0] == 1.0 and math.isclose(base[-1], want[-1] / 4, rel_tol=1e-12)
    parts, mag = ops.rotary_freqs(64, scaling="parts", factor=4.0, trained=2048, fast=32, slow=1)
    turns = 2048 * want / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], want[turns >= 32])
    assert torch.allclose(parts[turns <= 1], want[turns <= 1] / 4, rtol=1e-14, atol=0)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((parts < want) & (parts > want / 4))[mid].all()
    assert math.isclose(mag, 1 + 0.1 * math.log(4), rel_tol=1e-6)


@pytest.mark.parametrize("kw", [
    dict(rot=0), dict(rot=7), dict(rot=-2), dict(theta=1.0), dict(theta=float("nan")), dict(theta=float("inf")),
    dict(scaling="other"), dict(scaling="linear", factor=0.5), dict(scaling="base", rot=2, factor=2.0),
    dict(scaling="parts", factor=2.0), dict(scaling="parts", factor=2.0, trained=100, fast=1, slow=1)])
def test_frequencies_refuse(kw):
    with pytest.raises((ValueError, _lib.DCError)):
        ops.rotary_freqs(**dict(dict(rot=64), **kw))


def call(x=None, rows=4, heads=2, d=64, freqs=None, **kw):
    x = torch.zeros(4, 128) if x is None else x
    freqs = torch.ones(32, dtype=torch.float64) if freqs is None else freqs
    return ops.rotary(ops.Ctx("cpu", ws_mb=1), x, rows, heads, d, freqs, **kw)


@pytest.mark.parametrize("kw", [
    dict(rows=0), dict(heads=0), dict(d=0), dict(off=-1, t=4), dict(off=1, t=4), dict(freqs=torch.ones(33, dtype=torch.float64), t=4),
    dict(freqs=torch.ones(0, dtype=torch.float64), t=4), dict(freqs=torch.ones(32), t=4), dict(x=torch.zeros(4, 128).int(), t=4),
    dict(t=0), dict(pos=torch.zeros(4, dtype=torch.int64)), dict(t=4, mag=float("nan")), dict(t=4)])
def test_call_refuses(kw):
    with pytest.raises(ValueError):   # the last case: a context that is on no GPU
        call(**kw)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), 1), (dict(y=None), 1), (dict(freqs=None), 1), (dict(type=3), 1), (dict(rows=0), 1), (dict(heads=0), 1),
    (dict(d=0), 1), (dict(rot=0), 1), (dict(rot=3), 1), (dict(rot=66), 1), (dict(off=-1), 1), (dict(off=2), 1), (dict(ldx=127), 1),
    (dict(ldy=127), 1), (dict(t=0), 1), (dict(y=4096, ldy=136), 1), (dict(x=4097), 3), (dict(freqs=4100), 3), (dict(pos=4098), 3),
    (dict(rows=1 << 41), 1), (dict(heads=70000), 1)])
def test_entry_refuses(kw, status):
    a = dict(x=4096, ldx=128, y=8192, ldy=128, type=0, rows=4, heads=2, d=64, off=0, rot=64, freqs=4096, pos=None, pos0=0, t=4,
             mag=1.0, interleaved=0, inverse=0)
    assert _lib.load().dc_rotary(C.byref(_lib.RotaryDesc(**dict(a, **kw))), None) == status


def test_no_null_descriptor():
    assert _lib.load().dc_rotary(None, None) == 1


@pytest.mark.parametrize("rows,y", [(1 << 30, 8192), (1 << 27, 8194)])
def test_entry_refuses_more_threads_than_a_launch_has(rows, y):
    """2^32 packs of pairs, and as many single pairs where the rows start between two packs."""
    a = _lib.RotaryDesc(x=4096, ldx=128, y=y, ldy=128, type=0, rows=rows, heads=2, d=64, off=0, rot=64, freqs=4096, pos=None, pos0=0,
                        t=4, mag=1.0, interleaved=0, inverse=0)
    assert _lib.load().dc_rotary(C.byref(a), None) == 1
