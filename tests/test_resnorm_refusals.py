"""What the norms around a block refuse, in Python and at the C entry (CPU: nothing is launched)."""
import ctypes as C

import pytest
import torch

from depth_completion_amd import _lib, ops

X, V = torch.zeros(6, 64), torch.zeros(64)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("kw", [
    dict(rows=0), dict(c=0), dict(c=60), dict(c=8200), dict(first="batch"), dict(second="l2"), dict(first="none", w1=V),
    dict(second="none", b2=V, h=None), dict(eps=-1.0), dict(eps=float("nan")), dict(a=float("nan")), dict(s=float("inf")),
    dict(gate=torch.zeros(4, 64)), dict(gate=torch.zeros(0, 64)), dict(x=X.int()), dict()])
def test_python_refuses(kw, back):
    c = dict(dict(x=X, y=X, rows=6, c=64, r=X, h=X, stats=torch.zeros(6, 4), first="rms", second="rms"), **kw)
    h, r = c.pop("h"), c.pop("r")
    pos = [ops.Ctx("cpu", ws_mb=1), c.pop("x"), c.pop("y"), c.pop("rows"), c.pop("c")]
    stats = c.pop("stats")
    with pytest.raises(ValueError):   # the last case: a context that is on no GPU
        if back:
            ops.resnorm_bwd(*pos, stats, r, h, X, X, **c)
        else:
            ops.resnorm_fwd(*pos, r, h, stats, **c)


def descriptor(**kw):
    p = 4096
    base = dict(type=0, c=64, first=2, second=2, rows=6, gates=2, x=p, y=p, gate=p, w1=p, w2=p, ldx=64, ldy=64, ldg=64, ldr=64,
                ldh=64, a=1.0, s=1.0, eps=1e-5, r=p, h=p, stats=p, dr=p, dh=p, dx=p, dy=p, lddr=64, lddh=64, lddx=64, lddy=64,
                lddg=64)
    d = _lib.ResnormDesc()
    for k, v in dict(base, **kw).items():
        setattr(d, k, v)
    return d


ARG, ALIGN = 1, 3
BOTH = [(dict(type=3), ARG), (dict(type=-1), ARG), (dict(c=0), ARG), (dict(c=60), ARG), (dict(c=8200), ARG), (dict(rows=0), ARG),
        (dict(first=3), ARG), (dict(second=-1), ARG), (dict(x=None), ARG), (dict(y=None), ARG), (dict(stats=None), ARG),
        (dict(gate=None), ARG), (dict(gates=0), ARG), (dict(gates=4), ARG), (dict(gates=-2), ARG), (dict(first=0), ARG),
        (dict(second=0), ARG), (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG), (dict(ldx=56), ARG), (dict(ldg=56), ARG),
        (dict(rows=1 << 42), ARG), (dict(ldx=68), ALIGN), (dict(ldg=68), ALIGN), (dict(x=4104), ALIGN), (dict(gate=4104), ALIGN),
        (dict(w1=4098), ALIGN), (dict(stats=4100), ALIGN)]


@pytest.mark.parametrize("kw,status", BOTH + [(dict(r=None), ARG), (dict(h=None), ARG), (dict(ldr=56), ARG), (dict(ldh=68), ALIGN)])
def test_forward_entry_refuses(kw, status):
    assert _lib.load().dc_resnorm_fwd(C.byref(descriptor(**kw)), None) == status


@pytest.mark.parametrize("kw,status", BOTH + [
    (dict(dx=None), ARG), (dict(dy=None), ARG), (dict(dh=None), ARG), (dict(lddr=56), ARG), (dict(lddy=68), ALIGN),
    (dict(dgate=4096, lddg=56), ARG), (dict(dgate=4096, gates=0, gate=None), ARG), (dict(first=0, w1=None, dw1=4096), ARG),
    (dict(second=0, w2=None, dh=None, db2=4096), ARG), (dict(second=0, w2=None, dh=None, dr=None), ARG), (dict(dw1=4096), ARG)])
def test_backward_entry_refuses(kw, status):
    """The last wants scratch that the call does not bring."""
    assert _lib.load().dc_resnorm_bwd(C.byref(descriptor(**kw)), None, 0, None) == status


def test_no_null_descriptor():
    lib = _lib.load()
    assert lib.dc_resnorm_fwd(None, None) == ARG and lib.dc_resnorm_bwd(None, None, 0, None) == ARG
    assert lib.dc_resnorm_ws_bytes(None) == 0
    assert lib.dc_resnorm_bwd(C.byref(descriptor(dw1=4096)), 4100, 1 << 30, None) == ALIGN
