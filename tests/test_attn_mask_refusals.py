"""What the masked attention refuses, in Python and at the C entry (CPU: nothing is launched)."""
import ctypes as C

import pytest
import torch

from depth_completion_amd import _lib, ops

GOOD = dict(nb=1, tq=4, tk=8, heads=4, kv_heads=2, d=64)


def call(back=False, dtype=torch.bfloat16, **kw):
    c = dict(GOOD, **kw)
    ctx = ops.Ctx("cpu", ws_mb=1)
    h, g, d = c["heads"], c["kv_heads"], c["d"]
    q, k = torch.zeros(4, abs(h * d) + 1, dtype=dtype), torch.zeros(8, abs(g * d) + 1, dtype=dtype)
    lse = torch.zeros(64)
    if back:
        return ops.attn_mask_bwd(ctx, q, k, k, q, lse, q, q, k, k, **c)
    return ops.attn_mask_fwd(ctx, q, k, k, q, lse, **c)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("kw", [
    dict(nb=0), dict(tq=0), dict(tk=-1), dict(heads=0), dict(kv_heads=3), dict(d=60), dict(d=136), dict(d=0),
    dict(dtype=torch.float32), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")),
    dict(prefix=torch.zeros(1, dtype=torch.int32)), dict(doc_q=torch.zeros(4, dtype=torch.int32)),
    dict(doc_k=torch.zeros(8, dtype=torch.int32)), dict()])
def test_python_refuses(kw, back):
    with pytest.raises(ValueError):   # the last case: a context that is on no GPU
        call(back, **kw)


def test_row_views():
    t = torch.zeros(6, 40)
    view = lambda x, rows=6, cols=16: ops._row_view("t", x, rows, cols, torch.float32, -1)  # noqa: E731
    assert view(t) == (t.data_ptr(), 40)
    assert view(ops.S(t, 24)) == (t.data_ptr() + 96, 40)
    assert view(t[:, 8:24]) == (t.data_ptr() + 32, 40)
    assert view(t[:1, :13], 1, 13) == (t.data_ptr(), 16)   # one row: its stride is never used
    for bad in (t.double(), t[:5], ops.S(t, 25), ops.S(t, -8), t.t(), t[:, ::2], t.view(-1), t[None]):
        with pytest.raises(ValueError):
            view(bad)
    with pytest.raises(ValueError):
        ops._row_view("t", t, 6, 16, torch.float32, 0)   # another device
    for bad in (t[:, :3], t[:1], t.int()):
        with pytest.raises(ValueError):
            ops._flat("t", bad, 41, torch.float32, -1)
    assert ops._flat("t", None, 5, torch.float32, 0) == 0


def descriptor(**kw):
    base = dict(type=0, nb=1, tq=4, tk=8, heads=4, kv_heads=2, d=64, q=4096, k=4096, v=4096, o=4096, lse=4096, ldq=256, ldk=128,
                ldv=128, ldo=256, scale=0.125, dout=4096, dq=4096, dk=4096, dv=4096, lddo=256, lddq=256, lddk=128, lddv=128)
    d = _lib.AttnDesc()
    for k, v in dict(base, **kw).items():
        setattr(d, k, v)
    return d


ARG, ALIGN = 1, 3


@pytest.mark.parametrize("entry", ["dc_attn_mask_fwd", "dc_attn_mask_bwd"])
@pytest.mark.parametrize("kw,status", [
    (dict(type=2), ARG), (dict(type=-1), ARG), (dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(o=None), ARG),
    (dict(lse=None), ARG), (dict(nb=0), ARG), (dict(tq=0), ARG), (dict(tk=0), ARG), (dict(heads=3), ARG), (dict(d=4), ARG),
    (dict(d=136, ldq=544, ldo=544, ldk=272, ldv=272), ARG), (dict(scale=0.0), ARG), (dict(scale=float("nan")), ARG),
    (dict(scale=float("inf")), ARG), (dict(softcap=-1.0), ARG), (dict(softcap=float("nan")), ARG), (dict(prefix=4096), ARG),
    (dict(doc_q=4096), ARG), (dict(doc_k=4096), ARG), (dict(ldq=248), ARG), (dict(ldk=120), ARG), (dict(ldq=260), ALIGN),
    (dict(ldv=132), ALIGN), (dict(q=4098), ALIGN), (dict(v=4104), ALIGN),
    (dict(nb=1 << 20, tq=1 << 10), ARG), (dict(doc_q=4096, doc_k=4096, tk=1000), ARG), (dict(tq=1, tk=100000), ARG)])
def test_entry_refuses(entry, kw, status):
    """The last two want scratch that the call does not bring."""
    assert getattr(_lib.load(), entry)(C.byref(descriptor(**kw)), None, 0, None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dout=None), ARG), (dict(dq=None), ARG), (dict(dk=None), ARG), (dict(dv=None), ARG), (dict(lddo=248), ARG),
    (dict(lddk=132), ALIGN), (dict(dv=4098), ALIGN), (dict(), ARG)])
def test_backward_entry_refuses(kw, status):
    assert _lib.load().dc_attn_mask_bwd(C.byref(descriptor(**kw)), None, 0, None) == status


def test_entries_take_no_null_descriptor():
    lib = _lib.load()
    assert lib.dc_attn_mask_fwd(None, None, 0, None) == ARG and lib.dc_attn_mask_bwd(None, None, 0, None) == ARG
    assert lib.dc_attn_mask_ws_bytes(None, 0) == 0


def test_scratch_alignment():
    lib, d = _lib.load(), C.byref(descriptor())
    assert lib.dc_attn_mask_fwd(d, 4100, 1 << 30, None) == ALIGN and lib.dc_attn_mask_bwd(d, 4100, 1 << 30, None) == ALIGN


@pytest.mark.parametrize("desc,pack", [(_lib.AttnDesc, _lib.PACK_ATTN), (_lib.RotaryDesc, _lib.PACK_ROTARY),
                                       (_lib.ResnormDesc, _lib.PACK_RESNORM)])
def test_packed_descriptors(desc, pack):
    """The packed bytes are the structure's, field by field."""
    values = [i + 1 for i in range(len(desc._fields_))]
    d = desc(*values)
    assert pack.size == C.sizeof(desc) and pack.pack(*values) == bytes(d)


@pytest.mark.parametrize("kw", [
    dict(kv_heads=8), dict(kv_heads=3), dict(tq=0), dict(nb=1 << 30, heads=1 << 30, kv_heads=1 << 30, tq=16), dict(nb=1 << 22, tq=1)])
@pytest.mark.parametrize("back", [0, 1])
def test_scratch_of_impossible_shapes(kw, back):
    """More key heads than heads, products that pass 64 bits, more blocks than a launch has: no scratch, and no division by none."""
    d = descriptor(**kw)
    assert _lib.load().dc_attn_mask_ws_bytes(C.byref(d), back) == 0
    assert _lib.load().dc_attn_mask_fwd(C.byref(d), 4096, 1 << 40, None) == ARG


def test_fields_that_do_not_hold():
    """Numbers beyond a descriptor's fields are refused as arguments, not as an error of the packing."""
    fields = [0] * len(_lib.AttnDesc._fields_)
    for i, v in ((1, 1 << 31), (3, -1 << 40), (12, 1 << 31)):
        bad = list(fields)
        bad[i] = v
        with pytest.raises(ValueError, match="attn"):
            ops._pack(_lib.PACK_ATTN, "attn_mask", *bad)
    assert ops._pack(_lib.PACK_ATTN, "attn_mask", *fields) == bytes(_lib.AttnDesc())


def test_slopes_beside_no_scale():
    with pytest.raises(ValueError, match="slopes"):
        call(slopes=torch.zeros(4), scale=1e-31)
    d = descriptor(slopes=4096, scale=1e-31)
    assert _lib.load().dc_attn_mask_fwd(C.byref(d), 4096, 1 << 30, None) == ARG


def test_scratch_of_few_rows():
    """Documents of few query rows are looked at as their keys are read: without split keys the forward needs no scratch."""
    lib = _lib.load()
    few = descriptor(nb=64, tq=64, tk=600, heads=8, kv_heads=8, doc_q=4096, doc_k=4096)
    assert lib.dc_attn_mask_ws_bytes(C.byref(few), 0) == 0
    few.tq = 65
    assert lib.dc_attn_mask_ws_bytes(C.byref(few), 0) >= 64 * 10 * 16   # a summary of each tile of keys
