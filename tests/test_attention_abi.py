"""What norm_rope, attention_packed and attention_prefix refuse, through the C
ABI and the Python wrappers; no GPU needed (every refusal comes before any
device work)."""
import ctypes as C

import pytest
import torch

import mlk2_b200 as mb
from mlk2_b200 import api

P, Y = 1 << 20, 1 << 24  # aligned addresses that are never followed


class Heads(C.Structure):
    _fields_ = [("data", C.c_void_p), ("rows", C.c_int64), ("row_stride", C.c_int64),
                ("head_stride", C.c_int64)]


def heads(rows=10, row=1024, head=128, data=P):
    return Heads(data, rows, row, head)


def refs(*ops):
    return [C.addressof(o) if o is not None else None for o in ops]


def refused(status, part=""):
    assert status == mb.ERR_INVALID, status
    assert part in mb.lib().mlkb_last_error().decode()


def accepted(status):
    """All checks passed: the call got as far as asking for a device."""
    assert status == mb.ERR_NO_DEVICE, (status, mb.lib().mlkb_last_error().decode())


no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="the call would run on these addresses")


# ---- norm_rope ------------------------------------------------------------------

def norm_rope(q=None, k=None, qo=None, ko=None, heads_=8, kv=2, d=128, rot=128, qw=P, kw=P, eps=1e-6,
              table=P, table_rows=100, positions=P, stride=10, sections=None, axes=1, dtype=mb.F16):
    ops = [q or heads(), k or heads(), qo or heads(), ko or heads()]
    sec = (C.c_int32 * len(sections))(*sections) if sections else None
    return mb.lib().mlkb_norm_rope(*refs(*ops), heads_, kv, d, rot, qw, kw, eps, table, table_rows,
                                   positions, stride, sec, axes, 0, dtype, None)


@no_device
def test_norm_rope_accepts():
    accepted(norm_rope())
    accepted(norm_rope(qw=None, kw=None, dtype=mb.BF16))
    accepted(norm_rope(d=80, rot=48, axes=3, sections=[8, 0, 16]))
    accepted(norm_rope(kv=0, kw=None))
    accepted(norm_rope(q=heads(row=0, rows=1), k=heads(rows=1), qo=heads(rows=1, row=-8),
                       ko=heads(rows=1)))  # a single row's stride does not matter


def test_norm_rope_nothing_to_do():
    empty = heads(rows=0, data=None)
    assert norm_rope(q=empty, k=empty, qo=empty, ko=empty, table=None, positions=None) == mb.OK


@pytest.mark.parametrize("kw,part", [
    ({"dtype": mb.F32}, "dtype"), ({"heads_": 0}, "heads"), ({"kv": -1}, "heads"), ({"d": 136}, "d and rot"),
    ({"d": 528}, "d and rot"), ({"rot": 24}, "d and rot"), ({"rot": 144}, "d and rot"), ({"rot": 0}, "d and rot"),
    ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"qw": None}, "weights"), ({"kw": None}, "weights"),
    ({"qw": P + 8}, "aligned"), ({"table": None}, "table"), ({"table": P + 4}, "table"),
    ({"positions": None}, "positions"), ({"positions": P + 2}, "positions"), ({"table_rows": 0}, "table"),
    ({"axes": 0}, "axes"), ({"axes": 5, "sections": [64, 0, 0, 0, 0]}, "axes"), ({"axes": 2}, "sections"),
    ({"axes": 2, "sections": [32, 16]}, "sections"), ({"axes": 2, "sections": [80, -16]}, "section"),
    ({"axes": 2, "sections": [32, 32], "stride": -1}, "stride"),
    ({"q": heads(data=None)}, "norm_rope q: null"), ({"q": heads(data=P + 8)}, "aligned"),
    ({"k": heads(row=1020)}, "strides"), ({"k": heads(head=-128)}, "strides"), ({"k": heads(rows=9)}, "rows"),
    ({"qo": heads(rows=11)}, "rows"), ({"q": heads(rows=-1)}, "rows"), ({"q": heads(rows=2 ** 30 + 1)}, "rows"),
    ({"qo": heads(row=512)}, "overlap"), ({"ko": heads(head=64)}, "overlap"),
    ({"q": heads(row=2 ** 40)}, "strides")])
def test_norm_rope_refuses(kw, part):
    refused(norm_rope(**kw), part)


# ---- attention_packed ----------------------------------------------------------------

def packed(q=None, k=None, v=None, y=None, heads_=8, kv=2, d=128, qs=P, ks=P, n=3, scale=0.1,
           dtype=mb.F16, ws=None, size=0):
    ops = [q or heads(), k or heads(20), v or heads(20), y or heads(data=Y)]
    return mb.lib().mlkb_attention_packed(*refs(*ops), heads_, kv, d, qs, ks, n, 1, scale, dtype, ws, size,
                                          None)


@no_device
def test_packed_accepts():
    accepted(packed())
    accepted(packed(dtype=mb.BF16, d=8, k=heads(0, data=None), v=heads(0, data=None)))
    accepted(packed(heads_=128, kv=1, q=heads(row=128 * 128), y=heads(row=128 * 128, data=Y)))


def test_y_may_not_be_an_input():
    refused(packed(y=heads()), "overlap")
    refused(packed(y=heads(), q=heads(data=Y)), "overlap")
    refused(packed(y=heads(data=Y), v=heads(20, data=Y)), "overlap")
    refused(prefix(y=heads()), "overlap")


def test_packed_nothing_to_do():
    empty = heads(rows=0, data=None)
    assert packed(q=empty, y=empty) == mb.OK
    assert packed(n=0, qs=None, ks=None) == mb.OK


@pytest.mark.parametrize("kw,part", [
    ({"dtype": mb.F64}, "dtype"), ({"heads_": 7}, "heads"), ({"kv": 0}, "heads"), ({"heads_": 258}, "heads"),
    ({"d": 136}, "d must"), ({"d": 0}, "d must"), ({"d": 12}, "d must"), ({"scale": 0.0}, "scale"),
    ({"scale": -1.0}, "scale"), ({"scale": float("inf")}, "scale"), ({"scale": float("nan")}, "scale"),
    ({"scale": 1e-40}, "scale"), ({"qs": None}, "starts"), ({"ks": P + 1}, "starts"), ({"n": -1}, "sequences"),
    ({"v": heads(19)}, "rows"), ({"y": heads(11)}, "rows"), ({"y": heads(row=1016)}, "overlap"),
    ({"k": heads(20, data=P + 2)}, "aligned"), ({"k": heads(20, head=130)}, "strides"), ({"size": -1}, "")])
def test_packed_refuses(kw, part):
    refused(packed(**kw), part)


def test_packed_workspace():
    size = mb.lib().mlkb_attention_packed_workspace
    assert size(1, 16384, 1, 32, 4, 128) > 0          # one query over many keys
    assert size(1, 500, 1, 32, 4, 128) == 0           # few keys
    assert size(8192, 8192, 1, 32, 8, 128) == 0       # items enough
    assert size(0, 100, 3, 8, 2, 64) == 0
    for bad in ((-1, 1, 1, 8, 2, 64), (1, 1, 1, 7, 2, 64), (1, 1, 1, 8, 2, 256), (1, 1, 1, 8, 0, 64)):
        assert size(*bad) < 0


# ---- attention_prefix ----------------------------------------------------------------

def prefix(q=None, pk=None, pv=None, kp=None, vp=None, y=None, batch=5, steps=2, heads_=8, kv=2, d=128,
           page=16, wide=3, pages=P, lens=P, scale=0.1, dtype=mb.F16, ws=P, size=1 << 40):
    ops = [q or heads(), pk or heads(30), pv or heads(30), kp or heads(320), vp or heads(320), y or heads(data=Y)]
    return mb.lib().mlkb_attention_prefix(*refs(*ops), batch, steps, heads_, kv, d, page, wide, pages, lens,
                                          scale, dtype, ws, size, None)


@no_device
def test_prefix_accepts():
    accepted(prefix())
    accepted(prefix(pages=None, page=37, wide=1, kp=heads(5 * 37), vp=heads(5 * 37)))
    none = heads(0, data=None)
    accepted(prefix(pk=none, pv=none))
    accepted(prefix(kp=none, vp=none, page=0, wide=0, pages=None, lens=None))


def test_prefix_nothing_to_do():
    empty = heads(rows=0, data=None)
    assert prefix(q=empty, y=empty, batch=0, ws=None, size=0) == mb.OK


@pytest.mark.parametrize("kw,part", [
    ({"dtype": mb.F32}, "dtype"), ({"heads_": 9}, "heads"), ({"d": 132}, "d must"), ({"scale": 0.0}, "scale"),
    ({"batch": 4}, "rows"), ({"steps": 0}, "rows"), ({"batch": -5, "steps": -2}, "rows"),
    ({"pv": heads(31)}, "equal rows"), ({"vp": heads(336)}, "equal rows"), ({"page": 8}, "page size"),
    ({"page": 48}, "page size"), ({"page": 64, "kp": heads(330), "vp": heads(330)}, "page"),
    ({"page": -16}, "page"), ({"wide": -1}, "page"), ({"wide": 2 ** 29}, "2^30"),
    ({"pages": None}, "page table"), ({"pages": None, "wide": 1, "page": 60}, "page table"),
    ({"lens": None}, "lens"), ({"lens": P + 2}, "lens"), ({"pages": P + 2}, "lens"), ({"ws": None}, "workspace"),
    ({"ws": P + 8}, "workspace"), ({"size": 100}, "workspace"), ({"y": heads(head=64)}, "overlap"),
    ({"q": heads(data=None)}, "attention q: null"), ({"pk": heads(30, row=1020)}, "strides")])
def test_prefix_refuses(kw, part):
    if torch.cuda.is_available() and kw == {}:
        pytest.skip("would run")
    refused(prefix(**kw), part)


def test_prefix_workspace():
    size = mb.lib().mlkb_attention_prefix_workspace
    assert size(4, 1, 8, 2, 64, 0, 0, 0) >= 16
    assert size(4, 1, 8, 2, 64, 500, 61, 1) > size(2, 1, 8, 2, 64, 500, 61, 1) > 0
    for bad in ((4, 0, 8, 2, 64, 5, 16, 1), (4, 1, 8, 3, 64, 5, 16, 1), (4, 1, 8, 2, 200, 5, 16, 1),
                (-1, 1, 8, 2, 64, 5, 16, 1), (4, 1, 8, 2, 64, -5, 16, 1)):
        assert size(*bad) < 0
    # the largest shapes stay within 64 bits
    assert size(2 ** 20, 1, 128, 1, 128, 2 ** 30, 16, 2 ** 20) > 0


# ---- the wrappers -----------------------------------------------------------------------

def test_wrappers_refuse_host_tensors_and_other_types():
    q = torch.zeros(4, 8, 64, dtype=torch.float16)
    k = torch.zeros(4, 2, 64, dtype=torch.float16)
    pos, t = torch.zeros(4, dtype=torch.int32), torch.zeros(9, 64)
    s = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        api.norm_rope(q, k, q, k, t, pos)
    with pytest.raises(ValueError, match="CUDA device"):
        api.attention_packed(q, k, k, q, s, s, 0.1)
    with pytest.raises(ValueError, match="CUDA device"):
        api.attention_prefix(q[:, None], k, k, k[:, None], k[:, None], q[:, None], pos, 0.1)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        api.norm_rope(q.float(), k.float(), q.float(), k.float(), t, pos)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        api.attention_packed(q.float(), k, k, q, s, s, 0.1)
