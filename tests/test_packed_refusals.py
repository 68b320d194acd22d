"""CPU checks of the packed-sequence entry points: bad arguments are refused before any launch, with the documented
status at the C entries and with ValueError in the wrappers."""

import ctypes
import math

import pytest
import torch

from appcorr_amd import _lib
from appcorr_amd import kernels as K

P16 = ctypes.c_void_p(16)
NULL = ctypes.c_void_p(0)


def refused(status, fn, *args):
    with pytest.raises(_lib.OudjatKernelError) as e:
        _lib.call(fn, *args)
    assert e.value.status_name == status, str(e.value)


def plan_args(**kw):
    a = dict(q=P16, qw=0, k=P16, kw=0, S=2, rows=4, cap=8, packed=0, cu_q=P16, k_out=P16, cu_k=P16, bi=P16, ti=P16)
    a.update(kw)
    return (*a.values(), NULL)


@pytest.mark.parametrize("status,kw", [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(S=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(rows=-1)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(cap=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(q=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(cu_k=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(ti=NULL)),
    ("OUDJAT_ERR_TOO_LARGE", dict(S=4097)), ("OUDJAT_ERR_TOO_LARGE", dict(rows=1 << 31)),
    ("OUDJAT_ERR_TOO_LARGE", dict(cap=1 << 31)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(bi=ctypes.c_void_p(24))),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(q=ctypes.c_void_p(20), qw=1)),
])
def test_plan_refuses(status, kw):
    refused(status, "oudjat_packed_plan", *plan_args(**kw))


def rope_args(sections=(16, 16), **kw):
    host = (ctypes.c_int64 * len(sections))(*sections)
    a = dict(q=P16, q_rs=256, q_hs=64, k=P16, k_rs=256, k_hs=64, rows=4, Hq=4, Hk=4, Dh=64, dtype=0, pos=P16, kind=1,
             p_rs=2, p_as=1, axes=len(sections), freq=P16, sections=ctypes.addressof(host), qo=P16, qo_rs=256, qo_hs=64,
             ko=P16, ko_rs=256, ko_hs=64)
    a.update(kw)
    return host, (*a.values(), NULL)


@pytest.mark.parametrize("status,kw", [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(rows=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(dtype=2)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(kind=3)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(pos=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(q=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(ko=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(sections=(-8, 16))),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(sections=(16, 17))), ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(sections=(32, 8))),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(sections=(0, 0))),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(sections=(8, 8, 8, 4, 4))), ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(Dh=72)),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(Dh=528)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(q_rs=260)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(k=ctypes.c_void_p(8))),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(pos=ctypes.c_void_p(20))),
])
def test_rope_refuses(status, kw):
    kw = dict(kw)
    if isinstance(kw.get("sections"), tuple):
        host, args = rope_args(kw.pop("sections"), **kw)
    else:
        host, args = rope_args(**kw)
    refused(status, "oudjat_rope_axes", *args)


@pytest.mark.parametrize("kw", [dict(qo_rs=0), dict(ko_rs=0), dict(qo_hs=0), dict(qo_hs=56), dict(ko_rs=248),
                                dict(qo_rs=64, qo_hs=248), dict(ko_rs=-256), dict(qo_rs=1 << 62, rows=1 << 20, qo_hs=0)])
def test_rope_refuses_an_output_that_overlaps_itself(kw):
    host, args = rope_args(**kw)
    refused("OUDJAT_ERR_UNSUPPORTED_LAYOUT", "oudjat_rope_axes", *args)


def norm_args(sections=(16, 16), **kw):
    host = (ctypes.c_int64 * len(sections))(*sections)
    a = dict(x=P16, x_rs=512, rows=4, Hq=4, Hk=2, Dh=64, dtype=0, layer=0, qw=P16, qb=NULL, kw_=P16, kb=NULL, eps=1e-6,
             pos=P16, kind=1, p_rs=2, p_as=1, axes=len(sections), freq=P16, sections=ctypes.addressof(host), bi=P16,
             ti=P16, kv=P16, kv_bs=1024, kv_ns=256, kv_cs=128, B=2, N=4, qo=P16, qo_rs=256)
    a.update(kw)
    return host, (*a.values(), NULL)


@pytest.mark.parametrize("status,kw", [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(rows=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(Hq=0)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(dtype=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(eps=-1.0)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(eps=math.nan)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(qb=P16)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(kv=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(bi=NULL)),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(Dh=96)), ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(axes=0)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(x_rs=516)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(kv_cs=4)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(qw=ctypes.c_void_p(8))),
])
def test_norm_refuses(status, kw):
    host, args = norm_args(**kw)
    refused(status, "oudjat_qk_norm_rope_kv", *args)


@pytest.mark.parametrize("kw", [dict(qo_rs=0), dict(qo_rs=248), dict(kv_bs=0), dict(kv_ns=0), dict(kv_cs=0),
                                dict(kv_cs=120), dict(kv_ns=248), dict(kv_bs=1016), dict(kv_bs=256, kv_ns=504, kv_cs=128)])
def test_norm_refuses_outputs_that_overlap_themselves(kw):
    host, args = norm_args(**kw)
    refused("OUDJAT_ERR_UNSUPPORTED_LAYOUT", "oudjat_qk_norm_rope_kv", *args)


def attn_args(**kw):
    a = dict(q=P16, q_rs=256, q_hs=64, rows=4, Hq=4, Dh=64, k=P16, k_bs=0, k_rs=128, k_hs=64, v=P16, v_bs=0, v_rs=128,
             v_hs=64, Hk=2, cap=8, batched=0, cu=P16, cu_w=0, keys=P16, keys_w=0, S=1, scale=0.1, causal=1, dtype=0,
             out=P16, out_rs=256, ws=NULL, ws_elems=0)
    a.update(kw)
    return (*a.values(), NULL)


@pytest.mark.parametrize("status,kw", [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(rows=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(Hk=0)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(cap=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(dtype=3)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scale=0.0)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scale=-1.0)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scale=math.inf)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scale=math.nan)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(q=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(v=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(keys=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(out=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(ws_elems=-1)),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(Dh=96)), ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(Hq=5)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(k_rs=-128)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(q_hs=60)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(v=ctypes.c_void_p(24))),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(cu=ctypes.c_void_p(20), cu_w=1)),
    ("OUDJAT_ERR_TOO_LARGE", dict(rows=1 << 30)), ("OUDJAT_ERR_TOO_LARGE", dict(cap=1 << 30)),
    ("OUDJAT_ERR_TOO_LARGE", dict(k_rs=1 << 24)),
])
def test_attention_refuses(status, kw):
    refused(status, "oudjat_packed_attention", *attn_args(**kw))


@pytest.mark.parametrize("out_rs", [0, 248])
def test_attention_refuses_an_output_that_overlaps_itself(out_rs):
    refused("OUDJAT_ERR_UNSUPPORTED_LAYOUT", "oudjat_packed_attention", *attn_args(out_rs=out_rs))


def test_attention_refuses_a_missing_or_small_workspace():
    """Few rows over a long cache: the keys may be split, and the call needs what the library asks for."""
    shape = (4, 1, 4, 2, 64)
    need = _lib.load().oudjat_packed_attention_workspace_elems(*shape, 5000)
    assert need > 0 and _lib.load().oudjat_packed_attention_workspace_elems(*shape, 2048) == 0
    for ws, elems in ((NULL, need), (P16, need - 1), (ctypes.c_void_p(24), need)):
        refused("OUDJAT_ERR_INVALID_ARGUMENT", "oudjat_packed_attention", *attn_args(cap=5000, ws=ws, ws_elems=elems))


@pytest.mark.parametrize("rows,S,Hq,Hk,Dh,cap", [(1, 1, 1, 1, 64, 1 << 29), (32, 32, 32, 8, 128, 16385), (700, 3, 32, 8, 128, 9000),
                                                  (100, 70, 4, 1, 64, 4000), (1, 1, 64, 64, 128, 1 << 29)])
def test_attention_workspace_is_bounded(rows, S, Hq, Hk, Dh, cap):
    """A part is at most 256 rows of Dh + 2 floats and there are about as many as CUs and tiles together."""
    need = _lib.load().oudjat_packed_attention_workspace_elems(rows, S, Hq, Hk, Dh, cap)
    tiles = rows * (Hq // Hk) // 16 + min(S, rows)
    assert 0 < need <= (tiles * Hk + 2 * 256 + 2 * Hk) * (256 * (Dh + 2) + 4)


def test_nothing_to_do_is_no_error():
    _lib.call("oudjat_packed_attention", *attn_args(rows=0, q=NULL, out=NULL))
    _lib.call("oudjat_packed_attention", *attn_args(S=0, cu=NULL))
    host, args = rope_args(rows=0, q=NULL)
    _lib.call("oudjat_rope_axes", *args)
    host, args = norm_args(rows=0, x=NULL)
    _lib.call("oudjat_qk_norm_rope_kv", *args)


def test_wrappers_take_gpu_tensors_only():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU only"):
        K.packed_plan(n, n, 4, cache_len=4)
    with pytest.raises(ValueError, match="GPU only"):
        K.packed_attention(x, x, x, n, n, 0.1, causal=True)
    with pytest.raises(ValueError, match="GPU only"):
        K.apply_rope_axes(x, x, torch.zeros(2, 1), torch.zeros(32), (32,))
