"""CPU checks of the INT8 and NVFP4-cache entry points: bad arguments are refused before any launch, with the documented status at
the C entries and with ValueError in the wrappers; what the host decides about a call."""

import ctypes
import re
from collections import Counter

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


def quant_args(**kw):
    a = dict(x=P16, rows=4, K=64, x_rs=64, dtype=0, codes=ctypes.c_void_p(1 << 20), c_rs=64, scale=P16)
    a.update(kw)
    return (*a.values(), NULL)


@pytest.mark.parametrize("status,kw", [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(rows=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(K=-16)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(dtype=2)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(x=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(codes=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scale=NULL)),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(K=72)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(x_rs=68)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(x_rs=-64)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(c_rs=72)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(x=ctypes.c_void_p(8))), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(c_rs=0)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(c_rs=48)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(scale=ctypes.c_void_p(6))),
    ("OUDJAT_ERR_TOO_LARGE", dict(rows=1 << 26)), ("OUDJAT_ERR_TOO_LARGE", dict(K=1 << 30, x_rs=1 << 30, c_rs=1 << 30)),
])
def test_quantize_refuses(status, kw):
    refused(status, "oudjat_quantize_int8", *quant_args(**kw))


def linear_args(**kw):
    a = dict(A=P16, M=4, K=128, lda=128, sa=P16, W=P16, N=64, ldw=128, sw=P16, bias=NULL, epi=0, gamma=NULL, resid=NULL,
             ldr=0, C=P16, ldc=64, dtype=0)
    a.update(kw)
    return (*a.values(), NULL)


@pytest.mark.parametrize("status,kw", [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(M=-1)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(epi=1)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(epi=16)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(dtype=3)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(A=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(sw=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(epi=3)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(epi=2, gamma=P16)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(epi=4)), ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(K=96)),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(K=0)), ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(N=60)),
    ("OUDJAT_ERR_TOO_LARGE", dict(K=1 << 17, lda=1 << 17, ldw=1 << 17)), ("OUDJAT_ERR_TOO_LARGE", dict(lda=1 << 22)),
    ("OUDJAT_ERR_TOO_LARGE", dict(ldw=1 << 22)), ("OUDJAT_ERR_TOO_LARGE", dict(M=1 << 30)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(lda=136)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(ldc=68)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(ldc=56)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(ldc=0)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(W=ctypes.c_void_p(24))), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(lda=-128)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(bias=ctypes.c_void_p(8))), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(sw=ctypes.c_void_p(8))),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(epi=4, resid=P16, ldr=60)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(epi=4, resid=P16, ldr=-64)),
])
def test_linear_refuses(status, kw):
    refused(status, "oudjat_linear_int8", *linear_args(**kw))


@pytest.mark.parametrize("rows,K", [(1 << 24, 1040), (1 << 25, 8192), ((1 << 26) - 3, 64)])
def test_quantize_refuses_more_workgroups_than_a_launch_holds(rows, K):
    refused("OUDJAT_ERR_TOO_LARGE", "oudjat_quantize_int8", *quant_args(rows=rows, K=K, x_rs=K, c_rs=K))


@pytest.mark.parametrize("M,N,K", [(1 << 27, 16, 64), ((1 << 30) - 1, 64, 64), ((1 << 30) - 1, 8, 128)])
def test_linear_refuses_more_workgroups_than_a_launch_holds(M, N, K):
    refused("OUDJAT_ERR_TOO_LARGE", "oudjat_linear_int8", *linear_args(M=M, N=N, K=K, lda=K, ldw=K, ldc=N))


def cache_args(Dh=64, Hk=2, N=8, **kw):
    """A head-major cache's addresses and strides."""
    a = dict(codes=ctypes.c_void_p(1 << 20), c_bs=2 * Hk * N * Dh // 2, c_ns=Dh // 2, c_cs=Hk * N * Dh // 2,
             c_hs=N * Dh // 2, scales=ctypes.c_void_p(1 << 24), s_bs=2 * Hk * N * Dh // 16, s_ns=Dh // 16,
             s_cs=Hk * N * Dh // 16, s_hs=N * Dh // 16, ts=P16)
    a.update({k: v for k, v in kw.items() if k in a})
    return tuple(a.values())


CACHE_REFUSED = [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(codes=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scales=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(ts=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(Hk=0)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(dtype=2)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(rows=-1)),
    ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(Dh=96)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(c_ns=40)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(c_bs=-512)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(s_ns=2)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(s_hs=-32)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(codes=ctypes.c_void_p(24))),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(scales=ctypes.c_void_p(18))),
]


def write_args(Hk=2, Dh=64, **kw):
    a = dict(k=P16, k_rs=256, k_hs=64, v=P16, v_rs=256, v_hs=64, rows=4, Hk=Hk, Dh=Dh, dtype=0, bi=P16, ti=P16)
    a.update({k: v for k, v in kw.items() if k in a})
    return (*a.values(), *cache_args(Dh, max(Hk, 1), **kw), kw.get("B", 2), kw.get("N", 8), NULL)


@pytest.mark.parametrize("status,kw", CACHE_REFUSED + [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(k=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(ti=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(B=-1)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(k_rs=260)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(v_hs=-64)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(v=ctypes.c_void_p(8))),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(bi=ctypes.c_void_p(20))),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(c_ns=16)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(c_bs=0)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(c_cs=0)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(s_bs=0)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(s_hs=4)), ("OUDJAT_ERR_TOO_LARGE", dict(Hk=65536)),
    ("OUDJAT_ERR_TOO_LARGE", dict(rows=1 << 40)),
])
def test_write_refuses(status, kw):
    refused(status, "oudjat_kv_nvfp4_write", *write_args(**kw))


def read_args(Hk=2, Dh=64, **kw):
    a = dict(bi=P16, ti=P16, rows=4, dtype=0, ko=P16, vo=ctypes.c_void_p(1 << 16))
    a.update({k: v for k, v in kw.items() if k in a})
    return (*cache_args(Dh, max(Hk, 1), **kw), kw.get("B", 2), kw.get("N", 8), Hk, Dh, *a.values(), NULL)


@pytest.mark.parametrize("status,kw", CACHE_REFUSED + [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(ko=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(vo=P16)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(ko=ctypes.c_void_p(24))),
])
def test_read_refuses(status, kw):
    refused(status, "oudjat_kv_nvfp4_read", *read_args(**kw))


def attn_args(Hk=2, Dh=64, N=8, **kw):
    a = dict(q=P16, q_rs=256, q_hs=64, rows=4, Hq=4, Dh=Dh)
    b = dict(Hk=Hk, cap=N, cu=P16, cu_wide=0, keys=P16, keys_wide=0, S=2, scale=0.1, causal=1, dtype=0, out=P16, out_rs=256,
             ws=NULL, elems=0)
    a.update({k: v for k, v in kw.items() if k in a})
    b.update({k: v for k, v in kw.items() if k in b})
    return (*a.values(), *cache_args(Dh, max(Hk, 1), N, **kw), *b.values(), NULL)


@pytest.mark.parametrize("status,kw", CACHE_REFUSED + [
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(q=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(out=NULL)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(cu=NULL)), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scale=0.0)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scale=float("nan"))), ("OUDJAT_ERR_INVALID_ARGUMENT", dict(scale=float("inf"))),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(S=-1)), ("OUDJAT_ERR_UNSUPPORTED_SHAPE", dict(Hq=5)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(q_rs=260)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(q_hs=-64)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(out_rs=0)), ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(out_rs=248)),
    ("OUDJAT_ERR_UNSUPPORTED_LAYOUT", dict(cu=ctypes.c_void_p(20), cu_wide=1)), ("OUDJAT_ERR_TOO_LARGE", dict(c_ns=1 << 24)),
    ("OUDJAT_ERR_TOO_LARGE", dict(s_ns=1 << 24)), ("OUDJAT_ERR_TOO_LARGE", dict(rows=1 << 29)),
    ("OUDJAT_ERR_INVALID_ARGUMENT", dict(N=4096)),  # keys that are split need a workspace
])
def test_attention_refuses(status, kw):
    refused(status, "oudjat_packed_attention_nvfp4", *attn_args(**kw))


def test_nothing_to_do_is_no_error():
    _lib.call("oudjat_quantize_int8", *quant_args(rows=0, x=NULL, codes=NULL, scale=NULL))
    _lib.call("oudjat_linear_int8", *linear_args(M=0, A=NULL, C=NULL))
    _lib.call("oudjat_linear_int8", *linear_args(N=0, W=NULL, C=NULL))
    _lib.call("oudjat_kv_nvfp4_write", *write_args(rows=0))
    _lib.call("oudjat_kv_nvfp4_write", *write_args(B=0, codes=NULL, scales=NULL))
    _lib.call("oudjat_kv_nvfp4_read", *read_args(rows=0))
    _lib.call("oudjat_packed_attention_nvfp4", *attn_args(rows=0))
    _lib.call("oudjat_packed_attention_nvfp4", *attn_args(S=0))


@pytest.mark.parametrize("rows,S,Hq,Hk,Dh,cap", [
    (1, 1, 1, 1, 64, 1), (4, 4, 32, 8, 128, 16385), (512, 3, 32, 8, 128, 9000), (700, 3, 32, 8, 128, 9000),
    (100, 70, 4, 1, 64, 4000), (1, 1, 64, 64, 128, 1 << 29), (1 << 20, 64, 16, 16, 64, 1 << 20)])
def test_attention_workspace_is_bounded(rows, S, Hq, Hk, Dh, cap):
    elems = _lib.load().oudjat_packed_attention_nvfp4_workspace_elems(rows, S, Hq, Hk, Dh, cap)
    assert 0 <= elems <= (rows * Hq * Hk // Hk * 2 + 64 * (S + 600) * Hk * 16) * (Dh + 8)


def test_wrappers_refuse_cpu_tensors_and_bad_operands():
    x, i8 = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.int8)
    s = torch.ones(4)
    with pytest.raises(ValueError, match="GPU only"):
        K.quantize_int8(x)
    with pytest.raises(ValueError, match="GPU only"):
        K.linear_int8(i8, s, i8, s)
    cache = K.kv_nvfp4_cache(2, 8, 2, 64, "cpu")
    i = torch.zeros(4, dtype=torch.long)
    kv = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU only"):
        K.kv_nvfp4_write(kv, kv, i, i, cache)
    with pytest.raises(ValueError, match="GPU only"):
        K.kv_nvfp4_read(cache, i, i)
    with pytest.raises(ValueError, match="GPU only"):
        K.packed_attention_nvfp4(kv, cache, torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1.0,
                                 causal=True)


def test_a_cache_lays_a_heads_tokens_side_by_side():
    c = K.kv_nvfp4_cache(3, 10, 4, 128, "cpu", tensor_scale=0.25)
    assert c.codes.shape == (3, 10, 2, 4, 64) and c.scales.shape == (3, 10, 2, 4, 8)
    assert c.codes.stride() == (5120, 64, 2560, 640, 1) and c.scales.stride() == (640, 8, 320, 80, 1)
    assert c.scales.dtype == torch.float8_e4m3fn and (c.tensor_scale == 0.25).all() and c.tensor_scale.shape == (2, 4)
    own = torch.rand(2, 4)
    assert K.kv_nvfp4_cache(1, 1, 4, 64, "cpu", tensor_scale=own).tensor_scale is own


def test_gpu_tests_reach_every_tile_of_the_product():
    from tests.test_gpu_int8 import SHAPES

    plans = [(s, K.linear_int8_tile(*s)) for s in SHAPES]
    tiles = Counter(p[:2] for _, p in plans)
    assert set(tiles) == {(16, 16), (64, 64), (64, 128), (128, 128), (192, 256), (256, 256)}
    assert min(tiles.values()) >= 2
    split = [(s, p) for s, p in plans if p[2] != s[0]]  # rows in two launches, from either of the large tiles
    assert {p[0] for _, p in split} == {192, 256}
    assert all(0 < p[2] < s[0] and p[2] % p[0] == 0 for s, p in split)


def test_every_kernel_of_the_library_is_one_that_a_call_takes():
    blob = _lib.LIB_PATH.read_bytes()
    tiles = {tuple(map(int, re.findall(rb"\d+", m))) for m in
             re.findall(rb"int8_tile_kernelINS_9Quant(?:Bf16|Fp16)E((?:Li\d+E)+)E", blob)}
    assert {t[1:] for t in tiles} == {(64, 64, 2, 2, 4), (64, 128, 2, 4, 3), (128, 128, 2, 2, 2), (192, 256, 2, 4, 2),
                                      (256, 256, 2, 4, 2)}
    assert {t[0] for t in tiles} == {_lib.EPI_BIAS, _lib.EPI_BIAS_LS, _lib.EPI_BIAS_LS_RESID, _lib.EPI_BIAS_SILU_MUL}

    def attention(kernel):
        found = re.findall(kernel + rb"INS_8Elem(Bf16|Fp16)E((?:Li\d+E)+)E", blob)
        return {(e.decode(), *map(int, re.findall(rb"\d+", n))) for e, n in found}

    both = [(e,) for e in ("Bf16", "Fp16")]
    assert attention(rb"nvfp4_attn_keys_kernel") == {(*e, d, w) for e in both for d in (64, 128) for w in (4, 8)}
    assert attention(rb"nvfp4_attn_rows_kernel") == {(*e, d, w) for e in both for d, w in ((64, 4), (128, 4), (128, 8))}
    rows = {(e.decode(), m.decode(), int(u)) for m, e, u in
            re.findall(rb"kv_nvfp4_(write|read)_kernelINS_8Elem(Bf16|Fp16)ELb([01])EE", blob)}
    assert rows == {(e, m, u) for (e,) in both for m in ("write", "read") for u in (0, 1)}
