"""packed_attention_nvfp4 over split keys, the operator's one call with a workspace and a second launch: query rows that are not
finite go through the parts and their merge, and a call on a side stream waits for that stream's work and for nothing else's
scratch."""

import math

import pytest
import torch

from appcorr_amd import kernels as K
from tests import test_gpu_nvfp4_kv as KV
from tests.test_gpu_nvfp4_limits import FAR, offsets

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("case", range(len(FAR)))
def test_rows_that_are_not_finite(dev, case):
    """NaN and infinities in a query row give NaN there, whole or in parts, and no other row notices."""
    nq, nk, N, Hq, Hk, Dh = FAR[case]
    g = KV.gen(dev, case)
    cache = KV.filled(dev, len(nq), N, Hk, Dh, g)
    q = torch.randn(sum(nq), Hq, Dh, generator=g, device=dev).to(BF)
    cu, kl = offsets(dev, nq, nk)
    want = K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True).view(*q.shape)
    assert torch.isfinite(want).all()
    last = sum(nq) - 1
    q[0, 1, 5], q[last, 0, 0], q[last, Hq - 1, Dh - 1] = math.nan, math.inf, -math.inf
    got = K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True).view(*q.shape)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device=dev)
    bad[0, 1] = bad[last, 0] = bad[last, Hq - 1] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("nq,nk,Hq,Hk,Dh", [([1, 2], [5000, 4500], 16, 2, 128), ([1, 3], [4900, 5000], 4, 4, 64),
                                            ([300], [2600], 8, 2, 64), ([300], [2600], 8, 2, 128)])
def test_split_keys_on_another_stream(dev, nq, nk, Hq, Hk, Dh):
    """Behind work of the side stream that makes the queries and the cache, beside calls of the main stream with scratch of
    their own; the same bits as on the main stream alone."""
    N, S, g = 5000, len(nq), KV.gen(dev, 5)
    x = torch.randn(S * N, 2, Hk, Dh, generator=g, device=dev).to(BF)
    base = torch.randn(sum(nq), Hq, Dh, generator=g, device=dev)
    cu, kl = offsets(dev, nq, nk)
    i = torch.arange(S * N, device=dev)
    other = KV.filled(dev, S, N, Hk, Dh, g)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def made():
        q = base
        for _ in range(20):
            q = q * 1.01
        q = q.to(BF)
        cache = K.kv_nvfp4_cache(S, N, Hk, Dh, dev)
        K.kv_nvfp4_write(x[:, 0], x[:, 1], i // N, i % N, cache)
        return q, cache, K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True)

    elsewhere = torch.randn(sum(nq), Hq, Dh, generator=g, device=dev).to(BF)
    want_elsewhere = K.packed_attention_nvfp4(elsewhere, other, cu, kl, 0.1, causal=True)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(stream):
            q, cache, out = made()
        beside = [K.packed_attention_nvfp4(elsewhere, other, cu, kl, 0.1, causal=True) for _ in range(5)]
        torch.cuda.synchronize()
        assert all(torch.equal(b, want_elsewhere) for b in beside)
        ref, tol = KV.attend64(q, KV.values64(cache), nq, nk, 0.1, True, N)
        KV.check(out, ref, tol)
        assert torch.equal(out, made()[2])
