"""NVFP4 attention of finite queries whose scores are far beyond a trained model's.

With s the fp32 sum of the products and c the row's factor, a weight is 2^(c (s - s_ref)), so it is at most 2^15 in
fp16 whatever c s is, and that of the largest score is 2^7 or more: outputs are finite and lie between the least and the
largest visible value (half a step of the output's type, and (n / 32 + 40) 2^-24 of the sums, beside them). The scores themselves are
off by (Dh + 8) 2^-24 scale sum|q||k|; a row whose largest score is further than twice that and 40 above the others is that key's
value: the rest weighs n e^-40. Equal keys have equal scores, bit for bit, so their row is the mean of the values."""

import math

import pytest
import torch

from appcorr_amd import kernels as K
from tests import test_gpu_nvfp4_kv as KV

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16

# Rows, keys, cache length, heads, key heads, dims: the keys kernel, whole and with split keys; the rows kernel of 128 and of 256
# rows, whole and with split keys.
FAR = [([1] * 4, [1029, 7, 128, 129], 1030, 16, 4, 64), ([1, 2], [5000, 4500], 5000, 16, 2, 128),
       ([201, 33], [201, 700], 701, 28, 4, 128), ([100, 60], [100, 333], 400, 4, 4, 64), ([300], [2600], 2700, 8, 2, 64),
       ([300], [2600], 2700, 8, 2, 128)]


def offsets(dev, nq, nk):
    cu = torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device=dev)
    return cu, torch.tensor(nk, dtype=torch.int32, device=dev)


def rows_of(q, x, nq, nk):
    """(sequence's row range, head, queries, its keys and values, hidden) in 64 bits, causal."""
    Hq, Hk, at = q.shape[1], x.shape[3], 0
    for s, (a, b) in enumerate(zip(nq, nk)):
        hidden = torch.arange(b, device=q.device) > torch.arange(a, device=q.device)[:, None] + (b - a)
        for h in range(Hq):
            kh = h * Hk // Hq
            yield slice(at, at + a), h, q[at:at + a, h].double(), x[s, :b, 0, kh], x[s, :b, 1, kh], hidden
        at += a


def check_far(out, q, x, nq, nk, scale):
    M, Hq, Dh = q.shape
    out = out.view(M, Hq, Dh)
    assert torch.isfinite(out).all()
    u = KV.half_step(out.dtype)
    single = total = 0
    for rows, h, qq, k, v, hidden in rows_of(q, x, nq, nk):
        n = k.shape[0]
        got = out[rows, h].double()
        slack = (u + (n / 32 + 40) * 2.0 ** -23) * v.abs().amax(0) + 2.0 ** -24
        lo = torch.stack([v[~hid].amin(0) for hid in hidden])
        hi = torch.stack([v[~hid].amax(0) for hid in hidden])
        assert (got >= lo - slack).all() and (got <= hi + slack).all()
        z = (qq @ k.T * scale).masked_fill(hidden, -math.inf)
        off = (Dh + 8) * 2.0 ** -24 * (qq.abs() @ k.abs().T * scale).masked_fill(hidden, 0).amax(-1)
        top = torch.topk(torch.nn.functional.pad(z, (0, 1), value=-math.inf), 2, -1)
        alone = top.values[:, 0] - top.values[:, 1] > 2 * off + 40
        best = v[top.indices[:, 0]]
        near = (got - best).abs() <= (u + (n / 32 + 40) * 2.0 ** -23) * (best.abs() + v.abs().amax(0)) + 2.0 ** -24
        assert near[alone].all()
        single, total = single + int(alone.sum()), total + alone.numel()
    return single / total


@pytest.mark.parametrize("spread", [1e7, 2e8, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_far_scores(dev, case, spread):
    nq, nk, N, Hq, Hk, Dh = FAR[case]
    g = KV.gen(dev, case)
    cache = KV.filled(dev, len(nq), N, Hk, Dh, g)
    q = (torch.randn(sum(nq), Hq, Dh, generator=g, device=dev) * spread).to(BF)
    cu, kl = offsets(dev, nq, nk)
    out = K.packed_attention_nvfp4(q, cache, cu, kl, Dh ** -0.5, causal=True)
    # (two of n scores lie closer than 40 + 2e-4 of their size in a few rows of a hundred)
    assert check_far(out, q, KV.values64(cache), nq, nk, Dh ** -0.5) > 0.9


@pytest.mark.parametrize("case", range(len(FAR)))
def test_far_scores_of_fp16_queries(dev, case):
    """Large keys: a tensor scale of 2^14 times the usual one."""
    nq, nk, N, Hq, Hk, Dh = FAR[case]
    g = KV.gen(dev, case)
    cache = KV.filled(dev, len(nq), N, Hk, Dh, g)
    cache.tensor_scale[0] *= 2.0 ** 14
    q = (torch.randn(sum(nq), Hq, Dh, generator=g, device=dev) * 1e4).to(HF)
    cu, kl = offsets(dev, nq, nk)
    out = K.packed_attention_nvfp4(q, cache, cu, kl, 1.0, causal=True)
    assert check_far(out, q, KV.values64(cache), nq, nk, 1.0) > 0.9


@pytest.mark.parametrize("spread", [1.0, 1e5, 2e8, 1e9, 1e12, 3e37])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_equal_keys_weigh_the_same(dev, case, spread):
    nq, nk, N, Hq, Hk, Dh = FAR[case]
    B, g = len(nq), KV.gen(dev, case)
    cache = KV.cache_of(dev, B, N, Hk, Dh, g)
    key = torch.randn(1, Hk, Dh, generator=g, device=dev).to(BF).expand(B * N, Hk, Dh)
    v = (torch.randn(B * N, Hk, Dh, generator=g, device=dev) + 1).to(BF)
    i = torch.arange(B * N, device=dev)
    K.kv_nvfp4_write(key, v, i // N, i % N, cache)
    q = (torch.randn(sum(nq), Hq, Dh, generator=g, device=dev).clamp(-4, 4) * spread).to(BF)
    cu, kl = offsets(dev, nq, nk)
    out = K.packed_attention_nvfp4(q, cache, cu, kl, 3.0, causal=True).view(*q.shape)
    assert torch.isfinite(out).all()
    for rows, h, _, _, v64, hidden in rows_of(q, KV.values64(cache), nq, nk):
        w = (~hidden).double()
        mean, size = (w @ v64) / w.sum(-1, keepdim=True), (w @ v64.abs()) / w.sum(-1, keepdim=True)
        tol = (v64.shape[0] / 32 + 40) * 2.0 ** -24 * (size + mean.abs())
        assert ((out[rows, h].double() - mean).abs() <= tol + KV.half_step(BF) * (mean.abs() + tol)).all()


@pytest.mark.parametrize("base", [2.0 ** 10, 2.0 ** 18, 2.0 ** 24, 2.0 ** 25, 2.0 ** 26, 2.0 ** 27])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_scores_that_rise_by_less_than_the_reference_may_lag(dev, case, base):
    """A score of `base` (log2) by one dim, the same for all keys, and one that rises by up to 7.5 over the keys by another block:
    weights of 2^8 times the reference's meet references that are rounded."""
    nq, nk, N, Hq, Hk, Dh = FAR[case]
    B, g = len(nq), KV.gen(dev, case)
    cache = KV.cache_of(dev, B, N, Hk, Dh, g)
    k = torch.zeros(B * N, Hk, Dh, device=dev, dtype=BF)
    k[:, :, 0] = 6
    k[:, :, 16] = (torch.arange(B * N, device=dev) % N / N * 6)[:, None].to(BF)
    v = torch.randn(B * N, Hk, Dh, generator=g, device=dev).to(BF)
    i = torch.arange(B * N, device=dev)
    cache.tensor_scale.fill_(1.0)
    K.kv_nvfp4_write(k, v, i // N, i % N, cache)
    q = torch.zeros(sum(nq), Hq, Dh, device=dev, dtype=BF)
    q[:, :, 0], q[:, :, 16] = base / 6 * (1 + 0.5 * torch.rand(sum(nq), Hq, generator=g, device=dev)), 1.25
    cu, kl = offsets(dev, nq, nk)
    out = K.packed_attention_nvfp4(q, cache, cu, kl, 0.6931472, causal=True)
    check_far(out, q, KV.values64(cache), nq, nk, 0.6931472)
