"""packed_attention where scores are large. A weight is 2^(c (s - s_ref)) whatever c s is: equal keys weigh the same, so that their
row is the mean of the values, over any number of tiles, waves and parts; finite rows stay finite and between the least and the
largest visible value; a score that is alone at the top is that key's value (bounds: test_gpu_nvfp4_limits.py)."""

import pytest
import torch

from appcorr_amd import kernels as K
from tests import test_gpu_nvfp4_kv as KV
from tests.test_gpu_nvfp4_limits import FAR, check_far, offsets, rows_of

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype,spread", [(BF, 1e3), (BF, 2e4), (BF, 1e6), (BF, 1e15), (HF, 1e3), (HF, 8e3), (HF, 1.3e4)])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_far_scores(dev, case, dtype, spread):
    nq, nk, N, Hq, Hk, Dh = FAR[case]
    g = KV.gen(dev, case)
    x = torch.randn(len(nq), N, 2, Hk, Dh, generator=g, device=dev)
    x[:, :, 0] = x[:, :, 0].clamp(-4, 4) * spread
    x = x.to(dtype)
    q = (torch.randn(sum(nq), Hq, Dh, generator=g, device=dev).clamp(-4, 4) * spread).to(dtype)
    cu, kl = offsets(dev, nq, nk)
    out = K.packed_attention(q, x[:, :, 0], x[:, :, 1], cu, kl, Dh ** -0.5, causal=True)
    assert check_far(out, q, x.double(), nq, nk, Dh ** -0.5) > 0.9


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,size", [*((BF, x) for x in (1.0, 30.0, 80.0, 2e3, 2e4, 1e6, 1e12)),
                                        *((HF, x) for x in (30.0, 80.0, 2e3, 2e4))])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_equal_keys_weigh_the_same(dev, case, dtype, size, causal):
    nq, nk, N, Hq, Hk, Dh = FAR[case]
    B, g = len(nq), KV.gen(dev, case)
    x = torch.randn(B, N, 2, Hk, Dh, generator=g, device=dev) + 1
    x[:, :, 0] = torch.randn(Hk, Dh, generator=g, device=dev).clamp(-3, 3) * size
    x = x.to(dtype)
    q = (torch.randn(sum(nq), Hq, Dh, generator=g, device=dev).clamp(-3, 3) * size).to(dtype)
    cu, kl = offsets(dev, nq, nk)
    out = K.packed_attention(q, x[:, :, 0], x[:, :, 1], cu, kl, 0.5, causal=causal).view(*q.shape)
    assert torch.isfinite(out).all()
    for rows, h, _, _, v, hidden in rows_of(q, x.double(), nq, nk):
        w = (~hidden if causal else torch.ones_like(hidden)).double()
        mean, mag = (w @ v) / w.sum(-1, keepdim=True), (w @ v.abs()) / w.sum(-1, keepdim=True)
        tol = (v.shape[0] / 32 + 40) * 2.0 ** -24 * (mag + mean.abs())
        assert ((out[rows, h].double() - mean).abs() <= tol + KV.half_step(dtype) * (mean.abs() + tol)).all()
