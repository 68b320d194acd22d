"""NVFP4 writes with tensor scales whose significand is all ones, 2^j (1 - 2^-24): the correctly rounded reciprocal of such a
number is not what a Newton step arrives at, and a quotient by the wrong one is off where a value lies on a border between
codes, or a block's largest on one between scales. Codes and scales bit for bit as by IEEE division."""

import numpy as np
import pytest
import torch

from appcorr_amd import kernels as K
from tests import test_gpu_nvfp4_kv as KV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ones", [True, False])
def test_write_by_tensor_scales_hard_to_invert(dev, dtype, ones):
    js = np.arange(-6, 6)
    Hk = len(js)
    ts = (np.float32(1 - 2.0 ** -24) if ones else np.float32(1 + 2.0 ** -23)) * np.float32(2.0) ** js.astype(np.float32)
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    near = [[6.0, *borders, *-borders, 0.5]]  # the unit is all ones too: values on the borders
    near += [[6.0, *borders * np.float32(1 + d), *-borders, 1.0] for d in (2.0 ** -7, -2.0 ** -7, 2.0 ** -8)]
    # largest values whose sixth is half way between two scales, for all mantissas
    near += [[6.0 * (1 + (2 * i + 1) / 16), *borders * np.float32(1 + i / 8), *-borders, 2.0] for i in range(8)]
    x = np.array(near, np.float32)
    rows = len(x) // 4
    x = x.reshape(rows, 1, 64) * np.float32(2.0) ** js.astype(np.float32)[None, :, None]
    k = torch.from_numpy(x.astype(np.float32)).to(dev).to(dtype)
    v = -k.flip(0)
    cache = K.kv_nvfp4_cache(1, rows, Hk, 64, dev, tensor_scale=torch.from_numpy(np.stack([ts, ts])).to(dev))
    i = torch.arange(rows, device=dev)
    K.kv_nvfp4_write(k, v, i * 0, i, cache)
    both = torch.stack([k, v], 1).float().cpu().numpy().reshape(rows, 2, Hk, 4, 16)
    codes, s8 = KV.quantized(both, np.broadcast_to(ts[None, None, :, None], both.shape[:-1]))
    codes = codes.reshape(rows, 2, Hk, 64)
    assert torch.equal(cache.scales.view(torch.uint8)[0].cpu(), torch.from_numpy(s8))
    assert torch.equal(cache.codes[0].cpu(), torch.from_numpy(codes[..., 0::2] | codes[..., 1::2] << 4))
