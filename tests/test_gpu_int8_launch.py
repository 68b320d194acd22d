"""linear_int8 where the tile that would be fastest has more workgroups than a launch holds: larger ones do it."""

import pytest
import torch

from appcorr_amd import kernels as K
from tests import test_gpu_int8 as I8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,Kd", [(1 << 27, 16, 64), ((1 << 30) - 1, 8, 128)])
def test_more_rows_than_small_tiles_hold(dev, M, N, Kd):
    """One row of codes for all (stride 0), a scale for each: rows from both ends and from the middle."""
    g = I8.gen(dev, N)
    x8 = torch.randint(-127, 128, (1, Kd), generator=g, device=dev, dtype=torch.int8).expand(M, Kd)
    w8 = torch.randint(-127, 128, (N, Kd), generator=g, device=dev, dtype=torch.int8)
    sx, sw = torch.rand(M, generator=g, device=dev), torch.rand(N, generator=g, device=dev)
    out = K.linear_int8(x8, sx, w8, sw)
    rows = torch.cat([torch.arange(300, device=dev), torch.randint(0, M, (2000,), generator=g, device=dev),
                      torch.arange(M - 300, M, device=dev)])
    I8.check(out[rows], *I8.product64(x8[rows], sx[rows], w8, sw, None, None, None, "bias"))
