"""Packed sequences at the limits of their buffers: offsets that fall, lengths past the row buffer, the cache or the key
rows, groups as large as a tile, value rows that overlap, heads at the ends of the type's range."""

import math

import pytest
import torch

from appcorr_amd import _lib
from appcorr_amd import kernels as K
from tests.test_gpu_packed import BF, HF, attention64, gen, near

pytestmark = pytest.mark.gpu


def test_falling_offsets_leave_the_merge_inside_its_workspace(dev):
    """Offsets that rise and fall make 119 items of a key head where rows and sequences that follow one another make
    79 at the most. What lies behind the workspace, and what nothing wrote in it, is NaN."""
    rows, Hk, Dh, cap = 1, 2, 128, 20000
    cu = [1, 1, 1, 1, 1, 0, 0, 1, 0, 0, 1, 0, 1, 0, 0, 1, 1, 0, 1, 1, 1]
    cu_k = [0, 20000, 20000, 20000, 0, 0, 0, 20000, 0, 20000, 20000, 0, 20000, 0, 0, 0, 0, 0, 20000, 0, 0]
    S = len(cu) - 1
    g = gen(dev, 60)
    q = torch.randn(rows, Hk, Dh, generator=g, device=dev).to(BF)
    k = torch.randn(cap, Hk, Dh, generator=g, device=dev).to(BF)
    cu, cu_k = (torch.tensor(c, device=dev, dtype=torch.int32) for c in (cu, cu_k))
    need = _lib.load().oudjat_packed_attention_workspace_elems(rows, S, Hk, Hk, Dh, cap)
    ws = torch.full((3 * need,), math.nan, device=dev)
    out = torch.full((rows + 2, Hk * Dh), 5.0, device=dev, dtype=BF)
    _lib.call("oudjat_packed_attention", q.data_ptr(), Hk * Dh, Dh, rows, Hk, Dh, k.data_ptr(), 0, Hk * Dh, Dh,
              k.data_ptr(), 0, Hk * Dh, Dh, Hk, cap, 0, cu.data_ptr(), 0, cu_k.data_ptr(), 0, S, 0.1, 1, _lib.DTYPE_BF16,
              out[1].data_ptr(), Hk * Dh, ws.data_ptr(), need, _lib.stream_of(q))
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and (out[0] == 5).all() and (out[-1] == 5).all()
    assert torch.isnan(ws[need:]).all()
