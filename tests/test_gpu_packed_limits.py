"""Packed sequences at the limits of their buffers: offsets that fall, lengths past the row buffer, the cache or the key
rows, groups as large as a tile, value rows that overlap, heads at the ends of the type's range."""

import math

import pytest
import torch

from appcorr_amd import _lib
from appcorr_amd import kernels as K
from tests.test_gpu_packed import BF, HF, attention64, gen, near, packed_case

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


@pytest.mark.parametrize("m,n,Hq,Hk", [([2], [100], 16, 1), ([2], [100], 32, 2), ([3, 1], [70, 33], 16, 1),
                                       ([2, 0], [41, 9], 32, 1), ([1, 1, 2], [5, 64, 2500], 16, 1), ([2, 0], [2601, 9], 32, 1),
                                       ([2, 1], [3001, 2500], 16, 1)])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_values_of_a_group_that_fills_the_tile(dev, m, n, Hq, Hk, Dh, bad):
    """16 or 32 query heads of a key head, so that a tile of 16 rows is one token: the last token's value is not finite,
    and the tokens before it do not see it. The keys of the longer ones are split."""
    for dtype in (BF, HF):
        q, k, v, cu, keys = packed_case(dev, m, n, Hq, Hk, Dh, dtype, True, 61)
        v = v.clone()
        for s, b in enumerate(n):
            v[s, b - 1:] = bad
        got = K.packed_attention(q, k, v, cu, keys, Dh ** -0.5, causal=True).view(-1, Hq, Dh)
        at = 0
        for s, (a, b) in enumerate(zip(m, n)):
            if a:
                ref, slack = attention64(q[at:at + a - 1], k[s, :b - 1], v[s, :b - 1], a - 1, b - 1, Dh ** -0.5, True)
                near(got[at:at + a - 1], ref, slack, f"{dtype} sequence {s}")
                last = got[at + a - 1]
                assert (last.isnan() if math.isnan(bad) else last == bad).all()
            at += a


@pytest.mark.parametrize("m,Dh", [(1, 64), (1, 128), (100, 64), (40, 128), (300, 128)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_closer_than_a_row(dev, m, Dh, causal, bad):
    """A cache of one token, one value for every key and value rows that overlap: an infinite value that a row sees is
    that infinity in its dim, not NaN by meeting the weight 0 of keys past the last."""
    g = gen(dev, 62)
    for dtype in (BF, HF):
        q = torch.randn(m, 2, Dh, generator=g, device=dev).to(dtype)
        cu = torch.tensor([0, m], device=dev)
        k = torch.randn(1, 70, 2, Dh, generator=g, device=dev).to(dtype)
        one = torch.randn(1, 1, 2, Dh, generator=g, device=dev).to(dtype)
        overlapping = torch.randn(8 * 69 + 2 * Dh, generator=g, device=dev).to(dtype)
        one.view(-1)[1] = overlapping[8 * 69 + Dh - 1] = bad
        for n, v in ((1, one), (70, one.expand(1, 70, 2, Dh)),
                     (70, overlapping.as_strided((1, 70, 2, Dh), (0, 8, Dh, 1)))):
            keys = torch.tensor([n], device=dev)
            got = K.packed_attention(q, k[:, :n], v, cu, keys, Dh ** -0.5, causal=causal).view(m, 2, Dh)
            p = torch.ones(m, n, dtype=torch.bool, device=dev)
            if causal:
                p = torch.arange(n, device=dev) <= torch.arange(m, device=dev)[:, None] + n - m
            met = (p.double() @ (~torch.isfinite(v[0])).double().reshape(n, -1)).view(m, 2, Dh) > 0
            assert met.any()
            assert (got[met].isnan() if math.isnan(bad) else got[met] == bad).all()
            assert torch.isfinite(got[~met]).all()
