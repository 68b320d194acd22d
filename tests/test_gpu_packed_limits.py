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


def edge_reference(q, k, v, first, end, k0, k1, scale):
    """(out, slack) of the rows `first` .. `end` of a buffer, a sequence whose last row is end - 1 and whose keys are rows
    k0 .. k1 - 1 of a key buffer, causal: row r sees the key rows up to k1 - end + r. What lies outside a buffer is
    not there."""
    rows = range(max(0, first), min(end, q.shape[0]))
    outs = []
    for r in rows:
        lo, hi = max(0, k0), min(k.shape[0], k1 - end + r + 1)
        outs.append(attention64(q[r:r + 1], k[lo:max(lo, hi)], v[lo:max(lo, hi)], 1, max(0, hi - lo), scale, True))
    return rows, torch.cat([o for o, _ in outs]), torch.cat([s for _, s in outs])


@pytest.mark.parametrize("m,n,N,Hq,Hk,Dh", [
    ([4], [54], 50, 2, 2, 64), ([10, 1, 3], [54, 51, 40], 50, 4, 1, 128), ([70], [130], 100, 8, 2, 64),
    ([300, 2], [500, 90], 299, 4, 1, 128), ([5, 1], [2601, 1 << 40], 2500, 8, 1, 64), ([200], [4000], 3900, 2, 1, 128),
    ([90], [70], 64, 2, 1, 64), ([1] * 70, [40 + i for i in range(70)], 60, 2, 2, 64), ([9], [1 << 40], 33, 2, 2, 64)])
def test_causal_edge_of_sequences_longer_than_their_cache(dev, m, n, N, Hq, Hk, Dh):
    """Row i of m sees the keys up to its own token n - m + i, as far as the cache holds them."""
    for dtype in (BF, HF):
        q, k, v, cu, _ = packed_case(dev, m, [N] * len(m), Hq, Hk, Dh, dtype, True, 63)
        k, v = k[:, :N], v[:, :N]
        got = K.packed_attention(q, k, v, cu, torch.tensor(n, device=dev), Dh ** -0.5, causal=True).view(-1, Hq, Dh)
        at = 0
        for s, (a, b) in enumerate(zip(m, n)):
            rows, ref, slack = edge_reference(q, k[s], v[s], at, at + a, 0, b, Dh ** -0.5)
            near(got[rows.start:rows.stop], ref, slack, f"{dtype} sequence {s}")
            at += a


@pytest.mark.parametrize("cu,cu_k,M,Mk,Hq,Hk,Dh", [
    ([0, 3, 7, 12], [0, 10, 20, 30], 8, 30, 2, 2, 64), ([0, 60, 500], [0, 100, 2300], 200, 1500, 4, 2, 64),
    ([-5, 20, 45], [-4, 30, 70], 40, 60, 4, 1, 128), ([0, 2, 3], [0, 3000, 1 << 40], 3, 3500, 8, 1, 128),
    ([-(1 << 40), 5], [0, 20], 10, 20, 2, 1, 64), ([0, 700], [-300, 500], 400, 450, 2, 1, 128),
    (list(range(0, 140, 2)), list(range(0, 1400, 20)), 101, 1111, 2, 2, 64)])
def test_causal_edge_of_offsets_outside_the_buffers(dev, cu, cu_k, M, Mk, Hq, Hk, Dh):
    g = gen(dev, 64)
    for dtype in (BF, HF):
        q = torch.randn(M, Hq, Dh, generator=g, device=dev).to(dtype)
        kv = torch.randn(Mk, 2, Hk, Dh, generator=g, device=dev).to(dtype)
        k, v = kv[:, 0], kv[:, 1]
        out = torch.full((M, Hq * Dh), 5.0, device=dev, dtype=dtype)
        K.packed_attention(q, k, v, torch.tensor(cu, device=dev), torch.tensor(cu_k, device=dev), Dh ** -0.5, causal=True,
                           out=out)
        for s in range(len(cu) - 1):
            if max(cu[s], 0) >= min(cu[s + 1], M):
                continue
            rows, ref, slack = edge_reference(q, k, v, cu[s], cu[s + 1], cu_k[s], cu_k[s + 1], Dh ** -0.5)
            near(out.view(M, Hq, Dh)[rows.start:rows.stop], ref, slack, f"{dtype} sequence {s}")
        assert (out[min(cu[-1], M):] == 5.0).all()
