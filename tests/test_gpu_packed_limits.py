"""Packed sequences at the limits of their buffers: offsets that fall, lengths past the row buffer, the cache or the key
rows, groups as large as a tile, value rows that overlap, heads at the ends of the type's range."""

import math
import random

import pytest
import torch

from appcorr_amd import _lib
from appcorr_amd import kernels as K
from tests.test_gpu_packed import (BF, HF, angles64, attention64, gen, near, norm64, norm_case, packed_case,
                                   rotate64)

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


def plan_reference(q_lens, k_lens, rows, cache_len, key_rows):
    """Token by token: row i of a sequence is token k - q + i; rows past the buffer are not there, nor are their tokens."""
    cu_q, nk, cu_k, batch, token = [0], [], [0], [], []
    for s, (a, b) in enumerate(zip(q_lens, k_lens)):
        a, b = max(a, 0), max(b, 0)
        kept = min(a, rows - len(batch))
        n = max(0, b - (a - kept))
        fits = cache_len is not None or cu_k[-1] + n <= key_rows and (not nk or nk[-1] is not None)
        cap = key_rows if cache_len is None else cache_len
        for t in range(b - a, b - a + kept):
            there = fits and 0 <= t < cap
            batch.append(s if there else -1)
            token.append(t if there else -1)
        cu_q.append(len(batch))
        nk.append(min(n, (1 << 31) - 1) if fits else None)
        cu_k.append(cu_k[-1] + (min(n, cap) if fits else 0))
    pad = [-1] * (rows - len(batch))
    return cu_q, [n or 0 for n in nk], cu_k, batch + pad, token + pad


def check_plan(dev, q_lens, k_lens, rows, want=None, dtype=torch.int64, **cap):
    p = K.packed_plan(torch.tensor(q_lens, dtype=dtype, device=dev), torch.tensor(k_lens, dtype=dtype, device=dev), rows,
                      **cap)
    ref = plan_reference(q_lens, k_lens, rows, cap.get("cache_len"), cap.get("key_rows"))
    for i, name in enumerate(("cu_q", "k_lens", "cu_k", "batch_idx", "token_idx")):
        got = getattr(p, name).tolist()
        assert got == ref[i], name
        assert want is None or got == want[i], name


@pytest.mark.parametrize("q_lens,k_lens,rows,cap,want", [
    # The row buffer ends inside the third sequence: its first row is its token 5, and 5 earlier tokens are its keys.
    ([3, 4, 5], [10, 10, 10], 8, dict(cache_len=50),
     ([0, 3, 7, 8], [10, 10, 6], [0, 10, 20, 26], [0, 0, 0, 1, 1, 1, 1, 2], [7, 8, 9, 6, 7, 8, 9, 5])),
    # The second one's rows are all left out: what was cached of it stays.
    ([4, 3, 0], [4, 9, 2], 4, dict(cache_len=50), ([0, 4, 4, 4], [4, 6, 2], [0, 4, 10, 12], [0] * 4, [0, 1, 2, 3])),
    # Tokens 50 .. 53 of a cache of 50, and 48 .. 51: only the first two have a slot.
    ([4, 4], [54, 52], 8, dict(cache_len=50), ([0, 4, 8], [54, 52], [0, 50, 100], [-1] * 4 + [1, 1, -1, -1],
                                               [-1] * 4 + [48, 49, -1, -1])),
    # Both: of 9 new rows, tokens 45 .. 53, the buffer has 7.
    ([9], [54], 7, dict(cache_len=50), ([0, 7], [52], [0, 50], [0] * 5 + [-1] * 2, [45, 46, 47, 48, 49, -1, -1])),
    # Packed keys, rows cut: prompts of 3, 4 and 5 rows in buffers of 8.
    ([3, 4, 5], [3, 4, 5], 8, dict(key_rows=8), ([0, 3, 7, 8], [3, 4, 1], [0, 3, 7, 8], [0] * 3 + [1] * 4 + [2],
                                                 [0, 1, 2, 0, 1, 2, 3, 0])),
    # Packed keys, too few key rows for the second sequence and so for all behind it.
    ([2, 2, 1], [4, 7, 1], 5, dict(key_rows=10), ([0, 2, 4, 5], [4, 0, 0], [0, 4, 4, 4], [0, 0, -1, -1, -1],
                                                  [2, 3, -1, -1, -1])),
    # Lengths past 31 and 32 bits.
    ([1 << 40, 5], [1 << 40, 9], 3, dict(cache_len=20), ([0, 3, 3], [3, 4], [0, 3, 7], [0] * 3, [0, 1, 2])),
    ([2, 2], [(1 << 40) + 1, 2], 4, dict(cache_len=20), ([0, 2, 4], [(1 << 31) - 1, 2], [0, 20, 22], [-1, -1, 1, 1],
                                                       [-1, -1, 0, 1])),
    ([3, 1], [(1 << 31) - 1, 1], 4, dict(cache_len=(1 << 31) - 2),
     ([0, 3, 4], [(1 << 31) - 1, 1], [0, (1 << 31) - 2, (1 << 31) - 1], [0, 0, -1, 1],
      [(1 << 31) - 4, (1 << 31) - 3, -1, 0])),
    ([1 << 62], [1], 2, dict(cache_len=20), ([0, 2], [0], [0, 0], [-1, -1], [-1, -1])),
])
def test_plan_of_lengths_past_the_buffers(dev, q_lens, k_lens, rows, cap, want):
    check_plan(dev, q_lens, k_lens, rows, want, **cap)
    if max(q_lens + k_lens) < 1 << 31:
        check_plan(dev, q_lens, k_lens, rows, want, dtype=torch.int32, **cap)


@pytest.mark.parametrize("S", [1, 2, 7, 64, 65, 256, 257, 1000, 2048, 2049, 4096])
def test_plan_of_many_sequences_past_the_buffers(dev, S):
    rng = random.Random(S)
    q = [rng.choice([-1, 0, 1, rng.randrange(40)]) for _ in range(S)]
    k = [max(a, 0) + rng.randrange(-3, 100) for a in q]
    for rows in (sum(max(a, 0) for a in q) + 5, sum(max(a, 0) for a in q) // 3):
        check_plan(dev, q, k, rows, cache_len=90)
        check_plan(dev, q, k, rows, cache_len=1000)
        check_plan(dev, q, k, rows, key_rows=sum(max(b, 0) for b in k) // 2)
        check_plan(dev, q, k, rows, key_rows=sum(max(b, 0) for b in k))
        check_plan(dev, q, k, rows, key_rows=0)


@pytest.mark.parametrize("rows,N,key_rows", [(9, 50, None), (40, 50, None), (23, 30, None), (26, None, 90), (12, None, 60)])
def test_layer_of_sequences_past_the_buffers(dev, rows, N, key_rows):
    """Plan, rotation with the K/V write and attention of sequences that do not fit: every row meets the keys of its own
    past that are there, at their own tokens, and what was cached before stays."""
    Hq, Hk, Dh, g = 4, 2, 64, gen(dev, 65)
    new, total = [6, 1, 11, 8], [25, 31, 34, 20]
    plan = K.packed_plan(torch.tensor(new, device=dev), torch.tensor(total, device=dev), rows, cache_len=N,
                         key_rows=key_rows)
    qkv = torch.randn(rows, Hq + 2 * Hk, Dh, generator=g, device=dev).to(BF)
    q = torch.zeros(rows, Hq, Dh, device=dev, dtype=BF)
    pos = torch.zeros(rows, 1, device=dev, dtype=torch.int64)  # no rotation: keys are only normed
    freq = torch.ones(32, device=dev)
    n = N or max(total)
    old = torch.randn(4, n, 2, Hk, Dh, generator=g, device=dev).to(BF)
    kv = old.clone()
    K.qk_norm_rope_kv(qkv, Hq, Hk, (None, None), (None, None), 1e-6, pos, freq, (32,), plan.batch_idx, plan.token_idx,
                      kv, q)
    if N:
        got = K.packed_attention(q, kv[:, :, 0], kv[:, :, 1], plan.cu_q, plan.k_lens, Dh ** -0.5, causal=True)
    else:
        ck = plan.cu_k.tolist()
        flat = torch.cat([kv[s, :ck[s + 1] - ck[s]] for s in range(4)] + [torch.full_like(kv[0, :1], math.nan)])
        got = K.packed_attention(q, flat[:, 0], flat[:, 1], plan.cu_q, plan.cu_k, Dh ** -0.5, causal=True)
    normed = qkv[:, Hq:Hq + Hk].double()
    normed = normed / (normed.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
    r, room = 0, key_rows
    for s, (a, b) in enumerate(zip(new, total)):
        kept = min(a, rows - r)
        if room is not None:
            room -= b - a + kept
        fits = room is None or room >= 0
        for i in range(kept):
            t = b - a + i
            if fits and t < n:  # the row's own key and value lie at its token
                assert (kv[s, t, 0].double() - normed[r]).abs().max() <= 2.0 ** -7 * normed[r].abs().max()
                assert torch.equal(kv[s, t, 1], qkv[r, Hq + Hk:])
            seen = min(t + 1, n) if fits else 0
            ref, slack = attention64(q[r:r + 1], kv[s, :seen, 0], kv[s, :seen, 1], 1, seen, Dh ** -0.5, True)
            if fits and t < n:
                near(got[r:r + 1].view(1, Hq, Dh), ref, slack, f"sequence {s} row {i}")
            elif not fits:
                assert not got[r].any()
            r += 1
        assert torch.equal(kv[s, :min(n, b - a)], old[s, :min(n, b - a)]), "tokens cached before were written"


@pytest.mark.parametrize("Hq,Hk,Dh", [(2, 1, 64), (3, 2, 128)])
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -120, 1e-6, 2.0 ** 127])
def test_norm_of_heads_at_the_ends_of_the_range(dev, Hq, Hk, Dh, layer, eps):
    """Heads whose sums or squares pass fp32's largest value, or whose squares are below its smallest: bf16's largest
    values, its subnormals, both in one head. The bound is the norm's own (1e-6 + 30 * 2^-24 of the value's size, then
    half a step of 2^-8), and 2^-134 more: below 2^-126 bf16 values are 2^-133 apart, so that rounding one is off by up
    to 2^-134 whatever its size, and eps = 1e-6 leaves the smallest heads there."""
    qkv, qn, kn, pos, freq, sections, bi, ti, kv, q_out = norm_case(dev, 24, Hq, Hk, Dh, BF, layer, True, seed=66)
    x = qkv.float()
    sizes = [1e18, 1e19, 3e19, 1e25, 1e30, 5e37, 1e38] + [2.0 ** -e for e in (40, 50, 62, 70, 100, 126)]
    for i, size in enumerate(sizes):
        x[i] *= size
    top = torch.finfo(BF).max
    x[13] = torch.where(x[13] > 0, top, -top)
    x[14] = torch.where(x[14] > 0, top, top / 2)     # (a sum past the range)
    x[15, :, ::2] *= 1e30                            # half of the head negligible
    x[16, :, 1] = 2.0 ** 120
    x[17, :, 1:] *= 2.0 ** -110
    x[18] = torch.where(x[18] > 0, 1.0, -1.0) * 2.0 ** -133
    x = x.clamp(-top, top).to(BF)
    K.qk_norm_rope_kv(x, Hq, Hk, qn, kn, eps, pos, freq, sections, bi, ti, kv, q_out, layer_norm=layer)
    angle = angles64(pos, freq, sections)
    half = angle.shape[1]
    for got, heads, weights in ((q_out, x[:, :Hq], qn), (kv[bi, ti, 0], x[:, Hq:Hq + Hk], kn)):
        y, size = norm64(heads, *weights, eps, layer)
        ref, _ = rotate64(y, angle)
        pair = size[..., :half] + size[..., half:2 * half]
        slack = (1e-6 + 30 * 2.0 ** -24) * torch.cat([pair, pair, size[..., 2 * half:]], -1)
        assert torch.isfinite(got).all()
        assert ((got.double() - ref).abs() <= slack + 2.0 ** -8 * (ref.abs() + slack) + 2.0 ** -134).all()


def test_norm_of_heads_that_are_not_finite(dev):
    """As the formula has it: an infinite value makes its own quotient NaN and the others 0, a NaN all of them."""
    qkv, qn, kn, _, freq, sections, bi, ti, kv, q_out = norm_case(dev, 4, 1, 1, 64, BF, False, False, seed=67)
    pos = torch.zeros(4, len(sections), device=dev, dtype=torch.int64)
    qkv[0, 0, 3] = math.inf
    qkv[1, 0, 9] = -math.inf
    qkv[2, 0, 11] = math.nan
    qkv[3] = 0
    K.qk_norm_rope_kv(qkv, 1, 1, qn, kn, 0.0, pos, freq, sections, bi, ti, kv, q_out)
    y = q_out[:, 0].float()
    assert y[0].isnan().sum() == 2 and y[0, 3].isnan() and y[1].isnan().sum() == 2 and y[1, 9].isnan()
    assert (y[:2].nan_to_num() == 0).all() and y[2:].isnan().all()


def test_probed_sites_of_packed_sequences_are_their_own(dev):
    """The sites of the rectangular pass ("attention", "qkv_post") do not time the packed operators."""
    qkv, qn, kn, pos, freq, sections, bi, ti, kv, q_out = norm_case(dev, 6, 2, 1, 64, BF, False, True)
    cu = torch.tensor([0, 6], device=dev)

    def layer():
        K.packed_plan(cu[1:], cu[1:], 6, cache_len=9)
        K.apply_rope_axes(qkv[:, :2], qkv[:, 2:3], pos, freq, sections)
        K.qk_norm_rope_kv(qkv, 2, 1, qn, kn, 1e-6, pos, freq, sections, bi, ti, kv, q_out)
        K.packed_attention(q_out, kv[:1, :, 0], kv[:1, :, 1], cu, cu[1:], 0.1, causal=True)

    own = ("packed_plan", "rope_axes", "qk_norm_rope_kv", "packed_attention")
    try:
        for tags, want in ((("attention", "qkv_post"), {}), (own, {t: 1 for t in own})):
            K.set_probe(tags)
            layer()
            assert {t: len(e) for t, e in K.probe_events().items()} == want
    finally:
        K.set_probe(None)
