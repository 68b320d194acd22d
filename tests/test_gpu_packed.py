"""Packed sequences of different lengths: plan, rotation by positions, normed heads with the K/V write and grouped
attention, each against its formula in 64 bits, and the four together as a layer uses them.

Tolerances: a rounding to the type is off by at most u = finfo.eps / 2 of the value. The rotation's sines and cosines
are within 5e-7 (reduced angle 2^-25 turns, the sine's own 2 ulp) and its products and sum add three fp32 roundings,
so before the last rounding a rotated value is within 1e-6 (|a| + |b|); the norms' sums of Dh <= 128 fp32 values (20
in a row) and their root, quotient and products stay within 30 * 2^-24 of |x| + mean|x| in units of the normed value.
Attention: probabilities rounded to the type on both sides of the quotient, 2 u sum(p |v|), beside the scores' fp32
sums, (Dh + 8) 2^-24 scale sum|q||k| each way in the exponent, and 2^-25 per key where fp16 probabilities are
subnormal (the largest is at least 1)."""

import math
import random

import pytest
import torch

from appcorr_amd import graphs
from appcorr_amd import kernels as K

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, ref, slack, what=""):
    """|got - ref| <= slack + u (|ref| + slack), elementwise, in 64 bits; fp16 subnormals are 2^-24 apart."""
    u = half_step(got.dtype)
    d = (got.double() - ref).abs()
    lim = slack + u * (ref.abs() + slack) + (2.0 ** -25 if got.dtype == HF else 0.0)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = d > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / lim).max()):.3g} of the bound"


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


# ------------------------------------------------------------------------------------------------
# packed_plan
# ------------------------------------------------------------------------------------------------


def plan_reference(q_lens, k_lens, rows, cache_len, key_rows):
    cu_q, cu_k, nk, batch, token = [0], [0], [], [], []
    for s, (a, b) in enumerate(zip(q_lens, k_lens)):
        a, b = max(a, 0), max(b, 0)
        b = min(b, cache_len) if cache_len is not None else min(b, key_rows - cu_k[-1])
        a = min(a, rows - cu_q[-1])
        cu_q.append(cu_q[-1] + a)
        cu_k.append(cu_k[-1] + b)
        nk.append(b)
        for t in range(b - a, b):
            batch.append(s if t >= 0 else -1)
            token.append(t if t >= 0 else -1)
    pad = [-1] * (rows - len(batch))
    return cu_q, nk, cu_k, batch + pad, token + pad


def check_plan(dev, q_lens, k_lens, rows, cache_len=None, key_rows=None, dtype=torch.int64):
    p = K.packed_plan(torch.tensor(q_lens, dtype=dtype, device=dev), torch.tensor(k_lens, dtype=dtype, device=dev), rows,
                      cache_len=cache_len, key_rows=key_rows)
    ref = plan_reference(q_lens, k_lens, rows, cache_len, key_rows)
    for name, want in zip(("cu_q", "k_lens", "cu_k", "batch_idx", "token_idx"), ref):
        assert getattr(p, name).tolist() == want, name


@pytest.mark.parametrize("q_lens,k_lens,rows", [
    ([1], [1], 1), ([0], [0], 0), ([], [], 3), ([5], [9], 7), ([0, 3, 0, 2, 0], [4, 3, 0, 7, 5], 9),
    ([3, 4], [1, 2], 7),             # fewer keys than rows: the first have no token
    ([3, 4, 5], [10, 10, 10], 8),    # more rows than the buffer has
    ([-2, 4, -1], [3, -5, 8], 6),    # lengths below zero
    ([2, 2], [100, 100], 4),         # more keys than the cache has
])
def test_plan(dev, q_lens, k_lens, rows):
    for dtype in (torch.int32, torch.int64):
        check_plan(dev, q_lens, k_lens, rows, cache_len=50, dtype=dtype)
        check_plan(dev, q_lens, k_lens, rows, key_rows=13, dtype=dtype)
        check_plan(dev, q_lens, k_lens, rows, key_rows=0, dtype=dtype)


@pytest.mark.parametrize("S", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 4096])
def test_plan_many_sequences(dev, S):
    rng = random.Random(S)
    q = [rng.randrange(0, 40) for _ in range(S)]
    k = [a + rng.randrange(0, 100) for a in q]
    check_plan(dev, q, k, sum(q) + 5, cache_len=90)
    check_plan(dev, q, k, max(1, sum(q) - 3), key_rows=sum(k) // 2)


def test_plan_saturates(dev):
    """Lengths whose sum passes 32 and whose values pass 31 bits."""
    big = [1 << 40, 1 << 33, 5]
    check_plan(dev, big, big, 9, cache_len=20)
    check_plan(dev, [2, 3, 4], [(1 << 31) - 2] * 3, 9, cache_len=(1 << 31) - 2)


# ------------------------------------------------------------------------------------------------
# apply_rope_axes
# ------------------------------------------------------------------------------------------------


def angles64(positions, inv_freq, sections):
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    return positions.double()[:, axis] * inv_freq.double()


def rotate64(x, angle):
    """(rotated, |a| + |b| of each value's pair)."""
    half = angle.shape[1]
    x = x.double()
    a, b = x[..., :half], x[..., half:2 * half]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    size = a.abs() + b.abs()
    rest = x[..., 2 * half:]
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1), torch.cat([size, size, 0 * rest], -1)


def positions_of(kind, rows, axes, dev, g, top=1 << 20):
    if kind == torch.float32:
        return torch.rand(rows, axes, generator=g, device=dev) * 2 - 1
    return torch.randint(-5, top, (rows, axes), generator=g, device=dev).to(kind)


ROPE = [  # rows, Hq, Hk, Dh, sections
    (1, 1, 1, 64, (32,)), (3, 6, 6, 64, (16, 16)), (201, 16, 4, 64, (8, 12, 12)), (5, 32, 8, 128, (16, 24, 24)),
    (2, 3, 0, 128, (32,)), (7, 0, 2, 128, (4, 2, 0, 2)), (1030, 2, 1, 96, (8, 8)), (1025, 5, 5, 16, (8,)),
    (1500, 4, 1, 512, (128, 128)),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("rows,Hq,Hk,Dh,sections", ROPE)
def test_rope(dev, rows, Hq, Hk, Dh, sections, kind, dtype):
    g = gen(dev, rows + Dh)
    q = torch.randn(rows, Hq, Dh, generator=g, device=dev).to(dtype)
    k = torch.randn(rows, Hk, Dh, generator=g, device=dev).to(dtype)
    pos = positions_of(kind, rows, len(sections), dev, g)
    freq = (1000.0 ** -torch.rand(sum(sections), generator=g, device=dev)).float()
    got = K.apply_rope_axes(q, k, pos, freq, sections)
    angle = angles64(pos, freq, sections)
    for o, x in zip(got, (q, k)):
        ref, size = rotate64(x, angle)
        assert o.shape == x.shape and o.is_contiguous()
        near(o, ref, 1e-6 * size, f"rope {kind}")


def test_rope_views_and_in_place(dev):
    """q and k inside qkv rows, positions transposed and broadcast, results in place: what lies beside stays."""
    g = gen(dev, 3)
    qkv = torch.randn(70, 12, 64, generator=g, device=dev).to(BF)
    before = qkv.clone()
    q, k = qkv[:, :6], qkv[:, 6:9]
    pos = torch.randint(0, 99, (2, 70), generator=g, device=dev).t()
    freq = torch.rand(32, generator=g, device=dev)
    want = K.apply_rope_axes(q, k, pos, freq, (16, 16))
    assert torch.equal(qkv, before)
    got = K.apply_rope_axes(q, k, pos, freq, (16, 16), out=(q, k))
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 9:], before[:, 9:])
    one = pos[:1].expand(70, 2)
    q2, k2 = before[:, :6], before[:, 6:9]
    a = K.apply_rope_axes(q2, k2, one, freq, (16, 16))
    b = K.apply_rope_axes(q2, k2, one.contiguous(), freq, (16, 16))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_rope_position_zero_is_identity_and_far_positions(dev):
    g = gen(dev, 4)
    x = torch.randn(4, 2, 64, generator=g, device=dev).to(BF)
    freq = torch.ones(32, device=dev)
    z = K.apply_rope_axes(x, x, torch.zeros(4, 1, device=dev, dtype=torch.int64), freq, (32,))
    assert torch.equal(z[0], x) and torch.equal(z[1], x)
    far = torch.tensor([[0], [1 << 24], [(1 << 31) - 1], [-(1 << 31)]], device=dev)
    ref, size = rotate64(x, angles64(far, freq, (32,)))
    near(K.apply_rope_axes(x, x, far, freq, (32,))[0], ref, 1e-6 * size, "far")


def test_rope_empty(dev):
    x = torch.empty(0, 4, 64, device=dev, dtype=BF)
    a, b = K.apply_rope_axes(x, x, torch.empty(0, 1, device=dev), torch.ones(32, device=dev), (32,))
    assert a.shape == b.shape == x.shape


# ------------------------------------------------------------------------------------------------
# qk_norm_rope_kv
# ------------------------------------------------------------------------------------------------


def norm64(x, w, b, eps, layer):
    """(normed, size of the values whose roundings it carries)."""
    x = x.double()
    mean_abs = x.abs().mean(-1, keepdim=True)
    size = x.abs() + (mean_abs if layer else 0)
    if layer:
        x = x - x.mean(-1, keepdim=True)
    inv = 1 / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    w = 1.0 if w is None else w.double()
    y = x * inv * w
    size = size * inv * (w.abs() if torch.is_tensor(w) else w)
    if b is not None:
        y = y + b.double()
        size = size + b.double().abs()
    return y, size


def norm_case(dev, rows, Hq, Hk, Dh, dtype, layer, weights, kind=torch.int64, sections=None, seed=0, unused=0):
    g = gen(dev, seed + rows + Dh)
    qkv = (torch.randn(rows, Hq + 2 * Hk, Dh, generator=g, device=dev) * 3 + 0.5).to(dtype)
    sections = sections or (Dh // 8, Dh // 8, Dh // 4)
    pos = positions_of(kind, rows, len(sections), dev, g)
    freq = (1000.0 ** -torch.rand(sum(sections), generator=g, device=dev)).float()

    def weight(at):
        return (at + 0.3 * torch.randn(Dh, generator=g, device=dev)).to(dtype)

    qn, kn = [(weight(1) if weights else None, weight(0) if weights and layer else None) for _ in range(2)]
    B, N = 3, rows // 2 + 2
    slots = torch.randperm(B * N, generator=g, device=dev)[:rows]
    bi, ti = slots // N, slots % N
    if unused:
        bi[-unused:] = -1
        ti[-unused:] = -1
    kv = torch.randn(B, N, 2, Hk, Dh, generator=g, device=dev).to(dtype)
    q_out = torch.randn(rows, Hq, Dh, generator=g, device=dev).to(dtype)
    return qkv, qn, kn, pos, freq, sections, bi, ti, kv, q_out


def check_norm(qkv, Hq, Hk, qn, kn, eps, pos, freq, sections, bi, ti, kv, q_out, layer):
    kv0, q0 = kv.clone(), q_out.clone()
    K.qk_norm_rope_kv(qkv, Hq, Hk, qn, kn, eps, pos, freq, sections, bi, ti, kv, q_out, layer_norm=layer)
    angle = angles64(pos, freq, sections)
    ok = (bi >= 0) & (bi < kv.shape[0]) & (ti >= 0) & (ti < kv.shape[1])
    half = angle.shape[1]

    def turned(x, n):
        y, size = norm64(x, *n, eps, layer)
        ref, _ = rotate64(y, angle)
        pair = size[..., :half] + size[..., half:2 * half]
        return ref, torch.cat([pair, pair, size[..., 2 * half:]], -1)

    ref, size = turned(qkv[:, :Hq], qn)
    slack = 1e-6 + 30 * 2.0 ** -24
    near(q_out[ok], ref[ok], slack * size[ok], "q")
    assert torch.equal(q_out[~ok], q0[~ok]), "rows without a slot were written"
    ref, size = turned(qkv[:, Hq:Hq + Hk], kn)
    near(kv[bi[ok], ti[ok], 0], ref[ok], slack * size[ok], "k")
    assert torch.equal(kv[bi[ok], ti[ok], 1], qkv[ok, Hq + Hk:]), "values are copied"
    hit = torch.zeros(kv.shape[:2], dtype=torch.bool, device=kv.device)
    hit[bi[ok], ti[ok]] = True
    assert torch.equal(kv[~hit], kv0[~hit]), "cache rows of no slot were written"


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layer,weights", [(False, True), (True, True), (False, False), (True, False)])
@pytest.mark.parametrize("rows,Hq,Hk,Dh", [(1, 1, 1, 64), (3, 6, 6, 64), (33, 16, 4, 64), (32, 32, 8, 128),
                                            (77, 15, 5, 128), (1029, 3, 1, 128), (2000, 7, 7, 64)])
def test_norm(dev, rows, Hq, Hk, Dh, layer, weights, dtype):
    qkv, qn, kn, pos, freq, sections, bi, ti, kv, q_out = norm_case(dev, rows, Hq, Hk, Dh, dtype, layer, weights,
                                                                    unused=rows // 8)
    check_norm(qkv, Hq, Hk, qn, kn, 1e-6, pos, freq, sections, bi, ti, kv, q_out, layer)


@pytest.mark.parametrize("kind,sections", [(torch.float32, (16, 16)), (torch.int32, (8,)), (torch.int64, (0, 16, 0, 8))])
def test_norm_positions_partial_rotation_and_strides(dev, kind, sections):
    """Part of a head rotated; qkv rows, cache rows and q_out rows with gaps; slots far outside the cache."""
    Hq, Hk, Dh = 4, 2, 64
    qkv, qn, kn, pos, freq, sections, bi, ti, kv, q_out = norm_case(dev, 50, Hq, Hk, Dh, BF, False, True, kind, sections)
    wide = torch.zeros(50, Hq + 2 * Hk + 1, Dh, device=dev, dtype=BF)
    wide[:, :-1] = qkv
    kvw = torch.zeros(3, kv.shape[1], 2, Hk + 1, Dh, device=dev, dtype=BF)
    kvw[:, :, :, :Hk] = kv
    qw = torch.zeros(50, Hq + 3, Dh, device=dev, dtype=BF)
    bi[0], ti[1], bi[2], ti[3] = 3, kv.shape[1], 1 << 40, -(1 << 40)
    check_norm(wide[:, :-1], Hq, Hk, qn, kn, 1e-5, pos, freq, sections, bi, ti, kvw[:, :, :, :Hk], qw[:, :Hq], False)
    assert not kvw[:, :, :, Hk:].any() and not qw[:, Hq:].any()


def test_norm_of_zeros_and_large_values(dev):
    """A head of zeros is zero (eps keeps the quotient), one near the type's largest value does not overflow."""
    for dtype, big in ((BF, 1e15), (HF, 6e4)):
        qkv, qn, kn, pos, freq, sections, bi, ti, kv, q_out = norm_case(dev, 6, 2, 1, 64, dtype, False, True)
        qkv[0] = 0
        qkv[1] = big
        check_norm(qkv, 2, 1, qn, kn, 1e-6, pos, freq, sections, bi, ti, kv, q_out, False)
        assert not q_out[0].any()


def test_norm_without_rows(dev):
    qkv, qn, kn, pos, freq, sections, bi, ti, kv, q_out = norm_case(dev, 4, 2, 1, 64, BF, False, True)
    before = kv.clone()
    K.qk_norm_rope_kv(qkv[:0], 2, 1, qn, kn, 1e-6, pos[:0], freq, sections, bi[:0], ti[:0], kv, q_out[:0])
    assert torch.equal(kv, before)


# ------------------------------------------------------------------------------------------------
# packed_attention
# ------------------------------------------------------------------------------------------------


def attention64(q, k, v, m, n, scale, causal):
    """One sequence in 64 bits: q [m, Hq, Dh], k, v [n, Hk, Dh] -> (out, slack of the bound)."""
    Hq, Dh = q.shape[1:]
    G = Hq // k.shape[1]
    u = half_step(q.dtype)
    out = torch.zeros(m, Hq, Dh, dtype=torch.float64, device=q.device)
    slack = torch.zeros_like(out)
    if n == 0 or m == 0:
        return out, slack
    seen = torch.arange(m, device=q.device)[:, None] + (n - m)
    hidden = torch.arange(n, device=q.device) > seen if causal else torch.zeros(m, n, dtype=torch.bool, device=q.device)
    for h in range(Hq):
        qh, kh, vh = q[:, h].double(), k[:, h // G].double(), v[:, h // G].double()
        vh = torch.where(torch.isfinite(vh), vh, 0.0)
        kh = torch.where(torch.isfinite(kh), kh, 0.0)
        kt = kh.t().contiguous()
        s = (qh @ kt) * scale
        size = (qh.abs() @ kt.abs()) * scale
        size = size.masked_fill(hidden, 0.0).amax(-1, keepdim=True)
        s = s.masked_fill(hidden, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(hidden, 0.0, torch.exp(s - torch.where(torch.isfinite(top), top, 0.0)))
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        out[:, h] = p @ vh
        slack[:, h] = (p @ vh.abs()) * (2 * u + 2 * (Dh + 8) * 2.0 ** -24 * size + 2.0 ** -20)
        if q.dtype == HF:
            slack[:, h] += 2.0 ** -25 * (~hidden).double() @ vh.abs()
    return out, slack


def check_attention(q, k, v, m, n, scale, causal, got, what=""):
    """Every sequence of got [M, Hq Dh] against attention64; k, v packed or batched."""
    Hq, Dh = q.shape[1:]
    at = ak = 0
    for s, (a, b) in enumerate(zip(m, n)):
        ks, vs = (k[s, :b], v[s, :b]) if k.dim() == 4 else (k[ak:ak + b], v[ak:ak + b])
        ref, slack = attention64(q[at:at + a], ks, vs, a, b, scale, causal)
        near(got[at:at + a].view(a, Hq, Dh), ref, slack, f"{what} sequence {s}: {a} rows, {b} keys")
        at += a
        ak += b


def offsets(lens, dev, dtype=torch.int32):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=dtype, device=dev)


def packed_case(dev, m, n, Hq, Hk, Dh, dtype, batched, seed, sharp=1.0):
    g = gen(dev, seed)
    q = (torch.randn(sum(m), Hq, Dh, generator=g, device=dev) * sharp).to(dtype)
    if batched:
        kv = torch.randn(len(n), max(1, max(n)) + 3, 2, Hk, Dh, generator=g, device=dev).to(dtype)
        k, v = kv[:, :, 0], kv[:, :, 1]
        return q, k, v, offsets(m, dev), torch.tensor(n, dtype=torch.int32, device=dev)
    kv = torch.randn(sum(n), 2, Hk, Dh, generator=g, device=dev).to(dtype)
    return q, kv[:, 0], kv[:, 1], offsets(m, dev), offsets(n, dev)


LENS = [  # rows and keys of the sequences
    ([1], [1]), ([1], [64]), ([1], [65]), ([2, 1], [2, 700]), ([1, 1, 1], [31, 0, 33]), ([0, 0], [5, 0]),
    ([63], [63]), ([64], [64]), ([65], [65]), ([129], [129]), ([300], [300]), ([17, 0, 1, 200, 5], [17, 3, 1, 260, 900]),
    ([5, 9], [2, 0]),                       # causal: the first rows see nothing
    ([40], [1500]), ([1] * 9, [5, 1000, 2, 3000, 64, 63, 1, 130, 0]), ([3, 513], [2111, 513]),
]
HEADS = [(1, 1, 64), (4, 4, 64), (6, 2, 64), (8, 1, 128), (7, 1, 128), (8, 2, 128), (40, 1, 64)]


@pytest.mark.parametrize("Hq,Hk,Dh", HEADS)
@pytest.mark.parametrize("m,n", LENS)
@pytest.mark.parametrize("causal", [False, True])
def test_attention(dev, m, n, Hq, Hk, Dh, causal):
    for batched in (False, True):
        for dtype in (BF, HF):
            q, k, v, cu, keys = packed_case(dev, m, n, Hq, Hk, Dh, dtype, batched, len(m) + Dh)
            got = K.packed_attention(q, k, v, cu, keys, Dh ** -0.5, causal=causal)
            assert got.shape == (sum(m), Hq * Dh)
            check_attention(q, k, v, m, n, Dh ** -0.5, causal, got, f"batched={batched} {dtype}")


@pytest.mark.parametrize("m,n,Hq,Hk,Dh", [
    ([1000, 3, 700], [1000, 3, 700], 4, 4, 64), ([1, 1], [9000, 40], 8, 2, 128), ([600], [4101], 16, 4, 128),
    ([1029] * 4, [1029] * 4, 16, 16, 64), ([2000], [2000], 32, 8, 128), ([90, 4], [5000, 5000], 12, 12, 64),
    ([1] * 70, list(range(1, 71)), 4, 2, 128), ([40] * 70, [40 + 37 * i for i in range(70)], 2, 2, 64),
    ([1] * 100, [29 * i for i in range(1, 101)], 4, 2, 64), ([2] * 100, [2 + 29 * i for i in range(100)], 2, 1, 128),
    ([100, 30], [2600, 100], 2, 1, 64), ([1] * 300, [200 + i for i in range(300)], 8, 8, 64),
    ([33], [20000], 1, 1, 64), ([1], [50000], 4, 1, 128),
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_long(dev, m, n, Hq, Hk, Dh, causal):
    for dtype in (BF, HF):
        batched = m != n
        q, k, v, cu, keys = packed_case(dev, m, n, Hq, Hk, Dh, dtype, batched, sum(n))
        got = K.packed_attention(q, k, v, cu, keys, Dh ** -0.5, causal=causal)
        check_attention(q, k, v, m, n, Dh ** -0.5, causal, got, str(dtype))


@pytest.mark.parametrize("S,longest,Hq,Hk,Dh", [(65, 200, 4, 1, 64), (130, 40, 3, 3, 128), (300, 90, 8, 2, 64),
                                                (700, 3, 40, 4, 128), (5000, 2, 2, 1, 64)])
def test_attention_many_sequences(dev, S, longest, Hq, Hk, Dh):
    """Ragged lengths with empty sequences among them, the offsets starting inside the row buffer."""
    rng = random.Random(S)
    m = [rng.choice([0, 1, rng.randrange(longest + 1)]) for _ in range(S)]
    n = [a + rng.randrange(60) for a in m]
    q, k, v, cu, keys = packed_case(dev, m, n, Hq, Hk, Dh, BF, False, S)
    got = K.packed_attention(q, k, v, cu, keys, Dh ** -0.5, causal=True)
    some = rng.sample(range(S), 40)
    for s in some:
        at, ak = sum(m[:s]), sum(n[:s])
        ref, slack = attention64(q[at:at + m[s]], k[ak:ak + n[s]], v[ak:ak + n[s]], m[s], n[s], Dh ** -0.5, True)
        near(got[at:at + m[s]].view(m[s], Hq, Dh), ref, slack, f"sequence {s}")
    wide = torch.cat([q[:7], q, q[:9]])
    out = torch.full((wide.shape[0], Hq * Dh), 3.0, device=dev, dtype=BF)
    K.packed_attention(wide, k, v, cu + 7, keys, Dh ** -0.5, causal=True, out=out)
    assert torch.equal(out[7:-9], got) and (out[:7] == 3).all() and (out[-9:] == 3).all()


@pytest.mark.parametrize("scale", [1e-3, 0.6, 3.0])
def test_attention_sharp_and_flat_scores(dev, scale):
    m, n = [3, 200, 1], [400, 200, 3000]
    q, k, v, cu, keys = packed_case(dev, m, n, 4, 2, 64, BF, True, 5, sharp=2.0)
    check_attention(q, k, v, m, n, scale, True, K.packed_attention(q, k, v, cu, keys, scale, causal=True))


@pytest.mark.parametrize("m", [1, 50])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_of_many_small_weights(dev, m, Dh, dtype):
    """One key far above 20000 equal ones, whose weights (2^-15 and 2^-20 of its own, subnormal in fp16) add up to a
    large and to a small part of the sum."""
    n = 20001
    for octaves, at in ((15, 0), (15, n - 1), (20, 9000)):
        g = gen(dev, octaves)
        k = torch.zeros(1, n, 1, Dh, device=dev, dtype=dtype)
        k[0, at, 0, 0] = octaves
        v = torch.randn(1, n, 1, Dh, generator=g, device=dev).to(dtype) + 0.5
        q = torch.zeros(m, 2, Dh, device=dev, dtype=dtype)
        q[:, :, 0] = 1
        got = K.packed_attention(q, k, v, offsets([m], dev), torch.tensor([n], device=dev), math.log(2), causal=False)
        check_attention(q, k, v, [m], [n], math.log(2), False, got, f"{octaves} octaves")


@pytest.mark.parametrize("m", [1, 70])
@pytest.mark.parametrize("Dh", [64, 128])
def test_attention_of_tiny_and_huge_fp16_values(dev, m, Dh):
    """Values and keys below fp16's smallest normal number, and values near its largest."""
    q, k, v, cu, keys = packed_case(dev, [m], [300], 2, 2, Dh, HF, True, 6)
    for factor in (1e-5, 1.5e4):
        vf = (v.float() * factor).clamp(-65504, 65504).to(HF)  # (a value of 4.4 times the deviation would be infinite)
        got = K.packed_attention(q, k, vf, cu, keys, 0.1, causal=True)
        check_attention(q, k, vf, [m], [300], 0.1, True, got, f"values {factor}")
    small = (k.float() * 1e-5).to(HF)
    got = K.packed_attention(q, small, v, cu, keys, 1e4, causal=True)
    check_attention(q, small, v, [m], [300], 1e4, True, got, "keys")


@pytest.mark.parametrize("m,n,Hq,Hk,Dh", [([200, 7], [200, 7], 4, 4, 64), ([150, 60], [190, 333], 8, 1, 128),
                                          ([5, 1], [700, 90], 4, 2, 128), ([300], [300], 2, 2, 64),
                                          ([7, 3], [2500, 64], 4, 2, 64), ([6], [2400], 2, 1, 128),
                                          ([200], [2500], 4, 2, 64), ([150], [2600], 4, 2, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_keys_and_values_have_no_influence(dev, m, n, Hq, Hk, Dh, bad):
    """A NaN or infinite key or value is met by the rows that see it, and by no others: keys behind a sequence's
    last, other sequences' keys, and later tokens of the same sequence."""
    for dtype in (BF, HF):
        q, k, v, cu, keys = packed_case(dev, m, n, Hq, Hk, Dh, dtype, True, 8)
        want = K.packed_attention(q, k, v, cu, keys, Dh ** -0.5, causal=True)
        k, v = k.clone(), v.clone()
        for s, b in enumerate(n):
            k[s, b:] = bad
            v[s, b:] = bad
        got = K.packed_attention(q, k, v, cu, keys, Dh ** -0.5, causal=True)
        assert torch.equal(got, want)
        # One late token of every sequence that has rows before it.
        first_bad = [n[s] - (m[s] + 1) // 2 for s in range(len(m))]
        for s, t in enumerate(first_bad):
            if m[s] > 1:
                k[s, t, :, 1] = bad
                v[s, t, :, 3] = bad
                v[s, t, :, Dh - 1] = -bad
        got = K.packed_attention(q, k, v, cu, keys, Dh ** -0.5, causal=True)
        at = 0
        for s, a in enumerate(m):
            blind = first_bad[s] - (n[s] - a) if a > 1 else a   # rows that do not see it
            ref, slack = attention64(q[at:at + blind], k[s, :n[s] - a + blind], v[s, :n[s] - a + blind], blind,
                                     n[s] - a + blind, Dh ** -0.5, True)
            near(got[at:at + blind].view(blind, Hq, Dh), ref, slack, f"{dtype} sequence {s}")
            if math.isnan(bad):  # (an infinite key may weigh nothing)
                assert not torch.isfinite(got[at + blind:at + a].float()).all(-1).any()
            at += a


def test_visible_infinite_values(dev):
    """Rows that see an infinite value are that infinity in its dim, NaN where both signs meet, finite elsewhere."""
    q, k, v, cu, keys = packed_case(dev, [130], [130], 2, 2, 64, BF, False, 9)
    v = v.clone()
    v[100, :, 5] = math.inf
    v[110, :, 5] = -math.inf
    v[120, :, 6] = math.nan
    got = K.packed_attention(q, k, v, cu, keys, 0.01, causal=True).view(130, 2, 64).float()
    assert torch.isfinite(got[:100]).all() and (got[100:110, :, 5] == math.inf).all()
    assert torch.isnan(got[110:, :, 5]).all() and torch.isnan(got[120:, :, 6]).all()
    assert torch.isfinite(got[:, :, 7:]).all() and torch.isfinite(got[:120, :, 6]).all()


def test_attention_strides_and_rows_left_alone(dev):
    """q, k and v in one qkv row, keys of a cache with gaps, int64 offsets, a wide `out` whose other rows and
    columns stay; offsets that start and end inside the row buffer."""
    g = gen(dev, 10)
    m = [37, 0, 100]
    M = sum(m) + 9
    qkv = torch.randn(M, 12, 64, generator=g, device=dev).to(BF)
    q, k, v = qkv.split([8, 2, 2], 1)
    out = torch.full((M, 8 * 64 + 32), 7.0, device=dev, dtype=BF)
    cu = offsets(m, dev, torch.int64)
    got = K.packed_attention(q, k, v, cu, cu, 0.125, causal=True, out=out[:, :512])
    assert got.data_ptr() == out.data_ptr() and (out[:, 512:] == 7).all() and (out[sum(m):] == 7).all()
    check_attention(q[:sum(m)], k, v, m, m, 0.125, True, got[:sum(m)])
    out.fill_(7.0)
    K.packed_attention(q, k, v, cu + 4, cu + 4, 0.125, causal=True, out=out[:, :512])
    assert (out[:4] == 7).all() and (out[4 + sum(m):] == 7).all()
    check_attention(q[4:4 + sum(m)], k[4:], v[4:], m, m, 0.125, True, out[4:4 + sum(m), :512])
    one = k[:, :1].expand(M, 2, 64)  # one key head broadcast over two
    a = K.packed_attention(q[:sum(m)], one, v, cu, cu, 0.125, causal=False)
    assert torch.equal(a, K.packed_attention(q[:sum(m)], one.contiguous(), v.contiguous(), cu, cu, 0.125, causal=False))
    row = k[:1].expand(M, 2, 64)     # one key for every token
    a = K.packed_attention(q[:sum(m)], row, v, cu, cu, 0.125, causal=False)
    check_attention(q[:sum(m)], row, v, m, m, 0.125, False, a)


def test_attention_offsets_outside_the_buffers_are_cut(dev):
    q, k, v, _, _ = packed_case(dev, [20], [20], 2, 2, 64, BF, False, 11)
    cu = torch.tensor([-5, 8, 400], device=dev, dtype=torch.int32)
    got = K.packed_attention(q, k, v, cu, cu, 0.125, causal=False)
    check_attention(q, k, v, [8, 12], [8, 12], 0.125, False, got)
    kb = k[None].contiguous()
    got = K.packed_attention(q, kb, v[None].contiguous(), offsets([20], dev), torch.tensor([9999], device=dev), 0.125,
                             causal=False)
    check_attention(q, k, v, [20], [20], 0.125, False, got)
    none = K.packed_attention(q, kb, kb, offsets([20], dev), torch.tensor([-3], device=dev), 0.125, causal=False)
    assert not none.any()


def test_attention_offsets_that_fall(dev):
    """Offsets that rise and fall are no valid input: the call ends all the same and writes nothing outside `out`."""
    for S, Hk, Dh, cap in ((3, 2, 64, 3000), (200, 1, 128, 3000), (300, 2, 64, 100)):
        q, _, _, _, _ = packed_case(dev, [900], [900], 2 * Hk, Hk, Dh, BF, False, 14)
        g = gen(dev, 15)
        k = torch.randn(cap, Hk, Dh, generator=g, device=dev).to(BF)
        cu = torch.tensor([0, 20] + [900 if i % 2 else 0 for i in range(S - 1)], device=dev)
        cu_k = torch.tensor([0, 50] + [cap if i % 2 else 0 for i in range(S - 1)], device=dev)
        out = torch.full((902, 2 * Hk * Dh), 5.0, device=dev, dtype=BF)
        K.packed_attention(q, k, k, cu, cu_k, 0.1, causal=True, out=out[1:901])
        torch.cuda.synchronize()
        assert (out[0] == 5).all() and (out[901] == 5).all()


def test_attention_empty(dev):
    q = torch.empty(0, 4, 64, device=dev, dtype=BF)
    k = torch.empty(0, 2, 64, device=dev, dtype=BF)
    zero = torch.zeros(1, device=dev, dtype=torch.int32)
    assert K.packed_attention(q, k, k, zero, zero, 0.125, causal=True).shape == (0, 256)
    q1 = torch.ones(3, 4, 64, device=dev, dtype=BF)
    cu, ck = offsets([3], dev), offsets([0], dev)
    assert not K.packed_attention(q1, k, k, cu, ck, 0.125, causal=True).any()


@pytest.mark.parametrize("m,n", [([1], [3000]), ([40], [3000]), ([700], [700])])
def test_attention_is_deterministic(dev, m, n):
    q, k, v, cu, keys = packed_case(dev, m, n, 8, 2, 128, BF, True, 12)
    want = K.packed_attention(q, k, v, cu, keys, 0.1, causal=True)
    for _ in range(5):
        assert torch.equal(K.packed_attention(q, k, v, cu, keys, 0.1, causal=True), want)


def test_attention_cache_past_32_bits(dev):
    """One sequence whose keys span more than 4 GiB, another in a batch that starts past 2^31 elements."""
    N, Hk, Dh = 1100000, 8, 128
    kv = torch.zeros(2, N, 2, Hk, Dh, device=dev, dtype=BF)
    g = gen(dev, 13)
    near_end = torch.randn(2, 4000, 2, Hk, Dh, generator=g, device=dev).to(BF)
    kv[:, -4000:] = near_end
    q = (torch.randn(5, Hk, Dh, generator=g, device=dev) * 2).to(BF)
    cu = offsets([2, 3], dev)
    keys = torch.tensor([N, N], device=dev)
    got = K.packed_attention(q, kv[:, :, 0], kv[:, :, 1], cu, keys, Dh ** -0.5, causal=True)
    # The zero keys each weigh exp(0) and their values are zero: they only add N - 4000 to the sum.
    at = 0
    for s, m in enumerate((2, 3)):
        for h in range(Hk):
            kh, vh = near_end[s, :, 0, h].double(), near_end[s, :, 1, h].double()
            z = (q[at:at + m, h].double() @ kh.t().contiguous()) * Dh ** -0.5
            hid = torch.arange(4000, device=dev) > torch.arange(m, device=dev)[:, None] + 4000 - m
            top = torch.maximum(z.masked_fill(hid, -math.inf).amax(-1, keepdim=True), torch.zeros((), device=dev).double())
            p = torch.exp(z - top).masked_fill(hid, 0.0)
            total = p.sum(-1, keepdim=True) + (N - 4000) * torch.exp(-top)
            ref, size = p @ vh / total, p @ vh.abs() / total
            # the sum of N weights: each rounded by 2^-8, and fp32 additions of 64 at a time
            near(got[at:at + m].view(m, Hk, Dh)[:, h], ref, size * (2 * 2.0 ** -8 + 2.0 ** -9), f"sequence {s} head {h}")
        at += m


def test_attention_on_another_stream_and_in_graphs(dev):
    """Two graphs of one call each, replayed between eager calls after the lengths, rows and keys changed."""
    m, n = [1, 30, 4], [2000, 900, 64]
    states = []
    for seed in (20, 21):
        q, k, v, cu, keys = packed_case(dev, m, n, 8, 2, 128, BF, True, seed)
        k, v = k.clone(), v.clone()
        out = torch.empty(sum(m), 8 * 128, device=dev, dtype=BF)
        run = graphs.capture(lambda q=q, k=k, v=v, cu=cu, keys=keys, out=out: K.packed_attention(
            q, k, v, cu, keys, 0.09, causal=True, out=out))
        states.append((q, k, v, cu, keys, out, run))
    for turn in range(4):
        for q, k, v, cu, keys, out, run in states:
            q.copy_(torch.randn(q.shape, generator=gen(dev, turn), device=dev))
            if turn:
                m2 = [(2, 20, 13), (0, 35, 0), (11, 12, 12)][turn - 1]
                cu.copy_(offsets(m2, dev))
                keys.copy_(torch.tensor([1500, 64 * turn, 900], device=dev))
        torch.cuda.synchronize()
        side = [torch.cuda.Stream(device=dev) for _ in states]
        for st, s in zip(side, states):
            st.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(st):
                s[-1]()
        for st in side:
            torch.cuda.current_stream(dev).wait_stream(st)
        for q, k, v, cu, keys, out, run in states:
            assert torch.equal(out, K.packed_attention(q, k, v, cu, keys, 0.09, causal=True))
        torch.cuda.synchronize()


def test_attention_graphs_recorded_by_torch_own_their_scratch(dev):
    """torch records all its graphs on one stream; two of them, with split keys, replayed at once on two streams."""
    cases, runs = [], []
    for seed in (81, 82):
        q, k, v, cu, keys = packed_case(dev, [2, 1, 3], [5000, 4100, 4900], 8, 2, 128, BF, True, seed)
        out = torch.empty_like(q).flatten(1)
        want = K.packed_attention(q, k, v, cu, keys, 0.1, causal=True)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.packed_attention(q, k, v, cu, keys, 0.1, causal=True, out=out)
        cases.append((q, k, v, cu, keys, out, want))
        runs.append((g, torch.cuda.Stream()))
    for _ in range(4):
        for case in cases:
            case[5].fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, stream in runs:
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        for q, k, v, cu, keys, out, want in cases:
            assert torch.equal(out, want)
            assert torch.equal(K.packed_attention(q, k, v, cu, keys, 0.1, causal=True), want)


def test_attention_agrees_with_sparse_query_attention(dev):
    """Equal lengths, equal heads, no mask: the rectangular attention of the correction pass."""
    g = gen(dev, 30)
    B, T, N, H, Dh = 3, 70, 330, 6, 64
    q = torch.randn(B * T, H, Dh, generator=g, device=dev).to(BF)
    kv = torch.randn(B, N, 2, H, Dh, generator=g, device=dev).to(BF)
    want = K.sparse_query_attention(q, kv, T, 0.125)
    got = K.packed_attention(q, kv[:, :, 0], kv[:, :, 1], offsets([T] * B, dev), torch.full((B,), N, device=dev), 0.125,
                             causal=False)
    n = [N] * B
    check_attention(q, kv[:, :, 0], kv[:, :, 1], [T] * B, n, 0.125, False, want)
    check_attention(q, kv[:, :, 0], kv[:, :, 1], [T] * B, n, 0.125, False, got)


# ------------------------------------------------------------------------------------------------
# A layer: plan, qkv product, normed heads with the K/V write, attention; prompts first, then single tokens
# ------------------------------------------------------------------------------------------------


def test_layer_of_prompts_and_then_tokens(dev):
    """Three prompts of different lengths go into a cache, then each gets one token, then two get four: every step's
    output against the whole of its sequence computed at once in 64 bits from the step's own qkv rows."""
    Hq, Hk, Dh, C, N = 8, 2, 64, 256, 128
    g = gen(dev, 40)
    w = (torch.randn((Hq + 2 * Hk) * Dh, C, generator=g, device=dev) * 0.1).to(BF)
    qn, kn = [((1 + 0.2 * torch.randn(Dh, generator=g, device=dev)).to(BF), None) for _ in range(2)]
    freq = (100.0 ** -(torch.arange(32, device=dev) / 32)).float()
    kv = torch.full((3, N, 2, Hk, Dh), math.nan, device=dev, dtype=BF)
    have = [0, 0, 0]
    steps = [[70, 1, 33], [1, 1, 1], [4, 0, 4]]
    rows = 110  # a buffer longer than any step needs
    for new in steps:
        x = torch.randn(rows, C, generator=g, device=dev).to(BF)
        total = [a + b for a, b in zip(have, new)]
        plan = K.packed_plan(torch.tensor(new, device=dev), torch.tensor(total, device=dev), rows, cache_len=N)
        qkv = K.linear(x, w).view(rows, Hq + 2 * Hk, Dh)
        t = plan.token_idx.clamp(min=0)
        pos = torch.stack([t // 16, t % 16], 1)
        q = torch.zeros(rows, Hq, Dh, device=dev, dtype=BF)
        K.qk_norm_rope_kv(qkv, Hq, Hk, qn, kn, 1e-6, pos, freq, (16, 16), plan.batch_idx, plan.token_idx, kv, q)
        out = K.packed_attention(q, kv[:, :, 0], kv[:, :, 1], plan.cu_q, plan.k_lens, Dh ** -0.5, causal=True)
        used = sum(new)
        ok = plan.batch_idx >= 0
        assert ok[:used].all() and not ok[used:].any()
        y, _ = norm64(qkv[:, :Hq], *qn, 1e-6, False)
        ref, _ = rotate64(y, angles64(pos, freq, (16, 16)))
        assert (q[:used].double() - ref[:used]).abs().max() <= 2.0 ** -7 * ref[:used].abs().max()
        check_attention(q[:used], kv[:, :, 0], kv[:, :, 1], new, total, Dh ** -0.5, True, out[:used])
        have = total
    for s, n in enumerate(have):  # the cache holds the tokens that were given, and nothing else
        assert torch.isfinite(kv[s, :n]).all() and torch.isnan(kv[s, n:]).all()


def test_layer_in_a_graph(dev):
    """The three steps recorded once and replayed with other lengths, rows and caches, against eager calls."""
    Hq, Hk, Dh, N, rows, S = 8, 2, 128, 2300, 40, 5
    g = gen(dev, 50)
    qkv = torch.zeros(rows, Hq + 2 * Hk, Dh, device=dev, dtype=BF)
    new = torch.zeros(S, device=dev, dtype=torch.int64)
    total = torch.zeros(S, device=dev, dtype=torch.int64)
    w = torch.ones(Dh, device=dev, dtype=BF)
    freq = (100.0 ** -(torch.arange(64, device=dev) / 64)).float()
    pos = torch.randint(0, 1 << 20, (rows, 3), generator=g, device=dev)
    kv = torch.randn(S, N, 2, Hk, Dh, generator=g, device=dev).to(BF)
    q = torch.zeros(rows, Hq, Dh, device=dev, dtype=BF)
    out = torch.zeros(rows, Hq * Dh, device=dev, dtype=BF)

    def layer(kv, q, out):
        plan = K.packed_plan(new, total, rows, cache_len=N)
        K.qk_norm_rope_kv(qkv, Hq, Hk, (w, None), (w, None), 1e-6, pos, freq, (16, 24, 24), plan.batch_idx,
                          plan.token_idx, kv, q)
        K.packed_attention(q, kv[:, :, 0], kv[:, :, 1], plan.cu_q, plan.k_lens, Dh ** -0.5, causal=True, out=out)

    replay = graphs.capture(lambda: layer(kv, q, out))
    for turn, (a, b) in enumerate([([1] * 5, [2300, 1, 40, 700, 2000]), ([8, 0, 20, 3, 0], [8, 0, 2300, 1500, 9]),
                                   ([0] * 5, [0] * 5), ([40, 0, 0, 0, 0], [41, 0, 0, 0, 0])]):
        qkv.copy_(torch.randn(qkv.shape, generator=gen(dev, turn), device=dev))
        new.copy_(torch.tensor(a, device=dev))
        total.copy_(torch.tensor(b, device=dev))
        kv2, q2, out2 = kv.clone(), q.clone(), out.clone()
        layer(kv2, q2, out2)
        torch.cuda.synchronize()
        replay()
        torch.cuda.synchronize()
        assert torch.equal(kv, kv2) and torch.equal(q, q2) and torch.equal(out, out2), f"replay {turn}"


def test_outputs_in_other_orders(dev):
    """Outputs whose entries are apart in any order of dims: heads outside rows, a cache with K and V outside, every
    second row; what lies between stays."""
    g, Hq, Hk, Dh, M, B, N = gen(dev, 93), 4, 2, 64, 9, 2, 5
    pos, freq = torch.randint(0, 99, (M, 2), generator=g, device=dev), torch.rand(32, generator=g, device=dev)
    q, k = (torch.randn(M, h, Dh, generator=g, device=dev).to(BF) for h in (Hq, Hk))
    want = K.apply_rope_axes(q, k, pos, freq, (16, 16))
    oq = torch.full((Hq, 2 * M, Dh), 3.0, device=dev, dtype=BF)
    ok = torch.full((Hk, M, Dh), 3.0, device=dev, dtype=BF)
    K.apply_rope_axes(q, k, pos, freq, (16, 16), out=(oq[:, ::2].transpose(0, 1), ok.transpose(0, 1)))
    assert torch.equal(oq[:, ::2].transpose(0, 1), want[0]) and torch.equal(ok.transpose(0, 1), want[1])
    assert (oq[:, 1::2] == 3.0).all()

    qkv = torch.randn(M, Hq + 2 * Hk, Dh, generator=g, device=dev).to(BF)
    slot = torch.randperm(B * N, generator=g, device=dev)[:M]
    plain = torch.full((B, N, 2, Hk, Dh), 3.0, device=dev, dtype=BF)
    other = torch.full((2, N, B, Hk, Dh), 3.0, device=dev, dtype=BF)
    q1, q2 = torch.empty(M, Hq, Dh, device=dev, dtype=BF), torch.full((2 * M, Hq, Dh), 3.0, device=dev, dtype=BF)
    for cache, qo in ((plain, q1), (other.permute(2, 1, 0, 3, 4), q2[::2])):
        K.qk_norm_rope_kv(qkv, Hq, Hk, (None, None), (None, None), 1e-6, pos, freq, (16, 16), slot // N, slot % N, cache,
                          qo)
    assert torch.equal(other.permute(2, 1, 0, 3, 4), plain) and torch.equal(q2[::2], q1) and (q2[1::2] == 3.0).all()


@pytest.mark.parametrize("bad", [
    dict(q=(4, 4, 32)), dict(k=(9, 3, 64)), dict(v=(9, 2, 128)), dict(dtype=torch.float32), dict(cu=4), dict(keys=4),
    dict(scale=0.0), dict(scale=-0.1), dict(scale=math.nan), dict(out=(4, 255)), dict(kdtype=HF), dict(heads_strided=True),
    dict(k=(2, 9, 2, 64)), dict(cu_dtype=torch.float32), dict(odd=True),
])
def test_attention_refusals(dev, bad):
    """Arguments that do not fit are refused before a launch, ValueError by the wrapper or the library's status."""
    dtype = bad.get("dtype", BF)
    q = torch.zeros(bad.get("q", (4, 4, 64)), device=dev, dtype=dtype)
    k = torch.zeros(bad.get("k", (9, 2, 64)), device=dev, dtype=bad.get("kdtype", dtype))
    v = torch.zeros(bad.get("v", k.shape), device=dev, dtype=bad.get("kdtype", dtype))
    if bad.get("heads_strided"):
        k = torch.zeros(9, 2, 128, device=dev, dtype=dtype)[..., ::2]
    if bad.get("odd"):
        q = torch.zeros(4 * 4 * 64 + 1, device=dev, dtype=dtype)[1:].view(4, 4, 64)
    cu = torch.zeros(bad.get("cu", 4), device=dev, dtype=bad.get("cu_dtype", torch.int32))
    keys = torch.zeros(bad.get("keys", 4), device=dev, dtype=torch.int32)
    if bad.get("cu") == 4:
        keys = keys[:3]
    elif bad.get("keys") == 4:
        cu = cu[:3]
    out = torch.zeros(bad["out"], device=dev, dtype=dtype) if "out" in bad else None
    from appcorr_amd._lib import OudjatKernelError
    with pytest.raises((ValueError, OudjatKernelError)):
        K.packed_attention(q, k, v, cu, keys, bad.get("scale", 0.1), causal=True, out=out)


def test_row_operator_refusals(dev):
    from appcorr_amd._lib import OudjatKernelError
    x = torch.zeros(4, 6, 64, device=dev, dtype=BF)
    pos, freq = torch.zeros(4, 2, device=dev), torch.zeros(32, device=dev)
    n = torch.ones(3, device=dev, dtype=torch.int32)
    for call in (
        lambda: K.apply_rope_axes(x, x.to(HF), pos, freq, (16, 16)),
        lambda: K.apply_rope_axes(x.float(), x.float(), pos, freq, (16, 16)),
        lambda: K.apply_rope_axes(x, x[:3], pos, freq, (16, 16)),
        lambda: K.apply_rope_axes(x, x, pos, freq, (16, 8)),
        lambda: K.apply_rope_axes(x, x, pos, freq, (32,)),
        lambda: K.apply_rope_axes(x, x, pos.double(), freq, (16, 16)),
        lambda: K.apply_rope_axes(x, x, pos, freq.double(), (16, 16)),
        lambda: K.apply_rope_axes(x, x, pos, torch.zeros(40, device=dev), (20, 20)),
        lambda: K.apply_rope_axes(x, x, pos.cpu(), freq, (16, 16)),
        lambda: K.apply_rope_axes(x, x, pos, freq, (16, 16), out=(x, x[:, :3])),
        lambda: K.packed_plan(n, n[:2], 4, cache_len=4),
        lambda: K.packed_plan(n, n, 4),
        lambda: K.packed_plan(n, n, 4, cache_len=4, key_rows=4),
        lambda: K.packed_plan(n.float(), n, 4, cache_len=4),
        lambda: K.packed_plan(n, n, -1, cache_len=4),
        lambda: K.packed_plan(n, n, 4, cache_len=-1),
        lambda: K.packed_plan(torch.ones(4097, device=dev, dtype=torch.int32),
                              torch.ones(4097, device=dev, dtype=torch.int32), 4, cache_len=4),
    ):
        with pytest.raises((ValueError, OudjatKernelError)):
            call()
    w = torch.ones(64, device=dev, dtype=BF)
    slot = torch.zeros(4, device=dev, dtype=torch.int64)
    kv, q = torch.zeros(1, 8, 2, 1, 64, device=dev, dtype=BF), torch.zeros(4, 4, 64, device=dev, dtype=BF)

    def norm(qkv=x, heads=4, qn=(w, None), sections=(16, 16), bi=slot, ti=slot, kv=kv, q=q, eps=1e-6, **kw):
        K.qk_norm_rope_kv(qkv, heads, 1, qn, (None, None), eps, pos, freq, sections, bi, ti, kv, q, **kw)

    for kw in (dict(heads=5), dict(qkv=x.float()), dict(qn=(w[:32], None)), dict(qn=(w.float(), None)), dict(qn=(w, w)),
               dict(sections=(16,)), dict(bi=slot.int()), dict(ti=slot[:3]), dict(kv=kv[:, :, :1]), dict(kv=kv.to(HF)),
               dict(q=q[:3]), dict(q=q.to(HF)), dict(eps=-1.0), dict(eps=math.nan),
               dict(qkv=x.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises((ValueError, OudjatKernelError)):
            norm(**kw)
