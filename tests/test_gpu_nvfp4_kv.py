"""NVFP4 K/V caches: rows written and read back, and the attention over them, against their definitions in 64 bits.

The codes and scales that are written are compared bit for bit with a restatement in numpy (oracle.nvfp4's, whose rounding
goes by search over the code grids). What is read is e2m1 * e4m3 * tensor_scale: the first product is exact, the second is
rounded to fp32 and then to the type, half a step each.

Attention: the cached values are exact operands. Scores: the query is exact in fp16 but for bits below 2^-38 of the row's
largest value, sums of Dh products in fp32, (Dh + 8) 2^-24 scale sum|q||k| each way in the exponent. Probabilities are
rounded to fp16 with 2^-11 of their value at most (u16 on both sides of the quotient), or 2^-25 below fp16's normal range
where the largest is at least 2^7: 2^-32 per key. Sums of n weighted values in fp32, at most (n / 32 + 40) 2^-24 of sum(p |v|) with
32 keys a product. The output is rounded by half a step."""

import math
import random

import numpy as np
import pytest
import torch

from appcorr_amd import graphs
from appcorr_amd import kernels as K
from oracle import nvfp4 as ON

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------
# Write and read
# ------------------------------------------------------------------------------------------------


def quantized(x, ts):
    """(codes, scale bytes) of fp32 numpy blocks x [.., 16] with the tensor scales ts [..], in the steps of the format."""
    amax = np.abs(x).max(-1)
    scaled = np.clip((amax / np.float32(6)).astype(np.float32) / ts, ON.E4M3_EPS, ON.F8E4M3_MAX).astype(np.float32)
    s8 = ON.e4m3_encode(scaled)
    unit = (ts * ON.e4m3_decode(s8)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        codes = ON.e2m1_encode((x / unit[..., None]).astype(np.float32))
    return np.where(s8[..., None] == 0, 0, codes).astype(np.uint8), s8


def values64(cache):
    """The cache's values [B, N, 2, Hk, Dh] in 64 bits; scale bytes without their sign, 0x7f as 480."""
    codes = cache.codes.cpu().numpy()
    byte = cache.scales.contiguous().view(torch.uint8).cpu().numpy() & 0x7f
    s = np.where(byte == 0x7f, 480.0, ON.e4m3_decode(byte).astype(np.float64))
    both = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    x = ON.e2m1_decode(both).astype(np.float64) * np.repeat(s, 16, -1)
    return torch.from_numpy(x).to(cache.codes.device) * cache.tensor_scale.double()[:, :, None]


def cache_of(dev, B, N, Hk, Dh, g, layout="heads", garbage=True):
    """An empty cache of any bytes; layout: the order of its memory."""
    order = {"heads": (0, 2, 3, 1), "tokens": (0, 1, 2, 3), "planes": (2, 0, 3, 1)}[layout]
    sizes = (B, N, 2, Hk)
    back = [order.index(d) for d in range(4)]

    def make(last):
        shape = [sizes[d] for d in order] + [last]
        t = torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.uint8) if garbage else \
            torch.zeros(shape, device=dev, dtype=torch.uint8)
        return t.permute(*back, 4)

    ts = (0.5 + torch.rand(2, Hk, generator=g, device=dev)) / 448
    return K.KvNvfp4(make(Dh // 2), make(Dh // 16).view(torch.uint8), ts)


WRITE = [(1, 1, 64, 1, 5), (3, 6, 64, 2, 7), (201, 16, 64, 3, 100), (64, 8, 128, 64, 3), (1030, 5, 128, 2, 600),
         (77, 1, 128, 1, 80), (2500, 3, 64, 1, 2600)]


@pytest.mark.parametrize("layout", ["heads", "tokens", "planes"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,Hk,Dh,B,N", WRITE)
def test_write_and_read(dev, rows, Hk, Dh, B, N, dtype, layout):
    g = gen(dev, rows * 7 + Hk)
    cache = cache_of(dev, B, N, Hk, Dh, g, layout)
    qkv = torch.randn(rows, 3 * Hk + 1, Dh, generator=g, device=dev) * torch.exp(
        2 * torch.randn(rows, 3 * Hk + 1, 1, generator=g, device=dev))
    qkv = qkv.to(dtype)
    k, v = qkv[:, Hk:2 * Hk], qkv[:, 2 * Hk + 1:]
    slots = torch.randperm(B * N + rows, generator=g, device=dev)[:rows]
    inside = slots < B * N
    bi, ti = torch.where(inside, slots // N, -1), torch.where(inside, slots % N, -1)
    if rows > 2:  # outside in other ways
        bi[0], ti[0], inside[0] = B, 0, False
        bi[1], ti[1], inside[1] = 0, N, False
    before_c, before_s = cache.codes.clone(), cache.scales.clone()
    K.kv_nvfp4_write(k, v, bi, ti, cache)
    both = torch.stack([k, v], 1).float().cpu().numpy().reshape(rows, 2, Hk, Dh // 16, 16)
    ts = np.broadcast_to(cache.tensor_scale.cpu().numpy()[None, :, :, None], both.shape[:-1])
    codes, s8 = quantized(both, ts)
    codes = codes.reshape(rows, 2, Hk, Dh)
    want_c, want_s = before_c.clone(), before_s.clone()
    at = bi[inside], ti[inside]
    want_c[at] = torch.from_numpy(codes[..., 0::2] | codes[..., 1::2] << 4).to(dev)[inside]
    want_s[at] = torch.from_numpy(s8).to(dev)[inside]
    assert torch.equal(cache.scales, want_s)
    assert torch.equal(cache.codes, want_c)

    # Everything back, in another order, with slots outside among them.
    n = B * N + 3
    order = torch.randperm(n, generator=g, device=dev)
    rb, rt = order // N, order % N
    for out_type in (BF, HF):
        got = K.kv_nvfp4_read(cache, rb, rt, dtype=out_type)
        x = values64(cache)
        for which, y in enumerate(got):
            ref = torch.zeros(n, Hk, Dh, dtype=torch.float64, device=dev)
            ok = rb < B
            ref[ok] = x[rb[ok], rt[ok], which]
            lim = ref.abs() * (half_step(out_type) * (1 + 2.0 ** -20) + 2.0 ** -23)
            lim = lim + (2.0 ** -25 if out_type == HF else 0.0)
            assert ((y.double() - ref).abs() <= lim).all()


def test_write_at_the_ends_of_the_format(dev):
    """Zeros, infinities, NaN, values far above and far below what the tensor scale takes, ties."""
    for dtype in (BF, HF):
        big = 3e38 if dtype == BF else 65504.0
        tiny = 1e-40 if dtype == BF else 6e-8
        rows = [[0.0] * 16, [-0.0] * 16, [1.0] + [0.0] * 15, [big, -big] + [1.0] * 14, [tiny] * 16,
                [0.25, -0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, 6.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0],
                [448 * 6.0, -448 * 6.0, 448.0] + [1.0] * 13, [2.0 ** -12] * 16, [2.0 ** -9] * 16]
        x = torch.tensor(rows, device=dev).to(dtype)
        n = len(rows)
        k = torch.zeros(1, 3, 64, device=dev, dtype=dtype).view(-1)
        k[:16 * n] = x.view(-1)
        k = k.view(1, 3, 64)
        cache = K.kv_nvfp4_cache(1, 1, 3, 64, dev, tensor_scale=1.0)
        z = torch.zeros(1, dtype=torch.long, device=dev)
        K.kv_nvfp4_write(k, k, z, z, cache)
        codes, s8 = quantized(k.float().cpu().numpy().reshape(1, 3, 4, 16), np.ones((1, 3, 4), np.float32))
        codes = codes.reshape(1, 3, 64)
        for which in (0, 1):
            assert torch.equal(cache.scales.view(torch.uint8)[0, :, which].cpu(), torch.from_numpy(s8))
            assert torch.equal(cache.codes[0, :, which].cpu(), torch.from_numpy(codes[..., 0::2] | codes[..., 1::2] << 4))
    # What the format cannot hold: NaN is 0, infinities are the largest value, and the rest of the block is as it would be.
    x = torch.full((1, 1, 64), 6.0, device=dev, dtype=BF)
    x[0, 0, 0], x[0, 0, 17], x[0, 0, 18] = math.nan, math.inf, -math.inf
    cache = K.kv_nvfp4_cache(1, 1, 1, 64, dev, tensor_scale=0.5)
    K.kv_nvfp4_write(x, x, z, z, cache)
    k, v = K.kv_nvfp4_read(cache, z, z)
    for y in (k, v):
        y = y.flatten().tolist()
        assert y[0] == 0 and y[1:16] == [6.0] * 15 and y[17] == 1344.0 and y[18] == -1344.0 and y[32:] == [6.0] * 32
        assert y[16] == 0 and y[19:32] == [0.0] * 13  # next to an infinity, 6 is below half of the smallest step


def test_a_cache_nobody_has_written_reads_finite(dev):
    cache = cache_of(dev, 2, 50, 2, 64, gen(dev, 1))
    i = torch.arange(100, device=dev)
    for y in K.kv_nvfp4_read(cache, i // 50, i % 50, dtype=BF):
        assert torch.isfinite(y).all()


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------


def attend64(q, x, nq, nk, scale, causal, cap):
    """(outputs, tolerance before the last rounding) [M, Hq, Dh] of rows with counts nq over nk cached tokens."""
    M, Hq, Dh = q.shape
    Hk = x.shape[3]
    out = torch.zeros(M, Hq, Dh, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    at = 0
    for s, (a, b) in enumerate(zip(nq, nk)):
        n = min(b, cap)
        for h in range(Hq if a and n else 0):
            k, v = x[s, :n, 0, h * Hk // Hq], x[s, :n, 1, h * Hk // Hq]
            qq = q[at:at + a, h].double()
            z = qq @ k.T * scale
            hidden = torch.zeros(a, n, dtype=torch.bool, device=q.device)
            if causal:
                hidden = torch.arange(n, device=q.device) > torch.arange(a, device=q.device)[:, None] + (b - a)
            z = z.masked_fill(hidden, -math.inf)
            none = hidden.all(-1)
            p = torch.softmax(z, -1).masked_fill(none[:, None], 0.0)
            size = (qq.abs() @ k.abs().T * scale).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
            pv = p @ v.abs()
            o = p @ v
            rel = 2 * (Dh + 8) * 2.0 ** -24 * size + 2 * 2.0 ** -11 + (n / 32 + 40) * 2.0 ** -24 + 2 * 2.0 ** -20
            out[at:at + a, h] = o
            tol[at:at + a, h] = rel * (pv + o.abs()) + (n * 2.0 ** -32) * (v.abs().amax() + o.abs()) * (~none[:, None])
        at += a
    return out.view(M, -1), tol.view(M, -1)


def filled(dev, B, N, Hk, Dh, g, layout="heads"):
    cache = cache_of(dev, B, N, Hk, Dh, g, layout)
    x = torch.randn(B * N, 2, Hk, Dh, generator=g, device=dev, dtype=torch.float32).to(BF)
    i = torch.arange(B * N, device=dev)
    K.kv_nvfp4_write(x[:, 0], x[:, 1], i // N, i % N, cache)
    return cache


def check(got, ref, tol, what=""):
    u = half_step(got.dtype)
    lim = tol + u * (ref.abs() + tol) + (2.0 ** -25 if got.dtype == HF else 0.0)
    d = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = d > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / lim).max()):.3g} of the bound"


def run_attention(dev, nq, nk, N, Hq, Hk, Dh, dtype, causal, seed, layout="heads", extra=0, wide=False, spread=1.0):
    print(f"attention {nq[:4]}.. over {nk[:4]}.. of {N}, {Hq}/{Hk} x {Dh} {dtype} causal={causal} {layout}", flush=True)
    g = gen(dev, seed)
    S, M = len(nq), sum(nq) + extra
    cache = filled(dev, max(1, S), N, Hk, Dh, g, layout)
    q = (torch.randn(M, Hq, Dh, generator=g, device=dev) * spread).to(dtype)
    kind = torch.int64 if wide else torch.int32
    cu = torch.tensor([sum(nq[:i]) for i in range(S + 1)], dtype=kind, device=dev)
    kl = torch.tensor(nk, dtype=kind, device=dev)
    out = torch.full((M, Hq * Dh), 7.0, device=dev, dtype=dtype)
    K.packed_attention_nvfp4(q, cache, cu, kl, Dh ** -0.5, causal=causal, out=out)
    ref, tol = attend64(q, values64(cache), nq, nk, Dh ** -0.5, causal, N)
    end = sum(nq)
    check(out[:end], ref[:end], tol[:end])
    assert (out[end:] == 7.0).all()
    return q, cache, cu, kl, out


ATTN = [  # rows, keys, cache length, heads, key heads, dims
    ([1], [1], 1, 1, 1, 64), ([1], [5], 9, 3, 3, 128), ([1, 1, 1], [31, 32, 33], 40, 16, 4, 64),
    ([1] * 4, [1029, 7, 128, 129], 1030, 16, 16, 64), ([3, 0, 5], [3, 0, 9], 20, 6, 2, 128),
    ([2, 17, 1], [2, 300, 0], 300, 12, 12, 64), ([64], [64], 64, 8, 1, 64), ([201, 33], [201, 700], 701, 28, 4, 128),
    ([130, 1, 257], [130, 500, 300], 512, 4, 4, 64), ([300], [2600], 2700, 8, 2, 128), ([1] * 9, [2305] * 9, 2400, 8, 1, 128),
    ([40, 7], [4101, 3000], 4200, 15, 5, 128), ([1, 16], [5000, 4500], 5000, 16, 1, 64), ([1] * 70, [200] * 70, 210, 8, 2, 64),
    ([1] * 300, [37] * 300, 40, 4, 1, 64), ([513], [513], 600, 2, 2, 128), ([259, 128], [900, 4000], 4100, 2, 1, 64),
    ([5, 4], [2, 1], 8, 4, 2, 64),  # more rows than keys: the first see none
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(dev, case, dtype, causal):
    run_attention(dev, *ATTN[case], dtype, causal, case, extra=case % 3, wide=case % 2 == 1)


@pytest.mark.parametrize("layout", ["tokens", "planes"])
@pytest.mark.parametrize("case", [3, 7, 9, 11])
def test_attention_of_other_layouts(dev, case, layout):
    run_attention(dev, *ATTN[case], BF, True, case, layout=layout)


@pytest.mark.parametrize("spread", [2.0 ** -140, 1e-30, 1e-6, 30.0, 1e4])
def test_attention_of_small_and_large_queries(dev, spread):
    run_attention(dev, [3, 40, 200], [50, 300, 200], 300, 8, 2, 64, BF, True, 5, spread=spread)
    if 1e-7 < spread < 1e4:
        run_attention(dev, [3, 40, 200], [50, 300, 200], 300, 8, 2, 128, HF, True, 5, spread=spread)


def test_attention_equals_that_over_the_values(dev):
    """packed_attention over the cache read back in fp16 (exact with a power of two as tensor scale)."""
    g = gen(dev, 3)
    B, N, Hq, Hk, Dh = 3, 300, 8, 2, 128
    cache = filled(dev, B, N, Hk, Dh, g)
    cache.tensor_scale.fill_(2.0 ** -6)
    i = torch.arange(B * N, device=dev)
    k, v = (x.view(B, N, Hk, Dh) for x in K.kv_nvfp4_read(cache, i // N, i % N, dtype=HF))
    q = torch.randn(40, Hq, Dh, generator=g, device=dev, dtype=torch.float32).to(HF)
    cu = torch.tensor([0, 1, 25, 40], dtype=torch.int32, device=dev)
    kl = torch.tensor([300, 24, 211], dtype=torch.int32, device=dev)
    a = K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True).double()
    b = K.packed_attention(q, k, v, cu, kl, 0.1, causal=True).double()
    # Each is within its own roundings of the formula: probabilities 2 * 2^-11 of sum(p |v|) each, outputs 2^-11.
    top = float(v.abs().max())
    assert float((a - b).abs().max()) <= (4 * 2.0 ** -11 + 2 * 2.0 ** -11 + 2.0 ** -16) * top


def test_attention_hidden_and_unwritten_tokens(dev):
    """Tokens behind the last key hold any bytes, scale bytes of 0x7f and 0xff among them; they change nothing."""
    for Dh, nq, nk in ((64, [1, 40], [33, 40]), (128, [1, 1, 200], [70, 1, 200])):
        g = gen(dev, Dh)
        cache = filled(dev, len(nq), 256, 2, Dh, g)
        q = torch.randn(sum(nq), 8, Dh, generator=g, device=dev, dtype=torch.float32).to(BF)
        cu = torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device=dev)
        kl = torch.tensor(nk, dtype=torch.int32, device=dev)
        a = K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True)
        for byte in (0x7f, 0xff, 0x00):
            for s, n in enumerate(nk):
                cache.scales.view(torch.uint8)[s, n:] = byte
                cache.codes[s, n:] = 0x77
            assert torch.equal(K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True), a)


def test_attention_rows_that_are_not_finite(dev):
    g = gen(dev, 9)
    cache = filled(dev, 2, 100, 2, 64, g)
    q = torch.randn(41, 4, 64, generator=g, device=dev, dtype=torch.float32).to(BF)
    q[0, 1, 5], q[3, 0, 0], q[7, 3, 63] = math.nan, math.inf, -math.inf
    cu = torch.tensor([0, 1, 41], dtype=torch.int32, device=dev)
    kl = torch.tensor([90, 37], dtype=torch.int32, device=dev)  # the first three rows of the second see nothing
    out = K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True).view(41, 4, 64)
    bad = torch.zeros(41, 4, dtype=torch.bool, device=dev)
    bad[0, 1] = bad[7, 3] = True
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()
    assert (out[1:4] == 0).all()


def test_a_layer_in_a_graph(dev):
    """Plan, rotation, write and attention of prompts and then of single tokens, eager and replayed, against the formula."""
    g = gen(dev, 11)
    S, N, Hq, Hk, Dh, M = 3, 300, 8, 2, 64, 128
    cache = K.kv_nvfp4_cache(S, N, Hk, Dh, dev)
    new = torch.tensor([50, 1, 60], device=dev)
    total = torch.tensor([50, 1, 60], device=dev)
    qkv = torch.randn(M, Hq + 2 * Hk, Dh, generator=g, device=dev, dtype=torch.float32).to(BF)
    inv = (10000.0 ** -(torch.arange(32, device=dev) / 32)).float()
    out = torch.zeros(M, Hq * Dh, device=dev, dtype=BF)
    qr, kr = torch.empty(M, Hq, Dh, device=dev, dtype=BF), torch.empty(M, Hk, Dh, device=dev, dtype=BF)

    def layer():
        plan = K.packed_plan(new, total, M, cache_len=N)
        q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hk]
        K.apply_rope_axes(q, k, plan.token_idx.clamp(min=0).view(M, 1), inv, (32,), out=(qr, kr))
        K.kv_nvfp4_write(kr, qkv[:, Hq + Hk:], plan.batch_idx, plan.token_idx, cache)
        K.packed_attention_nvfp4(qr, cache, plan.cu_q, plan.k_lens, Dh ** -0.5, causal=True, out=out)

    replay = graphs.capture(layer)
    steps = [([50, 1, 60], [50, 1, 60]), ([1, 1, 1], [51, 2, 61]), ([1, 40, 1], [52, 42, 62]), ([1, 0, 1], [53, 42, 63])]
    for n_new, n_total in steps:
        new.copy_(torch.tensor(n_new))
        total.copy_(torch.tensor(n_total))
        qkv.copy_(torch.randn(M, Hq + 2 * Hk, Dh, generator=g, device=dev))
        out.fill_(0)
        replay()
        got = out.clone()
        ref, tol = attend64(qr[:sum(n_new)], values64(cache), n_new, n_total, Dh ** -0.5, True, N)
        check(got[:sum(n_new)], ref, tol)
        assert (got[sum(n_new):] == 0).all()
        layer()
        assert torch.equal(out, got)
