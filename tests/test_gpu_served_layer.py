"""A layer of packed sequences in 8 and 4 bits, as a server runs it: INT8 qkv product, rotation, K/V write into an NVFP4 cache,
attention, INT8 output product with LayerScale and residual. Each step is checked against its definition in 64 bits on
the tensors that it was given (tolerances: test_gpu_int8.py, test_gpu_nvfp4_kv.py), prompts first, then single tokens, eager and
replayed. And what calls at once, far addresses and other streams must not change."""

import pytest
import torch

from appcorr_amd import _lib, graphs
from appcorr_amd import kernels as K
from tests import test_gpu_int8 as I8
from tests import test_gpu_nvfp4_kv as KV

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


class Layer:
    def __init__(self, dev, S, N, M, Hq, Hk, Dh, dtype, seed):
        g = KV.gen(dev, seed)
        C = Hq * Dh
        self.Hq, self.Hk, self.Dh, self.M, self.N, self.dtype = Hq, Hk, Dh, M, N, dtype
        self.new = torch.zeros(S, dtype=torch.long, device=dev)
        self.total = torch.zeros(S, dtype=torch.long, device=dev)
        self.x = torch.zeros(M, C, device=dev, dtype=dtype)
        n = (Hq + 2 * Hk) * Dh
        self.wq, self.sq = K.quantize_int8((torch.randn(n, C, generator=g, device=dev) * C ** -0.5).to(dtype))
        self.bq = (0.1 * torch.randn(n, generator=g, device=dev)).to(dtype)
        self.wo, self.so = K.quantize_int8((torch.randn(C, C, generator=g, device=dev) * C ** -0.5).to(dtype))
        self.bo = (0.1 * torch.randn(C, generator=g, device=dev)).to(dtype)
        self.gamma = (1 + 0.1 * torch.randn(C, generator=g, device=dev)).to(dtype)
        self.inv = (10000.0 ** -(torch.arange(Dh // 2, device=dev) / (Dh // 2))).float()
        self.cache = K.kv_nvfp4_cache(S, N, Hk, Dh, dev)
        self.att = torch.zeros(M, C, device=dev, dtype=dtype)
        self.out = torch.zeros(M, C, device=dev, dtype=dtype)
        self.rows = g

    def step(self):
        plan = self.plan = K.packed_plan(self.new, self.total, self.M, cache_len=self.N)
        x8, sx = K.quantize_int8(self.x)
        qkv = self.qkv = K.linear_int8(x8, sx, self.wq, self.sq, self.bq, dtype=self.dtype).view(self.M, -1, self.Dh)
        self.before = qkv.clone()
        q, k, v = qkv.split([self.Hq, self.Hk, self.Hk], dim=1)
        K.apply_rope_axes(q, k, plan.token_idx.clamp(min=0).view(-1, 1), self.inv, (self.Dh // 2,), out=(q, k))
        K.kv_nvfp4_write(k, v, plan.batch_idx, plan.token_idx, self.cache)
        K.packed_attention_nvfp4(q, self.cache, plan.cu_q, plan.k_lens, self.Dh ** -0.5, causal=True, out=self.att)
        a8, sa = K.quantize_int8(self.att)
        K.linear_int8(a8, sa, self.wo, self.so, self.bo, epilogue=_lib.EPI_BIAS_LS_RESID, gamma=self.gamma, resid=self.x,
                      out=self.out, dtype=self.dtype)

    def check(self, new, total):
        n = sum(new)
        x8, sx = I8.quantized(self.x.float().cpu().numpy())
        x8, sx = (torch.from_numpy(t).to(self.x.device) for t in (x8, sx))
        I8.check(self.before.view(self.M, -1), *I8.product64(x8, sx, self.wq, self.sq, self.bq, None, None, "bias"), "qkv")
        values = KV.values64(self.cache)
        at = self.plan.batch_idx[:n], self.plan.token_idx[:n]
        # What was written is the rotated keys and the values, a rounding to four bits away: half the widest step (2 of 6) of the
        # block's scale, which is at most 1 / 16 above max / 6 of the block, plus that of the scale's own rounding.
        for which, rows in ((0, self.qkv[:n, self.Hq:self.Hq + self.Hk]), (1, self.qkv[:n, self.Hq + self.Hk:])):
            top = rows.double().unflatten(-1, (-1, 16)).abs().amax(-1).repeat_interleave(16, -1)
            assert ((values[at][:, which] - rows.double()).abs() <= top / 6 * (17 / 16) + top / 15).all()
        q = self.qkv[:n, :self.Hq]
        ref, tol = KV.attend64(q, values, new, total, self.Dh ** -0.5, True, self.N)
        KV.check(self.att[:n], ref, tol, "attention")
        a8, sa = I8.quantized(self.att.float().cpu().numpy())
        a8, sa = (torch.from_numpy(t).to(self.x.device) for t in (a8, sa))
        I8.check(self.out, *I8.product64(a8, sa, self.wo, self.so, self.bo, self.gamma, self.x, "ls_resid"), "output")


@pytest.mark.parametrize("Hq,Hk,Dh,dtype", [(8, 2, 64, BF), (4, 1, 128, BF), (6, 6, 64, HF)])
def test_layer_of_prompts_and_then_tokens(dev, Hq, Hk, Dh, dtype):
    layer = Layer(dev, 3, 200, 160, Hq, Hk, Dh, dtype, 5)
    replay = graphs.capture(layer.step)
    for step, (new, total) in enumerate([([60, 1, 70], [60, 1, 70]), ([1, 1, 1], [61, 2, 71]), ([1, 90, 0], [62, 92, 71]),
                                         ([1, 1, 1], [63, 93, 72])]):
        layer.new.copy_(torch.tensor(new))
        layer.total.copy_(torch.tensor(total))
        layer.x.copy_(torch.randn(layer.x.shape, generator=layer.rows, device=dev))
        layer.att.zero_()
        replay()
        got = layer.out.clone(), layer.att.clone()
        layer.att.zero_()
        layer.step()
        assert torch.equal(layer.out, got[0]) and torch.equal(layer.att, got[1]), step
        layer.check(new, total)
        assert (layer.att[sum(new):] == 0).all()  # rows behind the last sequence, as they were


def test_graphs_recorded_by_torch_own_their_scratch(dev):
    """Two graphs with split keys, recorded on torch's one capture stream, replayed at once on two streams."""
    cases, runs = [], []
    for seed, dh in ((81, 128), (82, 64)):
        g = KV.gen(dev, seed)
        cache = KV.filled(dev, 3, 5000, 2, dh, g)
        q = torch.randn(6, 8, dh, generator=g, device=dev).to(BF)
        cu = torch.tensor([0, 2, 3, 6], dtype=torch.int32, device=dev)
        kl = torch.tensor([5000, 4100, 4900], dtype=torch.int32, device=dev)
        out = torch.empty(6, 8 * dh, device=dev, dtype=BF)
        want = K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True, out=out)
        cases.append((q, cache, cu, kl, out, want))
        runs.append((graph, torch.cuda.Stream()))
    for _ in range(4):
        for case in cases:
            case[4].fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in runs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for q, cache, cu, kl, out, want in cases:
            assert torch.equal(out, want)
            assert torch.equal(K.packed_attention_nvfp4(q, cache, cu, kl, 0.1, causal=True), want)


def test_calls_on_another_stream(dev):
    """Each operator on a side stream, behind work of that stream that makes its inputs."""
    g = KV.gen(dev, 7)
    stream = torch.cuda.Stream()
    base = torch.randn(300, 512, generator=g, device=dev)
    w8, sw = K.quantize_int8(torch.randn(256, 512, generator=g, device=dev).to(BF))
    i = torch.arange(300, device=dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        x = base
        for _ in range(20):
            x = x * 1.01
        x = x.to(BF)
        y = K.linear_int8(*K.quantize_int8(x), w8, sw)
        cache = K.kv_nvfp4_cache(1, 300, 2, 64, dev)
        K.kv_nvfp4_write(x[:, :128].view(300, 2, 64), y[:, :128].view(300, 2, 64), i * 0, i, cache)
        k, v = K.kv_nvfp4_read(cache, i * 0, i)
    stream.synchronize()
    x2 = base
    for _ in range(20):
        x2 = x2 * 1.01
    x2 = x2.to(BF)
    assert torch.equal(x, x2)
    y2 = K.linear_int8(*K.quantize_int8(x2), w8, sw)
    assert torch.equal(y, y2)
    ref = KV.values64(cache)[0, :, 0].to(BF)
    assert torch.equal(k, ref.view(300, 2, 64)) and torch.isfinite(v).all()


def test_caches_beyond_4_gib(dev):
    """Tokens 16 KB apart: those from 262144 on lie past 4 GiB of their sequence's first. Written, read and attended to, by
    single tokens (split keys) and by a chunk (tiles of rows), and the same from a compact copy, bit for bit."""
    N, Hk, Dh = 270000, 1, 64
    buf = torch.zeros((N + 1) * 16384, device=dev, dtype=torch.uint8)
    codes = buf.as_strided((1, N, 2, Hk, Dh // 2), (N * 16384, 16384, 64, 64, 1))
    sbuf = torch.zeros((N + 1) * 16384, device=dev, dtype=torch.uint8)
    scales = sbuf.as_strided((1, N, 2, Hk, Dh // 16), (N * 16384, 16384, 64, 64, 1))
    far = K.KvNvfp4(codes, scales, torch.full((2, Hk), 1 / 448, device=dev))
    g = KV.gen(dev, 3)
    x = torch.randn(N, 2, Hk, Dh, generator=g, device=dev).to(BF)
    i = torch.arange(N, device=dev)
    K.kv_nvfp4_write(x[:, 0], x[:, 1], i * 0, i, far)
    near = K.kv_nvfp4_cache(1, N, Hk, Dh, dev)
    K.kv_nvfp4_write(x[:, 0], x[:, 1], i * 0, i, near)
    assert torch.equal(far.codes, near.codes) and torch.equal(far.scales, near.scales.view(torch.uint8))
    for a, b in zip(K.kv_nvfp4_read(far, i * 0, i), K.kv_nvfp4_read(near, i * 0, i)):
        assert torch.equal(a, b)
    for rows in (1, 200):
        q = torch.randn(rows, 2, Dh, generator=g, device=dev).to(BF)
        cu = torch.tensor([0, rows], dtype=torch.int32, device=dev)
        kl = torch.tensor([N], dtype=torch.int32, device=dev)
        a = K.packed_attention_nvfp4(q, far, cu, kl, 1.0, causal=True)
        assert torch.equal(a, K.packed_attention_nvfp4(q, near, cu, kl, 1.0, causal=True))
        if rows == 1:
            ref, tol = KV.attend64(q, KV.values64(near), [1], [N], 1.0, True, N)
            KV.check(a, ref, tol)


@pytest.mark.parametrize("M,N", [(70000, 64), (70000, 2304)])
def test_product_with_operands_beyond_4_gib(dev, M, N):
    """Rows 64 KB apart, the output's 64 KB too: the last tiles start past 4 GiB."""
    Kd, ld = 64, 65536
    g = KV.gen(dev, M)
    buf = torch.zeros(M * ld, device=dev, dtype=torch.int8)
    a = buf.as_strided((M, Kd), (ld, 1))
    x8 = torch.randint(-127, 128, (M, Kd), generator=g, device=dev, dtype=torch.int8)
    a.copy_(x8)
    w8 = torch.randint(-127, 128, (N, Kd), generator=g, device=dev, dtype=torch.int8)
    sx, sw = torch.rand(M, generator=g, device=dev), torch.rand(N, generator=g, device=dev)
    out = torch.zeros(M * (ld // 2), device=dev, dtype=BF).as_strided((M, N), (ld // 2, 1))
    K.linear_int8(a, sx, w8, sw, out=out)
    assert torch.equal(out, K.linear_int8(x8, sx, w8, sw))
    rows = torch.tensor([0, 1, M // 2, M - 2, M - 1], device=dev)
    I8.check(out[rows], *I8.product64(x8[rows], sx[rows], w8, sw, None, None, None, "bias"))
