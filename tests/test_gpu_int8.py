"""INT8 rows and products against their definitions in 64 bits.

Codes and scales are compared exactly with numpy's IEEE arithmetic. A product's sum is exact; as fp32 it is rounded once, the
two scales' product once, their product once, bias, gamma and residual once each: 8 * 2^-24 of the terms' sizes at most
(silu: the exponential 2 ulp, a sum, a quotient, 2^-21), then half a step of the output's type."""

import numpy as np
import pytest
import torch

from appcorr_amd import _lib, graphs
from appcorr_amd import kernels as K

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
EPI = {"bias": _lib.EPI_BIAS, "ls": _lib.EPI_BIAS_LS, "ls_resid": _lib.EPI_BIAS_LS_RESID, "silu": _lib.EPI_BIAS_SILU_MUL}


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def quantized(x):
    """(codes, scales) of fp32 numpy rows; codes 0 and scale NaN of a row that is not finite."""
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], np.float32(0), x)
    scale = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32) if x.shape[-1] else np.zeros(x.shape[:-1], np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.clip(np.rint((x / scale[..., None]).astype(np.float32)), -127, 127)
    return np.where(scale[..., None] > 0, q, 0).astype(np.int8), np.where(bad, np.float32(np.nan), scale)


def same(got, want):
    assert torch.equal(got[0].cpu(), torch.from_numpy(want[0]))
    assert np.array_equal(got[1].cpu().numpy(), want[1], equal_nan=True)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,Kd", [(1, 16), (3, 384), (5, 1024), (7, 1040), (201, 768), (2, 4096), (33, 4112), (9, 8192),
                                     (3, 8208), (2, 20000), (1025, 64), (4, 0), (0, 64)])
def test_quantize(dev, rows, Kd, dtype):
    g = gen(dev, rows + Kd)
    x = (torch.randn(rows, Kd, generator=g, device=dev) * torch.exp(3 * torch.randn(rows, 1, generator=g, device=dev))).to(dtype)
    if rows > 2:
        x[1] = 0
    same(K.quantize_int8(x), quantized(x.float().cpu().numpy()))


def test_quantize_ties_and_ends(dev):
    """x / scale on the borders between codes (scale a power of two), the ends of the types' ranges."""
    x = torch.arange(-127, 128, device=dev).float()
    x = torch.cat([x, x[:-1] + 0.5, torch.tensor([127.0, -127.0, 0.0], device=dev)])
    x = torch.nn.functional.pad(x, (0, 512 - x.numel()))
    for dtype in (BF, HF):
        y = (x * 2.0 ** -3).to(dtype)
        ones = torch.stack([y, y * 0.5, y * 2.0 ** -5])
        same(K.quantize_int8(ones), quantized(ones.float().cpu().numpy()))
    ends = torch.zeros(8, 64, device=dev)
    for i, v in enumerate((3.3e38, 1e-30, 1e-37, 2.0 ** -126, 2.0 ** -130, 2.0 ** -133, 1e30, 5e-25)):
        ends[i] = v * (torch.arange(64, device=dev) - 31) / 32
    for y in (ends.to(BF), torch.stack([ends[0] * 0 + 65504.0, torch.arange(64, device=dev) * 2.0 ** -24]).to(HF)):
        same(K.quantize_int8(y), quantized(y.float().cpu().numpy()))


def test_quantize_the_largest_values(dev):
    x = torch.linspace(-1, 1, 64, device=dev) * 3.3e38
    same(K.quantize_int8(x[None].to(BF)), quantized(x[None].to(BF).float().cpu().numpy()))


@pytest.mark.parametrize("Kd", [64, 4096, 9000 // 16 * 16])
def test_quantize_rows_that_are_not_finite(dev, Kd):
    for dtype in (BF, HF):
        x = torch.ones(5, Kd, device=dev, dtype=dtype)
        x[1, 3], x[2, Kd - 1], x[4, 0] = float("nan"), float("inf"), float("-inf")
        codes, scale = K.quantize_int8(x)
        assert torch.isnan(scale).tolist() == [False, True, True, False, True]
        assert (codes[[1, 2, 4]] == 0).all() and (codes[[0, 3]] == 127).all()


def test_quantize_strided(dev):
    x = torch.randn(9, 5, 256, device=dev, dtype=torch.float32).to(BF)
    same(K.quantize_int8(x[:, 2, :128]), quantized(x[:, 2, :128].float().cpu().numpy()))
    codes, scale = K.quantize_int8(x)
    same((codes.view(-1, 256), scale.view(-1)), quantized(x.view(-1, 256).float().cpu().numpy()))
    same(K.quantize_int8(x[0, 0]), quantized(x[0, 0].float().cpu().numpy()))
    same(K.quantize_int8(x[0, 0].expand(4, 256)), quantized(x[0, 0].expand(4, 256).float().cpu().numpy()))


def product64(x8, sx, w8, sw, bias, gamma, resid, epi):
    """(y, sum of the terms' sizes) in 64 bits."""
    y = (x8.double() @ w8.double().T) * sx.double()[:, None] * sw.double()
    size = y.abs()
    if bias is not None:
        y = y + bias.double()
        size = size + bias.double().abs()
    if epi == "silu":
        # silu's derivative is below 1.1
        return y * torch.sigmoid(y) * resid.double(), (1.1 * size + (y * torch.sigmoid(y)).abs() * 8) * resid.double().abs()
    if epi != "bias":
        y, size = y * gamma.double(), size * gamma.double().abs()
    if epi == "ls_resid":
        y, size = y + resid.double(), size + resid.double().abs()
    return y, size


def operands(dev, M, N, Kd, dtype, epi, seed):
    g = gen(dev, seed)
    x8 = torch.randint(-128, 128, (M, Kd), generator=g, device=dev, dtype=torch.int8)
    w8 = torch.randint(-128, 128, (N, Kd), generator=g, device=dev, dtype=torch.int8)
    sx = torch.rand(M, generator=g, device=dev) * 0.02 / Kd ** 0.5
    sw = torch.rand(N, generator=g, device=dev) * 0.02
    bias = torch.randn(N, generator=g, device=dev).to(dtype)
    gamma = torch.randn(N, generator=g, device=dev).to(dtype) if epi in ("ls", "ls_resid") else None
    resid = torch.randn(M, N, generator=g, device=dev).to(dtype) if epi in ("ls_resid", "silu") else None
    return x8, sx, w8, sw, bias, gamma, resid


def check(got, ref, size, what=""):
    u = torch.finfo(got.dtype).eps / 2
    slack = size * 8 * 2.0 ** -24
    lim = slack + u * (ref.abs() + slack) + (2.0 ** -25 if got.dtype == HF else 0.0)
    d = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    bad = d > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / lim).max()):.3g} of the bound"


SHAPES = [(1, 8, 64), (1, 4096, 4096), (2, 384, 384), (15, 200, 128), (16, 1024, 192), (17, 1032, 1024), (31, 64, 4160),
          (32, 8192, 1024), (33, 264, 576), (48, 768, 768), (64, 2048, 1024), (65, 136, 320), (100, 1000, 640), (127, 256, 256),
          (128, 128, 128), (129, 392, 448), (201, 384, 384), (255, 2304, 768), (300, 1536, 384), (513, 520, 64), (1044, 1024, 4096),
          (1656, 4096, 512), (2049, 776, 192), (4176, 1024, 1024)]


# Every tile at least twice, with ragged edges, one and several K tiles, whole ones and half ones at the end
# (test_int8_nvfp4_host.py says so); the widths of this package's blocks.
SHAPES += [(3531, 2184, 64), (2305, 5000, 192), (4117, 3896, 832), (2289, 4680, 192), (922, 11272, 320), (3000, 4104, 64),
           (3000, 4104, 192), (5243, 5448, 704), (1656, 8200, 576), (300, 1032, 2112)]
# The last rows in a second launch.
SHAPES += [(4116, 4096, 576), (12289, 2048, 448), (12309, 2056, 320)]


@pytest.mark.parametrize("epi", ["bias", "ls", "ls_resid", "silu"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,Kd", SHAPES)
def test_linear(dev, M, N, Kd, dtype, epi):
    print(f"linear_int8 {M} x {N} x {Kd} {dtype} {epi}", flush=True)
    x8, sx, w8, sw, bias, gamma, resid = operands(dev, M, N, Kd, dtype, epi, M + N + Kd)
    got = K.linear_int8(x8, sx, w8, sw, bias, epilogue=EPI[epi], gamma=gamma, resid=resid, dtype=dtype)
    check(got, *product64(x8, sx, w8, sw, bias, gamma, resid, epi))
    if epi == "ls_resid":  # in place of the residual
        out = resid.clone()
        K.linear_int8(x8, sx, w8, sw, bias, epilogue=EPI[epi], gamma=gamma, resid=out, out=out, dtype=dtype)
        assert torch.equal(out, got)


@pytest.mark.parametrize("epi", ["bias", "ls", "ls_resid", "silu"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_rows_result_does_not_depend_on_the_other_rows(dev, dtype, epi):
    """Rows of a product in two launches, and the same rows by themselves through other kernels: the same bits."""
    M, N, Kd = 4116, 4096, 576
    x8, sx, w8, sw, bias, gamma, resid = operands(dev, M, N, Kd, dtype, epi, 11)
    whole = K.linear_int8(x8, sx, w8, sw, bias, epilogue=EPI[epi], gamma=gamma, resid=resid, dtype=dtype)
    cuts = [(7, 8), (40, 60), (100, 200), (300, 800), (900, 2000), (2000, 4000), (4090, 4116)]
    assert len({K.linear_int8_tile(b - a, N, Kd)[:2] for a, b in cuts} | {K.linear_int8_tile(M, N, Kd)[:2]}) >= 5
    for a, b in cuts:
        part = K.linear_int8(x8[a:b], sx[a:b], w8, sw, bias, epilogue=EPI[epi], gamma=gamma,
                             resid=None if resid is None else resid[a:b], dtype=dtype)
        assert torch.equal(part, whole[a:b]), (a, b)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_is_exact_at_the_largest_sums(dev, M):
    """Codes of -128 everywhere, K just below 2^17: the sums come within 2^20 of 2^31."""
    Kd, N = (1 << 17) - 64, 72
    x8 = torch.full((M, Kd), -128, device=dev, dtype=torch.int8)
    w8 = torch.full((N, Kd), -128, device=dev, dtype=torch.int8)
    w8[1::2] = 127
    one = torch.ones(max(M, N), device=dev)
    got = K.linear_int8(x8, one[:M] * 2.0 ** -10, w8, one[:N] * 2.0 ** -10)
    want = torch.where(torch.arange(N, device=dev) % 2 == 0, 128 * 128 * Kd * 2.0 ** -20, -128 * 127 * Kd * 2.0 ** -20)
    assert torch.equal(got, want.to(BF).expand(M, N))


def test_linear_strided_operands(dev):
    """Rows of codes, weight, residual and output that are views; an output in one half of a wider buffer, the rest as it
    was; one row repeated (stride 0)."""
    M, N, Kd = 70, 136, 192
    x8, sx, w8, sw, bias, gamma, resid = operands(dev, M, N, Kd, BF, "ls_resid", 3)
    ref, size = product64(x8, sx, w8, sw, bias, gamma, resid, "ls_resid")
    xb = torch.zeros(M, 2, Kd, device=dev, dtype=torch.int8)
    wb = torch.full((N, 3, Kd), 99, device=dev, dtype=torch.int8)
    rb, ob = torch.zeros(M, 2 * N, device=dev, dtype=BF), torch.full((M, 2 * N), 5.0, device=dev, dtype=BF)
    xb[:, 1], wb[:, 2], rb[:, N:] = x8, w8, resid
    K.linear_int8(xb[:, 1], sx, wb[:, 2], sw, bias, epilogue=EPI["ls_resid"], gamma=gamma, resid=rb[:, N:], out=ob[:, N:])
    check(ob[:, N:], ref, size)
    assert (ob[:, :N] == 5.0).all()
    got = K.linear_int8(x8[:1].expand(M, Kd), sx, w8, sw)
    check(got, *product64(x8[:1].expand(M, Kd), sx, w8, sw, None, None, None, "bias"))
    three = K.linear_int8(x8.view(7, 10, Kd), sx.view(7, 10), w8, sw, bias)
    assert three.shape == (7, 10, N)
    check(three.view(M, N), *product64(x8, sx, w8, sw, bias, None, None, "bias"))


def test_strided_operands_in_two_launches(dev):
    """As above where the rows are dealt to two launches."""
    M, N, Kd = 4103, 4096, 256
    assert K.linear_int8_tile(M, N, Kd)[2] == 4096
    x8, sx, w8, sw, bias, gamma, resid = operands(dev, M, N, Kd, HF, "ls_resid", 5)
    ref, size = product64(x8, sx, w8, sw, bias, gamma, resid, "ls_resid")
    xb = torch.zeros(M, 2, Kd, device=dev, dtype=torch.int8)
    ob = torch.full((M + 1, N + 8), 5.0, device=dev, dtype=HF)
    xb[:, 1], ob[:M, :N] = x8, resid
    K.linear_int8(xb[:, 1], sx, w8, sw, bias, epilogue=EPI["ls_resid"], gamma=gamma, resid=ob[:M, :N], out=ob[:M, :N], dtype=HF)
    check(ob[:M, :N], ref, size)
    assert (ob[M] == 5.0).all() and (ob[:, N:] == 5.0).all()
    got = K.linear_int8(x8[:1].expand(M, Kd), sx, w8, sw, epilogue=EPI["ls_resid"], gamma=gamma, resid=resid[:1].expand(M, N),
                        dtype=HF)
    check(got, *product64(x8[:1].expand(M, Kd), sx, w8, sw, None, gamma, resid[:1].expand(M, N), "ls_resid"))


def test_rows_that_are_not_finite_give_nan(dev):
    x = torch.randn(20, 256, device=dev).to(BF)
    x[3, 7] = float("inf")
    w8, sw = K.quantize_int8(torch.randn(64, 256, device=dev).to(BF))
    y = K.linear_int8(*K.quantize_int8(x), w8, sw)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[[i for i in range(20) if i != 3]]).all()


def test_an_mlp_in_a_graph(dev):
    """Quantise, gate products, quantise, last product with the residual, as one block's SwiGLU runs them; replayed."""
    g = gen(dev, 4)
    M, C, H = 40, 256, 512
    x = torch.randn(M, C, generator=g, device=dev).to(BF)
    w1, w2, w3 = ((torch.randn(n, k, generator=g, device=dev) * k ** -0.5).to(BF) for n, k in ((H, C), (H, C), (C, H)))
    (c1, s1), (c2, s2), (c3, s3) = (K.quantize_int8(w) for w in (w1, w2, w3))
    gamma = torch.ones(C, device=dev, dtype=BF)
    out = torch.empty(M, C, device=dev, dtype=BF)

    def mlp():
        x8, sx = K.quantize_int8(x)
        a = K.linear_int8(x8, sx, c2, s2)
        h = K.linear_int8(x8, sx, c1, s1, epilogue=EPI["silu"], resid=a)
        K.linear_int8(*K.quantize_int8(h), c3, s3, epilogue=EPI["ls_resid"], gamma=gamma, resid=x, out=out)

    replay = graphs.capture(mlp)
    for seed in range(3):
        x.copy_(torch.randn(M, C, generator=gen(dev, seed), device=dev))
        replay()
        got = out.clone()
        mlp()
        assert torch.equal(got, out)
        xd = x.double()
        a, b = xd @ w1.double().T, xd @ w2.double().T
        ref = xd + (a * torch.sigmoid(a) * b) @ w3.double().T
        # Eight bits leave about one percent of a product's size.
        assert float((got.double() - ref).norm() / (ref - xd).norm()) < 0.05
