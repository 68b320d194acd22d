"""Workloads of a layer served in 8 and 4 bits: INT8 products with a scale for each token and channel, K/V in NVFP4.

A server that answers many streams reads its weights and its K/V caches for every token: both are kept in fewer bits.
Three passes, in the order in which a layer uses them:

  linear  quantize_int8 (rows of activations to 8 bits, a scale each) and linear_int8 (their product with a weight that was
          quantised the same way, a scale for each output channel), with the epilogues of the package's other products;
  store   kv_nvfp4_write (K/V rows into a cache of 4-bit values with a scale for each 16) and kv_nvfp4_read (rows of that
          cache in 16 bits again, as a stream that moves to a 16-bit cache needs them);
  attn    packed_attention_nvfp4: grouped-head attention of packed rows over such caches.

Widths, head counts and lengths are those of this package's configurations (16 x 64, 32 x 128, 6 x 64 heads; widths 384,
768, 1024 and 4096, SwiGLU of 8192; 201, 1029, 2305, 4101 tokens; 1656 selected rows) or generic ones (32 query heads over 8
key heads, powers of two). Queries and keys are N(0, 1) as normed heads are, values N(0, 1); activations N(0, 1) with a
few channels ten times as large, as the inputs of a block's products are, weights N(0, 1 / K).
"""

from __future__ import annotations

import math
import random

import torch

own = False  # False: elementary torch operations in 32 bits; True: this package's operators

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One token of one stream through the attention's output product of the largest backbone: latency.
        linear("linear_1_token", 1, 4096, 4096, "bias", "bf16"),
        # One token of each of 32 streams through the second gate product of its SwiGLU.
        linear("linear_32_tokens", 32, 8192, 4096, "silu", "bf16"),
        # A small image's rows through the smallest backbone's output product.
        linear("linear_201_rows", 201, 384, 384, "ls_resid", "fp16"),
        # The selected rows of four images of 1024 px through the fused qkv product.
        linear("linear_1656_rows", 1656, 12288, 4096, "bias", "bf16"),
        # All rows of four such images through the last product of the block: the largest product.
        linear("linear_16404_rows", 16404, 4096, 8192, "ls_resid", "bf16"),
        # One token of each of 32 streams.
        store("store_32_tokens", 32, 8, 128, 1029, "bf16"),
        # Four images of 512 px.
        store("store_4116_rows", 4116, 16, 64, 1029, "fp16"),
        # Four images of 1024 px, all heads of the largest backbone.
        store("store_16404_rows", 16404, 32, 128, 4101, "bf16"),
        # One token of each of four streams against short caches: latency.
        attn("attn_4_tokens", 4, 1, 1029, 16, 16, 64, "bf16", 3),
        # One token of each of 32 streams against caches of up to 16384 tokens.
        attn("attn_32_tokens_long", 32, 1, 16384, 32, 8, 128, "bf16", 4),
        # The next 512 rows at most of three long streams.
        attn("attn_3_chunks", 3, 512, 8192, 32, 8, 128, "fp16", 7),
        # Prompts of up to 4101 tokens that have just been written.
        attn("attn_4_prompts", 4, 4101, 0, 16, 16, 64, "bf16", 5),
    ]


def linear(name, rows, n, k, epilogue, dtype):
    return {"name": name, "kind": "linear", "rows": rows, "n": n, "k": k, "epilogue": epilogue, "dtype": dtype}


def store(name, rows, kv_heads, dim, cache_len, dtype):
    return {"name": name, "kind": "store", "rows": rows, "kv_heads": kv_heads, "dim": dim, "cache_len": cache_len,
            "dtype": dtype}


def attn(name, seqs, longest, past, heads, kv_heads, dim, dtype, lens):
    return {"name": name, "kind": "attn", "seqs": seqs, "longest": longest, "past": past, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "lens": lens}


def between(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


HEADS = [(6, 6, 64), (12, 12, 64), (16, 16, 64), (16, 4, 64), (8, 1, 64), (32, 32, 128), (32, 8, 128), (28, 4, 128),
         (15, 5, 128), (8, 8, 128)]


def draw(rng):
    kind = rng.choice(["linear", "linear", "store", "attn", "attn"])
    heads, kv_heads, dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    lens = rng.randrange(1 << 30)
    if kind == "linear":
        while True:
            case = linear("", between(rng, 1, 16404), 64 * between(rng, 1, 192), 64 * between(rng, 1, 128),
                          rng.choice(["bias", "ls", "ls_resid", "silu"]), dtype)
            if work(case)["flops"] <= work(listed()[4])["flops"] / 2:
                break
    elif kind == "store":
        case = store("", between(rng, 1, 16404), kv_heads, dim, rng.choice([1029, 2305, 4101]), dtype)
    else:
        form = rng.choice(["tokens", "tokens", "chunks", "prompts"])
        while True:
            if form == "tokens":
                case = attn("", between(rng, 1, 256), 1, between(rng, 1, 16384), heads, kv_heads, dim, dtype, lens)
            elif form == "chunks":
                case = attn("", between(rng, 1, 8), between(rng, 2, 512), between(rng, 1, 8192), heads, kv_heads, dim,
                            dtype, lens)
            else:
                case = attn("", between(rng, 1, 24), between(rng, 1, 4101), 0, heads, kv_heads, dim, dtype, lens)
            keys = case["longest"] + case["past"]
            if case["seqs"] * keys * kv_heads * dim <= 1 << 30 and case["seqs"] * heads * case["longest"] * keys <= 1 << 30:
                break
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------
# Lengths of a case's sequences (plain numbers of the case alone, so that every seed has the same shapes)
# ------------------------------------------------------------------------------------------------


def query_lengths(case):
    """New rows of each sequence, the longest among them; one in sixteen has a single one, one in sixteen none."""
    rng = random.Random(case["lens"])
    longest = case["longest"]
    n = [between(rng, max(1, longest // 32), longest) for _ in range(case["seqs"])]
    if longest > 1:
        n = [rng.choice([0, 1]) if rng.random() < 1 / 8 else v for v in n]
    n[rng.randrange(len(n))] = longest
    return n


def key_lengths(case):
    """Keys of each sequence, its new rows' among them."""
    rng = random.Random(case["lens"] + 1)
    q = query_lengths(case)
    if not case["past"]:
        return q
    past = [between(rng, max(1, case["past"] // 32), case["past"]) for _ in q]
    past[rng.randrange(len(past))] = case["past"]
    return [v + p for v, p in zip(q, past)]


def visible(nq, nk):
    """Query-key pairs of one sequence: row i sees the keys up to its own (the last row sees all)."""
    first = nk - nq + 1
    return nq * first + nq * (nq - 1) // 2


# ------------------------------------------------------------------------------------------------
# The two formats in 32 bits
# ------------------------------------------------------------------------------------------------

BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between the e2m1 magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def int8_rows(x):
    """(whole numbers -127 .. 127 as fp32, a scale for each row) of x [M, K]."""
    x = x.float()
    scale = x.abs().amax(-1, keepdim=True) / 127
    codes = torch.where(scale > 0, (x / scale).round().clamp(-127, 127), 0.0)
    return codes, scale[:, 0]


def nvfp4(x, tensor_scale):
    """(codes 0 .. 15 uint8 [.., D], block scales e4m3 [.., D / 16]) of x; tensor_scale broadcasts over [.., D / 16]."""
    x = x.float().unflatten(-1, (-1, 16))
    scale = (x.abs().amax(-1) / 6 / tensor_scale).clamp(2.0 ** -16, 448.0).to(torch.float8_e4m3fn)
    q = x / (tensor_scale * scale.float())[..., None]
    a = q.abs()
    # Ties go to the even code: up from 0.75, 1.75 and 3.5, down from the others.
    code = ((a > BORDERS[0]).to(torch.uint8) + (a >= BORDERS[1]) + (a > BORDERS[2]) + (a >= BORDERS[3])
            + (a > BORDERS[4]) + (a >= BORDERS[5]) + (a > BORDERS[6])) | (torch.signbit(x).to(torch.uint8) << 3)
    return torch.where(scale.float()[..., None] > 0, code, 0).flatten(-2), scale


def nvfp4_values(codes, scales, tensor_scale):
    """fp32 values of packed codes [.., D / 2] with scales [.., D / 16]."""
    both = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    x = table[both.int()].unflatten(-1, (-1, 16)) * scales.float()[..., None]
    return (x * tensor_scale[..., None, None]).flatten(-2)


def packed(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    state = {"case": case}
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    if case["kind"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        channel = torch.where(torch.rand(k, generator=g, device=dev) < 0.01, 10.0, 1.0)
        state["x"] = (normal(rows, k) * channel).to(dtype)
        codes, state["w_scale"] = int8_rows(normal(n, k) * k ** -0.5)
        state["w8"] = codes.to(torch.int8)
        state["bias"] = (0.1 * normal(n)).to(dtype)
        state["gamma"] = (1 + 0.1 * normal(n)).to(dtype) if case["epilogue"] in ("ls", "ls_resid") else None
        state["resid"] = normal(rows, n, dtype=dtype) if case["epilogue"] in ("ls_resid", "silu") else None
        return state
    hk, dim = case["kv_heads"], case["dim"]
    # Scales of the heads as a calibration leaves them: the largest value near the top of the format.
    state["tensor_scale"] = (1 + torch.rand(2, hk, generator=g, device=dev)) * (6.0 / (448 * 6))
    if case["kind"] == "store":
        rows, n = case["rows"], case["cache_len"]
        qkv = normal(rows, 3 * hk, dim, dtype=dtype)  # keys and values lie in the rows of the qkv product
        state["k"], state["v"] = qkv[:, hk:2 * hk], qkv[:, 2 * hk:]
        # Every row has a slot of its own; the last rows of the buffer belong to no sequence.
        used = rows - rows // 64
        batches = max(1, -(-used // n)) if rows > 64 else rows
        slots = torch.randperm(batches * n, generator=g, device=dev)[:used]
        outside = torch.full((rows - used,), -1, device=dev, dtype=torch.long)
        state["batch_idx"] = torch.cat([slots // n, outside])
        state["token_idx"] = torch.cat([slots % n, outside])
        state["used"] = used
        shape = (batches, 2, hk, n)
        # What is read afterwards: the rows written, in another order, and as many slots as may hold older tokens.
        older = torch.randint(0, batches * n, (used,), generator=g, device=dev)
        both = torch.cat([slots, older])[torch.randperm(2 * used, generator=g, device=dev)]
        state["read_batch"], state["read_token"] = both // n, both % n
        state["codes"] = torch.randint(0, 256, (*shape, dim // 2), generator=g, device=dev, dtype=torch.uint8)
        old = torch.randint(1, 120, (*shape, dim // 16), generator=g, device=dev, dtype=torch.uint8)
        state["scales"] = old.view(torch.float8_e4m3fn)
    else:
        nq, nk = query_lengths(case), key_lengths(case)
        state["nq"], state["nk"] = nq, nk
        state["cu_q"] = torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device=dev)
        state["k_lens"] = torch.tensor(nk, dtype=torch.int32, device=dev)
        state["q"] = normal(sum(nq), case["heads"], dim, dtype=dtype)
        made = [nvfp4(normal(2, hk, case["longest"] + case["past"], dim), state["tensor_scale"][:, :, None, None])
                for _ in nk]
        state["codes"] = torch.stack([packed(c) for c, _ in made])
        state["scales"] = torch.stack([s.view(torch.uint8) for _, s in made]).view(torch.float8_e4m3fn)
    # [B, N, 2, heads, ..] as the 16-bit caches are, a head's tokens side by side in memory.
    state["codes"], state["scales"] = (state[x].permute(0, 3, 1, 2, 4) for x in ("codes", "scales"))
    return state


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    return {"linear": run_linear, "store": run_store, "attn": run_attn}[case["kind"]](case, state)


def run_linear(case, state):
    x, w8, bias, gamma, resid = state["x"], state["w8"], state["bias"], state["gamma"], state["resid"]
    if own:
        from appcorr_amd import _lib
        from appcorr_amd import kernels as K

        epilogue = {"bias": _lib.EPI_BIAS, "ls": _lib.EPI_BIAS_LS, "ls_resid": _lib.EPI_BIAS_LS_RESID,
                    "silu": _lib.EPI_BIAS_SILU_MUL}[case["epilogue"]]
        x8, x_scale = K.quantize_int8(x)
        return K.linear_int8(x8, x_scale, w8, state["w_scale"], bias, epilogue=epilogue, gamma=gamma, resid=resid,
                             dtype=x.dtype)
    codes, scale = int8_rows(x)
    y = torch.matmul(codes, w8.float().t()) * (scale[:, None] * state["w_scale"]) + bias.float()
    if case["epilogue"] == "silu":
        y = y / (1 + torch.exp(-y)) * resid.float()
    elif case["epilogue"] != "bias":
        y = y * gamma.float()
        if resid is not None:
            y = y + resid.float()
    return y.to(x.dtype)


def run_store(case, state):
    k, v, codes, scales, ts = state["k"], state["v"], state["codes"], state["scales"], state["tensor_scale"]
    at = state["read_batch"], state["read_token"]
    if own:
        from appcorr_amd import kernels as K

        cache = K.KvNvfp4(codes, scales, ts)
        K.kv_nvfp4_write(k, v, state["batch_idx"], state["token_idx"], cache)
        return K.kv_nvfp4_read(cache, *at, dtype=k.dtype)
    used = state["used"]
    c, s = nvfp4(torch.stack([k[:used], v[:used]], dim=1), ts[:, :, None])
    to = state["batch_idx"][:used], state["token_idx"][:used]
    codes[to] = packed(c)
    scales.view(torch.uint8)[to] = s.view(torch.uint8)
    x = nvfp4_values(codes[at], scales.view(torch.uint8)[at].view(torch.float8_e4m3fn), ts).to(k.dtype)
    return x[:, 0], x[:, 1]


def run_attn(case, state):
    q, codes, scales, ts = state["q"], state["codes"], state["scales"], state["tensor_scale"]
    scale = case["dim"] ** -0.5
    if own:
        from appcorr_amd import kernels as K

        return K.packed_attention_nvfp4(q, K.KvNvfp4(codes, scales, ts), state["cu_q"], state["k_lens"], scale,
                                        causal=True)
    # All sequences at once, their rows padded to the longest.
    seqs, n, _, hk, _ = codes.shape
    d, longest, h = case["dim"], case["longest"], case["heads"]
    first, k_lens = state["cu_q"][:-1].long(), state["k_lens"].long()
    q_lens = state["cu_q"][1:].long() - first
    i = torch.arange(longest, device=q.device)
    there = i < q_lens[:, None]
    row = torch.where(there, first[:, None] + i, 0)
    qg = q.float()[row].view(seqs, longest, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(seqs * hk, -1, d)
    k = nvfp4_values(codes[:, :, 0], scales[:, :, 0], ts[0])
    kt = k.permute(0, 2, 3, 1).reshape(seqs * hk, d, n).contiguous()
    p = torch.bmm(qg, kt).view(seqs, hk, h // hk, longest, n) * scale
    del k, kt
    last = (k_lens - q_lens)[:, None] + i
    last = torch.minimum(last, k_lens[:, None] - 1)
    p.masked_fill_(torch.arange(n, device=q.device) > last[:, None, None, :, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    v = nvfp4_values(codes[:, :, 1], scales[:, :, 1], ts[1]).transpose(1, 2).reshape(seqs * hk, n, d)
    o = torch.bmm(p.view(seqs * hk, -1, n), v).view(seqs, hk, h // hk, longest, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(seqs * longest, h * d)
    # The rows back to where they came from; padding goes to a row past the end.
    out = torch.empty(q.shape[0] + 1, h * d, dtype=q.dtype, device=q.device)
    out[torch.where(there, row, q.shape[0]).view(-1)] = o.to(q.dtype)
    return out[:-1]


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without, and its values in 64 bits
# ------------------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        extra = {"bias": 0, "ls": 0, "ls_resid": 1, "silu": 1}[case["epilogue"]]
        side = 2 * n * (2 if case["epilogue"] in ("ls", "ls_resid") else 1) + 4 * n
        return {"bytes": 2 * rows * k + n * k + 2 * rows * n * (1 + extra) + side, "flops": 2 * rows * n * k}
    hk, dim = case["kv_heads"], case["dim"]
    row4 = 2 * hk * (dim // 2 + dim // 16)  # a token's keys and values in 4 bits with their scales
    if case["kind"] == "store":
        used = case["rows"] - case["rows"] // 64
        row16 = 2 * hk * dim * 2
        return {"bytes": used * (row16 + row4) + case["rows"] * 16 + 2 * used * (row4 + row16 + 16),
                "flops": 6 * used * hk * dim}
    nq, nk = query_lengths(case), key_lengths(case)
    pairs = sum(visible(a, b) for a, b in zip(nq, nk))
    keys = sum(b for a, b in zip(nq, nk) if a)
    return {"bytes": 4 * dim * case["heads"] * sum(nq) + row4 * keys, "flops": 4 * dim * case["heads"] * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    return {"linear": exact_linear, "store": exact_store, "attn": exact_attn}[case["kind"]](case, state)


def exact_linear(case, state):
    x = state["x"].double()
    # The scale is a number of 32 bits; a whole number is the one nearest to the quotient.
    step = (x.abs().max(dim=1).values / 127).float().double()
    whole = torch.round(x / step.clamp(min=1e-300)[:, None])
    w = state["w8"].double() * state["w_scale"].double()[:, None]
    y = (whole * step[:, None]) @ w.T + state["bias"].double()
    if case["epilogue"] == "silu":
        return y * torch.sigmoid(y) * state["resid"].double()
    if state["gamma"] is not None:
        y *= state["gamma"].double()
    return y if state["resid"] is None else y + state["resid"].double()


def e4m3_grid(device):
    """The positive values of e4m3 by code, 0 .. 126."""
    c = torch.arange(127, device=device, dtype=torch.float64)
    e, m = (c / 8).floor(), c % 8
    return torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7))


def nearest(values, grid):
    """Index of the grid's value nearest to each value >= 0, ties to the even index."""
    hi = torch.searchsorted(grid, values.contiguous()).clamp(1, len(grid) - 1)
    up, down = grid[hi] - values, values - grid[hi - 1]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def exact_values(codes, scales):
    """Values [.., D] of packed codes and scale bytes without the tensor scale, in 64 bits."""
    grid = e4m3_grid(codes.device)[scales.view(torch.uint8).long()]
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    level = torch.tensor(MAGNITUDES, dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes.long() >> (4 * half)) & 15
        out[..., half::2] = level[c % 8] * (1 - 2 * (c // 8))
    return out * grid.repeat_interleave(16, dim=-1)


def exact_store(case, state):
    ts = state["tensor_scale"].double()
    grid = e4m3_grid(ts.device)
    level = torch.tensor(MAGNITUDES, dtype=torch.float64, device=ts.device)
    used, n = state["used"], case["cache_len"]
    slot = state["batch_idx"][:used] * n + state["token_idx"][:used]
    wanted = state["read_batch"] * n + state["read_token"]
    written = torch.full((state["codes"].shape[0] * n,), -1, dtype=torch.long, device=ts.device)
    written[slot] = torch.arange(used, device=ts.device)
    source = written[wanted]
    at = state["read_batch"], state["read_token"]
    out = []
    for which, x in ((0, state["k"]), (1, state["v"])):
        x = x.double().unflatten(-1, (-1, 16))
        t = ts[which][:, None]
        s = grid[nearest((x.abs().amax(-1) / (6 * t)).clamp(max=448), grid)]
        # (the divisor of a block is a number of 32 bits)
        unit = (t * s).float().double()[..., None]
        y = torch.sign(x) * level[nearest(torch.where(unit > 0, x.abs() / unit, 0.0), level)] * (t * s)[..., None]
        old = exact_values(state["codes"][at][:, which], state["scales"].view(torch.uint8)[at][:, which]) \
            * ts[which][:, None]
        out.append(torch.where((source >= 0)[:, None, None], y.flatten(-2)[source.clamp(min=0)], old))
    return tuple(out)


def exact_attn(case, state):
    q, h, hk, d = state["q"], case["heads"], case["kv_heads"], case["dim"]
    ts = state["tensor_scale"].double()
    out = torch.zeros(q.shape[0], h, d, dtype=torch.float64, device=q.device)
    at = 0
    for s, (a, b) in enumerate(zip(state["nq"], state["nk"])):
        for j in range(hk if a else 0):
            k, v = (exact_values(state["codes"][s, :b, w, j], state["scales"][s, :b, w, j]) * ts[w, j] for w in (0, 1))
            kt = k.T.contiguous()
            for head in range(j * (h // hk), (j + 1) * (h // hk)):
                for r in range(0, a, 4096):  # rows in blocks
                    e = min(a, r + 4096)
                    z = q[at + r:at + e, head].double() @ kt / math.sqrt(d)
                    if e > r + 1 or a > 1:
                        seen = torch.arange(r, e, device=q.device)[:, None] + (b - a)
                        z.masked_fill_(torch.arange(b, device=q.device) > seen, -math.inf)
                    out[at + r:at + e, head] = torch.softmax(z, -1) @ v
        at += a
    return out.view(-1, h * d)
