"""Workloads of the packed-sequence operators: one layer's steps over crops, frames and streams of different lengths.

A server answers requests of different lengths side by side: their rows lie packed one after another, sequence s in
rows cu_q[s] .. cu_q[s + 1] - 1, and their keys either packed the same way (a prompt with nothing cached) or in a
[B, N, 2, H, Dh] K/V cache (sequence s in batch s). Four operators, in the order in which a layer uses them:

  plan  packed_plan: row offsets, key lengths and every row's cache slot from the requests' lengths;
  rope  apply_rope_axes: q and k rotated by positions with several axes (time, height, width);
  norm  qk_norm_rope_kv: per-head norm of q and k, rotation, K/V rows written into the cache, one pass;
  attn  packed_attention: grouped-head attention of every row over its own sequence's keys, causal or not.

Head counts and lengths are those of this package's configurations (16 x 64, 32 x 128, 6 x 64 heads; 201, 764, 1029
and 4101 tokens) or generic ones (32 query heads over 8 key heads, lengths of powers of two). Queries and keys are
N(0, 1) as normed heads are, values N(0, 1), positions those of frames cut into patches.
"""

from __future__ import annotations

import math
import random

import torch

own = False  # False: elementary torch operations in 32 (angles 64) bits; True: this package's operators

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # Four streams that add one token each to what they have cached: the smallest plan.
        plan("plan_4_tokens", 4, 1, 4, 1029, 1),
        # A burst of requests of up to 1029 tokens with a cache of 4101 each, the row buffer longer than they need.
        plan("plan_256_requests", 256, 1029, 131072, 4101, 2),
        # One small image (224 px, 201 tokens) of the smallest backbone, patch coordinates on two axes.
        rope("rope_201x6_image", 201, 6, 6, 64, "float", 2, "bf16"),
        # Four frames of 1024 px, (time, height, width), grouped keys, half of each head rotated.
        rope("rope_16404x32_grouped", 16404, 32, 8, 128, "long", 3, "fp16", rotated=64),
        # One token of each of 32 streams.
        norm("norm_32_tokens", 32, 32, 8, 128, "long", 3, "bf16", False, 1029),
        # Four images of 512 px with LayerNormed heads and patch coordinates.
        norm("norm_4116x16_layernorm", 4116, 16, 16, 64, "float", 2, "bf16", True, 1029),
        # Four images of 1024 px at the largest backbone's width, grouped keys.
        norm("norm_16404x32_grouped", 16404, 32, 8, 128, "long", 3, "bf16", False, 4101),
        # One token of each of four streams against short caches: latency.
        attn("attn_4_tokens", 4, 1, 1029, 16, 16, 64, "cache", True, "bf16", 3),
        # One token of each of 32 streams against caches of up to 16384 keys.
        attn("attn_32_tokens_long", 32, 1, 16384, 32, 8, 128, "cache", True, "bf16", 4),
        # Crops of up to 1029 tokens side by side, every token sees its crop: no mask, packed keys.
        attn("attn_24_crops", 24, 1029, 0, 16, 16, 64, "packed", False, "bf16", 5),
        # The next 512 rows at most of three long streams, whose earlier rows are cached.
        attn("attn_3_chunks", 3, 512, 8192, 32, 8, 128, "cache", True, "fp16", 7),
        # Prompts of up to 16384 tokens, causal, grouped heads: the largest.
        attn("attn_prompts_16384", 6, 16384, 0, 32, 8, 128, "packed", True, "bf16", 6),
    ]


def plan(name, seqs, longest, rows, cache_len, lens):
    return {"name": name, "kind": "plan", "seqs": seqs, "longest": longest, "rows": rows, "cache_len": cache_len,
            "lens": lens}


def rope(name, rows, heads, kv_heads, dim, positions, axes, dtype, rotated=0):
    return {"name": name, "kind": "rope", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotated": rotated or dim, "positions": positions, "axes": axes, "dtype": dtype}


def norm(name, rows, heads, kv_heads, dim, positions, axes, dtype, layer_norm, cache_len):
    return {"name": name, "kind": "norm", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotated": dim, "positions": positions, "axes": axes, "dtype": dtype, "layer_norm": layer_norm,
            "cache_len": cache_len}


def attn(name, seqs, longest, past, heads, kv_heads, dim, keys, causal, dtype, lens):
    return {"name": name, "kind": "attn", "seqs": seqs, "longest": longest, "past": past, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "keys": keys, "causal": causal, "dtype": dtype, "lens": lens}


def between(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


HEADS = [(6, 6, 64), (12, 12, 64), (16, 16, 64), (16, 4, 64), (8, 1, 64), (32, 32, 128), (32, 8, 128), (28, 4, 128),
         (15, 5, 128), (8, 8, 128)]


def draw(rng):
    kind = rng.choice(["plan", "rope", "norm", "attn", "attn", "attn"])
    heads, kv_heads, dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    positions, axes = rng.choice([("long", 1), ("long", 3), ("float", 2), ("long", 2)])
    lens = rng.randrange(1 << 30)
    if kind == "plan":
        seqs = between(rng, 1, 256)
        longest = between(rng, 1, 1029)
        case = plan("", seqs, longest, 1, between(rng, longest, 16384), lens)
        case["rows"] = min(131072, max(1, int(sum(query_lengths(case)) * rng.choice([1.0, 1.0, 1.3]))))
    elif kind == "rope":
        rows = between(rng, 1, 16404)
        case = rope("", rows, heads, kv_heads, dim, positions, axes, dtype, rng.choice([dim, dim, dim // 2]))
    elif kind == "norm":
        rows = between(rng, 1, 16404)
        case = norm("", rows, heads, kv_heads, dim, positions, axes, dtype, rng.choice([False, False, True]),
                    rng.choice([1029, 2305, 4101]))
    else:
        form = rng.choice(["tokens", "chunks", "prompts", "crops"])
        while True:
            if form == "tokens":
                case = attn("", between(rng, 1, 64), 1, between(rng, 1, 16384), heads, kv_heads, dim, "cache",
                            True, dtype, lens)
            elif form == "chunks":
                case = attn("", between(rng, 1, 8), between(rng, 2, 512), between(rng, 1, 8192), heads, kv_heads, dim,
                            "cache", True, dtype, lens)
            else:
                case = attn("", between(rng, 1, 24), between(rng, 1, 8192), 0, heads, kv_heads, dim, "packed",
                            form == "prompts", dtype, lens)
            at_most = work(listed()[-1])
            if case["seqs"] * (case["longest"] + case["past"]) * kv_heads * dim <= 1 << 30 and \
                    work(case)["flops"] <= at_most["flops"] / 4:
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


def visible(nq, nk, causal):
    """Query-key pairs of one sequence: row i sees the keys up to its own (the last row sees all)."""
    if not causal:
        return nq * nk
    first = nk - nq + 1  # keys that row 0 sees
    return sum_from(first, nq) if first >= 1 else sum_from(1, max(0, nk))


def sum_from(first, count):
    return count * first + count * (count - 1) // 2


def axis_sections(case):
    """How many of the rotated / 2 frequencies each axis has: time the fewest."""
    half, axes = case["rotated"] // 2, case["axes"]
    if axes == 1:
        return (half,)
    if axes == 2:
        return (half // 2, half - half // 2)
    t = half // 4
    h = (half - t) // 2
    return (t, h, half - t - h)


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    state = {"case": case}

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    if case["kind"] == "plan":
        # The new rows of the requests in another order for each seed, and what each has cached already.
        q_lens = torch.tensor(query_lengths(case), device=dev)[torch.randperm(case["seqs"], generator=g, device=dev)]
        past = torch.randint(0, case["cache_len"], (case["seqs"],), generator=g, device=dev)
        state["q_lens"], state["k_lens"] = q_lens, (q_lens + past).clamp(max=case["cache_len"])
        return state

    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("rope", "norm"):
        rows = case["rows"]
        # q, k and v lie side by side in the rows of the qkv product.
        state["qkv"] = normal(rows, heads + 2 * kv_heads, dim, dtype=dtype)
        if case["positions"] == "long":  # frame number, patch row, patch column; streams run for hours
            top = torch.tensor([1 << 20, 64, 64][:case["axes"]], device=dev)
            state["positions"] = (torch.rand(rows, case["axes"], generator=g, device=dev, dtype=torch.float64)
                                  * top).long()
        else:  # patch centres in -1 .. 1
            state["positions"] = torch.rand(rows, case["axes"], generator=g, device=dev) * 2 - 1
        half = case["rotated"] // 2
        span = torch.arange(half, dtype=torch.float64) / half
        freq = 10000.0 ** -span if case["positions"] == "long" else 2 * math.pi * 100.0 ** -span
        state["inv_freq"] = freq.float().to(dev)
        state["sections"] = axis_sections(case)
    if case["kind"] == "norm":
        for name in ("q", "k"):
            state[name + "_weight"] = (1 + 0.1 * normal(dim)).to(dtype)
            state[name + "_bias"] = (0.1 * normal(dim)).to(dtype) if case["layer_norm"] else None
        n = case["cache_len"]
        # Every row has a slot of its own; the last rows of the buffer belong to no sequence.
        used = rows - rows // 64
        batches = max(1, -(-used // n)) if rows > 64 else rows
        slots = torch.randperm(batches * n, generator=g, device=dev)[:used]
        outside = torch.full((rows - used,), -1, device=dev, dtype=torch.long)
        state["batch_idx"] = torch.cat([slots // n, outside])
        state["token_idx"] = torch.cat([slots % n, outside])
        state["used"] = used
        state["kv_cache"] = torch.zeros(batches, n, 2, kv_heads, dim, device=dev, dtype=dtype)
        state["q_out"] = torch.zeros(rows, heads, dim, device=dev, dtype=dtype)
    if case["kind"] == "attn":
        nq, nk = query_lengths(case), key_lengths(case)
        state["nq"], state["nk"] = nq, nk
        state["cu_q"] = torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device=dev)
        if case["keys"] == "packed":
            qkv = normal(sum(nq), heads + 2 * kv_heads, dim, dtype=dtype)
            state["q"], state["k"], state["v"] = qkv.split([heads, kv_heads, kv_heads], dim=1)
        else:
            state["q"] = normal(sum(nq), heads, dim, dtype=dtype)
            kv = normal(len(nk), case["longest"] + case["past"], 2, kv_heads, dim, dtype=dtype)
            state["k"], state["v"] = kv[:, :, 0], kv[:, :, 1]
            state["k_lens"] = torch.tensor(nk, dtype=torch.int32, device=dev)
    return state


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    return {"plan": run_plan, "rope": run_rope, "norm": run_norm, "attn": run_attn}[case["kind"]](case, state)


def run_plan(case, state):
    if own:
        from appcorr_amd import kernels as K

        p = K.packed_plan(state["q_lens"], state["k_lens"], case["rows"], cache_len=case["cache_len"])
        return p.cu_q, p.k_lens, p.cu_k, p.batch_idx, p.token_idx
    rows, n = case["rows"], case["cache_len"]
    zero = torch.zeros(1, dtype=torch.long, device=state["q_lens"].device)
    cu_q = torch.cat([zero, state["q_lens"].clamp(min=0).cumsum(0)]).clamp(max=rows)
    nk = state["k_lens"].clamp(0, n)
    cu_k = torch.cat([zero, nk.cumsum(0)])
    row = torch.arange(rows, device=cu_q.device)
    seq = torch.searchsorted(cu_q[1:].contiguous(), row, right=True)
    inside = seq < nk.numel()
    seq_in = seq.clamp(max=nk.numel() - 1)
    token = nk[seq_in] - cu_q[seq_in + 1] + row
    inside = inside & (token >= 0)
    return cu_q.int(), nk.int(), cu_k, torch.where(inside, seq, -1), torch.where(inside, token, -1)


def run_rope(case, state):
    qkv = state["qkv"]
    h, hk = case["heads"], case["kv_heads"]
    q, k = qkv[:, :h], qkv[:, h:h + hk]
    if own:
        from appcorr_amd import kernels as K

        return K.apply_rope_axes(q, k, state["positions"], state["inv_freq"], state["sections"])
    cos, sin = angles(state)
    return rotated(q.float(), cos, sin).to(q.dtype), rotated(k.float(), cos, sin).to(k.dtype)


def angles(state):
    """cos and sin [rows, 1, R / 2] of position (of the frequency's axis) times frequency, in 64 bits until here."""
    axis = torch.cat([torch.full((n,), a, dtype=torch.long, device=state["qkv"].device)
                      for a, n in enumerate(state["sections"])])
    angle = state["positions"].double()[:, axis] * state["inv_freq"].double()
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def rotated(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)


def run_norm(case, state):
    h, hk = case["heads"], case["kv_heads"]
    qkv = state["qkv"]
    if own:
        from appcorr_amd import kernels as K

        K.qk_norm_rope_kv(qkv, h, hk, (state["q_weight"], state["q_bias"]), (state["k_weight"], state["k_bias"]), 1e-6,
                          state["positions"], state["inv_freq"], state["sections"], state["batch_idx"],
                          state["token_idx"], state["kv_cache"], state["q_out"], layer_norm=case["layer_norm"])
        return state["q_out"], state["kv_cache"]
    cos, sin = angles(state)
    used = state["used"]
    q, k, v = qkv.split([h, hk, hk], dim=1)
    q = rotated(normed(q, state["q_weight"], state["q_bias"], case["layer_norm"]), cos, sin).to(qkv.dtype)
    k = rotated(normed(k, state["k_weight"], state["k_bias"], case["layer_norm"]), cos, sin).to(qkv.dtype)
    state["q_out"][:used] = q[:used]
    at = state["batch_idx"][:used], state["token_idx"][:used]
    state["kv_cache"][at] = torch.stack([k, v], dim=1)[:used]
    return state["q_out"], state["kv_cache"]


def normed(x, weight, bias, layer_norm):
    x = x.float()
    if layer_norm:
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    return x + bias.float() if bias is not None else x


def run_attn(case, state):
    q, k, v = state["q"], state["k"], state["v"]
    scale = case["dim"] ** -0.5
    packed = case["keys"] == "packed"
    if own:
        from appcorr_amd import kernels as K

        return K.packed_attention(q, k, v, state["cu_q"], state["cu_q"] if packed else state["k_lens"], scale,
                                  causal=case["causal"])
    if not packed:
        return attn_cached(case, state, scale)
    outs, at = [], 0
    for n in state["nq"]:  # sequence by sequence: padded to the longest they would not fit
        outs.append(attn_sequence(q[at:at + n], k[at:at + n], v[at:at + n], scale, case["causal"]))
        at += n
    return torch.cat(outs)


def attn_sequence(q, k, v, scale, causal):
    """Every row of q [n, H, D] over the keys k, v [n, Hk, D] of its sequence -> [n, H D]."""
    n, h, d = q.shape
    hk = k.shape[1]
    if n == 0:
        return q.reshape(0, h * d)
    qg = q.float().view(n, hk, h // hk, d).permute(1, 2, 0, 3).contiguous()
    kt = k.float().permute(1, 2, 0).contiguous()
    vg = v.float().transpose(0, 1).contiguous()
    hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1) if causal else None
    out = torch.empty_like(qg)
    for i in range(hk):  # a key head at a time keeps the scores of the longest sequence in memory
        p = torch.matmul(qg[i].view(-1, d), kt[i]).view(h // hk, n, n).mul_(scale)
        if causal:
            p.masked_fill_(hidden, -math.inf)
        p.sub_(p.amax(-1, keepdim=True)).exp_()
        total = p.sum(-1, keepdim=True)
        out[i] = torch.matmul(p.view(-1, n), vg[i]).view(h // hk, n, d) / total
    return out.permute(2, 0, 1, 3).reshape(n, h * d).to(q.dtype)


def attn_cached(case, state, scale):
    """All sequences at once, their rows padded to the longest."""
    q, k, v = state["q"], state["k"], state["v"]
    seqs, n, hk, d = k.shape
    longest, h = case["longest"], case["heads"]
    first, k_lens = state["cu_q"][:-1].long(), state["k_lens"].long()
    q_lens = state["cu_q"][1:].long() - first
    i = torch.arange(longest, device=q.device)
    there = i < q_lens[:, None]
    row = torch.where(there, first[:, None] + i, 0)
    qg = q.float()[row].view(seqs, longest, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(seqs * hk, -1, d)
    kt = k.float().permute(0, 2, 3, 1).reshape(seqs * hk, d, n).contiguous()
    p = torch.bmm(qg, kt).view(seqs, hk, h // hk, longest, n) * scale
    last = (k_lens - q_lens)[:, None] + i if case["causal"] else (k_lens - 1)[:, None].expand(-1, longest)
    last = torch.minimum(last, k_lens[:, None] - 1)
    p = p.masked_fill(torch.arange(n, device=q.device) > last[:, None, None, :, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    vg = v.float().transpose(1, 2).reshape(seqs * hk, n, d)
    o = torch.bmm(p.view(seqs * hk, -1, n), vg).view(seqs, hk, h // hk, longest, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(seqs * longest, h * d)
    # The rows back to where they came from; padding goes to a row past the end.
    out = torch.empty(q.shape[0] + 1, h * d, dtype=q.dtype, device=q.device)
    out[torch.where(there, row, q.shape[0]).view(-1)] = o.to(q.dtype)
    return out[:-1]


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without, and its values in 64 bits
# ------------------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "plan":
        return {"bytes": case["seqs"] * (16 + 4 + 4 + 8) + case["rows"] * 16, "flops": 2 * case["rows"]}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("rope", "norm"):
        rows = case["rows"]
        side = rows * case["axes"] * (8 if case["positions"] == "long" else 4) + case["rotated"] * 2
        if case["kind"] == "rope":
            n = rows * (heads + kv_heads) * dim
            return {"bytes": 4 * n + side, "flops": 3 * n}
        rows -= rows // 64
        n = rows * (heads + 2 * kv_heads) * dim
        return {"bytes": 4 * n + side + case["rows"] * 16 + 4 * dim, "flops": 7 * rows * (heads + kv_heads) * dim}
    nq, nk = query_lengths(case), key_lengths(case)
    pairs = sum(visible(a, b, case["causal"]) for a, b in zip(nq, nk))
    keys = sum(b for a, b in zip(nq, nk) if a)
    return {"bytes": 2 * dim * (2 * heads * sum(nq) + 2 * kv_heads * keys), "flops": 4 * dim * heads * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "plan":
        return exact_plan(case, state)
    if case["kind"] == "attn":
        return exact_attn(case, state)
    h, hk = case["heads"], case["kv_heads"]
    x = state["qkv"].double()
    turn, at = [], 0
    for axis, count in enumerate(state["sections"]):
        turn.append(state["positions"][:, axis].double().outer(state["inv_freq"][at:at + count].double()))
        at += count
    unit = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), torch.cat(turn, 1))[:, None]

    def turned(y):
        z = torch.complex(y[..., :at], y[..., at:2 * at]) * unit
        return torch.cat([z.real, z.imag, y[..., 2 * at:]], -1)

    if case["kind"] == "rope":
        return turned(x[:, :h]), turned(x[:, h:h + hk])
    parts = []
    for name, y in (("q", x[:, :h]), ("k", x[:, h:h + hk])):
        if case["layer_norm"]:
            y = y - y.sum(-1, keepdim=True) / case["dim"]
        y = y / ((y ** 2).sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt() * state[name + "_weight"].double()
        if case["layer_norm"]:
            y = y + state[name + "_bias"].double()
        parts.append(turned(y))
    used = state["used"]
    q_out, kv = state["q_out"].double(), state["kv_cache"].double()
    q_out[:used] = parts[0][:used]
    flat = kv.view(-1, 2, hk, case["dim"])
    slot = state["batch_idx"][:used] * case["cache_len"] + state["token_idx"][:used]
    flat[slot, 0] = parts[1][:used]
    flat[slot, 1] = x[:used, h + hk:]
    return q_out, kv


def exact_plan(case, state):
    rows, cu_q, cu_k, nk = case["rows"], [0], [0], []
    batch, token = [], []
    for s, (a, b) in enumerate(zip(state["q_lens"].tolist(), state["k_lens"].tolist())):
        b = min(b, case["cache_len"])
        a = min(a, rows - cu_q[-1])
        nk.append(b)
        cu_q.append(cu_q[-1] + a)
        cu_k.append(cu_k[-1] + b)
        where = range(b - a, b)
        batch += [s if t >= 0 else -1 for t in where]
        token += [t if t >= 0 else -1 for t in where]
    batch += [-1] * (rows - len(batch))
    token += [-1] * (rows - len(token))
    return (torch.tensor(cu_q, dtype=torch.int32), torch.tensor(nk, dtype=torch.int32), torch.tensor(cu_k),
            torch.tensor(batch), torch.tensor(token))


def exact_attn(case, state):
    q, k, v = state["q"], state["k"], state["v"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(q.shape[0], h, d, dtype=torch.float64, device=q.device)
    at = 0
    for s, (a, b) in enumerate(zip(state["nq"], state["nk"])):
        ks, vs = (k[at:at + b], v[at:at + b]) if case["keys"] == "packed" else (k[s, :b], v[s, :b])
        for head in range(h if b else 0):
            kk, vv = ks[:, head * hk // h].double(), vs[:, head * hk // h].double()
            for r in range(0, a, 4096):  # rows in blocks
                e = min(a, r + 4096)
                z = q[at + r:at + e, head].double() @ kk.T.contiguous() / math.sqrt(d)
                if case["causal"]:
                    seen = torch.arange(r, e, device=q.device)[:, None] + (b - a)
                    z = z.where(torch.arange(b, device=q.device) <= seen, torch.tensor(-math.inf, dtype=torch.float64,
                                                                                     device=q.device))
                    z = torch.softmax(z, -1).nan_to_num(0.0)
                else:
                    z = torch.softmax(z, -1)
                out[at + r:at + e, head] = z @ vv
        at += a
    return out.view(-1, h * d)
