"""What the decode-step operators are measured on: one token step of an attention block over a paged cache, with its products in block-scaled 8-bit floating point.

    quantize_blocks      x [M,K] -> e4m3 values and one fp32 scale per 1 x 128 (activations) or 128 x 128 (weights) block
    matmul_f8_blocks     C[M,N] = sum over 128-wide blocks of K of  a_scale * b_scale * (A_block . B_block^T)
    cache_append         rotates the new tokens' queries and keys by their positions and writes keys and values into cache pages
    sdpa_shared_prefix   attention of a batch whose sequences share one long prefix, each with a suffix of its own, over those pages

A case is a dict of plain values; `run` computes it in elementary torch operations, or - with `own` set - by the
library's operators.  Sizes are the weight-only and 8-bit configurations of bench.py (N = 14336, K = 4096, and the way
back), 32 query heads of 128 as in its attention, and ragged ones around them.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
#: A block's largest magnitude is taken to be at least this, so that neither its scale nor the scale's reciprocal leaves the normal fp32 range.
AMAX_FLOOR = 2.0 ** -110
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the activations of one token on their way into a product: launch latency
        {"name": "quantise 1 token", "op": "quantize", "m": 1, "k": 4096, "dtype": "bf16", "block_rows": 1},
        # the activations of a prefill in front of the way back from the wide layer: a stream through memory
        {"name": "quantise prefill", "op": "quantize", "m": 4096, "k": 14336, "dtype": "bf16", "block_rows": 1},
        # one token through the wide layer: the weights are read once
        {"name": "f8 product 1 token", "op": "matmul", "m": 1, "n": 14336, "k": 4096, "out": "bf16"},
        # a ragged batch of tokens, no extent a multiple of a tile
        {"name": "f8 product ragged", "op": "matmul", "m": 61, "n": 4100, "k": 4176, "out": "f16"},
        # a chunk of a prompt through the way back: few tiles, a long sum
        {"name": "f8 product 512 rows", "op": "matmul", "m": 512, "n": 4096, "k": 14336, "out": "bf16"},
        # a prefill through the wide layer: tensor-core rate
        {"name": "f8 product prefill", "op": "matmul", "m": 4096, "n": 14336, "k": 4096, "out": "bf16"},
        # a decode step's new tokens, eight of them padding of a captured batch: launch latency
        {"name": "append decode", "op": "append", "tokens": 64, "padding": 8, "hq": 32, "hkv": 8, "d": 128, "rotary": 128, "page": 16,
         "pages": 2048, "positions": 32768, "dtype": "bf16", "interleaved": False},
        # a prefill's tokens, half of each head rotated, pairs side by side
        {"name": "append prefill", "op": "append", "tokens": 8191, "padding": 0, "hq": 32, "hkv": 8, "d": 128, "rotary": 64, "page": 64,
         "pages": 256, "positions": 131072, "dtype": "f16", "interleaved": True},
        # four sequences behind a short instruction: latency
        {"name": "prefix 512, 4 sequences", "op": "prefix", "batch": 4, "queries": 1, "prefix": 512, "suffix": 64, "hq": 32, "hkv": 8,
         "d": 128, "page": 16, "dtype": "bf16"},
        # a decode batch behind a long document, suffixes of every length up to 1024
        {"name": "prefix 8192, 64 sequences", "op": "prefix", "batch": 64, "queries": 1, "prefix": 8192, "suffix": 1024, "hq": 32, "hkv": 8,
         "d": 128, "page": 16, "dtype": "bf16"},
        # up to five drafted tokens a sequence, an odd number of query heads per key head, a prefix that ends inside a page
        {"name": "prefix 4999, drafted", "op": "prefix", "batch": 48, "queries": 5, "prefix": 4999, "suffix": 300, "hq": 20, "hkv": 4,
         "d": 64, "page": 64, "dtype": "f16"},
        # a large batch behind a very long prefix: tensor-core rate
        {"name": "prefix 32768, 256 sequences", "op": "prefix", "batch": 256, "queries": 1, "prefix": 32768, "suffix": 512, "hq": 32, "hkv": 8,
         "d": 128, "page": 32, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number from [low, high], its logarithm uniform."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "append", "prefix", "prefix"])
    if op == "quantize":
        return {"op": op, "m": _spread(rng, 1, 4096), "k": _spread(rng, 64, 14336), "dtype": rng.choice(["bf16", "f16", "f32"]),
                "block_rows": rng.choice([1, 1, 128])}
    if op == "matmul":
        return {"op": op, "m": _spread(rng, 1, 4096), "n": _spread(rng, 512, 14336), "k": 16 * _spread(rng, 16, 256), "out": rng.choice(["bf16", "f16"])}
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "f16"])
    if op == "append":
        tokens = _spread(rng, 1, 8191)
        return {"op": op, "tokens": tokens, "padding": rng.choice([0, tokens // 4]), "hq": hq, "hkv": hkv, "d": d, "rotary": rng.choice([d, d // 2]),
                "page": page, "pages": (2 * tokens + page - 1) // page + 1, "positions": _spread(rng, 1024, 131072), "dtype": dtype,
                "interleaved": rng.random() < 0.5}
    return {"op": op, "batch": _spread(rng, 1, 192), "queries": rng.choice([1, 1, 1, 3]), "prefix": _spread(rng, 64, 16384),
            "suffix": _spread(rng, 4, 512), "hq": hq, "hkv": hkv, "d": d, "page": page, "dtype": dtype}


def _blocks(n, size=BLOCK):
    return -(-n // size)


def _prefix_layout(case):
    """(query counts, suffix lengths) of the case's sequences before they are put in an order: the lengths are spread evenly over
    [queries, suffix], the counts over [1, queries]."""
    b, most = case["batch"], case["queries"]
    counts = [1 + i % most for i in range(b)]
    low = min(most, case["suffix"])
    lengths = [low + (case["suffix"] - low) * (i + 1) // b for i in range(b)]
    return counts, lengths


# ------------------------------------------------------------------------------------------------ inputs

def _scaled_values(shape, block, generator, device):
    """What a quantiser leaves: e4m3 values whose blocks reach the format's largest magnitude, and their scales."""
    rows, cols = shape
    x = torch.randn(rows, cols, generator=generator, device=device)
    # channels of unequal strength, as activations and weights have them
    x *= torch.exp(0.5 * torch.randn(cols, generator=generator, device=device))
    q, scale = _quantize_plain(x, block)
    pitch = _blocks(cols, 16) * 16
    stored = torch.zeros(rows, pitch, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)[:, :cols]
    stored.view(torch.uint8).copy_(q.view(torch.uint8))
    return stored, scale


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "quantize":
        x = torch.randn(case["m"], case["k"], generator=g, device=device)
        x *= torch.exp(torch.randn(1, case["k"], generator=g, device=device))
        s["x"] = x.to(DTYPES[case["dtype"]])
    elif op == "matmul":
        s["a"], s["a_scale"] = _scaled_values((case["m"], case["k"]), 1, g, device)
        s["b"], s["b_scale"] = _scaled_values((case["n"], case["k"]), BLOCK, g, device)
    elif op == "append":
        t, hq, hkv, d, dtype = case["tokens"], case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
        # one projection's result: the three are views of it, as a fused product leaves them
        fused = torch.randn(t, (hq + 2 * hkv) * d, generator=g, device=device).to(dtype)
        s["q"], s["k"], s["v"] = (part.unflatten(1, (-1, d)) for part in fused.split([hq * d, hkv * d, hkv * d], dim=1))
        shape = (case["pages"], case["page"], hkv, d)
        s["k_cache"] = torch.randn(shape, generator=g, device=device).to(dtype)
        s["v_cache"] = torch.randn(shape, generator=g, device=device).to(dtype)
        s["slots"] = torch.randperm(case["pages"] * case["page"], generator=g, device=device)[:t].contiguous()
        if case["padding"]:
            s["slots"][t - case["padding"]:] = -1
        s["positions"] = torch.randint(0, case["positions"], (t,), generator=g, device=device)
        half = case["rotary"] // 2
        rate = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
        angle = torch.arange(case["positions"], dtype=torch.float64, device=device)[:, None] * rate
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
    else:
        b, hq, hkv, d, page, dtype = case["batch"], case["hq"], case["hkv"], case["d"], case["page"], DTYPES[case["dtype"]]
        counts, lengths = _prefix_layout(case)
        order = torch.randperm(b, generator=g, device=device)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)[order].contiguous()
        starts = torch.zeros(b + 1, dtype=torch.int32, device=device)
        starts[1:] = torch.tensor(counts, dtype=torch.int32, device=device)[order].cumsum(0)
        s["query_starts"] = starts if case["queries"] > 1 else None
        prefix_pages, width = _blocks(case["prefix"], page), _blocks(case["suffix"], page)
        pages = prefix_pages + b * width
        shape = (pages, page, hkv, d)
        s["k_cache"] = torch.randn(shape, generator=g, device=device, dtype=torch.float32).to(dtype)
        s["v_cache"] = torch.randn(shape, generator=g, device=device, dtype=torch.float32).to(dtype)
        where = torch.randperm(pages, generator=g, device=device).int()
        s["prefix_pages"] = where[:prefix_pages].contiguous()
        s["page_table"] = where[prefix_pages:].reshape(b, width).contiguous()
        s["q"] = torch.randn(sum(counts), hq, d, generator=g, device=device).to(dtype)
        s["scale"] = d ** -0.5
    return s


# ------------------------------------------------------------------------------------------------ one pass

_ops = None


def _operators():
    """torch.ops.vecops_b200, its library loaded once."""
    global _ops
    if _ops is None:
        from vecops_b200 import torch_ops

        torch_ops.load()
        _ops = torch.ops.vecops_b200
    return _ops


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        ops = _operators()
    if op == "quantize":
        return ops.quantize_blocks(s["x"], case["block_rows"]) if own else _quantize_plain(s["x"], case["block_rows"])
    if op == "matmul":
        dtype = DTYPES[case["out"]]
        if own:
            return ops.matmul_f8_blocks(s["a"], s["a_scale"], s["b"], s["b_scale"], dtype)
        return _matmul_plain(s["a"], s["a_scale"], s["b"], s["b_scale"], dtype)
    if op == "append":
        call = ops.cache_append if own else _append_plain
        q = call(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["positions"], s["cos_sin"], case["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    call = ops.sdpa_shared_prefix if own else _prefix_plain
    return call(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"], case["prefix"], s["page_table"], s["lengths"], s["scale"], s["query_starts"])


def _quantize_plain(x, block_rows):
    m, k = x.shape
    rows, cols = _blocks(m, block_rows), _blocks(k)
    padded = torch.nn.functional.pad(x.float(), (0, cols * BLOCK - k, 0, rows * block_rows - m))
    tiles = padded.view(rows, block_rows, cols, BLOCK)
    amax = tiles.abs().amax(dim=(1, 3)).clamp(AMAX_FLOOR, torch.finfo(torch.float32).max)
    scale = amax / E4M3_MAX
    q = (tiles / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(rows * block_rows, cols * BLOCK)[:m, :k], scale


def _matmul_plain(a, a_scale, b, b_scale, dtype):
    m, k = a.shape
    n = b.shape[0]
    af = a.float() * a_scale.repeat_interleave(BLOCK, dim=1)[:, :k]
    bf = b.float() * b_scale.repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
    return (af @ bf.t()).to(dtype)


def _rotate(x, cos, sin, interleaved):
    """x [T,H,D] with its first 2 * cos.shape[1] dims rotated."""
    half = cos.shape[1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if interleaved:
        first, second = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([first * cos - second * sin, second * cos + first * sin], dim=-1).flatten(-2)
    else:
        first, second = turned[..., :half], turned[..., half:]
        turned = torch.cat([first * cos - second * sin, second * cos + first * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _append_plain(q, k, v, k_cache, v_cache, slots, positions, cos_sin, interleaved):
    cos, sin = cos_sin[positions].chunk(2, dim=1)
    valid = slots >= 0
    q_out = (_rotate(q.float(), cos, sin, interleaved) * valid[:, None, None]).to(q.dtype)
    k_new = _rotate(k.float(), cos, sin, interleaved).to(k.dtype)
    # padding rows write what row 0 (a real one) writes, where it writes it
    target = torch.where(valid, slots, slots[0])
    k_cache.view(-1, *k.shape[1:])[target] = torch.where(valid[:, None, None], k_new, k_new[:1])
    v_cache.view(-1, *v.shape[1:])[target] = torch.where(valid[:, None, None], v, v[:1])
    return q_out


def _prefix_parts(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, lengths, query_starts, real):
    """Queries [T,Hkv,G,D], prefix keys and values [P,Hkv,D], each token's suffix keys and values [T,S,Hkv,D] and what it sees of them [T,S]."""
    t, hq, d = q.shape
    hkv, b = k_cache.shape[2], page_table.shape[0]
    queries = q.to(real).view(t, hkv, hq // hkv, d)
    prefix_k, prefix_v = (c[prefix_pages.long()].flatten(0, 1)[:prefix_len].to(real) for c in (k_cache, v_cache))
    token = torch.arange(t, device=q.device, dtype=torch.int32)
    starts = query_starts if query_starts is not None else torch.arange(b + 1, device=q.device, dtype=torch.int32)
    owner = torch.searchsorted(starts, token, right=True) - 1
    sees = lengths[owner] - (starts[owner + 1] - 1 - token)  # a sequence's newest token sees all of its suffix, the one before it one key less
    suffix_k, suffix_v = (c[page_table.long()].flatten(1, 2).to(real)[owner] for c in (k_cache, v_cache))
    seen = torch.arange(suffix_k.shape[1], device=q.device)[None, :] < sees[:, None]
    return queries, prefix_k, prefix_v, suffix_k, suffix_v, seen


def _prefix_plain(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, lengths, scale, query_starts):
    queries, pk, pv, sk, sv, seen = _prefix_parts(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, lengths, query_starts, torch.float32)
    t, hkv, group, d = queries.shape
    rows = queries.permute(1, 0, 2, 3).reshape(hkv, t * group, d)
    on_prefix = (rows @ pk.permute(1, 2, 0)).view(hkv, t, group, -1).transpose(0, 1) * scale
    on_suffix = (queries @ sk.permute(0, 2, 3, 1)) * scale
    on_suffix = on_suffix.masked_fill(~seen[:, None, None, :], -math.inf)
    scores = torch.cat([on_prefix, on_suffix], dim=-1)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    total = p.sum(dim=-1, keepdim=True)
    p_prefix, p_suffix = p[..., :prefix_len], p[..., prefix_len:]
    out = (p_prefix.transpose(0, 1).reshape(hkv, t * group, prefix_len) @ pv.transpose(0, 1)).view(hkv, t, group, d).transpose(0, 1)
    out = out + p_suffix @ sv.transpose(1, 2)
    return (out / total).reshape(t, hkv * group, d).to(q.dtype)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x, rows = s["x"].double(), case["block_rows"]
        m, k = x.shape
        row_block = torch.arange(m, device=x.device) // rows
        col_block = torch.arange(k, device=x.device) // BLOCK
        amax = torch.zeros(_blocks(m, rows) * _blocks(k), dtype=torch.float64, device=x.device)
        index = row_block[:, None] * _blocks(k) + col_block[None, :]
        amax.scatter_reduce_(0, index.reshape(-1), x.abs().reshape(-1), "amax")
        scale = amax.clamp(AMAX_FLOOR, torch.finfo(torch.float32).max) / E4M3_MAX
        # the values before their rounding to 8 bits: what they are measured against
        return x / scale[index], scale.view(_blocks(m, rows), _blocks(k))
    if op == "matmul":
        m, k = s["a"].shape
        n = s["b"].shape[0]
        col = torch.arange(k, device="cuda") // BLOCK
        a = s["a"].float().double() * s["a_scale"].double()[:, col]
        b = s["b"].float().double() * s["b_scale"].double()[torch.arange(n, device="cuda") // BLOCK][:, col]
        return torch.einsum("mk,nk->mn", a, b)
    if op == "append":
        table = s["cos_sin"].double()[s["positions"]]
        half = case["rotary"] // 2
        unit = torch.complex(table[:, :half], table[:, half:])[:, None, :]

        def turned(x):
            x = x.double().clone()
            lanes = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., lanes[0]], x[..., lanes[1]]) * unit
            x[..., lanes[0]], x[..., lanes[1]] = z.real, z.imag
            return x

        real = case["tokens"] - case["padding"]
        page, offset = s["slots"][:real] // case["page"], s["slots"][:real] % case["page"]
        q = turned(s["q"])
        q[real:] = 0
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        k_cache[page, offset] = turned(s["k"])[:real]
        v_cache[page, offset] = s["v"][:real].double()
        return q, k_cache, v_cache
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    starts = s["query_starts"].tolist() if s["query_starts"] is not None else list(range(case["batch"] + 1))
    page, group = case["page"], case["hq"] // case["hkv"]
    shared = torch.arange(case["prefix"], device="cuda")
    shared_pages = s["prefix_pages"].long()[shared // page]
    prefix_k = s["k_cache"][shared_pages, shared % page].double().permute(1, 2, 0)  # [Hkv,D,P]
    prefix_v = s["v_cache"][shared_pages, shared % page].double().transpose(0, 1)   # [Hkv,P,D]
    for i, length in enumerate(s["lengths"].tolist()):
        mine = torch.arange(length, device="cuda")
        pages = s["page_table"][i].long()[mine // page]
        keys = s["k_cache"][pages, mine % page].double().permute(1, 2, 0)
        values = s["v_cache"][pages, mine % page].double().transpose(0, 1)
        count = starts[i + 1] - starts[i]
        for j in range(count):
            sees = length - (count - 1 - j)
            x = s["q"][starts[i] + j].double().view(case["hkv"], group, case["d"]) * s["scale"]
            weights = torch.softmax(torch.cat([x @ prefix_k, x @ keys[..., :sees]], dim=-1), dim=-1)
            y = weights[..., :case["prefix"]] @ prefix_v + weights[..., case["prefix"]:] @ values[:, :sees]
            out[starts[i] + j] = y.reshape(case["hq"], case["d"])
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "quantize":
        m, k = case["m"], case["k"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": m * k * (size + 1) + 4 * _blocks(m, case["block_rows"]) * _blocks(k), "flops": 3 * m * k}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k + 2 * m * n + 4 * (m + _blocks(n)) * _blocks(k), "flops": 2 * m * n * k}
    if op == "append":
        real, d = case["tokens"] - case["padding"], case["d"]
        values = real * (case["hq"] + 2 * case["hkv"]) * d
        padding = case["padding"] * case["hq"] * d
        return {"bytes": 2 * 2 * values + 2 * padding + 16 * case["tokens"] + 4 * min(real, case["positions"]) * case["rotary"],
                "flops": 3 * real * (case["hq"] + case["hkv"]) * case["rotary"]}
    counts, lengths = _prefix_layout(case)
    tokens, keys, row = sum(counts), case["prefix"] + sum(lengths), case["hkv"] * case["d"] * 2
    # counts and lengths are paired anew by each seed: every token is given its sequence's mean suffix
    pairs = tokens * (case["prefix"] + sum(lengths) / len(lengths))
    return {"bytes": 2 * keys * row + 2 * tokens * case["hq"] * case["d"] * 2 + 4 * (_blocks(case["prefix"], case["page"]) + case["batch"]),
            "flops": 4 * pairs * case["hq"] * case["d"]}
