"""Plain 64-bit implementations of the decode-step operators, and how far a correct kernel may be from them.

A rounding to a type is off by at most half a step: torch.finfo(type).eps / 2 of the value.  An fp32 sum of n terms is
off by at most n * 2^-23 of the sum of their magnitudes (2^-24 per addition to nearest, twice that where an adder truncates).
"""
import math

import torch

F32_STEP = 2.0 ** -23


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def quantize(x, block_rows):
    """(e4m3 values, fp32 scales), in the formula's own fp32 operations; x on the CPU."""
    x = x.float()
    m, k = x.shape
    rows, cols = -(-m // block_rows), -(-k // 128)
    padded = torch.zeros(rows * block_rows, cols * 128)
    padded[:m, :k] = x
    tiles = padded.view(rows, block_rows, cols, 128)
    finite = torch.where(tiles.isnan(), torch.zeros_like(tiles), tiles.abs())
    amax = finite.amax(dim=(1, 3)).clamp(2.0 ** -110, torch.finfo(torch.float32).max)
    factor = (torch.tensor(448.0) / amax)[:, None, :, None]
    q = (tiles * factor).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(rows * block_rows, cols * 128)[:m, :k], amax / 448


def matmul_f8(a, a_scale, b, b_scale):
    """(C in fp64, the sum of its terms' magnitudes)."""
    k = a.shape[1]
    col = torch.arange(k, device=a.device) // 128
    row = torch.arange(b.shape[0], device=a.device) // 128
    x = a.float().double() * a_scale.double()[:, col]
    y = b.float().double() * b_scale.double()[row][:, col]
    return x @ y.t(), x.abs() @ y.abs().t()


def matmul_f8_tolerance(c, magnitude, k, dtype):
    """A block's 128 exact products are summed in fp32, scaled (three roundings) and added over the blocks; then one rounding.
    fp16 results below its normal range are off by half of its smallest step."""
    blocks = -(-k // 128)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return half_step(dtype) * c.abs() * 1.01 + (128 + blocks + 4) * F32_STEP * magnitude + tiny


def rotate(x, table, interleaved):
    """x [T,H,D] fp64, table [T,R] (cosines, then sines): (rotated, the sum of the magnitudes of what was added)."""
    half = table.shape[1] // 2
    cos, sin = table[:, None, :half].double(), table[:, None, half:].double()
    y, size = x.clone(), torch.zeros_like(x)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first], size[..., second] = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
    return y, size


def prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, lengths, scale, query_starts=None):
    """(out, tolerance) in fp64 for CPU tensors; a token's keys are gathered one by one."""
    t, hq, d = q.shape
    pages, page, hkv, _ = k_cache.shape
    batch = page_table.shape[0]
    starts = query_starts.tolist() if query_starts is not None else list(range(batch + 1))
    out = torch.zeros(t, hq, d, dtype=torch.float64)
    tolerance = torch.zeros_like(out)
    step = half_step(q.dtype)

    def slots(table, count):
        count = max(0, min(count, len(table) * page))
        return [(table[j // page], j % page) for j in range(count) if 0 <= table[j // page] < pages]

    shared = slots(prefix_pages.tolist(), prefix_len)
    for b in range(batch):
        length = int(lengths[b])
        if length < 0:
            continue
        for i in range(starts[b], starts[b + 1]):
            where = shared + slots(page_table[b].tolist(), length - (starts[b + 1] - 1 - i))
            if not where:
                continue
            index = torch.tensor(where)
            keys, values = k_cache[index[:, 0], index[:, 1]].double(), v_cache[index[:, 0], index[:, 1]].double()  # [n,Hkv,D]
            keys, values = keys.repeat_interleave(hq // hkv, dim=1), values.repeat_interleave(hq // hkv, dim=1)
            x = q[i].double()
            scores = torch.einsum("hd,nhd->hn", x, keys) * scale
            reach = torch.einsum("hd,nhd->hn", x.abs(), keys.abs()) * abs(scale)
            p = torch.softmax(scores, dim=-1)
            out[i] = torch.einsum("hn,nhd->hd", p, values)
            weight = torch.einsum("hn,nhd->hd", p, values.abs())
            n = len(where)
            # a score is off by (d + 4) fp32 steps of its terms, moving every p by e^(2 * that) at most; e^x itself by the
            # rounding of its argument (|x| steps) and 2^-22; p is rounded to q's type; sums of n terms; the result is rounded
            score = (d + 4) * F32_STEP * reach.amax(dim=-1) + 2 * F32_STEP * scores.abs().amax(dim=-1) + 2.0 ** -22
            relative = step + 3 * score[:, None] + (n + 64) * F32_STEP
            # fp16 probabilities below its normal range: half of its smallest step each, against a sum of at least 1
            tiny = n * 2.0 ** -25 * values.abs().amax(dim=0) if q.dtype == torch.float16 else 0.0
            tolerance[i] = weight * relative + tiny + step * out[i].abs() * 1.05 + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    return out, tolerance


def assert_within(got, want, tolerance):
    got, want = got.double().cpu(), want.cpu()
    bad = ~((got - want).abs() <= tolerance.cpu())
    if bad.any():
        where = bad.nonzero()[0].tolist()
        worst = ((got - want).abs() / tolerance.cpu().clamp_min(1e-300)).nan_to_num(math.inf).max().item()
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} values outside the tolerance (worst {worst:.3g} times), first at {where}: "
                             f"{got[tuple(where)].item()} for {want[tuple(where)].item()}")
