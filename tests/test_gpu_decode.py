"""The decode-step operators on the GPU against plain 64-bit implementations (tests/decode_reference.py), through torch.ops.vecops_b200."""
import math

import pytest
import torch

from tests import decode_reference as ref
from vecops_b200 import capi

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from vecops_b200 import torch_ops
    torch_ops.load()
    yield torch.ops.vecops_b200
    torch.cuda.synchronize()
    word, error = capi.c_uint32(0), capi.ErrorBuffer()
    capi.library().vecops_b200_take_device_status(0, capi.byref(word), capi.byref(error.record))
    assert word.value == 0, f"a bounded device wait ran out: {word.value:#x}"


def generator(seed):
    return torch.Generator().manual_seed(seed)


def same_bits(x, y):
    return torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


# ------------------------------------------------------------------------------------------------ quantiser

@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (1, 4096), (3, 127), (5, 129), (64, 200), (130, 1000), (257, 384)])
def test_quantizer(ops, m, k, block_rows, dtype):
    x = torch.randn(m, k, generator=generator(m * 1000 + k)) * torch.logspace(-3, 3, k)[None, :]
    x = x.clamp(-6e4, 6e4).to(dtype)
    want, want_scale = ref.quantize(x, block_rows)
    q, scale = ops.quantize_blocks(x.cuda(), block_rows)
    assert q.dtype == E4M3 and q.shape == (m, k) and q.stride(0) % 16 == 0
    assert torch.equal(scale.cpu(), want_scale)
    assert same_bits(q.cpu(), want)
    # and what they stand for is x to half an e4m3 step (2^-4 of a normal value, 2^-10 scales below)
    stands = q.cpu().double() * want_scale.double().repeat_interleave(block_rows, 0)[:m].repeat_interleave(128, 1)[:, :k]
    each = want_scale.double().repeat_interleave(block_rows, 0)[:m].repeat_interleave(128, 1)[:, :k]
    assert ((stands - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * each) * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantizer_special_values(ops, dtype):
    x = torch.zeros(6, 300, dtype=dtype)
    x[1, 5], x[1, 6] = math.nan, 3.0             # NaN stays and does not count
    x[2, 130], x[2, 131] = math.inf, -1.0        # infinity saturates
    x[3, :] = math.nan
    x[4, 0], x[4, 1] = 1e-38, -1e-38             # under the smallest scale
    x[5, 299] = -2.5
    for block_rows in (1, 128):
        want, want_scale = ref.quantize(x, block_rows)
        q, scale = ops.quantize_blocks(x.cuda(), block_rows)
        assert torch.equal(scale.cpu(), want_scale) and torch.isfinite(scale).all() and (scale > 0).all()
        got, expected = q.float().cpu(), want.float()
        assert torch.equal(got.isnan(), expected.isnan()) and torch.equal(got.nan_to_num(0.0), expected.nan_to_num(0.0))


def test_quantizer_reads_strided_and_unaligned_sources(ops):
    x = torch.randn(70, 300, generator=generator(3)).to(BF16)
    for view in (x.t(), x[1:, 1:], x[::2, ::3], x[:1].expand(5, 300)):
        device = view.cuda() if view.is_contiguous() else x.cuda().as_strided(view.shape, view.stride(), view.storage_offset())
        for block_rows in (1, 128):
            want, want_scale = ref.quantize(view, block_rows)
            q, scale = ops.quantize_blocks(device, block_rows)
            assert same_bits(q.cpu(), want) and torch.equal(scale.cpu(), want_scale)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantizer_of_many_rows_off_boundaries(ops, dtype, block_rows):
    # more blocks than the grid's warps have at once, every row's start at another offset, the last block ragged
    x = torch.randn(1500, 1999, generator=generator(5)).to(dtype)
    want, want_scale = ref.quantize(x, block_rows)
    q, scale = ops.quantize_blocks(x.cuda(), block_rows)
    assert torch.equal(scale.cpu(), want_scale) and same_bits(q.cpu(), want)


def test_quantizer_of_nothing(ops):
    for shape in ((0, 128), (4, 0)):
        q, scale = ops.quantize_blocks(torch.empty(shape, dtype=BF16, device="cuda"))
        assert q.shape == shape and scale.shape == (shape[0], -(-shape[1] // 128))


# ------------------------------------------------------------------------------------------------ block-scaled product

def product_operands(m, n, k, seed):
    g = generator(seed)
    a, a_scale = ref.quantize(torch.randn(m, k, generator=g) * torch.logspace(-1, 1, k)[None, :], 1)
    b, b_scale = ref.quantize(torch.randn(n, k, generator=g), 128)

    def pitched(x):
        pitch = -(-x.shape[1] // 16) * 16
        stored = torch.full((x.shape[0], pitch), 0x7f, dtype=torch.uint8)  # NaN in the padding: not to be read
        stored[:, :x.shape[1]] = x.view(torch.uint8)
        return stored.cuda().view(E4M3)[:, :x.shape[1]]
    return pitched(a), a_scale.cuda(), pitched(b), b_scale.cuda()


def check_product(ops, a, a_scale, b, b_scale, dtype):
    c = ops.matmul_f8_blocks(a, a_scale, b, b_scale, dtype)
    assert c.dtype == dtype and c.shape == (a.shape[0], b.shape[0])
    want, magnitude = ref.matmul_f8(a, a_scale, b, b_scale)
    ref.assert_within(c, want, ref.matmul_f8_tolerance(want, magnitude, a.shape[1], dtype))
    return c


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (1, 4096, 4096), (2, 130, 640), (7, 129, 1000), (16, 512, 2048), (17, 1000, 384), (33, 4100, 4176),
                                   (61, 777, 144), (64, 1024, 1024), (65, 300, 256), (128, 384, 512), (129, 256, 896), (200, 1111, 1040), (256, 512, 128),
                                   (300, 1025, 272), (512, 768, 2048), (1000, 2000, 528)])
def test_product(ops, m, n, k, dtype):
    check_product(ops, *product_operands(m, n, k, m + n + k), dtype)


@pytest.mark.parametrize("m", [3, 100, 400])
def test_product_repeats_bit_for_bit(ops, m):
    operands = product_operands(m, 1536, 4096, m)
    first = ops.matmul_f8_blocks(*operands)
    for _ in range(3):
        assert torch.equal(ops.matmul_f8_blocks(*operands), first)


@pytest.mark.parametrize("m", [5, 150])
def test_product_reads_strided_operands(ops, m):
    n, k = 260, 400
    a, a_scale, b, b_scale = product_operands(m, n, k, 9)
    # scales transposed in memory, operands on odd pitches, transposed, and from an odd address
    scale_t, b_scale_t = a_scale.t().contiguous().t(), b_scale.t().contiguous().t()
    raw = torch.zeros(m * 403 + 1, dtype=torch.uint8, device="cuda")
    odd = raw[1:].view(m, 403)[:, :k]
    odd.copy_(a.view(torch.uint8))
    a_t = a.view(torch.uint8).t().contiguous().t().view(E4M3)
    b_t = b.view(torch.uint8).t().contiguous().t().view(E4M3)
    want, magnitude = ref.matmul_f8(a, a_scale, b, b_scale)
    for x, xs, y, ys in ((a, scale_t, b, b_scale_t), (odd.view(E4M3), a_scale, b, b_scale), (a_t, a_scale, b, b_scale), (a, a_scale, b_t, b_scale)):
        c = ops.matmul_f8_blocks(x, xs, y, ys, F32)
        ref.assert_within(c, want, ref.matmul_f8_tolerance(want, magnitude, k, F32))


@pytest.mark.parametrize("m", [4, 200])
def test_product_keeps_nan_and_infinity_where_they_belong(ops, m):
    a, a_scale, b, b_scale = product_operands(m, 256, 256, 4)
    a.view(torch.uint8)[1, 7] = 0x7f
    b_scale[1, 1] = math.inf
    c = ops.matmul_f8_blocks(a, a_scale, b, b_scale, F32)
    assert c[1].isnan().all()
    rest = torch.cat([c[:1], c[2:]])
    assert torch.isfinite(rest[:, :128]).all() and not torch.isfinite(rest[:, 128:]).any()


def test_product_of_nothing(ops):
    empty = torch.empty(4, 0, device="cuda").to(E4M3)
    none = torch.empty(4, 0, device="cuda")
    c = ops.matmul_f8_blocks(empty, none, empty, none[:1])
    assert c.shape == (4, 4) and (c == 0).all()
    a, a_scale, b, b_scale = product_operands(4, 8, 64, 1)
    assert ops.matmul_f8_blocks(a[:0], a_scale[:0], b, b_scale).shape == (0, 8)
    assert ops.matmul_f8_blocks(a, a_scale, b[:0], b_scale[:0]).shape == (4, 0)


def test_product_refuses(ops):
    a, a_scale, b, b_scale = product_operands(4, 200, 300, 1)
    for bad in ((a, a_scale[:, :2], b, b_scale), (a, a_scale, b, b_scale[:1]), (a[:, :128], a_scale, b, b_scale), (a.float(), a_scale, b, b_scale),
                (a, a_scale.double(), b, b_scale), (a, a_scale.cpu(), b, b_scale)):
        with pytest.raises(RuntimeError):
            ops.matmul_f8_blocks(*bad)
    with pytest.raises(RuntimeError):
        ops.matmul_f8_blocks(a, a_scale, b, b_scale, torch.int32)


# ------------------------------------------------------------------------------------------------ cache append

def append_inputs(tokens, hq, hkv, d, rotary, page, pages, dtype, seed, positions=5000):
    g = generator(seed)
    make = lambda *shape: torch.randn(*shape, generator=g).to(dtype)
    q, k, v = make(tokens, hq, d), make(tokens, hkv, d), make(tokens, hkv, d)
    k_cache, v_cache = make(pages, page, hkv, d), make(pages, page, hkv, d)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    at = torch.randint(0, positions, (tokens,), generator=g)
    half = rotary // 2
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    return q, k, v, k_cache, v_cache, slots, at, torch.cat([angle.cos(), angle.sin()], dim=1).float()


def check_append(ops, inputs, interleaved, views=None):
    q, k, v, k_cache, v_cache, slots, positions, table = inputs
    dtype, step = q.dtype, ref.half_step(q.dtype)
    device = [t.cuda() for t in inputs] if views is None else views
    out = ops.cache_append(*device, interleaved)
    pages, page = k_cache.shape[:2]
    real = (slots >= 0) & (slots < pages * page)
    if table.shape[1]:
        real &= (positions >= 0) & (positions < table.shape[0])
    rows = table[positions.clamp(0, max(table.shape[0] - 1, 0))] if table.shape[1] else table[:0].new_zeros(len(slots), 0)
    rotary = table.shape[1]

    def check(got, x):
        want, size = ref.rotate(x.double(), rows[real], interleaved)
        tiny = 2.0 ** -25 if dtype == F16 else 0.0
        ref.assert_within(got, want, step * want.abs() * 1.01 + 2 * ref.F32_STEP * size + tiny)
        assert same_bits(got[..., rotary:].cpu(), x[..., rotary:])

    check(out[real.cuda()], q[real])
    assert (out[~real.cuda()] == 0).all()
    where = slots[real]
    for got, before, new, rotated in ((device[3], k_cache, k, True), (device[4], v_cache, v, False)):
        got = got.cpu()
        flat = got.reshape(pages * page, *got.shape[2:])
        untouched = torch.ones(pages * page, dtype=torch.bool)
        untouched[where] = False
        assert same_bits(flat[untouched], before.reshape(pages * page, *before.shape[2:])[untouched])
        if rotated:
            check(flat[where], new[real])
        else:
            assert same_bits(flat[where], new[real])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,hq,hkv,d,rotary,page", [(1, 32, 8, 128, 128, 16), (64, 32, 8, 128, 64, 16), (5, 7, 7, 64, 64, 1), (3, 4, 2, 80, 32, 7), (9, 6, 3, 96, 96, 32),
                                                         (2, 5, 1, 63, 20, 16), (130, 2, 1, 256, 256, 64), (4, 3, 1, 40, 0, 16), (700, 8, 2, 64, 32, 128)])
def test_append(ops, tokens, hq, hkv, d, rotary, page, dtype, interleaved):
    pages = -(-2 * tokens // page) + 1
    check_append(ops, append_inputs(tokens, hq, hkv, d, rotary, page, pages, dtype, tokens + d), interleaved)


@pytest.mark.parametrize("d,rotary", [(128, 128), (63, 20)])
def test_append_skips_padding_and_what_lies_outside(ops, d, rotary):
    inputs = list(append_inputs(12, 4, 2, d, rotary, 16, 4, BF16, 8))
    inputs[5][2], inputs[5][5], inputs[5][6], inputs[5][11] = -1, 64, 1 << 40, -(1 << 40)
    inputs[6][0], inputs[6][9] = -1, 5000
    inputs[6][3] = 4999
    check_append(ops, inputs, False)


def test_append_takes_strided_operands(ops):
    t, hq, hkv, d = 20, 8, 2, 64
    inputs = append_inputs(t, hq, hkv, d, 64, 16, 8, BF16, 5)
    q, k, v, k_cache, v_cache = inputs[:5]
    fused = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], dim=1).cuda()
    parts = [x.unflatten(1, (-1, d)) for x in fused.split([hq * d, hkv * d, hkv * d], dim=1)]
    for permuted in (False, True):  # [pages, heads, page, D] in memory, and one key and one value side by side
        if permuted:
            caches = [c.transpose(1, 2).contiguous().cuda().transpose(1, 2) for c in (k_cache, v_cache)]
        else:
            both = torch.stack([k_cache, v_cache], dim=3).cuda()
            caches = [both[:, :, :, 0], both[:, :, :, 1]]
        check_append(ops, inputs, False, [*parts, *caches, *(x.cuda() for x in inputs[5:])])
    # rows off 16-byte boundaries
    odd = torch.zeros(t, hq + 2 * hkv, d + 1, dtype=BF16, device="cuda")
    odd[..., 1:] = fused.unflatten(1, (-1, d))
    check_append(ops, inputs, True, [*odd[..., 1:].split([hq, hkv, hkv], dim=1), k_cache.cuda(), v_cache.cuda(), *(x.cuda() for x in inputs[5:])])


def test_append_writes_far_into_a_long_cache(ops):
    # element offsets past 2^32: 2^20 pages of 16 slots of 2 heads of 128, 8 GiB a cache
    pages, page, hkv, d = (1 << 20) + 3, 16, 2, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    q, k, v, _, _, _, positions, table = append_inputs(3, 4, hkv, d, 128, page, 1, BF16, 3)
    k_cache, v_cache = (torch.zeros(pages, page, hkv, d, dtype=BF16, device="cuda") for _ in range(2))
    slots = torch.tensor([5, pages * page - 1, (1 << 24) + 7])
    ops.cache_append(q.cuda(), k.cuda(), v.cuda(), k_cache, v_cache, slots.cuda(), positions.cuda(), table.cuda())
    flat = v_cache.view(-1, hkv, d)
    assert same_bits(flat[slots.cuda()].cpu(), v)
    want, size = ref.rotate(k.double(), table[positions], False)
    ref.assert_within(k_cache.view(-1, hkv, d)[slots.cuda()], want, 2.0 ** -8 * want.abs() * 1.01 + 2 * ref.F32_STEP * size)
    assert int((flat != 0).any(-1).any(-1).sum()) == 3


def test_append_refuses(ops):
    good = [t.cuda() for t in append_inputs(4, 4, 2, 64, 64, 16, 4, BF16, 1)]
    for i, bad in ((0, good[0].float()), (1, good[1][:, :1]), (2, good[2][:3]), (3, good[3].to(F16)), (5, good[5].int()), (6, good[6][:2]), (7, good[7].half()),
                   (4, good[4].transpose(2, 3)), (5, good[5].cpu()), (7, good[7][:, :3])):
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError):
            ops.cache_append(*args)


# ------------------------------------------------------------------------------------------------ shared-prefix attention

def prefix_inputs(counts, lengths, prefix, hq, hkv, d, page, dtype, seed, width=None, ragged=True, scale=None, spare=3):
    g = generator(seed)
    batch = len(lengths)
    width = width if width is not None else max(1, -(-max([*lengths, 1]) // page))
    shared = -(-prefix // page)
    pages = shared + batch * width + spare
    where = torch.randperm(pages, generator=g).int()
    k_cache, v_cache = (torch.randn(pages, page, hkv, d, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(sum(counts), hq, d, generator=g).to(dtype)
    starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
    return dict(q=q, k_cache=k_cache, v_cache=v_cache, prefix_pages=where[:shared].contiguous(), prefix_len=prefix,
                page_table=where[shared:shared + batch * width].reshape(batch, width).contiguous(), lengths=torch.tensor(lengths, dtype=torch.int32),
                scale=d ** -0.5 if scale is None else scale, query_starts=starts if ragged else None)


def on_device(inputs):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in inputs.items()}


def check_prefix(ops, inputs, device=None):
    out = ops.sdpa_shared_prefix(**(device or on_device(inputs)))
    ref.assert_within(out, *ref.prefix_attention(**inputs))
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("batch,prefix,suffix,hq,hkv,d,page", [
    (1, 1, 1, 1, 1, 64, 16), (1, 128, 1, 8, 8, 128, 16), (4, 512, 64, 32, 8, 128, 16), (3, 127, 5, 4, 4, 64, 32), (3, 129, 200, 4, 2, 64, 16), (2, 1000, 17, 6, 2, 128, 64),
    (33, 300, 40, 20, 4, 64, 16), (40, 260, 33, 8, 2, 128, 128), (5, 64, 300, 16, 1, 128, 16), (7, 250, 30, 12, 4, 96, 16), (2, 100, 50, 4, 2, 80, 8), (2, 60, 20, 4, 4, 256, 16),
    (3, 50, 20, 4, 2, 40, 7), (2, 33, 9, 2, 1, 63, 16), (6, 900, 100, 32, 1, 64, 256), (130, 384, 3, 4, 4, 64, 64), (2, 5000, 700, 4, 1, 128, 16)])
def test_prefix_attention_of_single_tokens(ops, batch, prefix, suffix, hq, hkv, d, page, dtype):
    lengths = [1 + (i * 37) % suffix for i in range(batch)]
    lengths[-1] = suffix
    check_prefix(ops, prefix_inputs([1] * batch, lengths, prefix, hq, hkv, d, page, dtype, batch + prefix, ragged=False))


@pytest.mark.parametrize("counts,lengths,prefix,hq,hkv,d", [
    ([1, 5, 2, 3], [9, 40, 2, 3], 200, 8, 2, 64), ([3, 0, 4], [100, 7, 130], 150, 4, 4, 128), ([17], [17], 64, 8, 1, 64), ([40, 1], [129, 300], 300, 6, 2, 128),
    ([4, 4], [2, 1], 100, 4, 1, 64),  # more new tokens than suffix keys: the first ones see the prefix alone
    ([200], [200], 0, 4, 2, 64)])
def test_prefix_attention_of_several_tokens(ops, counts, lengths, prefix, hq, hkv, d):
    for dtype in (BF16, F16):
        check_prefix(ops, prefix_inputs(counts, lengths, prefix, hq, hkv, d, 16, dtype, sum(counts)))


def test_prefix_attention_without_a_prefix_without_a_suffix_without_either(ops):
    check_prefix(ops, prefix_inputs([1] * 5, [3, 100, 1, 17, 64], 0, 8, 2, 64, 16, BF16, 1, ragged=False))
    check_prefix(ops, prefix_inputs([1] * 3, [0, 0, 0], 77, 8, 2, 64, 16, BF16, 2, ragged=False))
    check_prefix(ops, prefix_inputs([1] * 3, [0, 0, 0], 77, 8, 2, 64, 16, BF16, 2, width=0, ragged=False))
    inputs = prefix_inputs([1] * 3, [0, 5, 0], 0, 8, 2, 64, 16, BF16, 3, ragged=False)
    out = check_prefix(ops, inputs)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    # nothing at all: no cache page exists
    empty = torch.empty(0, 16, 2, 64, dtype=BF16, device="cuda")
    out = ops.sdpa_shared_prefix(inputs["q"].cuda(), empty, empty, inputs["prefix_pages"].cuda(), 0, inputs["page_table"].cuda(), inputs["lengths"].cuda(), 0.1)
    assert (out == 0).all()


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (4, 4, 128)])
def test_prefix_attention_of_padding(ops, hq, hkv, d):
    inputs = prefix_inputs([1] * 6, [5, -1, 40, -1, 0, -7], 200, hq, hkv, d, 16, BF16, 4, ragged=False)
    out = check_prefix(ops, inputs)
    assert (out[1] == 0).all() and (out[5] == 0).all() and not (out[4] == 0).all()
    # tokens behind the last sequence, and before the first
    inputs = prefix_inputs([2, 3], [10, 20], 130, hq, hkv, d, 16, BF16, 5)
    inputs["q"] = torch.cat([inputs["q"], inputs["q"]])
    inputs["query_starts"] = inputs["query_starts"] + 2
    out = check_prefix(ops, inputs)
    assert (out[:2] == 0).all() and (out[7:] == 0).all()


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (40, 16)])
def test_prefix_attention_never_uses_what_lies_behind_the_keys(ops, d, page):
    for counts, prefix in (([1] * 4, 203), ([3, 1, 2, 5], 203), ([3, 1, 2, 5], 128)):
        inputs = prefix_inputs(counts, [7, 65, 129, 30], prefix, 8, 2, d, page, BF16, 6)
        used = torch.zeros(inputs["k_cache"].shape[:2], dtype=torch.bool)
        for j in range(prefix):
            used[inputs["prefix_pages"][j // page], j % page] = True
        for b, length in enumerate(inputs["lengths"].tolist()):
            for j in range(length):
                used[inputs["page_table"][b, j // page], j % page] = True
        for poison in (math.nan, math.inf):
            for cache in (inputs["k_cache"], inputs["v_cache"]):
                cache[~used] = poison
            check_prefix(ops, inputs)


@pytest.mark.parametrize("d", [64, 128, 40])
def test_prefix_attention_keeps_a_later_tokens_nan_from_the_earlier_ones(ops, d):
    inputs = prefix_inputs([6], [50], 100, 8, 2, d, 16, BF16, 7)
    for name in ("k_cache", "v_cache"):  # the newest key, which only the newest token sees
        inputs[name][inputs["page_table"][0, 49 // 16], 49 % 16] = math.nan
    out = ops.sdpa_shared_prefix(**on_device(inputs))
    want, tolerance = ref.prefix_attention(**inputs)
    ref.assert_within(out[:5], want[:5], tolerance[:5])
    assert out[5].isnan().all()


@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (40, 16)])
def test_prefix_attention_drops_pages_outside_the_cache(ops, d, page):
    inputs = prefix_inputs([1, 2, 1], [70, 90, 33], 300, 8, 2, d, page, BF16, 8)
    pages = inputs["k_cache"].shape[0]
    inputs["prefix_pages"][1], inputs["prefix_pages"][-1] = pages, -1
    inputs["page_table"][0, 0], inputs["page_table"][1, 1], inputs["page_table"][2, 0] = -5, pages + 7, 1 << 30
    check_prefix(ops, inputs)
    inputs["prefix_pages"][:] = -1
    inputs["page_table"][:] = pages
    assert (check_prefix(ops, inputs) == 0).all()


def test_prefix_attention_length_past_the_table(ops):
    inputs = prefix_inputs([1, 1], [30, 20], 40, 4, 2, 64, 16, BF16, 9)
    inputs["lengths"][1] = 1000  # the table ends at 32 keys
    check_prefix(ops, inputs)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_prefix_attention_scales(ops, scale):
    check_prefix(ops, prefix_inputs([1, 3], [70, 20], 300, 8, 2, 64, 16, BF16, 10, scale=scale))


def test_prefix_attention_of_rising_and_falling_scores(ops):
    # the maximum moves at every tile, or never after the first
    for order in (1, -1):
        inputs = prefix_inputs([1, 1], [260, 100], 700, 4, 2, 64, 16, BF16, 11, ragged=False)
        ramp = torch.linspace(-3 * order, 3 * order, 700 + 260)
        for j in range(700):
            inputs["k_cache"][inputs["prefix_pages"][j // 16], j % 16] = float(ramp[j])
        for b in range(2):
            for j in range(int(inputs["lengths"][b])):
                inputs["k_cache"][inputs["page_table"][b, j // 16], j % 16] = float(ramp[700 + j])
        inputs["q"] = inputs["q"].abs()
        check_prefix(ops, inputs)


def test_prefix_attention_takes_strided_operands(ops):
    inputs = prefix_inputs([1, 2, 1], [70, 90, 33], 300, 8, 2, 64, 16, BF16, 12)
    device = on_device(inputs)
    q = torch.zeros(4, 8, 3, 64, dtype=BF16, device="cuda")
    q[:, :, 1] = device["q"]
    both = torch.stack([device["k_cache"], device["v_cache"]], dim=1)  # a page's keys, then its values
    heads_first = [device[name].transpose(1, 2).contiguous().transpose(1, 2) for name in ("k_cache", "v_cache")]
    odd = torch.zeros(*inputs["k_cache"].shape[:3], 67, dtype=BF16, device="cuda")
    odd[..., 1:65] = device["k_cache"]
    wide = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, :inputs["page_table"].shape[1]] = device["page_table"]
    want = ref.prefix_attention(**inputs)
    for change in (dict(q=q[:, :, 1]), dict(k_cache=both[:, 0], v_cache=both[:, 1]), dict(k_cache=heads_first[0], v_cache=heads_first[1]),
                   dict(k_cache=odd[..., 1:65]), dict(page_table=wide[:, :inputs["page_table"].shape[1]])):
        ref.assert_within(ops.sdpa_shared_prefix(**{**device, **change}), *want)


def test_prefix_attention_reads_far_into_a_long_cache(ops):
    pages, page, hkv, d = (1 << 20) + 3, 16, 2, 128  # 8 GiB a cache, element offsets past 2^32
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    inputs = prefix_inputs([1, 1], [30, 50], 200, 8, hkv, d, page, BF16, 13, ragged=False)
    small = inputs["k_cache"].shape[0]
    far = torch.arange(small, dtype=torch.int64) * 7 % 5 + pages - 5 * (torch.arange(small) // 5 + 1)  # distinct pages at the far end
    assert len(set(far.tolist())) == small and int(far.max()) == pages - 1
    device = on_device(inputs)
    for name in ("k_cache", "v_cache"):
        cache = torch.zeros(pages, page, hkv, d, dtype=BF16, device="cuda")
        cache[far.cuda()] = device[name]
        device[name] = cache
    for name in ("prefix_pages", "page_table"):
        device[name] = far[inputs[name].long()].int().cuda()
    check_prefix(ops, inputs, device)


def test_prefix_attention_repeats_bit_for_bit(ops):
    inputs = on_device(prefix_inputs([1] * 40, [1 + 13 * i for i in range(40)], 3000, 8, 2, 128, 16, BF16, 14, ragged=False))
    first = ops.sdpa_shared_prefix(**inputs)
    for _ in range(3):
        assert torch.equal(ops.sdpa_shared_prefix(**inputs), first)


def test_prefix_attention_refuses(ops):
    good = on_device(prefix_inputs([1, 1], [30, 50], 200, 8, 2, 64, 16, BF16, 15, ragged=False))
    for change in (dict(q=good["q"].float()), dict(q=good["q"][:1]), dict(q=good["q"][:, :7]), dict(k_cache=good["k_cache"].to(F16)), dict(v_cache=good["v_cache"][:1]),
                   dict(prefix_pages=good["prefix_pages"].long()), dict(prefix_len=400), dict(prefix_len=-1), dict(lengths=good["lengths"][:1]),
                   dict(page_table=good["page_table"].t()), dict(lengths=good["lengths"].cpu()), dict(query_starts=good["lengths"])):
        with pytest.raises(RuntimeError):
            ops.sdpa_shared_prefix(**{**good, **change})


@pytest.mark.parametrize("batch,counts,hq,hkv,d", [(2100, None, 2, 1, 64), (700, [0, 1, 0, 2, 0, 0, 3], 4, 2, 64), (33, [16, 17, 1], 1, 1, 128), (5, [1, 2], 48, 1, 64)])
def test_prefix_attention_of_many_and_of_uneven_sequences(ops, batch, counts, hq, hkv, d):
    """More sequences than a warp has lanes, by far; empty ones between; items of many tokens; more query heads per key head than an
    item has rows.  Lengths from nothing to two slices beside one long one."""
    lengths = [(7 * i) % 33 for i in range(batch)]
    lengths[batch // 2] = 900
    counts = [1] * batch if counts is None else [counts[i % len(counts)] for i in range(batch)]
    inputs = prefix_inputs(counts, lengths, 70, hq, hkv, d, 16, BF16, batch, ragged=max(counts) > 1)
    check_prefix(ops, inputs)


def test_prefix_attention_of_a_long_prefix_and_a_long_suffix(ops):
    check_prefix(ops, prefix_inputs([1], [9000], 40000, 4, 1, 128, 64, BF16, 16, ragged=False))
    check_prefix(ops, prefix_inputs([1] * 70, [5] * 70, 20000, 8, 2, 64, 128, F16, 17, ragged=False))


@pytest.mark.parametrize("page", [3, 24, 48, 128, 384])
def test_prefix_attention_of_page_sizes(ops, page):
    # pages that end inside a slice of sixteen keys, or inside a tile of 128, and pages longer than a tile
    check_prefix(ops, prefix_inputs([1, 1, 1], [50, 400, 129], 0, 8, 2, 64, page, BF16, page, ragged=False))
    check_prefix(ops, prefix_inputs([2, 1, 3], [50, 400, 129], 777, 8, 2, 64, page, BF16, page))


# ------------------------------------------------------------------------------------------------ the C ABI's own forms

def run_record(function, record):
    error = capi.ErrorBuffer()
    error.raise_for(getattr(capi.library(), function)(capi.byref(record), capi.byref(error.record)))


def f8_record(a, a_scale, b, b_scale, c, kernel):
    r = capi.VecopsB200MatmulF8(struct_size=capi.ctypes.sizeof(capi.VecopsB200MatmulF8), kernel=kernel, m=a.shape[0], n=b.shape[0], k=a.shape[1],
                                a=a.data_ptr(), a_stride_m=a.stride(0), a_stride_k=a.stride(1), a_scale=a_scale.data_ptr(),
                                a_scale_stride_m=a_scale.stride(0), a_scale_stride_k=a_scale.stride(1), b=b.data_ptr(), b_stride_n=b.stride(0),
                                b_stride_k=b.stride(1), b_scale=b_scale.data_ptr(), b_scale_stride_n=b_scale.stride(0),
                                b_scale_stride_k=b_scale.stride(1), c=c.data_ptr(), c_stride_m=c.stride(0), c_stride_n=c.stride(1),
                                c_dtype={BF16: capi.DTYPE_BF16, F16: capi.DTYPE_F16, F32: capi.DTYPE_F32}[c.dtype],
                                stream=torch.cuda.current_stream().cuda_stream, device_index=0)
    return r


@pytest.mark.parametrize("kernel", [capi.F8_GENERIC, capi.F8_STREAM, capi.F8_TILED])
@pytest.mark.parametrize("m,n,k", [(1, 130, 1024), (33, 700, 640), (128, 257, 2064)])
def test_every_kernel_of_the_product(ops, m, n, k, kernel):
    """The kernels on one problem, into rows with a gap behind them and into a transposed C; what lies between stays."""
    a, a_scale, b, b_scale = product_operands(m, n, k, m + n)
    want, magnitude = ref.matmul_f8(a, a_scale, b, b_scale)
    for dtype in (BF16, F32):
        for stored in (torch.full((m, n + 5), 7.0, dtype=dtype, device="cuda"), torch.full((n, m + 3), 7.0, dtype=dtype, device="cuda")):
            c = stored[:, :n] if stored.shape[0] == m and stored.shape[1] == n + 5 else stored.t()[:m]
            run_record("vecops_b200_matmul_f8_run", f8_record(a, a_scale, b, b_scale, c, kernel))
            ref.assert_within(c, want, ref.matmul_f8_tolerance(want, magnitude, k, dtype))
            rest = stored[:, n:] if c.stride(1) == 1 else stored[:, m:]
            assert (rest == 7.0).all()


def test_the_products_kernel_is_chosen_and_refused_by_rule(ops):
    for m, n, k, kernel in ((1, 128, 128, capi.F8_STREAM), (128, 4096, 4096, capi.F8_STREAM), (129, 256, 512, capi.F8_TILED)):
        a, a_scale, b, b_scale = product_operands(m, n, k, 1)
        c = torch.empty(m, n, device="cuda")
        chosen, error = capi.c_uint32(0), capi.ErrorBuffer()
        error.raise_for(capi.library().vecops_b200_matmul_f8_select(capi.byref(f8_record(a, a_scale, b, b_scale, c, capi.F8_AUTO)), capi.byref(chosen), capi.byref(error.record)))
        assert chosen.value == kernel
    with pytest.raises(capi.VecopsB200Error) as info:
        run_record("vecops_b200_matmul_f8_run", f8_record(a, a_scale, b, b_scale, c, capi.F8_STREAM))  # 129 rows
    assert info.value.code == capi.NOT_APPLICABLE
    odd = torch.zeros(130, 513, dtype=torch.uint8, device="cuda").view(E4M3)[:129, 1:]
    chosen = capi.c_uint32(0)
    error.raise_for(capi.library().vecops_b200_matmul_f8_select(capi.byref(f8_record(odd, a_scale, b, b_scale, c, capi.F8_AUTO)), capi.byref(chosen), capi.byref(error.record)))
    assert chosen.value == capi.F8_GENERIC


@pytest.mark.parametrize("kernel", [capi.F8_STREAM, capi.F8_TILED, capi.F8_GENERIC])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("row,col,start", [(1, 120, 0), (301, 1, 1), (900, 2, 3), (304, 1, 0)])
def test_product_stores_into_any_strides(ops, kernel, dtype, row, col, start):
    m, n, k = 117, 299, 400
    a, a_scale, b, b_scale = product_operands(m, n, k, 21)
    whole = torch.full((300 * 120 + 900 * 120 + 8,), -3.0, dtype=dtype, device="cuda")
    before = whole.clone()
    c = whole.as_strided((m, n), (row, col), start)
    r = f8_record(a, a_scale, b, b_scale, c, kernel)
    r.c_dtype = {BF16: capi.DTYPE_BF16, F16: capi.DTYPE_F16, F32: capi.DTYPE_F32}[dtype]
    run_record("vecops_b200_matmul_f8_run", r)
    want, magnitude = ref.matmul_f8(a, a_scale, b, b_scale)
    ref.assert_within(c, want, ref.matmul_f8_tolerance(want, magnitude, k, dtype))
    before.as_strided((m, n), (row, col), start).copy_(c)
    assert torch.equal(whole, before)  # and nothing beside them


def append_record(q, k, v, q_out, k_cache, v_cache, slots, positions, table):
    r = capi.VecopsB200CacheAppend(struct_size=capi.ctypes.sizeof(capi.VecopsB200CacheAppend), dtype=capi.DTYPE_BF16, tokens=k.shape[0], q_heads=q.shape[1] if q is not None else 0,
                                   kv_heads=k.shape[1], head_dim=k.shape[2], pages=k_cache.shape[0], page_size=k_cache.shape[1], max_positions=table.shape[0],
                                   rotary=table.shape[1], cos_sin_stride=table.stride(0), stream=torch.cuda.current_stream().cuda_stream, device_index=0)
    for name, tensor in dict(q=q, k=k, v=v, q_out=q_out, k_cache=k_cache, v_cache=v_cache, slots=slots, positions=positions, cos_sin=table).items():
        if tensor is not None:
            setattr(r, name, tensor.data_ptr())
    for name, tensor in dict(q=q, k=k, v=v, q_out=q_out).items():
        if tensor is not None:
            setattr(r, f"{name}_stride_token", tensor.stride(0)), setattr(r, f"{name}_stride_head", tensor.stride(1))
    r.k_stride_page, r.k_stride_slot, r.k_cache_stride_head = k_cache.stride()[:3]
    r.v_stride_page, r.v_stride_slot, r.v_cache_stride_head = v_cache.stride()[:3]
    return r


def test_append_in_place_and_without_queries(ops):
    device = [t.cuda() for t in append_inputs(70, 8, 2, 64, 64, 16, 12, BF16, 30)]
    q, k, v, k_cache, v_cache, slots, positions, table = device
    want_k, want_v = k_cache.clone(), v_cache.clone()
    want_q = ops.cache_append(q, k, v, want_k, want_v, slots, positions, table)
    mine_k, mine_v, in_place = k_cache.clone(), v_cache.clone(), q.clone()
    run_record("vecops_b200_cache_append", append_record(in_place, k, v, in_place, mine_k, mine_v, slots, positions, table))
    assert torch.equal(in_place, want_q) and torch.equal(mine_k, want_k) and torch.equal(mine_v, want_v)
    mine_k, mine_v = k_cache.clone(), v_cache.clone()
    run_record("vecops_b200_cache_append", append_record(None, k, v, None, mine_k, mine_v, slots, positions, table))
    assert torch.equal(mine_k, want_k) and torch.equal(mine_v, want_v)


def test_prefix_attention_refuses_scratch_that_is_too_small(ops):
    inputs = on_device(prefix_inputs([1] * 4, [30] * 4, 400, 8, 2, 64, 16, BF16, 31, ragged=False))
    out = torch.full_like(inputs["q"], 7.0)
    r = capi.VecopsB200PrefixAttention(struct_size=capi.ctypes.sizeof(capi.VecopsB200PrefixAttention), dtype=capi.DTYPE_BF16, tokens=4, batch=4, q_heads=8, kv_heads=2, head_dim=64,
                                       pages=inputs["k_cache"].shape[0], page_size=16, prefix_len=400, table_stride=2, table_width=2, scale=0.125,
                                       stream=torch.cuda.current_stream().cuda_stream, device_index=0)
    for name in ("q", "k_cache", "v_cache", "prefix_pages", "page_table", "lengths"):
        setattr(r, name, inputs[name].data_ptr())
    r.out = out.data_ptr()
    r.q_stride_token, r.q_stride_head, r.out_stride_token, r.out_stride_head = 512, 64, 512, 64
    r.k_stride_page, r.k_stride_slot, r.k_stride_head = r.v_stride_page, r.v_stride_slot, r.v_stride_head = inputs["k_cache"].stride()[:3]
    need, error = capi.c_uint64(0), capi.ErrorBuffer()
    error.raise_for(capi.library().vecops_b200_prefix_sdpa_workspace(capi.byref(r), capi.byref(need), capi.byref(error.record)))
    scratch = torch.empty(need.value + 256, dtype=torch.uint8, device="cuda")
    for at, size in ((0, 0), (scratch.data_ptr(), need.value - 1), (scratch.data_ptr() + 8, need.value)):
        r.workspace, r.workspace_size = at or None, size
        with pytest.raises(capi.VecopsB200Error) as info:
            run_record("vecops_b200_prefix_sdpa_run", r)
        assert info.value.code == capi.INVALID_ARGUMENT and "scratch" in info.value.message
    assert (out == 7.0).all()
    r.workspace, r.workspace_size = scratch.data_ptr(), need.value
    run_record("vecops_b200_prefix_sdpa_run", r)  # synchronous
    assert torch.equal(out, ops.sdpa_shared_prefix(**inputs))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("batch,prefix,hq,hkv,d", [(3, 900, 4, 2, 64), (40, 1000, 16, 2, 128)])
def test_prefix_attention_of_large_scores(ops, dtype, sign, batch, prefix, hq, hkv, d):
    # scores of +-(64 (d - 2) + 15) + r with r in eighths: exact in fp32, thousands away from zero and a few apart
    inputs = prefix_inputs([1] * batch, [40] * batch, prefix, hq, hkv, d, 16, dtype, 41, ragged=False, scale=1.0)
    inputs["q"][:], inputs["k_cache"][:] = 8.0 * sign, 8.0
    inputs["q"][..., d // 2] = 1.0
    inputs["q"][..., d // 2 + 1], inputs["k_cache"][..., d // 2 + 1] = sign, 15.0
    inputs["k_cache"][..., d // 2] = (torch.randint(-24, 25, inputs["k_cache"].shape[:3], generator=generator(42)) / 8).to(dtype)
    out = ops.sdpa_shared_prefix(**on_device(inputs))
    want, _ = ref.prefix_attention(**inputs)
    size, _ = ref.prefix_attention(**{**inputs, "v_cache": inputs["v_cache"].abs()})
    # In units of log2(e) a score is below 2^14: a product with the scale is off by 2^-11 (a key's own, or the maximum's it
    # is measured from), so a weight by 2 of them and the weights' sum by as much; p and the result are rounded to the type
    step = ref.half_step(dtype)
    relative = 4 * math.log(2) * 2.0 ** -11 + step + 2.0 ** -16
    tiny = 2.0 ** -25 * (prefix + 41) * 5 if dtype == F16 else 0.0
    ref.assert_within(out, want, 1.05 * (2 * relative * size + step * want.abs()) + tiny)


def test_prefix_attention_ignores_query_tokens_that_do_not_exist(ops):
    # starts before the first token and behind the last: the tokens there are nobody's
    for d in (64, 80, 72, 256):
        inputs = prefix_inputs([2, 3, 1], [40, 50, 20], 200, 8, 2, d, 16, BF16, 43)
        inside = dict(inputs, query_starts=torch.tensor([0, 2, 5, 6], dtype=torch.int32))
        whole = ops.sdpa_shared_prefix(**on_device(inside))
        outside = on_device(dict(inputs, query_starts=torch.tensor([-3, 2, 5, 9], dtype=torch.int32)))
        assert torch.equal(ops.sdpa_shared_prefix(**outside), whole), d


@pytest.mark.parametrize("page", [8, 16, 48, 128, 256])
@pytest.mark.parametrize("batch,prefix", [(3, 500), (160, 500), (3, 16), (160, 16), (1, 5000), (160, 128)])
def test_prefix_attention_whether_few_or_many_read_the_prefix(ops, batch, prefix, page):
    # 3 sequences read it in front of their suffixes, 160 by a kernel of its own; drafted tokens, idle slots, empty suffixes, absent pages, NaN behind the keys
    counts = [(1, 3, 0, 2)[i % 4] for i in range(batch)]
    lengths = [(5, 3, -1, 40)[i % 4] for i in range(batch)]
    if batch > 3:
        lengths[0], lengths[4] = 0, 0
    inputs = prefix_inputs(counts, lengths, prefix, 16, 8, 128, page, BF16, batch + prefix + page)
    if prefix > 2 * page:
        inputs["prefix_pages"][1] = -1
    if prefix % page:
        last = int(inputs["prefix_pages"][-1])
        if last >= 0:
            inputs["k_cache"][last, prefix % page:] = math.nan
            inputs["v_cache"][last, prefix % page:] = math.nan
    check_prefix(ops, inputs)


# ------------------------------------------------------------------------------------------------ together, captured, on other streams

def decode_step(ops, x, weights, k_cache, v_cache, tables, hq, hkv, d):
    """One token of every sequence through the attention block: product, append, attention, product."""
    w_in, s_in, w_out, s_out = weights
    prefix_pages, prefix_len, page_table, lengths, slots, positions, cos_sin = tables
    q8, qs = ops.quantize_blocks(x)
    qkv = ops.matmul_f8_blocks(q8, qs, w_in, s_in)
    q, k, v = (part.unflatten(1, (-1, d)) for part in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
    q = ops.cache_append(q, k, v, k_cache, v_cache, slots, positions, cos_sin)
    y = ops.sdpa_shared_prefix(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, lengths, d ** -0.5)
    y8, ys = ops.quantize_blocks(y.flatten(1))
    return qkv, q, y, ops.matmul_f8_blocks(y8, ys, w_out, s_out)


def step_state(ops, batch, hidden, hq, hkv, d, page, prefix, seed):
    g = generator(seed)
    w_in, s_in = ops.quantize_blocks(torch.randn((hq + 2 * hkv) * d, hidden, generator=g).cuda() / hidden ** 0.5, 128)
    w_out, s_out = ops.quantize_blocks(torch.randn(hidden, hq * d, generator=g).cuda() / (hq * d) ** 0.5, 128)
    inputs = prefix_inputs([1] * batch, [4] * batch, prefix, hq, hkv, d, page, BF16, seed, width=4, ragged=False)
    table = append_inputs(1, 1, 1, d, d, 1, 1, BF16, 1)[7]
    return (w_in, s_in, w_out, s_out), inputs, table


def step_tables(inputs, table, offset, batch, padding=0):
    page = inputs["k_cache"].shape[1]
    lengths = torch.tensor([offset + 1 + b % 3 for b in range(batch)], dtype=torch.int32)
    slots = torch.tensor([int(inputs["page_table"][b, (int(lengths[b]) - 1) // page]) * page + (int(lengths[b]) - 1) % page for b in range(batch)])
    positions = inputs["prefix_len"] + lengths.long() - 1
    if padding:
        lengths[batch - padding:], slots[batch - padding:] = -1, -1
    return inputs["prefix_pages"].cuda(), inputs["prefix_len"], inputs["page_table"].cuda(), lengths.cuda(), slots.cuda(), positions.cuda(), table.cuda()


def check_step(x, weights, before, after, tables, result, hq, hkv, d):
    """Each stage against its plain form on the stage's own inputs."""
    w_in, s_in, w_out, s_out = weights
    prefix_pages, prefix_len, page_table, lengths, slots, positions, cos_sin = tables
    qkv, q, y, out = result
    x8, xs = (t.cuda() for t in ref.quantize(x.cpu(), 1))
    want, magnitude = ref.matmul_f8(x8, xs, w_in, s_in)
    ref.assert_within(qkv, want, ref.matmul_f8_tolerance(want, magnitude, x.shape[1], BF16))
    parts = [part.unflatten(1, (-1, d)) for part in qkv.cpu().split([hq * d, hkv * d, hkv * d], dim=1)]
    real = (slots >= 0).cpu()
    rows = cos_sin.cpu()[positions.cpu()]
    for got, new in ((q.cpu(), parts[0]), (after[0].reshape(-1, hkv, d)[slots.cpu().clamp_min(0)], parts[1])):
        turned, size = ref.rotate(new.double(), rows, False)
        ref.assert_within(got[real], turned[real], (2.0 ** -8 * turned.abs() * 1.01 + 2 * ref.F32_STEP * size)[real])
    assert same_bits(after[1].reshape(-1, hkv, d)[slots.cpu()[real]], parts[2][real])
    keep = torch.ones(before[0].shape[0] * before[0].shape[1], dtype=torch.bool)
    keep[slots.cpu()[real]] = False
    for b, a in zip(before, after):
        assert same_bits(a.reshape(-1, hkv, d)[keep], b.reshape(-1, hkv, d)[keep])
    ref.assert_within(y, *ref.prefix_attention(q.cpu(), after[0], after[1], prefix_pages.cpu(), prefix_len, page_table.cpu(), lengths.cpu(), d ** -0.5))
    y8, ys = (t.cuda() for t in ref.quantize(y.flatten(1).cpu(), 1))
    want, magnitude = ref.matmul_f8(y8, ys, w_out, s_out)
    ref.assert_within(out, want, ref.matmul_f8_tolerance(want, magnitude, hq * d, BF16))


def test_a_decode_step_eager_and_captured(ops):
    """Three steps of a batch with padding: the operators in a row, then the same captured once and replayed with each step's
    lengths, slots, positions and activations written into its tensors."""
    batch, hidden, hq, hkv, d, page, prefix = 10, 512, 8, 2, 64, 16, 300
    weights, inputs, table = step_state(ops, batch, hidden, hq, hkv, d, page, prefix, 21)
    k_cache, v_cache = inputs["k_cache"].cuda(), inputs["v_cache"].cuda()
    static = list(step_tables(inputs, table, 0, batch))
    x = torch.zeros(batch, hidden, dtype=BF16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    decode_step(ops, x, weights, k_cache.clone(), v_cache.clone(), static, hq, hkv, d)  # warm-up outside the capture
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = decode_step(ops, x, weights, k_cache, v_cache, static, hq, hkv, d)
    eager_k, eager_v = inputs["k_cache"].cuda(), inputs["v_cache"].cuda()
    for step in range(3):
        tables = step_tables(inputs, table, 7 * step + 3, batch, padding=step)
        x.copy_(torch.randn(batch, hidden, generator=generator(step)).to(BF16))
        before = eager_k.cpu(), eager_v.cpu()
        result = decode_step(ops, x, weights, eager_k, eager_v, tables, hq, hkv, d)
        check_step(x, weights, before, (eager_k.cpu(), eager_v.cpu()), tables, result, hq, hkv, d)
        for old, new in zip(static, tables):
            if isinstance(old, torch.Tensor):
                old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for mine, theirs in zip(captured, result):
            assert torch.equal(mine, theirs)
        assert torch.equal(k_cache, eager_k) and torch.equal(v_cache, eager_v)


def test_steps_on_two_streams_at_once(ops):
    """Two batches on two streams, and two captured graphs replayed at once: no scratch of one call is another's."""
    states = []
    for seed in (31, 32):
        weights, inputs, table = step_state(ops, 6, 512, 8, 2, 64, 16, 2000, seed)
        x = torch.randn(6, 512, generator=generator(seed)).to(BF16).cuda()
        tables = step_tables(inputs, table, 20, 6)
        want = decode_step(ops, x, weights, inputs["k_cache"].cuda(), inputs["v_cache"].cuda(), tables, 8, 2, 64)
        states.append((x, weights, inputs["k_cache"].cuda(), inputs["v_cache"].cuda(), tables, 8, 2, 64, want))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    results = [[] for _ in states]
    for _ in range(5):
        for i, (stream, state) in enumerate(zip(streams, states)):
            with torch.cuda.stream(stream):
                results[i].append(decode_step(ops, *state[:-1]))
    torch.cuda.synchronize()
    graphs = []
    for stream, state in zip(streams, states):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = decode_step(ops, *state[:-1])
        graphs.append((graph, out))
    for _ in range(5):
        for stream, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for i, state in enumerate(states):
        for result in [*results[i], graphs[i][1]]:
            for mine, theirs in zip(result, state[-1]):
                assert torch.equal(mine, theirs)


def test_branches_of_a_captured_graph_join(ops):
    # products on one branch, attention on the other, a product behind both: launches that wait for more than one kernel
    inputs = on_device(prefix_inputs([1] * 6, [40, 3, 0, 17, 64, 9], 700, 8, 2, 64, 16, BF16, 51, ragged=False))
    g = generator(52)
    x = torch.randn(6, 512, generator=g).to(BF16).cuda()
    w, w_scale = ops.quantize_blocks(torch.randn(512, 512, generator=g).to(BF16).cuda(), 128)
    side = torch.cuda.Stream()

    def run():
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            y = ops.matmul_f8_blocks(*ops.quantize_blocks(x, 1), w, w_scale, BF16)
        o = ops.sdpa_shared_prefix(**inputs)
        here.wait_stream(side)
        z = ops.matmul_f8_blocks(*ops.quantize_blocks(o.view(6, 512), 1), w, w_scale, BF16)
        t = ops.sdpa_shared_prefix(**dict(inputs, q=z.view(6, 8, 64)))
        return y, o, z, t

    want = [r.clone() for r in run()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        for r in got:
            r.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for r, e in zip(got, want):
            assert torch.equal(r, e)
    del graph
