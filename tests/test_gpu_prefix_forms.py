"""Shared-prefix attention, each form on purpose: the prefix kernel with the suffixes behind it (three launches), the prefix read in
front of every suffix (two), and the simple kernel (one)."""
import pytest
import torch

from tests import decode_reference as ref
from tests.test_gpu_decode import (BF16, F16, check_step, decode_step, on_device, ops, prefix_inputs,  # noqa: F401  (ops is a fixture)
                                   step_state, step_tables)
from vecops_b200 import capi

pytestmark = pytest.mark.gpu

PREFIX_KERNEL, JOINED, SIMPLE = 3, 2, 1  # launches of a call


def attend(ops, inputs, form):  # noqa: F811
    """The attention of device tensors, by the form that is meant."""
    before = capi.library().vecops_b200_launch_count()
    out = ops.sdpa_shared_prefix(**inputs)
    assert capi.library().vecops_b200_launch_count() - before == form
    return out


# The prefix kernel cuts the prefix into chunks of 128-key tiles; on 148 SMs the cases have 1, 2, 3, 4, 5, 6, 7, 8 and 11 tiles to a
# chunk (and what is left to the last one).  With at most 128 rows to a key head the kernel's two halves take the tiles in turn.
CHUNKS = [(20, 8, 896), (5, 8, 4224), (5, 16, 2176), (5, 48, 896), (5, 48, 1152), (5, 48, 1400), (5, 48, 1664), (5, 48, 2048), (5, 48, 3968)]


@pytest.mark.parametrize("d", [64, 40, 128])
@pytest.mark.parametrize("batch,heads,prefix", CHUNKS)
def test_chunks_of_every_length_with_few_rows(ops, batch, heads, prefix, d):  # noqa: F811
    inputs = prefix_inputs([1] * batch, [1 + 7 * i for i in range(batch)], prefix, heads, heads, d, 64, BF16, prefix + d, ragged=False)
    ref.assert_within(attend(ops, on_device(inputs), PREFIX_KERNEL), *ref.prefix_attention(**inputs))


@pytest.mark.parametrize("hq,hkv,prefix", [(32, 8, 9600), (8, 8, 8832)])
def test_chunks_of_five_tiles_of_64_dims(ops, hq, hkv, prefix):  # noqa: F811
    inputs = prefix_inputs([1] * 16, [1 + 4 * i for i in range(16)], prefix, hq, hkv, 64, 64, F16, prefix, ragged=False)
    ref.assert_within(attend(ops, on_device(inputs), PREFIX_KERNEL), *ref.prefix_attention(**inputs))


# ------------------------------------------------------------------------------------------------ NaN and infinite scores

# (sequences, query heads, key heads, dims, prefix, page, form): 1 and 5 tiles a chunk with few rows, both row blocks, in front of the
# suffixes, and what the tensor-core kernels cannot address
FORMS = [(20, 8, 8, 64, 896, 64, PREFIX_KERNEL), (5, 48, 48, 64, 1152, 64, PREFIX_KERNEL), (40, 8, 2, 128, 3000, 16, PREFIX_KERNEL),
         (4, 8, 2, 64, 300, 16, JOINED), (150, 2, 1, 128, 200, 8, JOINED), (3, 4, 2, 63, 50, 16, SIMPLE), (3, 4, 2, 256, 40, 16, SIMPLE), (4, 4, 2, 64, 90, 24, SIMPLE)]


def form_inputs(batch, hq, hkv, d, prefix, page, form):
    # suffixes that end with one key in a slice of sixteen, and some that fill theirs
    return prefix_inputs([1] * batch, [(17, 1, 33, 16, 40)[i % 5] for i in range(batch)], prefix, hq, hkv, d, page, BF16, batch + d, ragged=False)


def same_but(out, clean, changed):
    """The rows [tokens, heads] marked in `changed` are NaN throughout, the others as they were, bit for bit."""
    assert out[changed].isnan().all()
    assert torch.equal(out[~changed], clean[~changed])


@pytest.mark.parametrize("case", FORMS)
def test_a_nan_in_a_query_reaches_its_row_and_no_other(ops, case):  # noqa: F811
    batch, hq, *_, form = case
    inputs = on_device(form_inputs(*case))
    clean = attend(ops, inputs, form)
    assert not clean.isnan().any()
    inputs["q"][1, 3 % hq, 5] = float("nan")
    inputs["q"][batch - 1, 0] = float("nan")
    changed = torch.zeros(batch, hq, dtype=torch.bool, device="cuda")
    changed[1, 3 % hq] = changed[batch - 1, 0] = True
    same_but(attend(ops, inputs, form), clean, changed)


@pytest.mark.parametrize("case", FORMS)
def test_a_nan_key_reaches_every_row_that_sees_it(ops, case):  # noqa: F811
    batch, hq, hkv, d, prefix, page, form = case
    inputs = on_device(form_inputs(*case))
    clean = attend(ops, inputs, form)
    group = hq // hkv
    for key in (0, prefix // 2, prefix - 1):  # of the prefix: every query of its head
        at = (int(inputs["prefix_pages"][key // page]), key % page, hkv - 1, 7)
        kept = inputs["k_cache"][at].clone()
        inputs["k_cache"][at] = float("nan")
        changed = torch.zeros(batch, hq, dtype=torch.bool, device="cuda")
        changed[:, (hkv - 1) * group:] = True
        same_but(attend(ops, inputs, form), clean, changed)
        inputs["k_cache"][at] = kept
    for sequence in range(3):  # 17, 1 and 33 keys: the last one is alone in its slice
        for key in {0, int(inputs["lengths"][sequence]) - 1}:
            at = (int(inputs["page_table"][sequence, key // page]), key % page, 0, 0)
            kept = inputs["k_cache"][at].clone()
            inputs["k_cache"][at] = float("nan")
            changed = torch.zeros(batch, hq, dtype=torch.bool, device="cuda")
            changed[sequence, :group] = True
            same_but(attend(ops, inputs, form), clean, changed)
            inputs["k_cache"][at] = kept


@pytest.mark.parametrize("d,form", [(64, JOINED), (128, JOINED), (63, SIMPLE)])
def test_a_nan_key_that_is_the_only_one(ops, d, form):  # noqa: F811
    for prefix, lengths in ((1, [0, 0, 0]), (0, [1, 0, 1])):
        inputs = on_device(prefix_inputs([1] * 3, lengths, prefix, 4, 2, d, 16, BF16, 3, ragged=False))
        inputs["k_cache"][:] = float("nan")
        out = attend(ops, inputs, form)
        if prefix:
            assert out.isnan().all()
        else:
            assert out[0].isnan().all() and (out[1] == 0).all() and out[2].isnan().all()


@pytest.mark.parametrize("case", FORMS)
def test_scores_of_minus_infinity(ops, case):  # noqa: F811
    batch, hq, hkv, d, prefix, page, form = case
    inputs = form_inputs(*case)
    inputs["q"][..., 3] = inputs["q"][..., 3].abs() + 0.5
    shared = inputs["prefix_pages"].long()
    own = inputs["page_table"].long()
    k_cache = inputs["k_cache"].clone()

    def at(pages, value):
        inputs["k_cache"] = k_cache.clone()
        for p in pages:
            inputs["k_cache"][p, :, :, 3] = value

    def dropped(**changes):  # a key whose score is -inf beside finite ones has no weight: as if it were not there
        return ref.prefix_attention(**{**inputs, "k_cache": k_cache, **changes})

    minus = float("-inf")
    at([shared], minus)  # the prefix, in front of finite suffixes
    ref.assert_within(attend(ops, on_device(inputs), form), *dropped(prefix_pages=torch.full_like(inputs["prefix_pages"], -1)))
    some = shared[: max(1, len(shared) // 2)]
    at([some], minus)  # the first half of the prefix's pages
    ref.assert_within(attend(ops, on_device(inputs), form), *dropped(prefix_pages=torch.where(torch.isin(shared, some), -1, shared).int()))
    at([own], minus)  # all suffixes, behind a finite prefix
    ref.assert_within(attend(ops, on_device(inputs), form), *dropped(page_table=torch.full_like(inputs["page_table"], -1)))
    at([shared, own], minus)  # everything: 0 / 0
    assert attend(ops, on_device(inputs), form).isnan().all()
    at([own], minus)  # ... and where the prefix is absent
    out = attend(ops, on_device({**inputs, "prefix_pages": torch.full_like(inputs["prefix_pages"], -1)}), form)
    assert out.isnan().all()
    at([shared[-1:]], float("inf"))
    assert attend(ops, on_device(inputs), form).isnan().all()


# ------------------------------------------------------------------------------------------------ the prefix kernel: operands, streams, graphs

# both row blocks; few rows and 128 dims; few rows and 64 dims in chunks of five tiles
SHAPES = [(40, 8, 2, 128, 3000), (20, 8, 8, 128, 896), (5, 48, 48, 64, 1152)]


def shape_inputs(shape, seed, page=16, **more):
    batch, hq, hkv, d, prefix = shape
    return prefix_inputs([1] * batch, [1 + 7 * i % 41 for i in range(batch)], prefix, hq, hkv, d, page, BF16, seed, **{"ragged": False, "width": 3, **more})


@pytest.mark.parametrize("shape", SHAPES)
def test_the_prefix_kernel_takes_strided_operands(ops, shape):  # noqa: F811
    batch, hq, hkv, d, _ = shape
    inputs = shape_inputs(shape, 61)
    device = on_device(inputs)
    want = ref.prefix_attention(**inputs)
    q = torch.zeros(batch, hq, 3, d, dtype=BF16, device="cuda")
    q[:, :, 1] = device["q"]
    heads_first = [device[name].transpose(1, 2).contiguous().transpose(1, 2) for name in ("k_cache", "v_cache")]
    both = torch.stack([device["k_cache"], device["v_cache"]], dim=3)  # a key beside its value
    wide = torch.full((batch, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, :3] = device["page_table"]
    for change in (dict(q=q[:, :, 1]), dict(k_cache=heads_first[0], v_cache=heads_first[1]), dict(k_cache=both[:, :, :, 0], v_cache=both[:, :, :, 1]),
                   dict(page_table=wide[:, :3])):
        ref.assert_within(attend(ops, {**device, **change}, PREFIX_KERNEL), *want)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_the_prefix_kernel_scales(ops, shape, scale):  # noqa: F811
    inputs = shape_inputs(shape, 62, scale=scale)
    ref.assert_within(attend(ops, on_device(inputs), PREFIX_KERNEL), *ref.prefix_attention(**inputs))


@pytest.mark.parametrize("shape", SHAPES)
def test_the_prefix_kernel_drops_absent_pages_and_never_uses_what_lies_behind_the_keys(ops, shape):  # noqa: F811
    page = 16
    inputs = shape_inputs((*shape[:-1], shape[-1] - 5), 63)  # ends inside a page
    pages = inputs["k_cache"].shape[0]
    inputs["prefix_pages"][1], inputs["prefix_pages"][2] = pages, -7
    inputs["prefix_pages"][8:16] = -1  # a whole tile of 128 keys
    inputs["lengths"][1] = -1
    used = torch.zeros(inputs["k_cache"].shape[:2], dtype=torch.bool)
    for j in range(inputs["prefix_len"]):
        at = int(inputs["prefix_pages"][j // page])
        if 0 <= at < pages:
            used[at, j % page] = True
    for b, length in enumerate(inputs["lengths"].tolist()):
        for j in range(max(0, length)):
            used[inputs["page_table"][b, j // page], j % page] = True
    for name in ("k_cache", "v_cache"):
        inputs[name][~used] = float("nan")
    ref.assert_within(attend(ops, on_device(inputs), PREFIX_KERNEL), *ref.prefix_attention(**inputs))


def test_the_prefix_kernel_reads_far_into_a_long_cache(ops):  # noqa: F811
    pages, page, hkv, d = (1 << 20) + 3, 16, 2, 128  # 8 GiB a cache, element offsets past 2^32
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    inputs = shape_inputs((40, 8, hkv, d, 3000), 64)
    small = inputs["k_cache"].shape[0]
    far = pages - small + torch.arange(small, dtype=torch.int64)
    device = on_device(inputs)
    for name in ("k_cache", "v_cache"):
        cache = torch.zeros(pages, page, hkv, d, dtype=BF16, device="cuda")
        cache[far.cuda()] = device[name]
        device[name] = cache
    for name in ("prefix_pages", "page_table"):
        device[name] = far[inputs[name].long()].int().cuda()
    ref.assert_within(attend(ops, device, PREFIX_KERNEL), *ref.prefix_attention(**inputs))


@pytest.mark.parametrize("shape", SHAPES)
def test_prefix_kernels_on_two_streams_at_once_repeat_bit_for_bit(ops, shape):  # noqa: F811
    states = [on_device(shape_inputs(shape, seed)) for seed in (65, 66)]
    want = [attend(ops, state, PREFIX_KERNEL).clone() for state in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    results = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(attend(ops, states[i], PREFIX_KERNEL))
    torch.cuda.synchronize()
    graphs = []
    for stream, state in zip(streams, states):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = [attend(ops, state, PREFIX_KERNEL) for _ in range(3)]  # one call's kernels start under the one before
        graphs.append((graph, out))
    for _ in range(5):
        for stream, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        for out in [*results[i], *graphs[i][1]]:
            assert torch.equal(out, want[i])


@pytest.mark.parametrize("shape", SHAPES)
def test_a_captured_prefix_kernel_follows_its_tensors(ops, shape):  # noqa: F811
    static = on_device(shape_inputs(shape, 67))
    attend(ops, static, PREFIX_KERNEL)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(ops, static, PREFIX_KERNEL)
    for seed in (68, 69):
        inputs = shape_inputs(shape, seed)
        inputs["lengths"] = (inputs["lengths"] * seed) % 49 - 1  # padding and empty suffixes among them
        for name, tensor in inputs.items():
            if isinstance(tensor, torch.Tensor):
                static[name].copy_(tensor)
        graph.replay()
        torch.cuda.synchronize()
        ref.assert_within(out, *ref.prefix_attention(**inputs))
        assert torch.equal(out, attend(ops, static, PREFIX_KERNEL))
    del graph


@pytest.mark.parametrize("batch,hq,hkv,d,prefix", [(40, 8, 2, 128, 3000), (20, 8, 8, 64, 1152)])
def test_a_decode_step_over_the_prefix_kernel_eager_and_captured(ops, batch, hq, hkv, d, prefix):  # noqa: F811
    hidden = 512
    weights, inputs, table = step_state(ops, batch, hidden, hq, hkv, d, 16, prefix, 71)
    k_cache, v_cache = inputs["k_cache"].cuda(), inputs["v_cache"].cuda()
    static = list(step_tables(inputs, table, 0, batch))
    x = torch.zeros(batch, hidden, dtype=BF16, device="cuda")
    before = capi.library().vecops_b200_launch_count()
    decode_step(ops, x, weights, k_cache.clone(), v_cache.clone(), static, hq, hkv, d)
    assert capi.library().vecops_b200_launch_count() - before == 5 + PREFIX_KERNEL
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = decode_step(ops, x, weights, k_cache, v_cache, static, hq, hkv, d)
    eager_k, eager_v = inputs["k_cache"].cuda(), inputs["v_cache"].cuda()
    for step in range(2):
        tables = step_tables(inputs, table, 7 * step + 3, batch, padding=step)
        x.copy_(torch.randn(batch, hidden, generator=torch.Generator().manual_seed(step)).to(BF16))
        earlier = eager_k.cpu(), eager_v.cpu()
        result = decode_step(ops, x, weights, eager_k, eager_v, tables, hq, hkv, d)
        check_step(x, weights, earlier, (eager_k.cpu(), eager_v.cpu()), tables, result, hq, hkv, d)
        for old, new in zip(static, tables):
            if isinstance(old, torch.Tensor):
                old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for mine, theirs in zip(captured, result):
            assert torch.equal(mine, theirs)
        assert torch.equal(k_cache, eager_k) and torch.equal(v_cache, eager_v)
    del graph


def test_branches_of_a_captured_graph_join_at_the_prefix_kernel(ops):  # noqa: F811
    # a product on one branch, attention on the other, a product and attention behind both
    inputs = on_device(shape_inputs((40, 4, 2, 128, 3000), 72))
    g = torch.Generator().manual_seed(73)
    x = torch.randn(40, 512, generator=g).to(BF16).cuda()
    w, w_scale = ops.quantize_blocks(torch.randn(512, 512, generator=g).to(BF16).cuda(), 128)
    side = torch.cuda.Stream()

    def run():
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            y = ops.matmul_f8_blocks(*ops.quantize_blocks(x, 1), w, w_scale, BF16)
        o = attend(ops, inputs, PREFIX_KERNEL)
        here.wait_stream(side)
        z = ops.matmul_f8_blocks(*ops.quantize_blocks(o.view(40, 512) + y, 1), w, w_scale, BF16)
        return y, o, z, attend(ops, dict(inputs, q=z.view(40, 4, 128)), PREFIX_KERNEL)

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


@pytest.mark.parametrize("shape", SHAPES)
def test_caches_whose_heads_or_pages_share_memory(ops, shape):  # noqa: F811
    hkv = shape[2]
    inputs = shape_inputs(shape, 81)
    one = {name: inputs[name][:, :, :1].contiguous() for name in ("k_cache", "v_cache")}
    device = on_device(inputs)
    shared = {name: cache.cuda().expand(-1, -1, hkv, -1) for name, cache in one.items()}
    # one head's keys, values or both for all heads
    for names in (("k_cache",), ("v_cache",), ("k_cache", "v_cache")):
        want = ref.prefix_attention(**{**inputs, **{name: one[name].expand(-1, -1, hkv, -1) for name in names}})
        ref.assert_within(attend(ops, {**device, **{name: shared[name] for name in names}}, PREFIX_KERNEL), *want)
    # one page for all, one key for all of a page's: left to the simple kernel
    pages, page = inputs["k_cache"].shape[:2]
    for name, few in (("k_cache", inputs["k_cache"][:1].expand(pages, -1, -1, -1)), ("v_cache", inputs["v_cache"][:, :1].expand(-1, page, -1, -1))):
        on_gpu = device[name][:1].expand(pages, -1, -1, -1) if name == "k_cache" else device[name][:, :1].expand(-1, page, -1, -1)
        assert 0 in on_gpu.stride()
        ref.assert_within(attend(ops, {**device, name: on_gpu}, SIMPLE), *ref.prefix_attention(**{**inputs, name: few}))
