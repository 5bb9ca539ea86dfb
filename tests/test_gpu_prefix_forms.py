"""Shared-prefix attention, each form on purpose: the prefix kernel with the suffixes behind it (three launches), the prefix read in
front of every suffix (two), and the simple kernel (one)."""
import pytest
import torch

from tests import decode_reference as ref
from tests.test_gpu_decode import BF16, F16, on_device, ops, prefix_inputs  # noqa: F401  (ops is a fixture)
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
