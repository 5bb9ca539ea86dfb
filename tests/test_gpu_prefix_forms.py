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
