"""Host-only checks of the decode-step entry points (include/vecops_b200/decode_cuda.h): record layouts, argument checks, and
the loud failure without a GPU.  No pointer in here is ever read: every call ends before a launch."""
import ctypes
import subprocess
from ctypes import byref
from pathlib import Path

import pytest
import torch

from vecops_b200 import capi

ROOT = Path(__file__).resolve().parents[1]
SOMEWHERE = 0x10000  # a non-null, aligned address


def test_records_match_the_header(tmp_path):
    names = ["VecopsB200QuantizeBlocks", "VecopsB200MatmulF8", "VecopsB200CacheAppend", "VecopsB200PrefixAttention"]
    lines = []
    for name in names:
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name}.{field} %zu\\n", offsetof({name}, {field}));' for field, _ in getattr(capi, name)._fields_]
    source = tmp_path / "layout.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "vecops_b200/decode_cuda.h"\nint main(void) {\n' + "\n".join(lines) + "\n  return 0;\n}\n")
    binary = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(source), "-o", str(binary)], check=True)
    for line in subprocess.run([str(binary)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, value = line.split()
        record, _, field = name.partition(".")
        record = getattr(capi, record)
        assert (getattr(record, field).offset if field else ctypes.sizeof(record)) == int(value), line


def quantize_record(**changes):
    r = capi.VecopsB200QuantizeBlocks(struct_size=ctypes.sizeof(capi.VecopsB200QuantizeBlocks), block_rows=1, rows=3, cols=200, src=SOMEWHERE,
                                      src_stride_row=200, src_stride_col=1, src_dtype=capi.DTYPE_BF16, dst=SOMEWHERE, dst_stride_row=208,
                                      scale=SOMEWHERE, scale_stride_row=2, scale_stride_col=1, device_index=-1)
    for key, value in changes.items():
        setattr(r, key, value)
    return r


def matmul_record(**changes):
    r = capi.VecopsB200MatmulF8(struct_size=ctypes.sizeof(capi.VecopsB200MatmulF8), m=16, n=256, k=512, a=SOMEWHERE, a_stride_m=512, a_stride_k=1,
                                a_scale=SOMEWHERE, a_scale_stride_m=4, a_scale_stride_k=1, b=SOMEWHERE, b_stride_n=512, b_stride_k=1,
                                b_scale=SOMEWHERE, b_scale_stride_n=4, b_scale_stride_k=1, c=SOMEWHERE, c_stride_m=256, c_stride_n=1,
                                c_dtype=capi.DTYPE_BF16, device_index=-1)
    for key, value in changes.items():
        setattr(r, key, value)
    return r


def append_record(**changes):
    r = capi.VecopsB200CacheAppend(struct_size=ctypes.sizeof(capi.VecopsB200CacheAppend), dtype=capi.DTYPE_BF16, tokens=4, q_heads=8, kv_heads=2,
                                   head_dim=64, pages=10, page_size=16, max_positions=100, rotary=64, cos_sin_stride=64, device_index=-1,
                                   q_stride_token=512, q_stride_head=64, k_stride_token=128, k_stride_head=64, v_stride_token=128, v_stride_head=64,
                                   q_out_stride_token=512, q_out_stride_head=64, k_stride_page=2048, k_stride_slot=128, k_cache_stride_head=64,
                                   v_stride_page=2048, v_stride_slot=128, v_cache_stride_head=64)
    for key in ("q", "k", "v", "q_out", "k_cache", "v_cache", "slots", "positions", "cos_sin"):
        setattr(r, key, SOMEWHERE)
    for key, value in changes.items():
        setattr(r, key, value)
    return r


def prefix_record(**changes):
    r = capi.VecopsB200PrefixAttention(struct_size=ctypes.sizeof(capi.VecopsB200PrefixAttention), dtype=capi.DTYPE_BF16, tokens=4, batch=4, q_heads=8,
                                       kv_heads=2, head_dim=64, q_stride_token=512, q_stride_head=64, out_stride_token=512, out_stride_head=64,
                                       k_stride_page=2048, k_stride_slot=128, k_stride_head=64, v_stride_page=2048, v_stride_slot=128,
                                       v_stride_head=64, pages=100, page_size=16, prefix_len=300, table_stride=8, table_width=8, scale=0.125,
                                       device_index=-1)
    for key in ("q", "out", "k_cache", "v_cache", "prefix_pages", "page_table", "lengths"):
        setattr(r, key, SOMEWHERE)
    for key, value in changes.items():
        setattr(r, key, value)
    return r


def code_of(function, record, *extra):
    error = capi.ErrorBuffer()
    code = getattr(capi.library(), function)(byref(record) if record is not None else None, *extra, byref(error.record))
    if code != capi.OK:
        assert error.text.value, "a refusal comes with a message"
    return code, error.text.value.decode()


@pytest.mark.parametrize("changes", [dict(block_rows=64), dict(src_dtype=capi.DTYPE_I8), dict(rows=-1), dict(cols=1 << 31), dict(src_stride_row=-1),
                                     dict(dst_stride_row=199), dict(src=None), dict(dst=None), dict(scale=None)])
def test_quantizer_refuses(library, changes):
    assert code_of("vecops_b200_quantize_blocks", quantize_record(**changes))[0] == capi.INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [dict(c_dtype=capi.DTYPE_I8), dict(m=-1), dict(k=1 << 31), dict(kernel=9), dict(a_stride_m=-1), dict(b_scale_stride_k=-4),
                                     dict(c_stride_n=0), dict(c_stride_m=0), dict(a=None), dict(b_scale=None), dict(c=None)])
def test_product_refuses(library, changes):
    assert code_of("vecops_b200_matmul_f8_run", matmul_record(**changes))[0] == capi.INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [dict(dtype=capi.DTYPE_F32), dict(tokens=-1), dict(rotary=63), dict(rotary=66), dict(rotary=-2), dict(interleaved=2),
                                     dict(k_stride_page=-1), dict(pages=1 << 40, page_size=1 << 30), dict(q=None), dict(q_out=None), dict(k=None),
                                     dict(v_cache=None), dict(slots=None), dict(positions=None), dict(cos_sin=None)])
def test_append_refuses(library, changes):
    assert code_of("vecops_b200_cache_append", append_record(**changes))[0] == capi.INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [dict(dtype=capi.DTYPE_F32), dict(tokens=5), dict(q_heads=7), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=257),
                                     dict(page_size=0), dict(prefix_len=-1), dict(prefix_len=1 << 31), dict(table_width=1 << 28), dict(k_stride_slot=-1),
                                     dict(q=None), dict(out=None), dict(k_cache=None), dict(prefix_pages=None), dict(page_table=None), dict(lengths=None)])
def test_prefix_attention_refuses(library, changes):
    need = ctypes.c_uint64(0)
    assert code_of("vecops_b200_prefix_sdpa_workspace", prefix_record(**changes), byref(need))[0] == capi.INVALID_ARGUMENT
    assert code_of("vecops_b200_prefix_sdpa_run", prefix_record(**changes))[0] == capi.INVALID_ARGUMENT


def test_outputs_that_share_memory_are_refused(library):
    for changes in (dict(scale_stride_row=0), dict(scale_stride_col=0)):
        code, message = code_of("vecops_b200_quantize_blocks", quantize_record(**changes))
        assert code == capi.INVALID_ARGUMENT and "share memory" in message, changes
    for name in ("k_stride_page", "k_stride_slot", "k_cache_stride_head", "v_stride_page", "v_stride_slot", "v_cache_stride_head", "q_out_stride_token", "q_out_stride_head"):
        code, message = code_of("vecops_b200_cache_append", append_record(**{name: 0}))
        assert code == capi.INVALID_ARGUMENT and "share memory" in message, name
    for name in ("out_stride_token", "out_stride_head"):
        code, message = code_of("vecops_b200_prefix_sdpa_run", prefix_record(**{name: 0}))
        assert code == capi.INVALID_ARGUMENT and "share memory" in message, name


def test_extents_past_the_grids_are_refused_or_left_to_the_simple_kernel(library):
    code, message = code_of("vecops_b200_prefix_sdpa_run", prefix_record(tokens=1 << 30, batch=1 << 30, q_heads=1 << 15, kv_heads=1 << 15))
    assert code == capi.INVALID_ARGUMENT and "too many" in message
    need = ctypes.c_uint64(7)
    many = prefix_record(tokens=1 << 23, batch=1 << 23, q_heads=8, kv_heads=1)  # 2^26 rows of one head: more blocks than a grid has
    assert code_of("vecops_b200_prefix_sdpa_workspace", many, byref(need))[0] == capi.OK and need.value == 0
    huge = 1 << 62  # (its double is negative)
    assert code_of("vecops_b200_cache_append", append_record(kv_heads=huge))[0] == capi.INVALID_ARGUMENT


ENTRIES = [("vecops_b200_quantize_blocks", quantize_record), ("vecops_b200_matmul_f8_run", matmul_record), ("vecops_b200_cache_append", append_record),
           ("vecops_b200_prefix_sdpa_run", prefix_record)]


@pytest.mark.parametrize("function,record", ENTRIES)
def test_short_records_are_an_abi_mismatch(library, function, record):
    assert code_of(function, None)[0] == capi.ABI_MISMATCH
    assert code_of(function, record(struct_size=16))[0] == capi.ABI_MISMATCH


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses in these records are not real")
@pytest.mark.parametrize("function,record", ENTRIES)
def test_calls_without_a_gpu_fail_loudly(library, function, record):
    r = record()
    if record is prefix_record:
        need = ctypes.c_uint64(0)
        assert code_of("vecops_b200_prefix_sdpa_workspace", r, byref(need))[0] == capi.OK
        r.workspace, r.workspace_size = SOMEWHERE, need.value
    code, message = code_of(function, r)
    assert code == capi.EXECUTION_ERROR and "no CPU fallback" in message


@pytest.mark.parametrize("function,record", [("vecops_b200_quantize_blocks", quantize_record(rows=0)), ("vecops_b200_quantize_blocks", quantize_record(cols=0)),
                                             ("vecops_b200_matmul_f8_run", matmul_record(m=0)), ("vecops_b200_matmul_f8_run", matmul_record(n=0)),
                                             ("vecops_b200_cache_append", append_record(tokens=0)),
                                             ("vecops_b200_prefix_sdpa_run", prefix_record(tokens=0, batch=0))])
def test_empty_calls_succeed_and_touch_nothing(library, function, record):
    assert code_of(function, record)[0] == capi.OK


def test_torch_operators_are_registered_and_refuse_cpu_tensors():
    from vecops_b200 import _build, torch_ops
    _build.build_torch_bridge()
    torch_ops.load()
    ops = torch.ops.vecops_b200
    assert "Tensor(a!) k_cache, Tensor(b!) v_cache" in str(ops.cache_append.default._schema)
    assert "Tensor? query_starts=None" in str(ops.sdpa_shared_prefix.default._schema)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.quantize_blocks(torch.zeros(4, 4))
    x = torch.zeros(4, 4).to(torch.float8_e4m3fn)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.matmul_f8_blocks(x, torch.zeros(4, 1), x, torch.zeros(1, 1))


def test_refusals_of_the_torch_operators_carry_their_numbers():
    # the C++ behind the operator called directly, as a CUDA tensor would reach it: a message with a formatted number in it comes
    # back as an exception (it ended the process when the bridge carried a C++ runtime of its own)
    from vecops_b200 import _build, torch_ops
    _build.build_torch_bridge()
    torch_ops.load()
    with pytest.raises(RuntimeError, match="block_rows is 1 or 128, not 64"):
        torch.ops.vecops_b200.quantize_blocks.default._op_dk(torch._C.DispatchKey.CUDA, torch.zeros(4, 4), 64)
