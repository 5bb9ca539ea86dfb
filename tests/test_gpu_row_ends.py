"""Dense products into rows of C that end off a 16-byte boundary while their pitch is a multiple of 16 bytes: what lies behind a row's end
stays.  The result is the one that a C without a gap gets, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32, I8, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int32


@pytest.fixture(scope="module")
def ops():
    from vecops_b200 import torch_ops
    torch_ops.load()
    return torch.ops.vecops_b200


def operand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    if dtype == I8:
        return torch.randint(-100, 101, shape, generator=g, dtype=I8).cuda()
    return torch.randn(shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("a_type,b_type,c_type", [(BF16, BF16, BF16), (BF16, BF16, F32), (F16, F16, F16), (I8, I8, I32), (BF16, I8, BF16), (BF16, I8, F32), (F32, F32, F32)])
@pytest.mark.parametrize("m,n,k", [(300, 299, 512), (128, 1003, 256), (64, 4097, 1024), (700, 2050, 768), (1500, 1021, 2048), (129, 3, 128), (1000, 65, 256)])
def test_rows_that_end_off_boundaries_leave_what_follows(ops, a_type, b_type, c_type, m, n, k):
    a, b = operand((m, k), a_type, m + k), operand((n, k), b_type, n)
    scale = torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda() if a_type != b_type else None
    plain = torch.empty(m, n, dtype=c_type, device="cuda")
    ops.matmul_out(a, b, plain, scale)
    pitch = -(-n // 16) * 16 + 16
    whole = torch.full((m, pitch), 7, dtype=c_type, device="cuda")
    ops.matmul_out(a, b, whole[:, :n], scale)
    assert torch.equal(whole[:, :n], plain)
    assert (whole[:, n:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,col0", [(504, 0), (504, 504), (40, 768), (300, 64)])
def test_a_gathered_slab_ends_with_its_own_columns(ops, dtype, n, col0):
    # a slab that is no whole number of 128-byte pieces: the next rank's columns, which start right behind it, are another kernel's to write
    from vecops_b200 import sharding
    m, k, n_total = 200, 256, 1536
    a, b = operand((m, k), BF16, 5), operand((n, k), BF16, 6)
    full = [torch.full((m, n_total), -3.0, dtype=dtype, device="cuda") for _ in range(2)]
    gemm = sharding.FusedGatherGemm(a, b, [t.data_ptr() for t in full], n_total, n_total, col0, dtype)
    gemm.launch()
    torch.cuda.synchronize()
    want = ops.matmul(a, b, out_dtype=dtype)
    end = col0 + -(-n // (16 // want.element_size())) * (16 // want.element_size())
    for t in full:
        assert torch.equal(t[:, col0:col0 + n], want)
        assert (t[:, :col0] == -3).all() and (t[:, end:] == -3).all()
