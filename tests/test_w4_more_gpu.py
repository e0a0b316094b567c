"""4-bit weights at the edges of the calls: outputs in an operand's memory, sizes beyond 32 bits, the
type of an output that is given, matrices and rows that are not there, every count of row tiles, and
elements of A near the format's lower end."""
import pytest
import torch
from test_w4_gpu import check_product, make, values

from helixml_b200 import _lib as L
from helixml_b200 import ops

pytestmark = pytest.mark.gpu


def test_shared_memory_is_refused_and_parts_of_one_buffer_are_not():
    gen = torch.Generator().manual_seed(1)
    m = ops.w4_quantize(torch.randn(48, 96, generator=gen).cuda(), 32, zero_points=True)
    buf = torch.randn(5, 160, generator=gen).cuda()
    a = buf[:, :96]
    want = ops.gemm_w4(a, m)
    assert torch.equal(ops.gemm_w4(a, m, out=buf[:, 100:148]), want)
    bias = torch.randn(48, generator=gen).cuda()
    for call in (lambda: ops.gemm_w4(a, m, out=buf[:, 90:138]), lambda: ops.gemm_w4(a, m, out=buf[:, :48]),
                 lambda: ops.gemm_w4(a[:1], m, bias=bias, out=bias[None])):
        with pytest.raises(L.HxError) as e:
            call()
        assert e.value.status == 10 and "share memory" in str(e.value)


def test_sizes_beyond_32_bits_are_refused():
    many = (1 << 32) + 3
    m = ops.w4_quantize(torch.randn(3, 32, generator=torch.Generator().manual_seed(2)).cuda(), 32)
    row = torch.zeros(1, 32, device="cuda")
    for call in (lambda: ops.gemm_w4(row.expand(many, 32), m, out=torch.zeros(1, 3, device="cuda").expand(many, 3)),
                 lambda: ops.w4_quantize(row.expand(many, 32), 32),
                 lambda: ops.w4_pack(row.to(torch.uint8).expand(many, 32), torch.ones(1, 1, device="cuda").expand(many, 1)),
                 lambda: ops.W4Matrix(many, 32, 32, torch.ones(1, 1, device="cuda").expand(many, 1), None)):
        with pytest.raises(L.HxError) as e:
            call()
        assert e.value.status == 2


def test_values_in_the_type_of_the_output_given():
    m = ops.w4_quantize(torch.randn(7, 64, generator=torch.Generator().manual_seed(3)).cuda(), 32)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.empty(7, 64, device="cuda", dtype=dtype)
        assert ops.w4_dequantize(m, out=out) is out and torch.equal(out, ops.w4_dequantize(m, dtype))
    assert ops.w4_dequantize(m).dtype == torch.float32
    for code, call in ((4, lambda: ops.w4_dequantize(m, torch.float32, out=torch.empty(7, 64, device="cuda", dtype=torch.bfloat16))),
                       (4, lambda: ops.w4_dequantize(m, out=torch.empty(7, 64, device="cuda", dtype=torch.float16)))):
        with pytest.raises(L.HxError) as e:
            call()
        assert e.value.status == code


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("zeros", [False, True])
def test_nothing_to_do(zeros, dtype):
    """No rows of weights, no rows of A, and a matrix without columns: it can be made and read back, a product with it is refused."""
    none = ops.w4_quantize(torch.empty(0, 64, device="cuda", dtype=dtype), 32, zero_points=zeros)
    assert none.codes.shape == (0, 64) and none.scale.shape == (0, 2) and ops.w4_dequantize(none).shape == (0, 64)
    assert ops.gemm_w4(torch.ones(3, 64, device="cuda", dtype=dtype), none).shape == (3, 0)
    packed = ops.w4_pack(torch.empty(0, 64, device="cuda", dtype=torch.uint8), torch.empty(0, 2, device="cuda", dtype=dtype))
    assert packed.group == 32 and ops.w4_dequantize(packed, dtype).shape == (0, 64)
    m = ops.w4_quantize(torch.ones(5, 64, device="cuda", dtype=dtype), 32, zero_points=zeros)
    assert ops.gemm_w4(torch.empty(0, 64, device="cuda", dtype=dtype), m).shape == (0, 5)
    narrow = ops.w4_quantize(torch.empty(5, 0, device="cuda", dtype=dtype), 32, zero_points=zeros)
    assert ops.w4_dequantize(narrow, dtype).shape == (5, 0)
    with pytest.raises(L.HxError) as e:
        ops.gemm_w4(torch.empty(3, 0, device="cuda", dtype=dtype), narrow)
    assert e.value.status == 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K,group", [(300, 416, 32), (2500, 256, 64), (70, 2048, 128)])
def test_every_count_of_row_tiles(N, K, group, dtype):
    """Rows of A up to, at and behind each multiple of 8 below 64, NaN in the memory behind the last one; the bound is check_product's."""
    codes, scale, zero = make(N, N, K, group, dtype, True)
    m, w = ops.w4_pack(codes.cuda(), scale.cuda(), zero.cuda()), values(codes, scale, zero, group)
    full = torch.full((72, K), float("nan"), device="cuda", dtype=dtype)
    for M in (9, 16, 17, 24, 25, 32, 33, 39, 40, 41, 48, 49, 55, 56, 57, 64, 65):
        full[:M] = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype).cuda()
        out = torch.full((72, N), 7.0, device="cuda", dtype=torch.float32)
        ops.gemm_w4(full[:M], m, out=out[:M])
        check_product(out[:M], full[:M], w, None)
        assert (out[M:] == 7).all()


@pytest.mark.parametrize("M", [1, 8])
def test_few_rows_too_long_to_be_staged(M):
    codes, scale, zero = make(3, 40, 65536, 128, torch.bfloat16, True)
    m = ops.w4_pack(codes.cuda(), scale.cuda(), zero.cuda())
    a = torch.randn(M, 65536, generator=torch.Generator().manual_seed(M)).bfloat16().cuda()
    check_product(ops.gemm_w4(a, m, out_dtype=torch.float32), a, values(codes, scale, zero, 128), None)


def test_small_elements_of_fp32_rows():
    """From 2^-110 on every bit of an element counts; below, what is left of it after cutting to a multiple of 2^-133."""
    K, N = 128, 24
    codes, _, zero = make(8, N, K, 64, torch.float32, True)
    scale = torch.full((N, K // 64), 2.0 ** 100)
    m, w = ops.w4_pack(codes.cuda(), scale.cuda(), zero.cuda()), values(codes, scale, zero, 64)
    a = torch.randn(12, K, generator=torch.Generator().manual_seed(9)) * 2.0 ** -torch.arange(104.0, 140.0, 3.0)[:, None]
    c = a.double() @ w.t()
    tol = 2 * 2.0 ** -24 * (18 + K / 16) * (a.double().abs() @ w.abs().t())
    tol += (a.abs() < 2.0 ** -110).double() @ w.abs().t() * 2.0 ** -133
    for rows in (slice(0, 12), slice(3, 4)):
        assert ((ops.gemm_w4(a[rows].cuda(), m).double().cpu() - c[rows]).abs() <= tol[rows]).all()
