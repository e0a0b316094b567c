"""4-bit weights at the edges of the calls: outputs in an operand's memory, sizes beyond 32 bits."""
import pytest
import torch

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
