"""4-bit weights at the edges of the calls: outputs in an operand's memory."""
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
