"""Weights in 4 bits: quantising, laying out, reading back, and the product of a few rows with them.

The codes, scales and zero points are held to equality with the definition, evaluated in exact arithmetic on 64-bit numbers
(a quotient of two 24-bit numbers cannot round across a half in 53 bits).  The product: u = 2^-24; each C[m,n] is a sum of K
products that are exact in fp32 (bf16 times a code of at most 4 bits and sign), or rounded once (fp32: parts of 8 bits, also exact),
accumulated over at most 16 + K / 16 dependent additions, each off by at most 2 u of the sum's magnitude (a tensor core may truncate),
then scaled: so |error| <= 2 u (18 + K / 16) sum |a| |w|, and the result's own rounding."""
import numpy as np
import pytest
import torch

from helixml_b200 import _lib as L
from helixml_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(seed, N, K, group, scale_dtype, zeros):
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (N, K), generator=gen, dtype=torch.uint8)
    scale = ((0.5 + torch.rand(N, K // group, generator=gen)) * 2.0 ** -4).to(scale_dtype)
    zero = torch.randint(0, 16, (N, K // group), generator=gen, dtype=torch.uint8) if zeros else None
    return codes, scale, zero


def values(codes, scale, zero, group):
    """The matrix in 64 bits."""
    z = torch.full_like(scale, 8.0, dtype=torch.float64) if zero is None else zero.double()
    wide = lambda t: t.double().repeat_interleave(group, 1)
    return (codes.double() - wide(z)) * wide(scale)


def unpack(m):
    """Codes from the documented layout, on the host."""
    raw = m.codes.cpu().numpy()
    out = np.zeros((m.rows, m.cols), dtype=np.uint8)
    for k in range(m.cols):
        r = k % 128
        at = (k // 128) * 64 + 16 * ((r % 32) // 8) + 4 * (r // 32)
        p = (r % 8) // 2 + 4 * (r % 2)
        out[:, k] = (raw[:, at + p // 2] >> (4 * (p % 2))) & 15
    return torch.from_numpy(out)


# ------------------------------------------------------------------ layout and values
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,groups", [(1, 1), (3, 3), (17, 5), (70, 8)])
def test_pack_and_dequantize(N, groups, group, zeros):
    K = groups * group
    codes, scale, zero = make(1, N, K, group, torch.float32, zeros)
    wide = torch.zeros(N, K + 5, dtype=torch.uint8)
    wide[:, 3:3 + K] = codes + 16   # bits above the low four do not count; rows at odd addresses
    m = ops.w4_pack(wide.cuda()[:, 3:3 + K], scale.cuda(), None if zero is None else zero.cuda())
    assert m.group == group and m.codes.shape == (N, L.lib().hx_w4_row_bytes(K))
    assert torch.equal(unpack(m), codes)
    if K % 128:   # the last block is filled up with code 8
        full = ops.W4Matrix(N, (K + 127) // 128 * 128, 32, torch.zeros(N, (K + 127) // 128 * 4, device="cuda"), None)
        full.codes = m.codes
        assert (unpack(full)[:, K:] == 8).all()
    want = values(codes, scale, zero, group)
    assert torch.equal(ops.w4_dequantize(m).cpu(), want.float())
    assert torch.equal(ops.w4_dequantize(m, torch.bfloat16).cpu(), want.float().bfloat16())
    out = torch.full((N, K + 3), 7.0, device="cuda")
    ops.w4_dequantize(m, out=out[:, 1:1 + K])
    assert torch.equal(out[:, 1:1 + K].cpu(), want.float()) and (out[:, 0] == 7).all() and (out[:, 1 + K:] == 7).all()


def definition(w, group, zeros, scale_dtype):
    """Codes, scale and zero point as the header defines them, in 64 bits."""
    N, K = w.shape
    v = w.double().view(N, K // group, group)
    if zeros:
        lo, hi = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
        scale = ((hi - lo) / 15).float()
    else:
        scale = (v.abs().amax(2) / 7).float()
    scale = scale.to(scale_dtype)
    s = scale.double()
    none = s == 0
    div = torch.where(none, 1.0, s)
    zero = (-lo / div).round().clamp(0, 15) if zeros else torch.full_like(s, 8.0)
    code = ((v / div[:, :, None]).round() + zero[:, :, None]).clamp(0 if zeros else 1, 15)
    zero = torch.where(none, 8.0, zero)
    code = torch.where(none[:, :, None], 8.0, code)
    return code.view(N, K).to(torch.uint8), scale, zero.to(torch.uint8) if zeros else None


def check_quantize(w, group, zeros, scale_dtype):
    m = ops.w4_quantize(w, group, zero_points=zeros, scale_dtype=scale_dtype)
    code, scale, zero = definition(w.cpu(), group, zeros, scale_dtype)
    assert torch.equal(m.scale.cpu(), scale)
    if zeros:
        assert torch.equal(m.zero.cpu(), zero)
    else:
        assert m.zero is None
    assert torch.equal(unpack(m), code)
    return m


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("wdt,sdt", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (5, 96, 32), (33, 192, 64), (16, 384, 128), (257, 1024, 64), (3, 4096, 128)])
def test_quantize(N, K, group, wdt, sdt, zeros):
    gen = torch.Generator().manual_seed(N + K)
    w = (torch.randn(N, K, generator=gen) * torch.logspace(-3, 3, N)[:, None]).to(DT[wdt]).cuda()
    check_quantize(w, group, zeros, DT[sdt])
    wide = torch.zeros(N, K + 3, dtype=DT[wdt], device="cuda")
    wide[:, 1:K + 1] = w   # rows off every vector's alignment
    a, b = ops.w4_quantize(w, group, zeros, DT[sdt]), ops.w4_quantize(wide[:, 1:K + 1], group, zeros, DT[sdt])
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scale, b.scale)


@pytest.mark.parametrize("sdt", ["f32", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_on_and_beside_the_halves(zeros, sdt):
    """Weights on every half step of their scale and one unit in the last place to either side."""
    steps = torch.arange(-15, 16).double() / 2
    rows = []
    for s in (1.0, 0.75, 0.1, 1.7e-5, 333.0):
        s = torch.tensor(s).to(DT[sdt]).double().item()
        at = (steps * s).float()
        up = torch.nextafter(at, torch.tensor(float("inf")))
        down = torch.nextafter(at, torch.tensor(float("-inf")))
        for v in (at, up, down):
            lim = torch.tensor([7 * s], dtype=torch.float64).float()   # the largest weight, so that the scale comes out as s
            rows.append(torch.cat([torch.clamp(v, -lim.item(), lim.item()), lim]))
    check_quantize(torch.stack(rows).cuda(), 32, zeros, DT[sdt])


@pytest.mark.parametrize("sdt", ["f32", "bf16"])
@pytest.mark.parametrize("wdt", ["f32", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_short_numbers(zeros, wdt, sdt):
    """Weights and scales of few bits, whose quotients are often exactly a half, at ordinary and at extreme sizes."""
    gen = torch.Generator().manual_seed(3)
    w = torch.randn(640, 1024, generator=gen)
    w[:320] = (w[:320] * 8).round() / 8
    w[320:480] = (w[320:480] * 100).round()
    w = w * torch.tensor([1.0, 2.0 ** -100, 2.0 ** -118, 2.0 ** 100]).repeat(160)[:, None]
    check_quantize(w.to(DT[wdt]).cuda(), 64, zeros, DT[sdt])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (4, 4), (8, 8), (8, 24), (1, 0), (16, 16)])
def test_dequantize_at_every_alignment(offset, pad, dtype):
    codes, scale, zero = make(9, 11, 96, 32, torch.float32, True)
    m = ops.w4_pack(codes.cuda(), scale.cuda(), zero.cuda())
    flat = torch.full((offset + 11 * (96 + pad) + 32,), 7.0, device="cuda", dtype=DT[dtype])
    out = flat[offset:offset + 11 * (96 + pad)].view(11, 96 + pad)
    ops.w4_dequantize(m, DT[dtype], out=out[:, :96])
    assert torch.equal(out[:, :96].cpu(), values(codes, scale, zero, 32).float().to(DT[dtype]))
    assert (out[:, 96:] == 7).all() and (flat[:offset] == 7).all() and (flat[offset + 11 * (96 + pad):] == 7).all()


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_of_unusual_groups(zeros):
    """Groups of zeros, of one sign, of one value, of denormals, with the largest numbers; infinities and NaN spoil their group."""
    w = torch.randn(12, 64, generator=torch.Generator().manual_seed(2))
    w[0] = 0.0
    w[1] = w[1].abs() + 1
    w[2] = -w[2].abs() - 1
    w[3] = 3.0
    w[4] *= 1e-42
    w[5, :32] = 1e-45
    w[6] = 3.4e38 * torch.sign(w[6])
    w[7] = -0.0
    for sdt in (torch.float32, torch.bfloat16):
        check_quantize(w.cuda(), 32, zeros, sdt)
    w[8, 3], w[9, 40], w[10, 5], w[10, 60] = float("inf"), float("-inf"), float("nan"), 1.0
    m = ops.w4_quantize(w.cuda(), 32, zero_points=zeros)
    back = ops.w4_dequantize(m).cpu()
    bad = torch.zeros(12, 2, dtype=torch.bool)
    bad[8, 0] = bad[9, 1] = bad[10, 0] = True
    assert torch.equal(torch.isnan(m.scale.cpu()), bad)
    assert torch.equal(torch.isnan(back), bad.repeat_interleave(32, 1))


# ------------------------------------------------------------------ the product
def activation(c, epilogue):
    if epilogue == L.EPI_SILU:
        return c * torch.sigmoid(c)
    return torch.nn.functional.softplus(c) if epilogue == L.EPI_SOFTPLUS else c


def check_product(got, a, w, bias, epilogue=L.EPI_NONE):
    a, w = a.double().cpu(), w
    c = a @ w.t()
    tol = 2 * U * (18 + w.shape[1] / 16) * (a.abs() @ w.abs().t())
    if bias is not None:
        c, tol = c + bias.double().cpu(), tol + U * (c.abs() + bias.double().cpu().abs())
    if epilogue != L.EPI_NONE:   # slopes of at most 1.1, and a few units of the functions themselves
        c, tol = activation(c, epilogue), 1.1 * tol + 16 * U * (c.abs() + 1)
    eps = torch.finfo(got.dtype).eps / 2
    err = (got.double().cpu() - c).abs() - (tol * (1 + eps) + eps * c.abs() + 2.0 ** -126)
    assert not torch.isnan(got).any()
    assert err.max().item() <= 0, err.max().item()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("adt", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(1, 1, 32, 32), (1, 7, 64, 64), (1, 16, 128, 128), (2, 33, 96, 32), (7, 100, 320, 64), (8, 64, 1536, 64),
                                         (9, 40, 384, 128), (16, 129, 1024, 32), (17, 48, 2048, 128), (24, 257, 768, 32), (33, 31, 640, 64),
                                         (64, 200, 512, 128), (65, 20, 256, 64), (130, 72, 160, 32), (1, 768, 1536, 64), (3, 5, 8192, 128),
                                         (1, 2500, 256, 32), (5, 4, 16416, 32), (12, 1000, 4096, 64)])
def test_product(M, N, K, group, adt, zeros):
    codes, scale, zero = make(M + N + K, N, K, group, DT[adt], zeros)
    m = ops.w4_pack(codes.cuda(), scale.cuda(), None if zero is None else zero.cuda())
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(DT[adt]).cuda()
    w = values(codes, scale, zero, group)
    got = ops.gemm_w4(a, m)
    assert got.dtype == a.dtype and got.shape == (M, N)
    check_product(got, a, w, None)
    assert torch.equal(got, ops.gemm_w4(a, m))
    assert L.device_status() == 0


@pytest.mark.parametrize("adt", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(8, 40, 16384, 128), (2, 768, 12288, 64), (1, 300, 16384, 32), (20, 2600, 1056, 32), (50, 900, 4096, 128)])
def test_product_shared_by_clusters(M, N, K, group, adt):
    """Long rows and few outputs: the columns are cut over CTAs, or the rows are too long to be staged whole."""
    codes, scale, zero = make(M + N + K, N, K, group, DT[adt], True)
    m = ops.w4_pack(codes.cuda(), scale.cuda(), zero.cuda())
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(DT[adt]).cuda()
    got = ops.gemm_w4(a, m, out_dtype=torch.float32)
    check_product(got, a, values(codes, scale, zero, group), None)
    assert torch.equal(got, ops.gemm_w4(a, m, out_dtype=torch.float32))


@pytest.mark.parametrize("epilogue", [L.EPI_NONE, L.EPI_SILU, L.EPI_SOFTPLUS])
@pytest.mark.parametrize("adt,cdt,sdt", [("f32", "f32", "bf16"), ("f32", "bf16", "f32"), ("bf16", "f32", "f32"), ("bf16", "bf16", "bf16")])
def test_product_types_bias_and_epilogue(adt, cdt, sdt, epilogue):
    for M, N, K, group in ((3, 50, 256, 64), (20, 24, 160, 32)):
        codes, scale, zero = make(4, N, K, group, DT[sdt], True)
        m = ops.w4_pack(codes.cuda(), scale.cuda(), zero.cuda())
        gen = torch.Generator().manual_seed(5)
        a, bias = torch.randn(M, K, generator=gen).to(DT[adt]).cuda(), torch.randn(N, generator=gen).cuda()
        got = ops.gemm_w4(a, m, bias=bias, out_dtype=DT[cdt], epilogue=epilogue)
        check_product(got, a, values(codes, scale, zero, group), bias, epilogue)


@pytest.mark.parametrize("adt", ["f32", "bf16"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (0, 8), (1, 1), (2, 6), (4, 4), (3, 5)])
def test_product_on_views(adt, offset, pad):
    """Rows at every alignment; what lies between the rows of A may be NaN, what lies between those of C stays."""
    for M in (1, 3, 20):
        N, K, group = 37, 288, 32
        codes, scale, zero = make(6, N, K, group, torch.float32, False)
        m = ops.w4_pack(codes.cuda(), scale.cuda())
        flat = torch.full((offset + M * (K + pad) + 64,), float("nan"), device="cuda", dtype=DT[adt])
        a = flat[offset:offset + M * (K + pad)].view(M, K + pad)[:, :K]
        a.copy_(torch.randn(M, K, generator=torch.Generator().manual_seed(7)).to(DT[adt]))
        out = torch.full((offset + M * (N + pad) + 64,), 7.0, device="cuda", dtype=DT[adt])
        c = out[offset:offset + M * (N + pad)].view(M, N + pad)
        ops.gemm_w4(a, m, out=c[:, :N])
        check_product(c[:, :N], a, values(codes, scale, None, group), None)
        assert (c[:, N:] == 7).all() and (out[:offset] == 7).all() and (out[offset + M * (N + pad):] == 7).all()
    one = torch.randn(1, K, generator=torch.Generator().manual_seed(8)).to(DT[adt]).cuda()
    assert torch.equal(ops.gemm_w4(one.expand(5, K), m), ops.gemm_w4(one.expand(5, K).contiguous(), m))   # one row five times


def test_product_of_more_rows_than_a_grid_holds():
    codes, scale, _ = make(14, 5, 32, 32, torch.float32, False)
    m = ops.w4_pack(codes.cuda(), scale.cuda())
    M = 65535 * 64 + 70
    a = torch.zeros(M, 32, device="cuda", dtype=torch.bfloat16)
    for r in (0, 63, 65535 * 64 - 1, 65535 * 64, M - 1):
        a[r] = torch.randn(32, generator=torch.Generator().manual_seed(r)).bfloat16()
    c = ops.gemm_w4(a, m, out_dtype=torch.float32)
    w = values(codes, scale, None, 32)
    rows = torch.tensor([0, 63, 64, 65535 * 64 - 1, 65535 * 64, M - 2, M - 1])
    check_product(c[rows.cuda()], a[rows.cuda()], w, None)
    assert (c != 0).any(1).sum().item() == 5


def test_product_keeps_fp32_operands():
    """fp32 rows whose bf16 part cancels: what is left is in the bits below."""
    K = 256
    codes = torch.full((16, K), 9, dtype=torch.uint8)   # value 1
    m = ops.w4_pack(codes.cuda(), torch.ones(16, K // 64, device="cuda"))
    a = torch.ones(2, K)
    a[:, 1::2] = -1.0
    a[0, ::2] += 2.0 ** -20
    a[1, ::2] += 2.0 ** -12
    got = ops.gemm_w4(a.cuda(), m)
    assert torch.equal(got[0].cpu(), torch.full((16,), 128 * 2.0 ** -20)) and torch.equal(got[1].cpu(), torch.full((16,), 128 * 2.0 ** -12))
    scales = torch.tensor([[1e-30, 1.0], [1e30, 1e-38]])   # groups of very different scale keep their own
    m = ops.w4_pack(torch.full((2, 128), 10, dtype=torch.uint8).cuda(), scales.cuda())
    a = torch.zeros(1, 128)
    a[0, 0], a[0, 64] = 1e10, 1e-10
    got = ops.gemm_w4(a.cuda(), m).cpu().double()
    want = a.double() @ (2 * scales.double().repeat_interleave(64, 1)).t()
    # 2 * 1e30 * 1e10 is beyond fp32's 3.4e38: infinity is its rounding there
    over = want.abs() > torch.finfo(torch.float32).max
    assert over.sum() == 1 and torch.equal(got[over], torch.sign(want[over]) * float("inf"))
    assert ((got - want)[~over].abs() <= 4 * U * want[~over].abs()).all()


@pytest.mark.parametrize("adt", ["f32", "bf16"])
def test_product_of_infinities_and_nan(adt):
    """They stay in their row of A and their column of C."""
    codes, scale, _ = make(9, 20, 256, 64, torch.float32, False)
    codes[codes == 8] = 9   # no weight of zero: inf * 0 would be NaN
    scale[7, 1] = float("nan")
    scale[11, 2] = float("inf")
    m = ops.w4_pack(codes.cuda(), scale.cuda())
    a = torch.randn(6, 256, generator=torch.Generator().manual_seed(10)).to(DT[adt])
    a[2, 100], a[4, 3] = float("inf"), float("nan")
    clean = torch.randn(6, 256, generator=torch.Generator().manual_seed(10)).to(DT[adt])
    got = ops.gemm_w4(a.cuda(), m).cpu()
    assert torch.isnan(got[4]).all() and torch.isnan(got[:, 7]).all()
    cols = [n for n in range(20) if n not in (7, 11)]
    rows = [0, 1, 3, 5]
    w = values(codes, scale, None, 64)
    sign = torch.sign(w[:, 100])
    assert torch.equal(got[2, cols].double(), (sign * float("inf"))[cols])
    assert not torch.isfinite(got[:, 11]).any()
    check_product(got[rows][:, cols], clean[rows], w[cols], None)


def test_offsets_beyond_32_bits():
    """More than 2^31 codes in one matrix: the last rows are read where they are."""
    N, K = 16400, 131072 + 128
    assert N * K > 1 << 31
    m = ops.W4Matrix(N, K, 128, torch.ones(N, K // 128, device="cuda"), None)
    m.codes.fill_(0x88)
    m.codes[-1] = 0x99   # every code 9: the value 1
    a = torch.ones(1, K, device="cuda")
    c = ops.gemm_w4(a, m)
    assert (c[0, :-1] == 0).all() and c[0, -1].item() == K
    del c
    out = torch.empty(N, K, device="cuda", dtype=torch.bfloat16)
    ops.w4_dequantize(m, torch.bfloat16, out=out)
    assert (out[-1] == 1).all() and (out[-2] == 0).all()
    m2 = ops.w4_quantize(out, 128)
    assert torch.equal(m2.codes[-1], torch.full_like(m2.codes[-1], 0xFF)) and (m2.codes[-2] == 0x88).all()


def test_streams_and_graphs():
    codes, scale, zero = make(11, 600, 512, 64, torch.float32, True)
    m = ops.w4_pack(codes.cuda(), scale.cuda(), zero.cuda())
    a = torch.randn(4, 512, device="cuda")
    want = ops.gemm_w4(a, m)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [ops.gemm_w4(a, m) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = ops.gemm_w4(a, m)
    for seed in range(3):
        a.copy_(torch.randn(4, 512, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        assert torch.equal(c, ops.gemm_w4(a, m))


def test_refusals():
    codes, scale, zero = (t.cuda() if t is not None else None for t in make(12, 8, 256, 64, torch.float32, True))
    m = ops.w4_pack(codes, scale, zero)
    a = torch.zeros(2, 256, device="cuda")
    for code, call in [
        (1, lambda: ops.w4_pack(codes, scale[:, :3])),
        (1, lambda: ops.w4_pack(codes, scale[:4])),
        (1, lambda: ops.w4_pack(codes, scale[:, :1])),       # a group of 256
        (4, lambda: ops.w4_pack(codes.int(), scale)),
        (4, lambda: ops.w4_pack(codes, scale.half())),
        (4, lambda: ops.w4_pack(codes, scale, zero.int())),
        (3, lambda: ops.w4_pack(codes, scale.cpu())),
        (3, lambda: ops.w4_pack(codes.cpu(), scale.cpu())),
        (1, lambda: ops.w4_quantize(a, 48)),
        (1, lambda: ops.w4_quantize(a[:, :80], 32)),
        (1, lambda: ops.w4_quantize(a[0], 32)),
        (1, lambda: ops.w4_quantize(a.t(), 32)),
        (4, lambda: ops.w4_quantize(a.half(), 32)),
        (4, lambda: ops.w4_quantize(a, 32, scale_dtype=torch.float16)),
        (3, lambda: ops.w4_quantize(a.cpu(), 32)),
        (4, lambda: ops.w4_dequantize(m, torch.float16)),
        (1, lambda: ops.w4_dequantize(m, out=a)),
        (1, lambda: ops.gemm_w4(a[:, :128], m)),
        (1, lambda: ops.gemm_w4(a[0], m)),
        (4, lambda: ops.gemm_w4(a.half(), m)),
        (4, lambda: ops.gemm_w4(a, m, out_dtype=torch.float16)),
        (1, lambda: ops.gemm_w4(a, m, bias=torch.zeros(7, device="cuda"))),
        (4, lambda: ops.gemm_w4(a, m, bias=torch.zeros(8, device="cuda").bfloat16())),
        (1, lambda: ops.gemm_w4(a, m, out=torch.zeros(2, 7, device="cuda"))),
        (1, lambda: ops.gemm_w4(a, m, out=torch.zeros(1, 8, device="cuda").expand(2, 8))),
        (10, lambda: ops.gemm_w4(a, m, epilogue=3)),
        (3, lambda: ops.gemm_w4(a.cpu(), m)),
    ]:
        with pytest.raises(L.HxError) as e:
            call()
        assert e.value.status == code


# ------------------------------------------------------------------ used together
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_recurrent_layer_served_with_4_bit_weights(dtype):
    """A gated recurrent layer: prefill of a ragged batch through the dense products and the scan, then tokens one by one
    through 4-bit products and the step, against the layer in 64 bits on the same 4-bit weights."""
    B, Lq, M, E, T = 3, 40, 96, 160, 6
    dt = DT[dtype]
    gen = torch.Generator().manual_seed(13)
    w_in, w_out = (ops.w4_quantize((torch.randn(n, k, generator=gen) * k ** -0.5).to(dt).cuda(), 32, zero_points=True)
                   for n, k in ((2 * E, M), (M, E)))
    lengths = torch.tensor([40, 17, 1], dtype=torch.int32)
    tokens = torch.randn(B, Lq + T, M, generator=gen).to(dt).cuda()
    d_in, d_out = ops.w4_dequantize(w_in, dt), ops.w4_dequantize(w_out, dt)
    xg = ops.gemm(tokens[:, :Lq].reshape(-1, M), d_in).view(B, Lq, 2 * E)
    h, state = ops.gated_scan(xg[:, :, :E], xg[:, :, E:], lengths=lengths.cuda(), return_state=True)
    ops.gemm(h.view(-1, E), d_out)
    outs = []
    for t in range(T):
        xg1 = ops.gemm_w4(tokens[:, Lq + t], w_in)
        y = ops.gated_scan_step(xg1[:, :E], xg1[:, E:], state)
        outs.append(ops.gemm_w4(y, w_out))
    # 64 bits; bf16 rounds the dequantised weights of the prefill, the projections, y and the output
    W_in, W_out = ops.w4_dequantize(w_in).double().cpu(), ops.w4_dequantize(w_out).double().cpu()
    x = tokens.double().cpu()
    ref = torch.zeros(B, E, dtype=torch.float64)
    for b in range(B):
        for t in list(range(int(lengths[b]))) + list(range(Lq, Lq + T)):
            p = W_in @ x[b, t]
            a = torch.sigmoid(p[E:])
            ref[b] = a * ref[b] + (1 - a) * p[:E]
            if t >= Lq:
                want = W_out @ ref[b]
                # relative errors of p (2 roundings of 2^-8 on sqrt(M) terms), y and the output add up to a few eps of the norms
                tol = (1e-4 if dtype == "f32" else 8 * 2.0 ** -8) * (1 + want.abs().max())
                assert (outs[t - Lq][b].double().cpu() - want).abs().max() <= tol
