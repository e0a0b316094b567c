"""The gated linear recurrence, its gradients and its single-token step against the recurrence in 64 bits.

Tolerances.  u = 2^-24.  With M_t = |a_t| M_{t-1} + |b_t| (all signs taken away) and W_t = |a_t| (W_{t-1} + M_{t-1}), W_t is the sum
over the inputs of their weight in M_t times the number of steps they are old.  Whatever the order in which the recurrence is
associated, an input that is s steps old has gone through s products and s sums, each rounded (2 u a step), and through s decays
that are themselves off: by 4 u where the sigmoid is computed with expf (2 ulp = 4 u of an e <= 1 that enters 1 + e with weight
e / (1 + e) <= 1/2, the sum and the division 1 u each), by 7 u with the hardware's exp2 and reciprocal (|g| + 5 u of e with the same
weight, 4 u for sum and reciprocal).  So h_t is within 16 u W_t + 64 u M_t of the exact value, where the second term covers the
input's own coefficient (1 - a is off by up to (|g| + 13) u, |g| <= 40 here) and the first sum; the result's rounding adds
eps / 2 |h_t|.  The same holds for delta backwards in time."""
import numpy as np
import pytest
import torch

from helixml_b200 import _lib as L
from helixml_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def coefficients(x, g, gate):
    """a, b in 64 bits, and 1 - a for the sigmoid."""
    if gate == "decay":
        return g, x, None
    return torch.sigmoid(g), torch.sigmoid(-g) * x, torch.sigmoid(-g)


def recur(a, b, h0):
    """h, and the M and W of the module's comment, over axis 1; 64 bits, one step after the other."""
    h, m, w = h0.clone(), h0.abs(), torch.zeros_like(h0)
    hs, ms, ws = [], [], []
    for t in range(a.shape[1]):
        w = a[:, t].abs() * (w + m)
        m = a[:, t].abs() * m + b[:, t].abs()
        h = a[:, t] * h + b[:, t]
        hs.append(h), ms.append(m), ws.append(w)
    return (torch.stack(v, 1) if v else b.new_zeros(b.shape) for v in (hs, ms, ws))


def masked(lengths, B, Lq):
    n = torch.full((B,), Lq) if lengths is None else torch.as_tensor(lengths).clamp(0, Lq)
    return (torch.arange(Lq)[None] < n[:, None])[:, :, None]


def reference(x, g, h0, gate, lengths=None):
    """(h, tolerance of h, h_last, tolerance) on the CPU from the very values the kernel gets."""
    x, g, h0 = x.double().cpu(), g.double().cpu(), h0.double().cpu()
    B, Lq, D = x.shape
    inside = masked(lengths, B, Lq)
    x, g = torch.where(inside, x, 0.0), torch.where(inside, g, 0.0)
    a, b, _ = coefficients(x, g, gate)
    a, b = torch.where(inside, a, 1.0), torch.where(inside, b, 0.0)
    h, m, w = recur(a, b, h0)
    tol = 16 * U * w + 64 * U * m
    last = h[:, -1] if Lq else h0
    last_tol = tol[:, -1] if Lq else torch.zeros_like(h0)
    return torch.where(inside, h, 0.0), torch.where(inside, tol, 0.0), last, last_tol


def reference_bwd(dh, x, g, h0, dh_last, gate, lengths=None):
    """((dx, tol), (dg, tol), (dh0, tol)) without the results' own rounding."""
    dh, x, g, h0, dh_last = (t.double().cpu() for t in (dh, x, g, h0, dh_last))
    B, Lq, D = x.shape
    inside = masked(lengths, B, Lq)
    x, g, dh = torch.where(inside, x, 0.0), torch.where(inside, g, 0.0), torch.where(inside, dh, 0.0)
    a, b, rest = coefficients(x, g, gate)
    a, b = torch.where(inside, a, 1.0), torch.where(inside, b, 0.0)
    h, m, w = recur(a, b, h0)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    before_tol = torch.cat([torch.zeros_like(h0)[:, None], (16 * U * w + 64 * U * m)[:, :-1]], 1)
    before_m = torch.cat([h0.abs()[:, None], m[:, :-1]], 1)
    # delta_t = dh_t + a_{t+1} delta_{t+1}
    nxt = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1).flip(1)
    delta, dm, dw = (v.flip(1) for v in recur(nxt, dh.flip(1), dh_last))
    dtol = 16 * U * dw + 64 * U * dm
    if gate == "decay":
        dx, dx_tol = delta, dtol
        dg, dg_tol = delta * before, dtol * before.abs() + dm * before_tol
    else:
        ar = a * rest
        dx, dx_tol = delta * rest, (dtol + 64 * U * dm) * rest
        dg = delta * (before - x) * ar
        dg_tol = (dtol * (before - x).abs() + dm * (before_tol + 128 * U * (before_m + x.abs()))) * ar
    dh0 = a[:, 0] * delta[:, 0]
    z = lambda t: torch.where(inside, t, 0.0)
    return (z(dx), z(dx_tol)), (z(dg), z(dg_tol)), (dh0, a[:, 0].abs() * (dtol[:, 0] + 16 * U * dm[:, 0]))


def assert_within(got, want, tol, what=""):
    eps = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    # 2^-126: results below the smallest normal number may be flushed
    err = (got - want).abs() - (tol * (1 + eps) + want.abs() * eps + 2.0 ** -126)
    assert not torch.isnan(got).any(), what
    worst = err.max().item() if err.numel() else 0.0
    assert worst <= 0, f"{what}: over the tolerance by {worst:.3g} at {np.unravel_index(int(err.argmax()), err.shape)}"


def inputs(seed, B, Lq, D, dtype, gate, shift=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, Lq, D, generator=gen)
    g = shift + 2.0 * torch.randn(B, Lq, D, generator=gen)
    if gate == "decay":
        g = torch.sigmoid(g) * torch.where(torch.rand(B, Lq, D, generator=gen) < 0.1, -1.0, 1.0)
    h0, dh_last = torch.randn(B, D, generator=gen), torch.randn(B, D, generator=gen)
    dh = torch.randn(B, Lq, D, generator=gen)
    dev = lambda t: t.to(DT[dtype]).cuda()
    return dev(x), dev(g), h0.cuda(), dev(dh), dh_last.cuda()


def check(x, g, h0, dh, dh_last, gate, lengths=None, out=None, grads=None):
    """Forward and backward of one call, both held against the reference."""
    B, Lq, D = x.shape
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    states = ops.gated_scan_states(B, Lq, D)
    h, last = ops.gated_scan(x, g, h0=h0, gate=gate, lengths=n, return_state=True, states=states, out=out)
    want, tol, want_last, last_tol = reference(x, g, h0, gate, lengths)
    assert_within(h, want, tol, "h")
    assert_within(last, want_last, last_tol, "h_last")
    got = ops.gated_scan_bwd(dh, x, g, states, gate=gate, lengths=n, dh_last=dh_last, out=grads)
    for name, t, (w, wt) in zip(("dx", "dg", "dh0"), got, reference_bwd(dh, x, g, h0, dh_last, gate, lengths)):
        assert_within(t, w, wt, name)
    assert L.device_status() == 0
    return h, last, got


SHAPES = [(1, 1, 1), (2, 7, 5), (1, 63, 33), (1, 64, 128), (3, 65, 130), (2, 200, 96), (1, 1000, 257), (9, 129, 64), (1, 4133, 40),
          (2, 2048, 256), (40, 3, 8), (1, 511, 1000), (300, 70, 64), (3, 96, 1536)]


@pytest.mark.parametrize("gate", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(shape, dtype, gate):
    check(*inputs(sum(shape), *shape, dtype, gate), gate)


@pytest.mark.parametrize("gate", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_memory_over_many_tiles(dtype, gate):
    """Decays near one: a state of the first tile is still there thousands of steps later."""
    x, g, h0, dh, dh_last = inputs(5, 1, 5000, 72, dtype, gate, shift=9.0)
    check(x, g, h0, dh, dh_last, gate)


@pytest.mark.parametrize("dtype,gate,shape,lengths", [("f32", "decay", (1, 22500, 1030), None),
                                                      ("bf16", "sigmoid", (3, 16000, 1000), [16000, 37, 11001])])
def test_inputs_larger_than_the_cache(dtype, gate, shape, lengths):
    """Long sequences of few channels are worked off span by span; a row may end in any of them."""
    x, g, h0, dh, dh_last = inputs(6, *shape, dtype, gate, shift=6.0)
    check(x, g, h0, dh, dh_last, gate, lengths=lengths)


def test_infinity_across_spans():
    """A state that has become infinite in the first span is what the last one starts from, and a gradient the other way."""
    Lq, D = 24000, 1024
    a = torch.full((1, Lq, D), 0.5, device="cuda")
    x, dh = torch.zeros(1, Lq, D, device="cuda"), torch.zeros(1, Lq, D, device="cuda")
    x[0, 3, 7], dh[0, Lq - 5, 9] = float("inf"), float("-inf")
    a[0, :, 11], x[0, 12000:, 11] = 2.0, 1.0          # a product that overflows over a state of zero
    states = ops.gated_scan_states(1, Lq, D)
    h, last = ops.gated_scan(x, a, gate="decay", states=states, return_state=True)
    assert torch.isposinf(h[0, 3:, 7]).all() and (h[0, :3, 7] == 0).all() and torch.isposinf(last[0, 7])
    assert (h[0, :12000, 11] == 0).all() and h[0, 12003, 11].item() == 15.0 and torch.isposinf(last[0, 11])
    others = [c for c in range(D) if c not in (7, 11)]
    assert (h[0][:, others] == 0).all()
    dx, dg, dh0 = ops.gated_scan_bwd(dh, x, a, states, gate="decay")
    assert torch.isneginf(dx[0, :Lq - 4, 9]).all() and (dx[0, Lq - 4:, 9] == 0).all() and torch.isneginf(dh0[0, 9])


@pytest.mark.parametrize("gate", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_padded_batches(dtype, gate):
    """Rows behind a sequence's end hold NaN and infinity; lengths 0, 1, around tile edges, full, and beyond the range."""
    lengths = [0, 1, 63, 64, 65, 300, 299, 128, -3, 1000]
    x, g, h0, dh, dh_last = inputs(7, len(lengths), 300, 70, dtype, gate)
    for i, n in enumerate(lengths):
        n = min(max(n, 0), 300)
        for t, v in ((x, float("nan")), (g, float("inf")), (dh, float("-inf"))):
            t[i, n:] = v
            t[i, n + 1::2] = float("nan")
    h, last, (dx, dg, dh0) = check(x, g, h0, dh, dh_last, gate, lengths=lengths)
    assert torch.equal(last[0], h0[0]) and torch.equal(dh0[0], dh_last[0])
    for t in (h, dx, dg):
        assert (t[0] == 0).all() and (t[1, 1:] == 0).all() and (t[8] == 0).all()


def test_without_state_and_optional_operands():
    x, g, h0, dh, _ = inputs(8, 2, 150, 40, "f32", "sigmoid")
    zero = torch.zeros_like(h0)
    assert torch.equal(ops.gated_scan(x, g), ops.gated_scan(x, g, h0=zero))
    states = ops.gated_scan_states(2, 150, 40)
    h = ops.gated_scan(x, g, states=states)
    assert torch.equal(h, ops.gated_scan(x, g))
    for a, b in zip(ops.gated_scan_bwd(dh, x, g, states), ops.gated_scan_bwd(dh, x, g, states, dh_last=zero)):
        assert torch.equal(a, b)
    tol = 1e-5
    for t, row in ((0, 0), (16, 1), (64, 4), (144, 9)):
        want = zero if t == 0 else h[:, t - 1]
        assert (states[:, row] - want).abs().max().item() <= tol


@pytest.mark.parametrize("gate", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_without_workspace_the_sequence_is_walked_whole(dtype, gate, monkeypatch):
    x, g, h0, dh, dh_last = inputs(18, 2, 777, 70, dtype, gate)
    monkeypatch.setattr(ops, "_gated_scan_workspace", lambda *a: None)
    check(x, g, h0, dh, dh_last, gate)


@pytest.mark.parametrize("empty", [(0, 5, 8), (2, 0, 8), (2, 5, 0)])
def test_empty(empty):
    B, Lq, D = empty
    x = torch.zeros(empty, device="cuda")
    h0 = torch.randn(B, D, device="cuda")
    states = ops.gated_scan_states(B, Lq, D)
    h, last = ops.gated_scan(x, x, h0=h0, return_state=True, states=states)
    assert h.shape == x.shape and torch.equal(last, h0)
    dx, dg, dh0 = ops.gated_scan_bwd(x, x, x, states, dh_last=h0)
    assert dx.shape == x.shape and torch.equal(dh0, h0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (0, 8), (1, 3), (2, 2), (4, 4), (3, 1)])
def test_views(dtype, offset, pad):
    """Halves of one buffer at every alignment; outputs into halves of another, whose other elements stay as they were."""
    B, Lq, D = 3, 130, 52
    x, g, h0, dh, dh_last = inputs(9, B, Lq, D, dtype, "sigmoid")
    W = 2 * D + pad
    flat = torch.zeros(offset + B * Lq * W, device="cuda", dtype=DT[dtype])
    buf = flat[offset:].view(B, Lq, W)
    buf[:, :, :D], buf[:, :, D:2 * D] = x, g
    grads = torch.full((offset + B * Lq * W,), 7.0, device="cuda", dtype=DT[dtype])
    gv = grads[offset:].view(B, Lq, W)
    out = torch.full((offset + B * Lq * W,), 7.0, device="cuda", dtype=DT[dtype])
    ov = out[offset:].view(B, Lq, W)
    h, _, (dx, dg, _) = check(buf[:, :, :D], buf[:, :, D:2 * D], h0, dh, dh_last, "sigmoid", out=ov[:, :, D:2 * D],
                              grads=(gv[:, :, :D], gv[:, :, D:2 * D]))
    assert (ov[:, :, :D] == 7).all() and (ov[:, :, 2 * D:] == 7).all() and (out[:offset] == 7).all()
    assert (gv[:, :, 2 * D:] == 7).all() and (grads[:offset] == 7).all()


@pytest.mark.parametrize("D", [64, 37])
def test_fp32_operands_off_eight_bytes(D):
    """Contiguous states, h0 and dh_last that begin one element into a buffer."""
    x, g, h0, dh, dh_last = inputs(19, 2, 100, D, "bf16", "sigmoid")
    off = lambda t: torch.cat([torch.zeros(1, device="cuda"), t.flatten()])[1:].view(t.shape)
    st = ops.gated_scan_states(2, 100, D)
    flat = torch.full((st.numel() + 2,), 7.0, device="cuda")
    shifted = flat[1:-1].view(st.shape)
    want = ops.gated_scan(x, g, h0=h0, states=st)
    assert torch.equal(ops.gated_scan(x, g, h0=off(h0), states=shifted), want)
    assert torch.equal(shifted, st) and flat[0] == 7 and flat[-1] == 7
    for a, b in zip(ops.gated_scan_bwd(dh, x, g, shifted, dh_last=off(dh_last)), ops.gated_scan_bwd(dh, x, g, st, dh_last=dh_last)):
        assert torch.equal(a, b)
    h, other = off(h0), off(torch.zeros_like(h0))
    y = ops.gated_scan_step(x[:, 0], g[:, 0], h, h_out=other)
    assert torch.equal(y, ops.gated_scan_step(x[:, 0], g[:, 0], h0)) and torch.equal(other, h0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_time_major_and_broadcast_views(dtype):
    x, g, h0, dh, dh_last = inputs(10, 4, 100, 36, dtype, "decay")
    tm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(100, 4, 36, device="cuda", dtype=DT[dtype]).transpose(0, 1)
    grads = tuple(torch.empty(100, 4, 36, device="cuda", dtype=DT[dtype]).transpose(0, 1) for _ in range(2))
    check(tm(x), tm(g), h0, tm(dh), dh_last, "decay", out=out, grads=grads)
    # one gate row for all steps, one for all rows
    check(x, g[:, :1].expand(-1, 100, -1), h0, dh, dh_last, "decay")
    check(x, g[:1].expand(4, -1, -1), h0, dh[:1, :1].expand(4, 100, -1), dh_last, "decay")


def test_offsets_beyond_32_bits():
    """The second batch row lies more than 2^32 bytes and 2^31 elements behind the first."""
    Lq, D = 70, 64
    stride = (1 << 31) + 64
    flat = torch.empty(stride + Lq * D, device="cuda", dtype=torch.bfloat16)
    far = lambda t: (lambda v: v.copy_(t))(flat.as_strided((2, Lq, D), (stride, D, 1)))
    x, g, h0, dh, dh_last = inputs(11, 2, Lq, D, "bf16", "sigmoid")
    h = ops.gated_scan(x, g, h0=h0)
    assert torch.equal(ops.gated_scan(far(x), g, h0=h0), h)
    out = flat.as_strided((2, Lq, D), (stride, D, 1))
    assert torch.equal(ops.gated_scan(x, g, h0=h0, out=out), h) and torch.equal(out, h)


# ------------------------------------------------------------------ values at the edges of the format
def sequential_f32(a, b, h0):
    out, h = [], h0.clone()
    for t in range(a.shape[1]):
        h = a[:, t] * h + b[:, t]
        out.append(h)
    return torch.stack(out, 1)


def same_special(got, want):
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    ok = torch.isfinite(want)
    assert ((got - want)[ok].abs() <= 1e-4 * (1 + want[ok].abs())).all()


def test_infinities_and_nan_are_those_of_the_recurrence():
    """An infinite input stays in the state however small the product of decays gets, a zero decay of it is NaN, a NaN stays;
    a state of zero under growing decays stays zero; every other channel is untouched."""
    B, Lq, D = 2, 700, 200
    gen = torch.Generator().manual_seed(3)
    a, x = 0.2 + 0.7 * torch.rand(B, Lq, D, generator=gen), torch.randn(B, Lq, D, generator=gen)
    inf, nan = float("inf"), float("nan")
    x[0, 5, 0], x[0, 70, 1], x[0, 300, 2], x[1, 0, 3] = inf, -inf, nan, inf
    x[1, 400, 3] = -inf                       # inf - inf
    x[0, 10, 4], a[0, 600, 4] = inf, 0.0      # 0 * inf
    a[0, 20:30, 5] = 0.0                      # forgets
    a[:, :, 6], x[:, :600, 6] = 2.0, 0.0      # 2^600 overflows over a state of zero
    a[:, :, 7], x[:, :, 7] = -1.0, 0.0
    a[0, 100, 8], x[0, :101, 8] = inf, 0.0    # inf * 0
    x[0, 650, 9], x[0, 651, 9] = 3e38, 3e38   # overflows in between
    a[0, 1:, 10], x[0, :, 10] = 1e-30, 0.0    # underflows
    h0 = torch.zeros(B, D)
    h0[0, 10], h0[1, 11] = 1.0, inf
    want = sequential_f32(a, x, h0)
    h, last = ops.gated_scan(x.cuda(), a.cuda(), h0=h0.cuda(), gate="decay", return_state=True)
    same_special(h.cpu(), want)
    same_special(last.cpu(), want[:, -1])


def test_infinite_gradients_are_those_of_the_recurrence():
    B, Lq, D = 2, 500, 150
    gen = torch.Generator().manual_seed(4)
    a, x, dh = 0.2 + 0.7 * torch.rand(B, Lq, D, generator=gen), torch.randn(B, Lq, D, generator=gen), torch.randn(B, Lq, D, generator=gen)
    dh[0, 450, 0], dh[1, 3, 1], dh[0, 200, 2] = float("inf"), float("-inf"), float("nan")
    a[:, :, 3], dh[:, 100:, 3] = 2.0, 0.0
    a[0, 40, 4], dh[0, 490, 4] = 0.0, float("inf")
    x[1, 30, 5] = float("inf")
    h0, dh_last = torch.randn(B, D), torch.zeros(B, D)
    dh_last[0, 6] = float("inf")
    h = sequential_f32(a, x, h0)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    nxt = torch.cat([a[:, 1:], torch.ones(B, 1, D)], 1)
    delta = sequential_f32(nxt.flip(1), dh.flip(1), dh_last).flip(1)
    states = ops.gated_scan_states(B, Lq, D)
    ops.gated_scan(x.cuda(), a.cuda(), h0=h0.cuda(), gate="decay", states=states)
    dx, dg, dh0 = ops.gated_scan_bwd(dh.cuda(), x.cuda(), a.cuda(), states, gate="decay", dh_last=dh_last.cuda())
    same_special(dx.cpu(), delta)
    same_special(dh0.cpu(), a[:, 0] * delta[:, 0])
    want = delta * before
    keep = torch.isfinite(before) & (before.abs() < 1e30)   # channel 3's states overflow: their products follow no tolerance
    same_special(torch.where(keep, dg.cpu(), 0.0), torch.where(keep, want, 0.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_at_the_ends_of_the_range(dtype):
    """sigmoid gates of +-infinity, of the type's largest and lowest value, and 1 - a where a rounds to 1."""
    big = torch.finfo(DT[dtype]).max
    vals = torch.tensor([float("inf"), float("-inf"), big, -big, 0.0, 80.0, -80.0, 17.0, -17.0, 100.0, -100.0, 30.0])
    g = vals[None, None].expand(1, 80, -1).contiguous().to(DT[dtype]).cuda()
    x = torch.full_like(g, 2.0)
    h0, ones = torch.ones(1, len(vals), device="cuda"), torch.ones_like(g)
    states = ops.gated_scan_states(1, 80, len(vals))
    h = ops.gated_scan(x, g, h0=h0, states=states)
    want, tol, _, _ = reference(x, g, h0, "sigmoid")
    assert_within(h, want, tol, "h")
    assert (h[0, :, 0] == 1).all() and (h[0, :, 1] == 2).all()
    got = ops.gated_scan_bwd(ones, x, g, states, dh_last=h0)
    for t, (w, wt) in zip(got, reference_bwd(ones, x, g, h0, h0, "sigmoid")):
        # |g| = 100: e is good to (|g| + 5) u
        assert_within(t, w, wt + 128 * U * w.abs(), "gradient")


# ------------------------------------------------------------------ gradients against differences
@pytest.mark.parametrize("gate", ["decay", "sigmoid"])
def test_gradients_against_differences(gate):
    """L = sum w h + sum v h_last, differenced through the kernel's own forward in f32.  L is linear in x and in h0, and in a
    single decay; for the sigmoid the third derivative is at most 1/8 of the gradient's scale, so a step of 2^-6 leaves
    2^-12 / 48 of it.  Rounding: L is a sum of a few hundred terms of size ~1, off by 1e-5; divided by the step 2^-5: 1e-3."""
    B, Lq, D = 1, 90, 3
    x, g, h0, w, v = inputs(12, B, Lq, D, "f32", gate, shift=1.0)
    states = ops.gated_scan_states(B, Lq, D)
    ops.gated_scan(x, g, h0=h0, gate=gate, states=states)
    grads = ops.gated_scan_bwd(w, x, g, states, gate=gate, dh_last=v)

    def loss(x, g, h0):
        h, last = ops.gated_scan(x, g, h0=h0, gate=gate, return_state=True)
        return ((h.double() * w.double()).sum() + (last.double() * v.double()).sum()).item()

    step = 2.0 ** -6
    for which, at in [(0, (0, 0, 0)), (0, (0, 63, 1)), (0, (0, 89, 2)), (1, (0, 0, 0)), (1, (0, 64, 1)), (1, (0, 89, 2)), (1, (0, 40, 0)),
                      (2, (0, 1))]:
        args = [x, g, h0]
        diff = []
        for sign in (1, -1):
            moved = args[which].clone()
            moved[at] += sign * step
            diff.append(loss(*[moved if i == which else t for i, t in enumerate(args)]))
        got = grads[which][at].item()
        assert abs((diff[0] - diff[1]) / (2 * step) - got) <= 1e-3 * (1 + abs(got)), (which, at)


# ------------------------------------------------------------------ single steps, parts, streams, graphs
@pytest.mark.parametrize("gate", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,D", [(1, 1), (3, 70), (1, 1536), (17, 257), (64, 512)])
def test_step(B, D, dtype, gate):
    """Rows of a projection's output, the state in place and into another buffer."""
    xg = torch.empty(B, 2 * D, device="cuda", dtype=DT[dtype])
    x, g, h0, _, _ = inputs(13, B, 1, D, dtype, gate)
    xg[:, :D], xg[:, D:] = x[:, 0], g[:, 0]
    want, tol, _, _ = reference(x, g, h0, gate)
    h, other = h0.clone(), torch.empty_like(h0)
    y = ops.gated_scan_step(xg[:, :D], xg[:, D:], h, gate=gate, h_out=other)
    assert torch.equal(h, h0)
    assert_within(other, want[:, 0], tol[:, 0], "state")
    assert_within(y, want[:, 0], tol[:, 0], "y")
    y2 = ops.gated_scan_step(xg[:, :D], xg[:, D:], h, gate=gate)
    assert torch.equal(y2, y) and torch.equal(h, other)
    wide = torch.full((B, 2 * D), 7.0, device="cuda", dtype=DT[dtype])
    ops.gated_scan_step(xg[:, :D], xg[:, D:], h0, gate=gate, h_out=other, out=wide[:, D:])
    assert torch.equal(wide[:, D:], y) and (wide[:, :D] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prefill_then_steps_and_parts(dtype):
    """A ragged prefill followed by single tokens, and a sequence in two parts, against the whole one."""
    B, Lq, D = 3, 140, 100
    x, g, h0, dh, dh_last = inputs(14, B, Lq, D, dtype, "sigmoid")
    want, tol, want_last, last_tol = reference(x, g, h0, "sigmoid")
    n = [100, 37, 1]
    _, h = ops.gated_scan(x, g, h0=h0, lengths=torch.tensor(n, dtype=torch.int32, device="cuda"), return_state=True)
    for k in range(39):
        at = [v + k for v in n]
        xt = torch.stack([x[i, t] for i, t in enumerate(at)])
        gt = torch.stack([g[i, t] for i, t in enumerate(at)])
        y = ops.gated_scan_step(xt, gt, h)
        assert_within(y, torch.stack([want[i, t] for i, t in enumerate(at)]), torch.stack([tol[i, t] for i, t in enumerate(at)]), f"step {k}")
    first, mid = ops.gated_scan(x[:, :77], g[:, :77], h0=h0, return_state=True)
    second, last = ops.gated_scan(x[:, 77:], g[:, 77:], h0=mid, return_state=True)
    assert_within(torch.cat([first, second], 1), want, tol, "parts")
    assert_within(last, want_last, last_tol, "last")


def test_same_result_every_time_and_on_two_streams():
    x, g, h0, dh, dh_last = inputs(15, 4, 1500, 300, "bf16", "sigmoid")
    states = ops.gated_scan_states(4, 1500, 300)
    h = ops.gated_scan(x, g, h0=h0, states=states)
    grads = ops.gated_scan_bwd(dh, x, g, states, dh_last=dh_last)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                st = ops.gated_scan_states(4, 1500, 300)
                got.append((ops.gated_scan(x, g, h0=h0, states=st), ops.gated_scan_bwd(dh, x, g, st, dh_last=dh_last)))
        torch.cuda.synchronize()
        for hh, gg in got:
            assert torch.equal(hh, h) and all(torch.equal(a, b) for a, b in zip(gg, grads))


def test_captured_into_graphs():
    """Two graphs of the same operators on their own tensors, replayed in turn with new inputs."""
    sets = []
    for seed in (16, 17):
        x, g, h0, dh, dh_last = inputs(seed, 2, 333, 96, "bf16", "decay")
        out, states = torch.empty_like(x), ops.gated_scan_states(2, 333, 96)
        grads = (torch.empty_like(x), torch.empty_like(x))
        n = torch.tensor([333, 200], dtype=torch.int32, device="cuda")
        ops.gated_scan(x, g, h0=h0, gate="decay", lengths=n, out=out, states=states)   # loads the kernels before the capture
        ops.gated_scan_bwd(dh, x, g, states, gate="decay", lengths=n, dh_last=dh_last, out=grads)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.gated_scan(x, g, h0=h0, gate="decay", lengths=n, out=out, states=states)
            _, _, dh0 = ops.gated_scan_bwd(dh, x, g, states, gate="decay", lengths=n, dh_last=dh_last, out=grads)
            h_next = torch.empty_like(h0)
            y = ops.gated_scan_step(x[:, 0], g[:, 0], h0, gate="decay", h_out=h_next)
        sets.append((graph, x, g, h0, dh, dh_last, n, out, grads, dh0, y, h_next))
    for turn in range(3):
        for i, (graph, x, g, h0, dh, dh_last, n, out, grads, dh0, y, h_next) in enumerate(sets):
            for t, v in zip((x, g, h0, dh, dh_last), inputs(20 + 2 * turn + i, 2, 333, 96, "bf16", "decay")):
                t.copy_(v)
            n.copy_(torch.tensor([333 - turn, 100 * turn], dtype=torch.int32))
            graph.replay()
            st = ops.gated_scan_states(2, 333, 96)
            assert torch.equal(out, ops.gated_scan(x, g, h0=h0, gate="decay", lengths=n, states=st))
            want = ops.gated_scan_bwd(dh, x, g, st, gate="decay", lengths=n, dh_last=dh_last)
            assert all(torch.equal(a, b) for a, b in zip((*grads, dh0), want))
            assert torch.equal(h_next, g[:, 0].float() * h0 + x[:, 0].float()) or (h_next - (g[:, 0].float() * h0 + x[:, 0].float())).abs().max() < 1e-6


def test_refusals():
    x = torch.zeros(2, 5, 8, device="cuda")
    st = ops.gated_scan_states(2, 5, 8)
    for code, call in [
        (4, lambda: ops.gated_scan(x, x.bfloat16())),
        (1, lambda: ops.gated_scan(x, x[:, :4])),
        (1, lambda: ops.gated_scan(x.transpose(1, 2), x.transpose(1, 2))),
        (10, lambda: ops.gated_scan(x, x, gate="tanh")),
        (4, lambda: ops.gated_scan(x.to(torch.uint8), x.to(torch.uint8))),
        (4, lambda: ops.gated_scan(x.half(), x.half())),
        (4, lambda: ops.gated_scan(x, x, h0=torch.zeros(2, 8, device="cuda", dtype=torch.bfloat16))),
        (1, lambda: ops.gated_scan(x, x, h0=torch.zeros(8, device="cuda"))),
        (4, lambda: ops.gated_scan(x, x, lengths=torch.zeros(2, device="cuda", dtype=torch.int64))),
        (1, lambda: ops.gated_scan(x, x, lengths=torch.zeros(3, device="cuda", dtype=torch.int32))),
        (3, lambda: ops.gated_scan(x, x, lengths=torch.zeros(2, dtype=torch.int32))),
        (3, lambda: ops.gated_scan(x.cpu(), x.cpu())),
        (1, lambda: ops.gated_scan(x, x, states=torch.zeros(2, 2, 8, device="cuda"))),
        (1, lambda: ops.gated_scan(x, x, out=x[:1].expand(2, 5, 8))),
        (1, lambda: ops.gated_scan(x, x, out=torch.zeros(2, 1, 8, device="cuda").expand(2, 5, 8))),
        (1, lambda: ops.gated_scan_bwd(x, x, x, torch.zeros(2, 5, 8, device="cuda"))),
        (1, lambda: ops.gated_scan_bwd(x[:, :4], x, x, st)),
        (1, lambda: ops.gated_scan_bwd(x, x, x, st, out=(x, torch.zeros(2, 1, 8, device="cuda").expand(2, 5, 8)))),
        (1, lambda: ops.gated_scan_step(x[:, 0], x[:, 0], torch.zeros(3, 8, device="cuda"))),
        (4, lambda: ops.gated_scan_step(x[:, 0], x[:, 0], torch.zeros(2, 8, device="cuda").bfloat16())),
        (1, lambda: ops.gated_scan_step(x[0, :, 0], x[0, :, 0], torch.zeros(5, device="cuda"))),
    ]:
        with pytest.raises(L.HxError) as e:
            call()
        assert e.value.status == code
