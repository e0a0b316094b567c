"""The gated recurrence and its gradients over sequences that are cut into segments, where numbers leave the format or come near its
ends.  A call without a workspace walks the steps one by one and is what the cut call has to agree with: infinities and NaN exactly,
other numbers within the bound of either one's rounding.

Tolerances.  u = 2^-24; M_t = |a_t| M_{t-1} + |v_t| and W_t = |a_t| (W_{t-1} + M_{t-1}) as in test_gated_scan_gpu.py, where each way
of associating the sums is within 16 u W_t + 64 u M_t of the exact value, so two ways are within twice that of one another.  Where a
segment hands its state on, numbers below 2^-126 may be taken as zero: 2^-126 a segment, of which an input meets at most 128, so
2^-119 in all.  bf16 results add their own rounding, 2^-8 of the value on either side."""
import pytest
import torch

from helixml_b200 import _lib as L_
from helixml_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
INF, NAN = float("inf"), float("nan")
TILE = 64        # channels that one warp owns: every special channel gets a tile of its own, with ordinary neighbours


def walked(monkeypatch, call):
    with monkeypatch.context() as m:
        m.setattr(ops, "_gated_scan_workspace", lambda *a: None)
        return call()


def bound(a, v, start, reverse=False):
    """2 (16 u W + 64 u M) + 2^-119 for every row, and behind the last one, in 64 bits."""
    a, v = a.double().abs().nan_to_num(0, 0, 0), v.double().abs().nan_to_num(0, 0, 0)
    m, w = start.double().abs().nan_to_num(0, 0, 0), torch.zeros_like(start, dtype=torch.float64)
    rows = []
    for t in (range(a.shape[1] - 1, -1, -1) if reverse else range(a.shape[1])):
        if reverse:      # delta_t = dh_t + e_{t+1}, e_t = a_t delta_t
            m = m + v[:, t]
            rows.append(32 * U * w + 128 * U * m)
            w, m = a[:, t] * (w + m), a[:, t] * m
        else:
            w = a[:, t] * (w + m)
            m = a[:, t] * m + v[:, t]
            rows.append(32 * U * w + 128 * U * m)
    rows = torch.stack(rows[::-1] if reverse else rows, 1)
    return rows + 2.0 ** -119, 32 * U * w + 128 * U * m + 2.0 ** -119


def agree(got, want, tol, what):
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(torch.isinf(got), torch.isinf(want)), what
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), what
    ok = torch.isfinite(want)
    eps = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps
    err = (got.double() - want.double()).abs() - tol * (1 + eps) - eps * want.double().abs()
    assert not (err[ok] > 0).any(), (what, err[ok].max().item())


def decay_cases(L):
    """name -> function that edits one channel's (a, v, h0) in place; 1-d tensors over time and a number."""
    def two_large(a, v):
        v[650] = v[651] = 3e38                       # overflows in the middle of a segment

    def late_large(a, v):
        v[L - 300], v[L - 299], a[L - 299] = 3e38, 3e38, 1.0

    def large_then_halves(a, v):
        a[:], v[:] = 0.5, 0.0
        v[100] = 1e30                                # 160 halvings later 6.8e-19

    def halves_of_start(a, v):
        a[:], v[:] = 0.5, 0.0
        return 1e30

    def grows_over_zero(a, v):
        a[:] = 2.0
        v[:L - 100] = 0.0                            # the products overflow, the state is zero

    def there_and_back(a, v):
        a[:], v[:] = 1.0, 0.0
        a[3:43], a[43:83] = 2.0, 0.5                 # 1e30 2^40 is infinite, the product of the decays is one
        return 1e30

    def shrinks_after_growth(a, v):
        a[:], v[:] = 1.0, 0.0
        a[10], a[20], a[21], a[500] = 1e20, 1e-25, 1e-25, 1e20   # 1e10 -> 1e30 -> 1e-20 -> 1; the products alone underflow
        return 1e10

    def grows_after_shrinking(a, v):
        a[:], v[:] = 1.0, 0.0
        a[10], a[20], a[21], a[30] = 1e-20, 1e-20, 1e20, 1e20    # 1 -> 1e-40 -> 1
        return 1e3

    def forgets(a, v):
        v[5], a[40] = 1e37, 0.0

    def infinite(a, v):
        a[:] = 0.5
        v[7] = INF

    def infinite_forgotten(a, v):
        v[7], a[900] = -INF, 0.0

    def not_a_number(a, v):
        v[300] = NAN

    def gate_not_a_number(a, v):
        a[1000] = NAN

    def infinite_gate(a, v):
        a[100] = INF
        v[:101] = 0.0

    def large_and_steady(a, v):
        v *= 1e36

    def over_the_largest(a, v):
        v *= 8e37                                    # sums that overflow now and then

    def alternates(a, v):
        a[::2], a[1::2] = -1.0, 1.0

    def small(a, v):
        v *= 1e-36

    def wild(a, v):
        a.copy_(torch.randn(L, generator=torch.Generator().manual_seed(9)))

    def sparse(a, v):
        keep = v[::700].clone()
        a[:], v[:] = 0.4, 0.0
        v[::700] = keep * 1e20

    def regrows(a, v):
        a[:], v[:], v[10] = 1.0, 0.0, 1e30
        a[24], a[25], a[26], a[27] = 1e-30, 1e-30, 1e30, 1e30    # 1e30 -> 1 -> 1e-30 -> 1 -> 1e30
        a[30:110] = 0.25                                         # 6.8e-19 from there on

    return {f.__name__: f for f in (two_large, late_large, large_then_halves, halves_of_start, grows_over_zero, there_and_back,
                                    shrinks_after_growth, grows_after_shrinking, forgets, infinite, infinite_forgotten, not_a_number,
                                    gate_not_a_number, infinite_gate, large_and_steady, over_the_largest, alternates, small, wild, sparse,
                                    regrows)}


def decay_inputs(B, L, dtype, reverse):
    """a, v and the start; the case of tile k is in its third channel.  reverse: as the recurrence from the end meets them."""
    cases = decay_cases(L)
    D = TILE * (len(cases) + 1)
    gen = torch.Generator().manual_seed(L)
    a, v = 0.2 + 0.7 * torch.rand(B, L, D, generator=gen), torch.randn(B, L, D, generator=gen)
    start = torch.randn(B, D, generator=gen)
    for k, f in enumerate(cases.values()):
        at, vt = a[0, :, TILE * k + 2].clone(), v[0, :, TILE * k + 2].clone()
        s = f(at, vt)
        start[0, TILE * k + 2] = 0.0 if s is None else s
        a[0, :, TILE * k + 2], v[0, :, TILE * k + 2] = at, vt
    if reverse:
        a, v = a.flip(1), v.flip(1)
    return a.to(DT[dtype]).cuda(), v.to(DT[dtype]).cuda(), start.cuda()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,lengths", [(1, 4096, None), (2, 4096, [4000, 1733]), (4, 4001, None)])
def test_decays_forward(B, L, lengths, dtype, monkeypatch):
    a, v, h0 = decay_inputs(B, L, dtype, False)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def call():
        st = ops.gated_scan_states(B, L, a.shape[2])
        st.zero_()   # rows of blocks behind a length are not written
        return *ops.gated_scan(v, a, h0=h0, gate="decay", lengths=n, return_state=True, states=st), st

    (h, last, st), (want, want_last, want_st) = call(), walked(monkeypatch, call)
    if lengths is not None:
        inside = (torch.arange(L, device="cuda")[None] < n[:, None])[:, :, None]
        a, v = torch.where(inside, a, 1.0), torch.where(inside, v, 0.0)
    tol, last_tol = bound(a, v, h0)
    agree(h, want, tol, "h")
    agree(last, want_last, last_tol, "h_last")
    before = torch.cat([torch.full_like(tol[:, :1], 2.0 ** -119), tol[:, :-1]], 1)[:, ::16]
    agree(st, want_st, before, "states")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,lengths", [(1, 4096, None), (2, 4096, [4096, 1733]), (4, 4001, None)])
def test_decays_backward(B, L, lengths, dtype, monkeypatch):
    a, dh, dh_last = decay_inputs(B, L, dtype, True)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    x = torch.randn(B, L, a.shape[2], generator=torch.Generator().manual_seed(1)).to(DT[dtype]).cuda()
    st = ops.gated_scan_states(B, L, a.shape[2])
    walked(monkeypatch, lambda: ops.gated_scan(x, a, gate="decay", lengths=n, states=st))
    call = lambda: ops.gated_scan_bwd(dh, x, a, st, gate="decay", lengths=n, dh_last=dh_last)
    (dx, dg, dh0), (want, want_dg, want0) = call(), walked(monkeypatch, call)
    if lengths is not None:
        inside = (torch.arange(L, device="cuda")[None] < n[:, None])[:, :, None]
        a, dh = torch.where(inside, a, 1.0), torch.where(inside, dh, 0.0)
    tol, tol0 = bound(a, dh, dh_last, reverse=True)
    agree(dx, want, tol, "dx")
    agree(dh0, want0, tol0, "dh0")
    for same in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(same(dg), same(want_dg))


def sigmoid_inputs(B, L, dtype):
    D = TILE * 8
    gen = torch.Generator().manual_seed(L)
    g, x, h0 = torch.randn(B, L, D, generator=gen), torch.randn(B, L, D, generator=gen), torch.randn(B, D, generator=gen)
    c = lambda k: TILE * k + 2
    g[0, :, c(0)], x[0, :, c(0)], h0[0, c(0)] = 0.0, 0.0, 1e30         # halves of a large start
    g[0, :, c(1)], x[0, :, c(1)], x[0, 100, c(1)] = 0.0, 0.0, 1e30     # of a large input
    x[0, 200, c(2)] = INF
    x[0, 333, c(3)] = NAN
    g[0, 333, c(4)] = NAN
    g[0, :, c(5)] = -30.0                                              # forgets everything within a step
    x[0, 500, c(5)], h0[0, c(5)] = 1e37, 1e37
    x[0, :, c(6)] *= 8e36
    return g.to(DT[dtype]).cuda(), x.to(DT[dtype]).cuda(), h0.cuda()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,L", [(1, 5000), (4, 4096)])
def test_sigmoid(B, L, dtype, monkeypatch):
    g, x, h0 = sigmoid_inputs(B, L, dtype)
    call = lambda: ops.gated_scan(x, g, h0=h0, return_state=True)
    (h, last), (want, want_last) = call(), walked(monkeypatch, call)
    tol, last_tol = bound(torch.sigmoid(g.double()), torch.sigmoid(-g.double()) * x.double(), h0)
    agree(h, want, tol, "h")
    agree(last, want_last, last_tol, "h_last")
    # the same numbers as gradients
    st = ops.gated_scan_states(B, L, g.shape[2])
    ones = torch.ones_like(x)
    walked(monkeypatch, lambda: ops.gated_scan(ones, g, states=st))
    call = lambda: ops.gated_scan_bwd(x.flip(1).contiguous(), ones, g, st, dh_last=h0)
    (dx, dg, dh0), (want, want_dg, want0) = call(), walked(monkeypatch, call)
    tol, tol0 = bound(torch.sigmoid(g.double()), x.flip(1), h0, reverse=True)
    agree(dx, want, tol, "dx")
    agree(dh0, want0, tol0, "dh0")
    for same in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(same(dg), same(want_dg))


def test_across_spans(monkeypatch):
    """Inputs beyond the cache go span by span; the cases lie in the first and the last of them."""
    L, D = 24000, 1024
    gen = torch.Generator().manual_seed(5)
    a, v = 0.2 + 0.7 * torch.rand(1, L, D, generator=gen), torch.randn(1, L, D, generator=gen)
    h0 = torch.randn(1, D, generator=gen)
    c = lambda k: TILE * k + 2
    a[0, :, c(0)], v[0, :, c(0)], h0[0, c(0)] = 0.999, 0.0, 1e30
    v[0, 650, c(1)] = v[0, 651, c(1)] = v[0, L - 651, c(2)] = v[0, L - 650, c(2)] = 3e38
    a[0, :, c(3)], v[0, :, c(3)], v[0, L - 4000, c(3)] = 0.5, 0.0, 1e30
    a[0, :, c(4)], v[0, :L - 90, c(4)], h0[0, c(4)] = 2.0, 0.0, 0.0
    a, v, h0 = a.cuda(), v.cuda(), h0.cuda()
    call = lambda: ops.gated_scan(v, a, h0=h0, gate="decay", return_state=True)
    (h, last), (want, want_last) = call(), walked(monkeypatch, call)
    assert torch.isinf(want[0, -1, [c(1), c(2)]]).all() and want[0, L - 3900, c(3)] != 0
    tol, last_tol = bound(a, v, h0)
    agree(h, want, tol, "h")
    agree(last, want_last, last_tol, "h_last")
    st = ops.gated_scan_states(1, L, D)
    ones = torch.ones_like(v)
    walked(monkeypatch, lambda: ops.gated_scan(ones, a, gate="decay", states=st))
    call = lambda: ops.gated_scan_bwd(v, ones, a, st, gate="decay", dh_last=h0)
    (dx, _, dh0), (want, _, want0) = call(), walked(monkeypatch, call)
    tol, tol0 = bound(a, v, h0, reverse=True)
    agree(dx, want, tol, "dx")
    agree(dh0, want0, tol0, "dh0")


@pytest.mark.parametrize("gate", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_channel_does_not_depend_on_its_neighbours(dtype, gate):
    """Infinities, NaN and numbers that leave the format in some channels of a tile leave every bit of the others as it was."""
    B, L, D = 2, 3000, 130
    gen = torch.Generator().manual_seed(8)
    x, g, dh = (torch.randn(B, L, D, generator=gen) for _ in range(3))
    if gate == "decay":
        g = 0.9 + 0.1 * torch.rand(B, L, D, generator=gen)
    h0, dh_last = torch.randn(B, D, generator=gen).cuda(), torch.randn(B, D, generator=gen).cuda()

    def call(x, g, dh):
        x, g, dh = (t.to(DT[dtype]).cuda() for t in (x, g, dh))
        st = ops.gated_scan_states(B, L, D)
        h, last = ops.gated_scan(x, g, h0=h0, gate=gate, states=st, return_state=True)
        return h, last, st, *ops.gated_scan_bwd(dh, x, g, st, gate=gate, dh_last=dh_last)

    want = call(x, g, dh)
    bad = [5, 36, 127]
    x[0, 9, 5], x[0, 1500, 36], x[1, 300, 127] = INF, NAN, -INF
    dh[0, 2990, 5], dh[0, 1500, 36], dh[1, 2000, 127] = -INF, NAN, INF
    x[1, 700:702, 5] = dh[1, 2000:2002, 5] = 3e38
    others = [c for c in range(D) if c not in bad]
    for name, got, w in zip(("h", "h_last", "states", "dx", "dg", "dh0"), call(x, g, dh), want):
        assert torch.equal(got[..., others], w[..., others]), name
        assert not torch.equal(got[..., bad], w[..., bad]), name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_small_decays_of_large_states(dtype):
    """sigmoid(g) of a strongly negative gate is good relative to itself, down to the smallest normal number: e = exp(-g) is off by
    (|g| + 5) u, the sum, the reciprocal and the product with the state by 6 u at most, so a h by (|g| + 16) u of itself; below 2^-126
    a may be zero.  A gate of minus infinity leaves nothing of an infinite state but NaN."""
    g = torch.arange(-86.5, 0.0, 0.25)
    D = g.numel()
    g = g[None, None].expand(1, 200, -1).to(DT[dtype]).cuda()
    h0 = torch.full((1, D), 3e38, device="cuda")
    x = torch.zeros(1, 200, D, dtype=DT[dtype], device="cuda")
    want = torch.sigmoid(g[:, 0].double()) * h0.double()
    tol = (g[:, 0].double().abs() + 16) * U * want
    _, last = ops.gated_scan(x[:, :1], g[:, :1], h0=h0, return_state=True)
    assert ((last.double() - want).abs() <= tol).all()
    _, last = ops.gated_scan(x, g, h0=h0, lengths=torch.ones(1, dtype=torch.int32, device="cuda"), return_state=True)
    assert ((last.double() - want).abs() <= tol).all()
    state = h0.clone()
    ops.gated_scan_step(x[:, 0], g[:, 0], state)
    assert ((state.double() - want).abs() <= tol).all()
    st = ops.gated_scan_states(1, 1, D)
    ops.gated_scan(x[:, :1], g[:, :1], states=st)
    _, _, dh0 = ops.gated_scan_bwd(x[:, :1], x[:, :1], g[:, :1], st, dh_last=h0)
    assert ((dh0.double() - want).abs() <= tol).all()
    for gate in (-INF, -90.0, torch.finfo(DT[dtype]).min):
        gt = torch.full((1, 1, 4), gate, dtype=DT[dtype], device="cuda")
        one, inf = torch.ones_like(gt), torch.full((1, 4), INF, device="cuda")
        _, last = ops.gated_scan(one, gt, h0=torch.full_like(inf, 3e38), return_state=True)
        assert (last == 1).all()
        _, last = ops.gated_scan(one, gt, h0=inf, return_state=True)
        assert torch.isnan(last).all()
        ops.gated_scan_step(one[:, 0], gt[:, 0], inf)
        assert torch.isnan(inf).all()


def test_shared_memory_is_refused_and_parts_of_one_buffer_are_not():
    B, L, D = 2, 900, 40
    buf = torch.randn(B, L, 5 * D, generator=torch.Generator().manual_seed(2)).cuda()
    part = lambda i: buf[:, :, i * D:(i + 1) * D]
    want = ops.gated_scan(part(0), part(1))
    st = ops.gated_scan_states(B, L, D)
    assert torch.equal(ops.gated_scan(part(0), part(1), out=part(2), states=st), want)
    x, g, dh = (part(i).clone() for i in (0, 1, 2))
    dx, dg, _ = ops.gated_scan_bwd(dh, x, g, st)
    ops.gated_scan_bwd(part(2), part(0), part(1), st, out=(part(3), part(4)))
    assert torch.equal(part(3), dx) and torch.equal(part(4), dg)
    first = x[:, :1].expand(B, L, D)      # an input without a stride, and an output among the rows around it
    assert torch.equal(ops.gated_scan(buf[:, :1, :D].expand(B, L, D), g, out=part(4)), ops.gated_scan(first, g))
    h = torch.randn(B, D, device="cuda")
    y = ops.gated_scan_step(x[:, 0], g[:, 0], h.clone())
    xt = x[:, 0].contiguous()
    assert torch.equal(ops.gated_scan_step(xt, g[:, 0], h, out=xt), y) and torch.equal(xt, y)
    before = buf.clone()
    for call in (lambda: ops.gated_scan(part(0), part(1), out=part(0)), lambda: ops.gated_scan(part(0), part(1), out=part(1)),
                 lambda: ops.gated_scan(part(0), part(1), out=buf[:, :, 3:D + 3]), lambda: ops.gated_scan(x, g, out=x),
                 lambda: ops.gated_scan(x[:, 1:], g[:, 1:], out=x[:, :-1]), lambda: ops.gated_scan_bwd(dh, x, g, st, out=(dh, dg)),
                 lambda: ops.gated_scan_bwd(dh, x, g, st, out=(dx, dx)), lambda: ops.gated_scan_bwd(dh, x, g, st, out=(dx, g)),
                 lambda: ops.gated_scan_step(buf[:, 0, :D], g[:, 0], h, out=buf[:, 0, 1:D + 1])):
        with pytest.raises(L_.HxError) as e:
            call()
        assert e.value.status == 10 and "share memory" in str(e.value)
    assert torch.equal(buf, before)


def test_sizes_beyond_32_bits_are_refused():
    """Views that repeat one element 2^32 + 5 times: the sizes reach the library in 32 bits."""
    many = (1 << 32) + 5
    one = torch.zeros(1, 1, 1, device="cuda")
    x = one.expand(1, many, 1)
    for call in (lambda: ops.gated_scan(x, x), lambda: ops.gated_scan_bwd(x, x, x, ops.gated_scan_states(1, 5, 1)),
                 lambda: ops.gated_scan(one.expand(many, 1, 1), one.expand(many, 1, 1)),
                 lambda: ops.gated_scan_step(one[0].expand(many, 1), one[0].expand(many, 1), torch.zeros(5, 1, device="cuda"))):
        with pytest.raises(L_.HxError) as e:
            call()
        assert e.value.status == 2


def random_extremes(seed, B, L, D):
    """Stretches of constant decay, growth by up to 1e30 that is taken back within 50 steps, and inputs and starts over the whole range."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=gen, device="cuda")
    choice = torch.tensor([1.0, 0.5, 0.25, 0.9, 0.99, 0.75, 1.0, 0.05], device="cuda")
    stretch = (r(B, L, D) < 0.01).cumsum(1)
    a = choice[(r(1, 1, D) * 8 + stretch * (1 + (r(1, 1, D) * 7).long())).long() % 8]
    for _ in range(6 * (seed % 2)):
        t, k = (r(B, 1, D) * (L - 60)).long(), 1 + (r(B, 1, D) * 50).long()
        u = (60 * r(B, 1, D) - 30) * (r(B, 1, D) < 0.5)
        a.scatter_(1, t, 10 ** u)
        a.scatter_(1, t + k, 10 ** -u)
    size = 38.4 * r(1, 1, D)
    v = torch.where(r(B, L, D) < 10 ** (-1 - 2.3 * r(1, 1, D)), 10 ** (size * (r(B, L, D) * 1.5 - 0.5)) * torch.sign(r(B, L, D) - 0.5), 0.0)
    v = torch.where(r(1, 1, D) < 0.3, v + torch.randn(B, L, D, generator=gen, device="cuda"), v)
    start = 10 ** (38 * (2 * r(B, D) - 1)) * torch.sign(r(B, D) - 0.5)
    return a, v.clamp(-3e38, 3e38), start


def hold(got, want, a, v, start, reverse=False):
    """2 (16 u W + 64 u M) as above, and 2^-125 a step for what may be taken as zero, under the decays behind it.  Where that reaches the
    largest number, either way of summing may overflow; what comes after is not compared."""
    a, v = a.double().abs(), v.double().abs()
    m, w, z = start.double().abs(), torch.zeros_like(start, dtype=torch.float64), torch.full_like(start, 2.0 ** -125, dtype=torch.float64)
    border = torch.zeros_like(start, dtype=torch.bool)
    wrong = compared = torch.zeros((), dtype=torch.int64, device="cuda")
    for t in (range(a.shape[1] - 1, -1, -1) if reverse else range(a.shape[1])):
        if reverse:
            m = m + v[:, t]
        else:
            w, m, z = a[:, t] * (w + m), a[:, t] * m + v[:, t], a[:, t] * z + 2.0 ** -125
        tol = 32 * U * w + 128 * U * m + z
        g, h = got[:, t].double(), want[:, t].double()
        border = border | (tol + h.abs().nan_to_num(0, 0, 0) >= 0.999 * torch.finfo(torch.float32).max)
        same = torch.where(torch.isfinite(h), (g - h).abs() <= tol, (g == h) | (torch.isnan(g) & torch.isnan(h)))
        wrong, compared = wrong + (~same & ~border).sum(), compared + (~border).sum()
        if reverse:
            w, m, z = a[:, t] * (w + m), a[:, t] * m, a[:, t] * z + 2.0 ** -125
    assert wrong.item() == 0 and compared.item() > 0.4 * got.numel(), (wrong.item(), compared.item())


@pytest.mark.parametrize("seed,B,L,D", [(0, 2, 3000, 1024), (1, 1, 1500, 2048), (2, 4, 2001, 1408), (3, 1, 6000, 512)])
def test_random_extremes(seed, B, L, D, monkeypatch):
    a, v, start = random_extremes(seed, B, L, D)
    call = lambda: ops.gated_scan(v, a, h0=start, gate="decay")
    hold(call(), walked(monkeypatch, call), a, v, start)
    zeros = torch.zeros_like(v)
    st = ops.gated_scan_states(B, L, D).zero_()
    call = lambda: ops.gated_scan_bwd(v, zeros, a, st, gate="decay", dh_last=start)[0]
    hold(call(), walked(monkeypatch, call), a, v, start, reverse=True)
