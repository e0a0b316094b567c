"""Performance cases of the gated recurrence and of the products with 4-bit weights.

  scan      the gated linear recurrence over whole sequences: h_t = a_t h_{t-1} + x_t with the decay a_t given ("decay"), or
            h_t = a_t h_{t-1} + (1 - a_t) x_t with a_t = sigmoid(g_t) ("sigmoid")
  scan_bwd  its gradients with respect to x, g and the state it started from
  step      one token of it per sequence, on a kept state
  gemm_w4   C = A W^T (+ bias) for a few rows, W in 4 bits with one scale (and zero point) per group of a row
  quantize  weights brought into that form and read back

A case is a dict of plain values; listed() holds the fixed ones and draw() gives more of the same ranges.  Where `own` is
false, run() computes the operators in elementary torch operations, in 32 bits (the quotients that decide a 4-bit code: in 64)."""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one layer's forward in training, bench.py's batch at its inner width; the states its backward pass needs are kept
        {"name": "scan bf16 32x2048x1536", "kind": "scan", "batch": 32, "seq_len": 2048, "width": 1536, "dtype": "bf16",
         "gate": "sigmoid", "ragged": False, "train": True},
        # one long document, carried on from the state of an earlier part: few chains, many steps
        {"name": "scan f32 1x32768x1536", "kind": "scan", "batch": 1, "seq_len": 32768, "width": 1536, "dtype": "f32",
         "gate": "decay", "ragged": False, "train": False},
        # prompts of different lengths in one padded batch, a width that is not a multiple of a tile
        {"name": "scan bf16 7x731x1000", "kind": "scan", "batch": 7, "seq_len": 731, "width": 1000, "dtype": "bf16",
         "gate": "sigmoid", "ragged": True, "train": False},
        # the gradients of the first case
        {"name": "scan_bwd bf16 32x2048x1536", "kind": "scan_bwd", "batch": 32, "seq_len": 2048, "width": 1536, "dtype": "bf16",
         "gate": "sigmoid", "ragged": False},
        # gradients of a padded batch in f32, odd length and width
        {"name": "scan_bwd f32 5x1003x1001", "kind": "scan_bwd", "batch": 5, "seq_len": 1003, "width": 1001, "dtype": "f32",
         "gate": "decay", "ragged": True},
        # one user's token: latency
        {"name": "step bf16 1x1536", "kind": "step", "batch": 1, "width": 1536, "dtype": "bf16", "gate": "sigmoid"},
        # a large serving batch of a wide layer
        {"name": "step f32 256x4096", "kind": "step", "batch": 256, "width": 4096, "dtype": "f32", "gate": "decay"},
        # the block's output projection for one token: latency
        {"name": "gemm_w4 bf16 1x768x1536", "kind": "gemm_w4", "rows": 1, "outs": 768, "ins": 1536, "group": 64, "dtype": "bf16",
         "zeros": False, "bias": False},
        # one token through a large projection: a stream over the weights
        {"name": "gemm_w4 bf16 1x16384x4096", "kind": "gemm_w4", "rows": 1, "outs": 16384, "ins": 4096, "group": 128,
         "dtype": "bf16", "zeros": False, "bias": False},
        # a batch of completions, zero points, small groups, an odd number of outputs
        {"name": "gemm_w4 f32 24x5001x8192", "kind": "gemm_w4", "rows": 24, "outs": 5001, "ins": 8192, "group": 32, "dtype": "f32",
         "zeros": True, "bias": True},
        # a checkpoint's matrix when it is loaded
        {"name": "quantize f32 8192x8192", "kind": "quantize", "outs": 8192, "ins": 8192, "group": 128, "dtype": "f32", "zeros": False},
        # a small one, with zero points
        {"name": "quantize bf16 1000x1536", "kind": "quantize", "outs": 1000, "ins": 1536, "group": 32, "dtype": "bf16", "zeros": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan_bwd", "scan_bwd", "step", "gemm_w4", "gemm_w4", "quantize"])
    dtype = rng.choice(["bf16", "f32"])
    gate = rng.choice(["sigmoid", "decay"])
    if kind in ("scan", "scan_bwd"):
        seq_len = _log_int(rng, 1, 16384 if kind == "scan" else 8192)
        width = _log_int(rng, 16, 4096)
        batch = _log_int(rng, 1, max(1, min(32, 40_000_000 // (seq_len * width))))
        case = {"kind": kind, "batch": batch, "seq_len": seq_len, "width": width, "dtype": dtype, "gate": gate,
                "ragged": rng.random() < 0.4}
        if kind == "scan":
            case["train"] = rng.random() < 0.5
        return case
    if kind == "step":
        return {"kind": kind, "batch": _log_int(rng, 1, 256), "width": _log_int(rng, 64, 4096), "dtype": dtype, "gate": gate}
    if kind == "gemm_w4":
        group = rng.choice([32, 64, 128])
        return {"kind": kind, "rows": _log_int(rng, 1, 64), "outs": _log_int(rng, 64, 12288),
                "ins": group * _log_int(rng, 2, 8192 // group), "group": group, "dtype": dtype, "zeros": rng.random() < 0.4,
                "bias": rng.random() < 0.3}
    group = rng.choice([32, 64, 128])
    return {"kind": kind, "outs": _log_int(rng, 64, 8192), "ins": group * _log_int(rng, 2, 8192 // group), "group": group,
            "dtype": dtype, "zeros": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind in ("scan", "scan_bwd"):
        B, L, D = case["batch"], case["seq_len"], case["width"]
        # x and the gate are the halves of one projection's output; gates that remember tens to hundreds of steps
        xg = torch.empty(B, L, 2 * D, device="cuda", dtype=dt)
        xg[:, :, :D] = rnd(B, L, D).to(dt)
        gate = 3.0 + 1.5 * rnd(B, L, D)
        xg[:, :, D:] = (torch.sigmoid(gate) if case["gate"] == "decay" else gate).to(dt)
        s.update(x=xg[:, :, :D], g=xg[:, :, D:], h0=rnd(B, D), lengths=None)
        if case["ragged"]:
            n = torch.randint(1, L + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
            n[0] = L
            s["lengths"] = n
        if kind == "scan_bwd":
            s.update(dh=rnd(B, L, D).to(dt), dh_last=rnd(B, D))
        if own:
            from helixml_b200 import ops
            if kind == "scan_bwd" or case["train"]:
                s["states"] = ops.gated_scan_states(B, L, D)
            if kind == "scan_bwd":  # what the forward pass of the same step has left
                ops.gated_scan(s["x"], s["g"], h0=s["h0"], gate=case["gate"], lengths=s["lengths"], states=s["states"])
    elif kind == "step":
        B, D = case["batch"], case["width"]
        xg = torch.empty(B, 2 * D, device="cuda", dtype=dt)
        xg[:, :D] = rnd(B, D).to(dt)
        gate = 3.0 + 1.5 * rnd(B, D)
        xg[:, D:] = (torch.sigmoid(gate) if case["gate"] == "decay" else gate).to(dt)
        s.update(x=xg[:, :D], g=xg[:, D:], h=rnd(B, D), h_next=torch.empty(B, D, device="cuda"))
    elif kind == "gemm_w4":
        M, N, K, G = case["rows"], case["outs"], case["ins"], case["group"]
        s.update(a=rnd(M, K).to(dt), bias=rnd(N) if case["bias"] else None,
                 codes=(8 + 2.5 * rnd(N, K)).round().clamp(0, 15).to(torch.uint8),
                 scale=(0.2 + 0.1 * torch.rand(N, K // G, device="cuda", generator=gen)) * K ** -0.5,
                 zero=torch.randint(6, 11, (N, K // G), device="cuda", generator=gen, dtype=torch.uint8) if case["zeros"] else None)
        if case["dtype"] == "bf16":
            s["scale"] = s["scale"].to(dt)
        if own:  # a serving program lays its weights out when it loads them
            from helixml_b200 import ops
            s["w4"] = ops.w4_pack(s["codes"], s["scale"], zero=s["zero"])
    else:
        N, K = case["outs"], case["ins"]
        s["w"] = (rnd(N, K) * K ** -0.5).to(dt)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from helixml_b200 import ops
    case, kind = s["case"], s["case"]["kind"]
    if kind == "scan":
        return ops.gated_scan(s["x"], s["g"], h0=s["h0"], gate=case["gate"], lengths=s["lengths"], return_state=True,
                              states=s.get("states"))
    if kind == "scan_bwd":
        return ops.gated_scan_bwd(s["dh"], s["x"], s["g"], s["states"], gate=case["gate"], lengths=s["lengths"],
                                  dh_last=s["dh_last"])
    if kind == "step":
        y = ops.gated_scan_step(s["x"], s["g"], s["h"], gate=case["gate"], h_out=s["h_next"])
        return y, s["h_next"]
    if kind == "gemm_w4":
        return ops.gemm_w4(s["a"], s["w4"], bias=s["bias"])
    w4 = ops.w4_quantize(s["w"], case["group"], zero_points=case["zeros"], scale_dtype=s["w"].dtype)
    values = ops.w4_dequantize(w4, s["w"].dtype)
    return (values, w4.scale, w4.zero) if case["zeros"] else (values, w4.scale)


def _decay_and_input(s):
    """a_t and b_t of h_t = a_t h_{t-1} + b_t in 32 bits, what lies behind a sequence's end as a = 1, b = 0; and which rows count."""
    x, g = s["x"].float(), s["g"].float()
    if s["case"]["gate"] == "decay":
        a, b = g, x
    else:
        a = 1.0 / (1.0 + torch.exp(-g))
        b = x / (1.0 + torch.exp(g))
    valid = None
    if s.get("lengths") is not None:
        valid = (torch.arange(x.shape[1], device=x.device)[None, :] < s["lengths"][:, None])[:, :, None]
        a, b = torch.where(valid, a, 1.0), torch.where(valid, b, 0.0)
    return x, a, b, valid


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "scan":
        x, a, b, valid = _decay_and_input(s)
        h, out = s["h0"], torch.empty_like(b)
        for t in range(x.shape[1]):
            h = torch.addcmul(b[:, t], a[:, t], h, out=out[:, t])
        last = h.clone()
        return (out if valid is None else torch.where(valid, out, 0.0)).to(s["x"].dtype), last
    if kind == "scan_bwd":
        x, a, b, valid = _decay_and_input(s)
        L = x.shape[1]
        before = torch.empty_like(b)  # h_{t-1}
        before[:, 0] = s["h0"]
        for t in range(L - 1):
            torch.addcmul(b[:, t], a[:, t], before[:, t], out=before[:, t + 1])
        delta = s["dh"].float()
        if valid is not None:
            delta = torch.where(valid, delta, 0.0)
        delta = delta.clone()
        delta[:, L - 1] += s["dh_last"]
        for t in range(L - 2, -1, -1):
            torch.addcmul(delta[:, t], a[:, t + 1], delta[:, t + 1], out=delta[:, t])
        dh0 = a[:, 0] * delta[:, 0]
        if case["gate"] == "decay":
            dx, dg = delta, delta * before
        else:
            rest = 1.0 / (1.0 + torch.exp(s["g"].float()))
            dx, dg = delta * rest, delta * (before - x) * a * rest
        if valid is not None:
            dx, dg = torch.where(valid, dx, 0.0), torch.where(valid, dg, 0.0)
        return dx.to(s["x"].dtype), dg.to(s["x"].dtype), dh0
    if kind == "step":
        x, g = s["x"].float(), s["g"].float()
        if case["gate"] == "decay":
            h = g * s["h"] + x
        else:
            h = s["h"] / (1.0 + torch.exp(-g)) + x / (1.0 + torch.exp(g))
        return h.to(s["x"].dtype), h
    if kind == "gemm_w4":
        G = case["group"]
        q = s["codes"].float().view(case["outs"], -1, G)
        z = 8.0 if s["zero"] is None else s["zero"].float()[:, :, None]
        w = ((q - z) * s["scale"].float()[:, :, None]).view(case["outs"], -1)
        c = s["a"].float() @ w.t()
        return (c if s["bias"] is None else c + s["bias"]).to(s["a"].dtype)
    # the quotients in 64 bits: a code changes at w / scale = k + 1/2, and weights do lie there
    dt = s["w"].dtype
    w = s["w"].double().view(case["outs"], -1, case["group"])
    if case["zeros"]:
        lo, hi = w.amin(2).clamp(max=0.0), w.amax(2).clamp(min=0.0)
        scale = ((hi - lo) / 15.0).float().to(dt)
        div = torch.where(scale == 0, 1.0, scale.double())
        zero = torch.where(scale == 0, 8.0, (-lo / div).round().clamp(0, 15))
        code = ((w / div[:, :, None]).round() + zero[:, :, None]).clamp(0, 15)
        code = torch.where(scale[:, :, None] == 0, 8.0, code)
        values = ((code - zero[:, :, None]).float() * scale.float()[:, :, None]).to(dt).view(case["outs"], -1)
        return values, scale, zero.to(torch.uint8)
    scale = (w.abs().amax(2) / 7.0).float().to(dt)
    div = torch.where(scale == 0, 1.0, scale.double())
    code = (w / div[:, :, None]).round().clamp(-7, 7)
    values = (code.float() * scale.float()[:, :, None]).to(dt).view(case["outs"], -1)
    return values, scale


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    kind = case["kind"]
    if kind in ("scan", "scan_bwd"):
        n, chains = case["batch"] * case["seq_len"] * case["width"], case["batch"] * case["width"]
        if kind == "scan":
            return {"bytes": 3 * n * e + 8 * chains, "flops": n * (2 if case["gate"] == "decay" else 7)}
        return {"bytes": 5 * n * e + 12 * chains, "flops": n * (5 if case["gate"] == "decay" else 14)}
    if kind == "step":
        n = case["batch"] * case["width"]
        return {"bytes": n * (3 * e + 8), "flops": n * (2 if case["gate"] == "decay" else 7)}
    if kind == "gemm_w4":
        M, N, K, groups = case["rows"], case["outs"], case["ins"], case["outs"] * (case["ins"] // case["group"])
        return {"bytes": N * K // 2 + groups * (e + (1 if case["zeros"] else 0)) + (M * K + M * N) * e + (4 * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    N, K, groups = case["outs"], case["ins"], case["outs"] * (case["ins"] // case["group"])
    return {"bytes": 2 * N * K * e + N * K // 2 + groups * (e + (1 if case["zeros"] else 0)), "flops": 4 * N * K}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _recur(a, b, start):
    """h_t = a_t h_{t-1} + b_t for all t, by doubling: after step k every row holds the product and the sum over its last 2^k steps."""
    a, b = a.clone(), b.clone()
    b[:, 0] += a[:, 0] * start
    k = 1
    while k < a.shape[1]:
        b[:, k:] = b[:, k:] + a[:, k:] * b[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return b


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("scan", "scan_bwd"):
        x, g = s["x"].double(), s["g"].double()
        a = g if case["gate"] == "decay" else torch.sigmoid(g)
        scale = 1.0 if case["gate"] == "decay" else torch.sigmoid(-g)
        inside = torch.ones(x.shape[:2], dtype=torch.bool, device=x.device)
        if s["lengths"] is not None:
            inside = torch.arange(x.shape[1], device=x.device)[None] < s["lengths"][:, None].long()
        inside = inside[:, :, None].expand_as(x)
        decay = a.masked_fill(~inside, 1.0)
        h = _recur(decay, (scale * x).masked_fill(~inside, 0.0), s["h0"].double())
        if kind == "scan":
            return h.masked_fill(~inside, 0.0), h[:, -1].clone()
        before = torch.cat([s["h0"].double()[:, None], h[:, :-1]], dim=1)
        del h
        dh = s["dh"].double().masked_fill(~inside, 0.0)
        # e_t = a_t (dh_t + e_{t+1}) from the end; delta_t = dh_t + e_{t+1}
        e = _recur(decay.flip(1), (decay * dh).flip(1), s["dh_last"].double()).flip(1)
        delta = dh + torch.cat([e[:, 1:], s["dh_last"].double()[:, None]], dim=1)
        if case["gate"] == "decay":
            dx, dg = delta, delta * before
        else:
            dx, dg = delta * scale, delta * (before - x) * a * scale
        return dx.masked_fill(~inside, 0.0), dg.masked_fill(~inside, 0.0), e[:, 0].clone()
    if kind == "step":
        g, x, h = s["g"].double(), s["x"].double(), s["h"].double()
        if case["gate"] == "decay":
            h = g * h + x
        else:
            h = torch.sigmoid(g) * h + torch.sigmoid(-g) * x
        return h, h
    if kind == "gemm_w4":
        group = torch.arange(case["ins"], device="cuda") // case["group"]
        c = torch.zeros(case["rows"], case["outs"], dtype=torch.float64, device="cuda")
        for n0 in range(0, case["outs"], 2048):  # a part of the outputs at a time
            part = slice(n0, n0 + 2048)
            w = s["codes"][part].double() - (8.0 if s["zero"] is None else s["zero"][part].double()[:, group])
            c[:, part] = s["a"].double() @ (w * s["scale"][part].double()[:, group]).t()
        return c if s["bias"] is None else c + s["bias"].double()
    dt = s["w"].dtype
    group = torch.arange(case["ins"], device="cuda") // case["group"]
    n_groups = case["ins"] // case["group"]
    w = s["w"].double()
    by_group = lambda how: torch.stack([how(w[:, j * case["group"]:(j + 1) * case["group"]]) for j in range(n_groups)], dim=1)
    if case["zeros"]:
        top, bottom = by_group(lambda v: v.amax(1)).clamp(min=0), by_group(lambda v: v.amin(1)).clamp(max=0)
        scale = ((top - bottom) / 15).float().to(dt).double()
        zero = torch.round(-bottom / scale).clamp(0, 15)
    else:
        scale = (by_group(lambda v: v.abs().amax(1)) / 7).float().to(dt).double()
        zero = torch.full_like(scale, 8.0)
    wide, z = scale[:, group], zero[:, group]
    code = torch.clamp(torch.round(w / wide) + z, 0 if case["zeros"] else 1, 15)
    values = (code - z) * wide
    return (values, scale, zero.to(torch.uint8)) if case["zeros"] else (values, scale)
