"""The operators of a routed-expert block with 4-bit weights, as cases that can be timed and compared.

The operators: `route` (the grouped router: scores, a bias for balance, groups, top k, weights), `quant` (rows to
microscaled 4-bit floating point and back to the values they stand for), `linear` (a dense product with such weights)
and `routed` (the experts' product with such weights, each row with the experts that its route chose).

A microscaled 4-bit value (MXFP4): 32 consecutive elements of a row share a scale 2^(s - 127), s a byte; an element is a
4-bit code (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6), two to a byte, the even element low.

`own` false: the plain form, elementary torch operations in 32 bits. `own` true: the calls of furykernel_b200."""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SUFFIX = {"f32": "", "bf16": "_xbf16", "f16": "_xf16"}
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One new token's route over a small set of experts, softmax scores: the smallest call, latency alone.
        {"name": "route_decode", "op": "route", "m": 1, "n": 64, "k": 4, "groups": 1, "top_groups": 1, "group_by": 1,
         "score": "softmax", "bias": False, "renorm": True, "factor": 1.0, "dtype": "f32"},
        # A long prompt's rows over 256 experts in 8 groups, sigmoid scores with a balance bias.
        {"name": "route_prompt", "op": "route", "m": 8192, "n": 256, "k": 8, "groups": 8, "top_groups": 4,
         "group_by": 2, "score": "sigmoid", "bias": True, "renorm": True, "factor": 2.5, "dtype": "f32"},
        # A few odd rows (an adapter's, or one expert's slice) to 4 bits and back.
        {"name": "quant_rows", "op": "quant", "rows": 33, "k": 1056, "dtype": "f32"},
        # A layer's gate and up weights, loaded in bf16, to 4 bits and back.
        {"name": "quant_layer", "op": "quant", "rows": 22016, "k": 4096, "dtype": "bf16"},
        # A decode step's projection for one sequence: the weights' bytes are the cost.
        {"name": "linear_decode", "op": "linear", "m": 1, "n": 11008, "k": 4096, "dtype": "f32"},
        # The same at a batch of 16 sequences.
        {"name": "linear_batch", "op": "linear", "m": 16, "n": 11008, "k": 4096, "dtype": "f32"},
        # A 511-row prompt through the gate and up projections.
        {"name": "linear_prompt", "op": "linear", "m": 511, "n": 22016, "k": 4096, "dtype": "f32"},
        # A vocabulary head over a batch of bf16 rows.
        {"name": "linear_head", "op": "linear", "m": 32, "n": 32000, "k": 4096, "dtype": "bf16"},
        # One new token through its 4 experts of 64.
        {"name": "routed_decode", "op": "routed", "m": 1, "k": 4, "entries": 64, "n": 1408, "kk": 2048,
         "per_rank": False, "dtype": "f32"},
        # A batch's down projection: each (row, rank) has an input of its own.
        {"name": "routed_batch", "op": "routed", "m": 16, "k": 4, "entries": 64, "n": 2048, "kk": 1408,
         "per_rank": True, "dtype": "f32"},
        # A 511-row prompt through two of 8 wide experts, the down projection.
        {"name": "routed_prompt", "op": "routed", "m": 511, "k": 2, "entries": 8, "n": 4096, "kk": 11008,
         "per_rank": True, "dtype": "f32"},
        # A long prompt in bf16 through 8 of 64 experts.
        {"name": "routed_long", "op": "routed", "m": 2048, "k": 8, "entries": 64, "n": 2816, "kk": 2048,
         "per_rank": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "quant", "linear", "routed"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        per = rng.randint(2, 64) if groups > 1 else rng.randint(8, 512)
        n = groups * per
        top_groups = rng.randint(1, groups)
        return {"op": op, "m": _log(rng, 1, 8192), "n": n, "k": rng.randint(1, min(8, top_groups * per)),
                "groups": groups, "top_groups": top_groups, "group_by": rng.choice([1, 2]),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "renorm": rng.random() < 0.7,
                "factor": rng.choice([1.0, 2.5]), "dtype": dtype}
    if op == "quant":
        return {"op": op, "rows": _log(rng, 1, 20000), "k": 32 * rng.randint(1, 128), "dtype": dtype}
    if op == "linear":
        m = _log(rng, 1, 511)
        return {"op": op, "m": m, "n": _log(rng, 100, 22016), "k": 32 * _log(rng, 8, 128), "dtype": dtype}
    entries = rng.choice([8, 16, 32, 64])
    k = rng.randint(1, 8)
    return {"op": op, "m": _log(rng, 1, 511), "k": k, "entries": entries, "n": _log(rng, 100, 2816),
            "kk": 32 * _log(rng, 4, 64), "per_rank": rng.random() < 0.5, "dtype": dtype}


# ---------------------------------------------------------------------------
# Inputs


def _widened(codes, scales):
    """The values that codes [.., k / 2] with scales [.., k / 32] stand for, [.., k] f32."""
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float32, device=codes.device)
    v = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1)
    v = v.reshape(*scales.shape, 32)
    return (v * torch.exp2(scales.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _quantised(x):
    """(signed codes, scale exponents) of x [.., k] f32, [.., k / 32, 32] and [.., k / 32]: the scale is the largest
    magnitude's power of two over 4, the elements rounded to nearest, ties to even, past 6 to 6."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1)
    e = ((amax.view(torch.int32) >> 23) - 129).clamp(min=-127)
    t = b * torch.exp2(-e.float()).unsqueeze(-1)
    a = t.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, t), e


def _packed(x):
    """The codes [.., k / 2] u8 and scales [.., k / 32] u8 of x."""
    v, e = _quantised(x)
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), (e + 127).to(torch.uint8)


def _weights(g, entries, n, k):
    """Weights as a model has them, N(0, 0.02), packed an expert at a time: [entries, n, ..]."""
    codes = torch.empty(entries, n, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(entries, n, k // 32, dtype=torch.uint8, device="cuda")
    for i in range(entries):
        codes[i], scales[i] = _packed(torch.randn(n, k, device="cuda", generator=g) * 0.02)
    return codes, scales


def _rows(g, m, k, dtype):
    """Activations: normal, some channels larger by an order of magnitude."""
    s = torch.exp(0.7 * torch.randn(k, device="cuda", generator=g))
    return (torch.randn(m, k, device="cuda", generator=g) * s).to(_TYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    t = _TYPES[case.get("dtype", "f32")]
    if case["op"] == "route":
        m, n = case["m"], case["n"]
        s["x"] = (1.5 * torch.randn(m, n, device="cuda", generator=g)).to(t)
        s["bias"] = 0.1 * torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        s["ids"] = torch.empty(m, case["k"], dtype=torch.int32, device="cuda")
        s["ws"] = torch.empty(m, case["k"], device="cuda")
        return s
    if case["op"] == "quant":
        rows, k = case["rows"], case["k"]
        s["x"] = (0.02 * torch.randn(rows, k, device="cuda", generator=g)).to(t)
        s["codes"] = torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(rows, k // 32, dtype=torch.uint8, device="cuda")
        s["y"] = torch.empty(rows, k, device="cuda")
        return s
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["w"], s["ws"] = (v[0] for v in _weights(g, 1, n, k))
        s["x"] = _rows(g, m, k, case["dtype"])
        s["y"] = torch.empty(m, n, dtype=t, device="cuda")
        s["work"] = torch.empty(_work_bytes(1, m, 1, n, k), dtype=torch.uint8, device="cuda")
        return s
    m, k, entries, n, kk = (case[v] for v in ("m", "k", "entries", "n", "kk"))
    s["w"], s["ws"] = _weights(g, entries, n, kk)
    s["x"] = _rows(g, m * k if case["per_rank"] else m, kk, case["dtype"])
    # Every row's ranks are distinct experts, the popular ones more often, as routes are.
    liking = torch.randn(m, entries, device="cuda", generator=g) + 0.5 * torch.randn(entries, device="cuda", generator=g)
    s["ids"] = liking.argsort(dim=-1, descending=True)[:, :k].to(torch.int32).contiguous()
    s["y"] = torch.empty(m, k, n, dtype=t, device="cuda")
    s["work"] = torch.empty(_work_bytes(entries, m, k, n, kk), dtype=torch.uint8, device="cuda")
    return s


def _work_bytes(entries, m, k, n, kk):
    """The products' workspace, as furykernel_b200 states it for every type: the (row, rank) inputs in parts, partial
    sums of few rows, and the lists that group the pairs by expert."""
    return 5 * m * k * kk + 16 * min(m * k, 512) * n + 16 * m * k + 64 * entries + 65536


# ---------------------------------------------------------------------------
# One pass


_context = None


def _ctx():
    global _context
    if _context is None:
        from furykernel_b200 import _native

        _context = _native.Context(torch.cuda.current_device())
    return _context


def _run_own(s):
    c = s["case"]
    ctx, sfx = _ctx(), _SUFFIX[c["dtype"]]
    p = lambda *names: [s[v].data_ptr() for v in names]  # noqa: E731
    if c["op"] == "route":
        params = {"m": c["m"], "n": c["n"], "k": c["k"], "groups": c["groups"], "top_groups": c["top_groups"],
                  "group_by": c["group_by"], "sigmoid": int(c["score"] == "sigmoid"), "renorm": int(c["renorm"]),
                  "ldx": c["n"], "factor": c["factor"]}
        if c["bias"]:
            ctx.launch("route_grouped_bias" + sfx, params, p("x", "bias", "ids", "ws"))
        else:
            ctx.launch("route_grouped" + sfx, params, p("x", "ids", "ws"))
        return {"ids": s["ids"], "weights": s["ws"]}
    if c["op"] == "quant":
        ctx.launch("quant_mxfp4" + sfx, {"rows": c["rows"], "k": c["k"], "ldx": c["k"]}, p("x", "codes", "scales"))
        ctx.launch("widen_mxfp4", {"rows": c["rows"], "k": c["k"], "ldy": c["k"]}, p("codes", "scales", "y"))
        return s["y"]
    if c["op"] == "linear":
        ctx.launch("linear_mxfp4" + sfx, {"n": c["n"], "k": c["k"], "m": c["m"], "ldx": c["k"], "ldy": c["n"]},
                   p("w", "ws", "x", "y", "work"))
        return s["y"]
    ctx.launch("linear_routed_mxfp4" + sfx,
               {"entries": c["entries"], "n": c["n"], "kk": c["kk"], "m": c["m"], "k": c["k"],
                "ldx": c["kk"] * (c["k"] if c["per_rank"] else 1), "ldy": c["k"] * c["n"],
                "per_rank": int(c["per_rank"])}, p("w", "ws", "ids", "x", "y", "work"))
    return s["y"]


def _run_route(s):
    """Scores in 32 bits, each exponential and each row's sum of them rounded once from 64: whole numbers come out of
    comparing them, so both forms have to have the same scores."""
    c, x = s["case"], s["x"].float()
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x.double()).float())
    else:
        e = torch.exp((x - x.amax(-1, keepdim=True)).double()).float()
        score = e / e.double().sum(-1, keepdim=True).float()
    choice = score + s["bias"] if c["bias"] else score
    if c["top_groups"] < c["groups"]:
        grouped = choice.view(c["m"], c["groups"], -1)
        best = grouped.sort(dim=-1, descending=True).values[..., : c["group_by"]].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, : c["top_groups"]]
        out = torch.ones_like(best, dtype=torch.bool).scatter_(1, kept, False)
        choice = grouped.masked_fill(out.unsqueeze(-1), -math.inf).view(c["m"], -1)
    ids = choice.sort(dim=-1, descending=True, stable=True).indices[:, : c["k"]]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": w * c["factor"]}


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "route":
        return _run_route(s)
    if c["op"] == "quant":
        v, e = _quantised(s["x"].float())
        return (v * torch.exp2(e.float()).unsqueeze(-1)).flatten(-2)
    x = s["x"].float()
    if c["op"] == "linear":
        return (x @ _widened(s["w"], s["ws"]).t()).to(s["x"].dtype)
    ids = s["ids"].long()
    m, k, kk = c["m"], c["k"], c["kk"]
    if m * k < c["entries"]:  # the chosen experts alone
        w = _widened(s["w"][ids], s["ws"][ids])
        y = w @ (x.view(m, k, kk, 1) if c["per_rank"] else x.view(m, 1, kk, 1))
        return y.squeeze(-1).to(s["x"].dtype)
    y = x @ _widened(s["w"], s["ws"]).transpose(1, 2)  # every row with every expert
    if c["per_rank"]:
        pair = torch.arange(m * k, device="cuda")
        return y[ids.view(-1), pair].view(m, k, -1).to(s["x"].dtype)
    return y[ids, torch.arange(m, device="cuda").unsqueeze(-1)].to(s["x"].dtype)


def work(case):
    c = case
    e = {"f32": 4, "bf16": 2, "f16": 2}[c["dtype"]]
    if c["op"] == "route":
        return {"bytes": e * c["m"] * c["n"] + 8 * c["m"] * c["k"] + (4 * c["n"] if c["bias"] else 0),
                "flops": 8 * c["m"] * c["n"]}
    if c["op"] == "quant":  # read, 4.25 bits out, read again, f32 out
        n = c["rows"] * c["k"]
        return {"bytes": n * (e + 4) + 2 * n * 17 / 32, "flops": 4 * n}
    if c["op"] == "linear":
        return {"bytes": c["n"] * c["k"] * 17 / 32 + e * c["m"] * (c["k"] + c["n"]),
                "flops": 2 * c["m"] * c["n"] * c["k"]}
    pairs = c["m"] * c["k"]
    taken = c["entries"] * (1 - (1 - c["k"] / c["entries"]) ** c["m"])  # the experts that some row chose, expected
    rows = pairs if c["per_rank"] else c["m"]
    return {"bytes": taken * c["n"] * c["kk"] * 17 / 32 + e * (rows * c["kk"] + pairs * c["n"]) + 4 * pairs,
            "flops": 2 * pairs * c["n"] * c["kk"]}


# ---------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_values(codes, scales):
    """The values, a decimal digit of the definition at a time: sign, exponent and mantissa bits of each code."""
    codes = codes.cpu().numpy()
    c = np.empty(codes.shape[:-1] + (2 * codes.shape[-1],), np.uint8)
    c[..., 0::2], c[..., 1::2] = codes % 16, codes // 16
    ex, mant = (c >> 1) & 3, (c & 1).astype(np.float32)
    v = np.where(ex == 0, mant / 2, np.exp2(ex.astype(np.float32) - 1) * (1 + mant / 2)) * np.where(c >= 8, -1, 1)
    scale = np.exp2(scales.cpu().numpy().astype(np.float64) - 127)
    return torch.from_numpy(v.astype(np.float32)).cuda().double() * torch.from_numpy(scale).cuda().repeat_interleave(
        32, -1)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "route":
        x = s["x"].float().cpu().numpy()
        x64 = x.astype(np.float64)
        # Which experts: by the 32-bit scores of the definition. Their weights: in 64 bits.
        if c["score"] == "sigmoid":
            f32 = np.float32(1) / (np.float32(1) + np.exp(-x64).astype(np.float32))
            f64 = 1 / (1 + np.exp(-x64))
        else:
            top = x.max(-1, keepdims=True)
            e = np.exp((x - top).astype(np.float64)).astype(np.float32)
            f32 = e / e.astype(np.float64).sum(-1, keepdims=True).astype(np.float32)
            e = np.exp(x64 - top)
            f64 = e / e.sum(-1, keepdims=True)
        choice = f32 + s["bias"].cpu().numpy() if c["bias"] else f32
        per = c["n"] // c["groups"]
        ids, w = [], []
        for r in range(c["m"]):
            by_group = [np.sort(choice[r, q * per:(q + 1) * per])[::-1] for q in range(c["groups"])]
            best = [v[0] + v[1] if c["group_by"] == 2 and per > 1 else v[0] for v in by_group]
            kept = sorted(range(c["groups"]), key=lambda q: (-best[q], q))[: c["top_groups"]]
            among = [i for q in sorted(kept) for i in range(q * per, (q + 1) * per)]
            got = sorted(among, key=lambda i: (-choice[r, i], i))[: c["k"]]
            v = f64[r, got]
            ids.append(got)
            w.append((v / v.sum() if c["renorm"] else v) * c["factor"])
        return {"ids": np.array(ids, np.int32), "weights": np.array(w)}
    if c["op"] == "quant":
        # The nearest of the grid's values by distance; of two as near, the one whose mantissa bit is 0.
        x = s["x"].double().view(c["rows"], -1, 32)
        amax = x.abs().amax(-1, keepdim=True)
        scale = torch.exp2((torch.floor(torch.log2(amax)) - 2).clamp(min=-127))
        near = torch.full_like(x, math.inf)
        got = torch.zeros_like(x)
        for v in (0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):
            d = (x.abs() / scale - v).abs()
            got = torch.where(d < near, v, got)
            near = torch.minimum(d, near)
        return torch.copysign(got * scale, x).view(c["rows"], -1)
    w = _exact_values(s["w"], s["ws"])
    x = s["x"].double()
    if c["op"] == "linear":
        return x @ w.t()
    y = torch.empty(c["m"] * c["k"], c["n"], dtype=torch.float64, device="cuda")
    flat = s["ids"].long().view(-1)
    for i in range(c["entries"]):
        pairs = (flat == i).nonzero().view(-1)
        y[pairs] = x[pairs if c["per_rank"] else pairs // c["k"]] @ w[i].t()
    return y.view(c["m"], c["k"], c["n"])
