"""Operators of the MXFP4 format and of the few-token mixture-of-experts layer: cases, plain forms and exact results.

Three operators, reached through the package's ops modules where `own` is set:

* quantize: rows -> MXFP4 (e2m1 values, one power-of-two scale per 32 elements along K) and back, `mxfp4.quantize` and
  `mxfp4.dequantize`;
* linear: y = x @ w.T with x quantised to MXFP4 on the way in and w held in MXFP4, `mxfp4.quantize` and
  `gemm.linear_mxfp4`, with a plain store or SiLU(gate) * up as its epilogue;
* layer: a whole mixture-of-experts layer for up to 16 tokens: router logits, top-k, the chosen experts' two products
  with their activation, weighted sum (+ the shared expert's rows), `moe.layer_forward`.

The plain forms are elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def listed() -> list:
    return [
        # one chat user's normed row in front of a projection: latency
        _quantize("quantize-1x5120", 1, 5120, "bf16"),
        # rows of a wider buffer (a slice of a fused projection), ragged prefill chunk
        _quantize("quantize-301x2688-strided", 301, 2688, "bf16", pad=1024),
        # the MLP's inner activations of a 2048-token prompt
        _quantize("quantize-2048x17408", 2048, 17408, "bf16"),
        # a full-precision weight matrix on its way into the format
        _quantize("quantize-weight-fp32", 17408, 5120, "fp32"),
        # one user: qkv projection of the 27B geometry, bound by the weight stream
        _linear("linear-1x7168x5120", 1, 7168, 5120),
        # 64 users: gate and up with SiLU
        _linear("linear-64x34816x5120-silu", 64, 34816, 5120, silu=True),
        # a ragged prefill chunk through the down projection
        _linear("linear-301x5120x17408", 301, 5120, 17408),
        # time to first token of a 2048-token prompt: gate and up with SiLU
        _linear("linear-2048x34816x5120-silu", 2048, 34816, 5120, silu=True),
        # one user of the 512-expert layer of width 2560 with its shared expert
        _layer("layer-1-mxfp4", 1, 512, 10, 2560, 640, "swiglu", "mxfp4", shared=True),
        # four users of a latent layer: the router reads the hidden rows, the experts the latent ones; sigmoid scores
        _layer("layer-4-nvfp4-latent", 4, 512, 22, 1024, 2688, "relu2", "nvfp4", sigmoid=True, route_width=4096),
        # a small layer in bf16, as before quantisation
        _layer("layer-7-bf16", 7, 64, 8, 2048, 768, "swiglu", "bf16"),
        # sixteen rows (users or a verify block): most of the time streams a quarter of all experts
        _layer("layer-16-mxfp4", 16, 512, 10, 2560, 640, "swiglu", "mxfp4", shared=True),
    ]


def _quantize(name, rows, k, dtype, pad=0):
    return {"name": name, "op": "quantize", "rows": rows, "k": k, "dtype": dtype, "pad": pad}


def _linear(name, m, n, k, silu=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "silu": silu}


def _layer(name, tokens, experts, topk, hidden, inter, act, fmt, sigmoid=False, shared=False, route_width=0):
    return {"name": name, "op": "layer", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden,
            "inter": inter, "act": act, "fmt": fmt, "sigmoid": sigmoid, "shared": shared, "route_width": route_width}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(("quantize", "linear", "layer"))
    if op == "quantize":
        k = 32 * _log(rng, 1, 17408 // 32)
        rows = _log(rng, 1, min(8192, 17408 * 5120 // k))
        case = _quantize("", rows, k, rng.choice(("bf16", "bf16", "fp16", "fp32")), pad=rng.choice((0, 8, 1000)))
    elif op == "linear":
        m, k = _log(rng, 1, 2048), 32 * _log(rng, 4, 17408 // 32)
        n = 16 * _log(rng, 4, 34816 // 16)
        while m * n * k > 2048 * 34816 * 5120 or n * k > 34816 * 5120:
            n = max(64, n // 32 * 16)
            if n == 64:
                m = max(1, m // 2)
        case = _linear("", m, n, k, silu=rng.random() < 0.5)
    else:
        experts = _log(rng, 8, 512)
        fmt, act = rng.choice(("mxfp4", "mxfp4", "nvfp4", "bf16")), rng.choice(("swiglu", "relu2"))
        hidden, inter = 128 * _log(rng, 2, 32), 128 * _log(rng, 1, 21)
        while experts * hidden * inter > 512 * 2560 * 640 // (4 if fmt == "bf16" else 1):
            if hidden > inter:
                hidden = max(256, hidden // 256 * 128)
            else:
                inter = max(128, inter // 256 * 128)
            if hidden == 256 and inter == 128:
                break
        case = _layer("", _log(rng, 1, 16), experts, min(_log(rng, 1, 22), experts, 10 if act == "swiglu" else 22),
                      hidden, inter, act, fmt, sigmoid=rng.random() < 0.5, shared=rng.random() < 0.5,
                      route_width=rng.choice((0, 0, 1536, 4096)))
    del case["name"]
    return case


# ---- inputs: the same on both sides, from the seed alone


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _rows(g, rows, k, dtype=torch.bfloat16, ld=0):
    """Normed activations: N(0, 1) with a few loud channels, as trained models have them."""
    x = torch.randn(rows, k, generator=g, device=DEVICE)
    loud = torch.rand(k, generator=g, device=DEVICE) < 0.004
    x = torch.where(loud, x * 20, x)
    if not ld:
        return x.to(dtype)
    buf = torch.zeros(rows, k + ld, dtype=dtype, device=DEVICE)
    buf[:, :k] = x.to(dtype)
    return buf[:, :k]


def _packed(g, rows, k):
    """Two e2m1 codes a byte, low nibble first."""
    return torch.randint(0, 256, (rows, k // 2), generator=g, device=DEVICE, dtype=torch.uint8)


def _inputs(case, seed) -> dict:
    g = _generator(seed)
    if case["op"] == "quantize":
        if case["dtype"] == "fp32":
            return {"x": torch.randn(case["rows"], case["k"], generator=g, device=DEVICE) * 0.02}
        return {"x": _rows(g, case["rows"], case["k"], TYPES[case["dtype"]], case["pad"])}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"x": _rows(g, m, k), "codes": _packed(g, n, k),
                "scales": torch.randint(117, 122, (n, k // 32), generator=g, device=DEVICE, dtype=torch.uint8)}
    t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inter"]
    n1 = 2 * i if case["act"] == "swiglu" else i
    d = {"x": _rows(g, t, h), "route_x": _rows(g, t, case["route_width"]) if case["route_width"] else None,
         "router": (torch.randn(e, case["route_width"] or h, generator=g, device=DEVICE) * 0.02).bfloat16(),
         "sel_bias": torch.randn(e, generator=g, device=DEVICE) * 0.05 if case["sigmoid"] else None,
         "shared": _rows(g, t, h) if case["shared"] else None}
    for name, n, k in (("fc1", n1, h), ("fc2", h, i)):
        if case["fmt"] == "bf16":
            d[name] = torch.empty(e * n, k, dtype=torch.bfloat16, device=DEVICE).normal_(0, 0.03, generator=g)
            continue
        d[name + "_codes"] = _packed(g, e * n, k)
        shape = (e * n, k // BLOCK[case["fmt"]])
        if case["fmt"] == "mxfp4":
            d[name + "_scales"] = torch.randint(117, 122, shape, generator=g, device=DEVICE, dtype=torch.uint8)
        else:      # e4m3 bytes between 64 and 240, a scale per expert
            d[name + "_scales"] = torch.randint(0x68, 0x78, shape, generator=g, device=DEVICE, dtype=torch.uint8)
            d[name + "_gscale"] = torch.rand(e, generator=g, device=DEVICE) * 4e-5 + 4e-5
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    state = {"case": dict(case), **d}
    if not own:
        return state
    from hibana_b200.ops import moe, mxfp4, nvfp4
    if case["op"] == "linear":
        state["w"] = mxfp4.from_blocks(d["codes"], d["scales"])
    elif case["op"] == "layer":
        e, h, i, fmt = case["experts"], case["hidden"], case["inter"], case["fmt"]
        if fmt == "bf16":
            ew = moe.ExpertWeights(e, h, i, case["act"], fmt, d["fc1"], d["fc2"])
        elif fmt == "mxfp4":
            ew = moe.ExpertWeights(e, h, i, case["act"], fmt, mxfp4.from_blocks(d["fc1_codes"], d["fc1_scales"]),
                                   mxfp4.from_blocks(d["fc2_codes"], d["fc2_scales"]))
        else:
            in_scale = torch.full((1,), 48.0 / (6 * 448), device=DEVICE)
            fc1, fc2 = (nvfp4.Nvfp4Tensor(d[f + "_codes"], nvfp4.swizzle_sf(d[f + "_scales"]), d[f + "_gscale"],
                                          d[f + "_codes"].shape[0], k) for f, k in (("fc1", h), ("fc2", i)))
            ew = moe.ExpertWeights(e, h, i, case["act"], fmt, fc1, fc2, fc1.gscale * in_scale, fc2.gscale * in_scale,
                                   in_scale, in_scale)
        state["experts"] = ew
    for key in ("codes", "scales", "fc1", "fc2", "fc1_codes", "fc2_codes", "fc1_scales", "fc2_scales"):
        state.pop(key, None)
    return state


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from hibana_b200.ops import gemm, moe, mxfp4
    c = s["case"]
    if c["op"] == "quantize":
        return mxfp4.dequantize(mxfp4.quantize(s["x"]), s["x"].dtype)
    if c["op"] == "linear":
        return gemm.linear_mxfp4(mxfp4.quantize(s["x"]), s["w"],
                                 epilogue=gemm.EPI_SILU_MUL if c["silu"] else gemm.EPI_STORE, static_weight=True)
    return moe.layer_forward(s["x"], s["router"], s["experts"], c["topk"], sigmoid=c["sigmoid"], sel_bias=s["sel_bias"],
                             renorm=True, scale=2.5 if c["sigmoid"] else 1.0, shared=s["shared"], route_x=s["route_x"])


# ---- the plain forms: elementary torch operations in 32 bits


def _quantized(x):
    """Rows in 32 bits -> the values their MXFP4 form stands for. The scale of a block of 32 is 2^(floor(log2(max)) - 2)
    (that of zeros 2^-127), elements are rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it (ties to the even
    code) and saturate."""
    rows, k = x.shape
    b = x.float().view(rows, k // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(amax).exponent - 1 - 2).clamp_min(-127)
    exponent = torch.where(amax > 0, exponent, torch.full_like(exponent, -127))
    y = torch.ldexp(b, -exponent)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp_max(6.0)
    return torch.ldexp(torch.copysign(q, y), exponent).view(rows, k)


def _decode(codes, scales, fmt, gscale=None):
    """Packed codes [..., k / 2] and scale bytes [..., k / block] -> values in 32 bits."""
    table = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), device=codes.device)
    c = codes.int()
    v = torch.stack((table[c & 15], table[c >> 4]), -1).flatten(-2)
    if fmt == "mxfp4":
        s = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    else:
        s = scales.view(torch.float8_e4m3fn).float() * gscale
    return (v.unflatten(-1, (-1, BLOCK[fmt])) * s.unsqueeze(-1)).flatten(-2)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        return _quantized(s["x"]).to(s["x"].dtype)
    if c["op"] == "linear":
        y = _quantized(s["x"]) @ _decode(s["codes"], s["scales"], "mxfp4").t()
        if c["silu"]:
            y = y[:, 0::2] / (1 + torch.exp(-y[:, 0::2])) * y[:, 1::2]
        return y.to(torch.bfloat16)
    t, e, k = c["tokens"], c["experts"], c["topk"]
    x = s["x"].float()
    logits = (x if s["route_x"] is None else s["route_x"].float()) @ s["router"].float().t()
    if c["sigmoid"]:
        score = 1 / (1 + torch.exp(-logits))
        order = score + s["sel_bias"]
    else:
        score = torch.exp(logits - logits.amax(-1, keepdim=True))
        score = order = score / score.sum(-1, keepdim=True)
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[:, :k]
    w = score.gather(1, ids)
    w = w / w.sum(-1, keepdim=True) * (2.5 if c["sigmoid"] else 1.0)

    def experts(name, n):
        if c["fmt"] == "bf16":
            return s[name].view(e, n, -1)[ids].float()
        scale = s[name + "_gscale"][ids][..., None, None] if c["fmt"] == "nvfp4" else None
        return _decode(s[name + "_codes"].view(e, n, -1)[ids], s[name + "_scales"].view(e, n, -1)[ids], c["fmt"], scale)

    n1 = 2 * c["inter"] if c["act"] == "swiglu" else c["inter"]
    h1 = (experts("fc1", n1) @ x[:, None, :, None])[..., 0]
    if c["act"] == "swiglu":
        mid = h1[..., 0::2] / (1 + torch.exp(-h1[..., 0::2])) * h1[..., 1::2]
    else:
        mid = h1.clamp_min(0) ** 2
    y = (experts("fc2", c["hidden"]) @ mid[..., None])[..., 0]
    out = (y * w[..., None]).sum(1)
    if s["shared"] is not None:
        out = out + s["shared"].float()
    return out.to(torch.bfloat16)


# ---- the definitions in 64 bits


def _exact_blocks(x):
    """MXFP4 values of rows in 64 bits, by search over the format's grid."""
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    out = torch.empty_like(x)
    for r in range(0, x.shape[0], 256):
        b = x[r:r + 256].reshape(-1, 32)
        top = b.abs().max(1).values
        e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
        e = torch.where(torch.pow(2.0, e) > top, e - 1, e)               # log2 rounds: settle next to powers of two
        e = torch.where(torch.pow(2.0, e + 1) <= top, e + 1, e)
        scale = torch.pow(2.0, torch.where(top > 0, e - 2, torch.full_like(e, -127.0)).clamp_min(-127))
        a = (b / scale[:, None]).abs()
        # of two grid points equally near, the one with the even code: walk up, moving on to an odd code only when nearer
        best = torch.zeros_like(a)
        for code in range(1, 8):
            middle = (grid[code] + grid[code - 1]) / 2
            best = torch.where((a > middle) | ((a == middle) & (code % 2 == 0)), grid[code], best)
        out[r:r + 256] = (torch.where(b < 0, -best, best) * scale[:, None]).view(-1, x.shape[1])
    return out


def _exact_values(codes, scales, fmt, gscale=1.0):
    low, high = (codes & 15).long(), (codes >> 4).long()
    v = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=codes.device)
    for start, c in ((0, low), (1, high)):
        v[..., start::2] = grid[c % 8] * (1 - 2 * (c // 8))
    if fmt == "mxfp4":
        s = torch.pow(2.0, scales.double() - 127)
    else:
        b = scales.long()
        s = torch.pow(2.0, (b >> 3 & 15).double() - 7) * (1 + (b & 7).double() / 8) * gscale      # (normal numbers only)
    return v * s.repeat_interleave(BLOCK[fmt], -1)


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "quantize":
        return _exact_blocks(d["x"].double())
    if case["op"] == "linear":
        x, rows = _exact_blocks(d["x"].double()), []
        for r in range(0, case["n"], 2048):
            rows.append(x @ _exact_values(d["codes"][r:r + 2048], d["scales"][r:r + 2048], "mxfp4").t())
        y = torch.cat(rows, 1)
        return y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2] if case["silu"] else y
    x = d["x"].double()
    logits = (d["x"] if d["route_x"] is None else d["route_x"]).double() @ d["router"].double().t()
    if case["sigmoid"]:
        score = torch.sigmoid(logits)
        order = score + d["sel_bias"].double()
    else:
        score = order = torch.softmax(logits, -1)
    out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=DEVICE)
    chosen = torch.argsort(order, dim=-1, descending=True, stable=True)[:, :case["topk"]]
    e, h, i = case["experts"], case["hidden"], case["inter"]
    n1 = 2 * i if case["act"] == "swiglu" else i

    def matrix(name, n, expert):
        rows = slice(expert * n, (expert + 1) * n)
        if case["fmt"] == "bf16":
            return d[name][rows].double()
        g = float(d[name + "_gscale"][expert]) if case["fmt"] == "nvfp4" else 1.0
        return _exact_values(d[name + "_codes"][rows], d[name + "_scales"][rows], case["fmt"], g)

    for expert in sorted(set(chosen.flatten().tolist())):
        tokens, place = (chosen == expert).nonzero(as_tuple=True)
        h1 = x[tokens] @ matrix("fc1", n1, expert).t()
        mid = h1[:, 0::2] * torch.sigmoid(h1[:, 0::2]) * h1[:, 1::2] if case["act"] == "swiglu" else torch.relu(h1) ** 2
        share = score[tokens, chosen[tokens, place]] / score[tokens[:, None], chosen[tokens]].sum(1)
        out[tokens] += (mid @ matrix("fc2", h, expert).t()) * (share * (2.5 if case["sigmoid"] else 1.0))[:, None]
    return out + d["shared"].double() if d["shared"] is not None else out


def work(case) -> dict:
    if case["op"] == "quantize":
        n, size = case["rows"] * case["k"], TYPES[case["dtype"]].itemsize
        return {"bytes": 2 * n * size, "flops": 3 * n}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k * 17 // 32 + 2 * m * (n // 2 if case["silu"] else n), "flops": 2 * m * n * k}
    t, e, k, h, i = (case[x] for x in ("tokens", "experts", "topk", "hidden", "inter"))
    per_expert = h * i * (3 if case["act"] == "swiglu" else 2)
    size = {"bf16": 2.0, "nvfp4": 9 / 16, "mxfp4": 17 / 32}[case["fmt"]]
    distinct = e * (1 - (1 - k / e) ** t)                     # experts that some token chooses, on average
    width = case["route_width"] or h
    rows = t * (2 * h + (h if case["shared"] else 0) + case["route_width"])
    return {"bytes": int(distinct * per_expert * size + 2 * e * width + 2 * rows),
            "flops": 2 * t * (k * per_expert + e * width)}
