"""A mixture-of-experts layer for a few tokens against a plain computation in 64 bits; MXFP4 experts."""
import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200.ops import moe, mxfp4


def _experts(e, h, inter, act, fmt, seed=0, std=0.05, h_out=None, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    n1 = 2 * inter if act == "swiglu" else inter
    fc1 = torch.randn(e, n1, h, generator=g) * std
    fc2 = torch.randn(e, h_out or h, inter, generator=g) * std
    return moe.ExpertWeights.create(fc1, fc2, act, fmt, in_amax=5.0, mid_amax=2.0).to(dev)


def _case(t, e, h, act, fmt, inter, seed=0, wide=0, shared=True, **kw):
    ew = _experts(e, h, inter, act, fmt, seed, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(t, h, generator=g).bfloat16()
    rx = torch.randn(t, wide, generator=g).bfloat16() if wide else None
    router = (torch.randn(e, wide or h, generator=g) * 0.2).bfloat16()
    bias = torch.randn(e, generator=g) * 0.1
    sh = torch.randn(t, ew.fc2_rows, generator=g).bfloat16() if shared else None
    return ew, x, rx, router, bias, sh


def _exact(ew, x, rx, router, topk, sigmoid, bias, scale, shared, renorm=True):
    """(out, allowed error before the final rounding), float64, by the definition."""
    lg = (x if rx is None else rx).double() @ router.double().t()
    score = torch.sigmoid(lg) if sigmoid else torch.softmax(lg, -1)
    order = torch.argsort(score + (bias.double() if sigmoid else 0), dim=-1, descending=True, stable=True)
    ids = order[:, :topk]
    w = score.gather(1, ids)
    w = w / w.sum(-1, keepdim=True) * scale if renorm else w * scale
    w1, w2 = ew.dense(1).double(), ew.dense(2).double()
    out = torch.zeros(x.shape[0], ew.fc2_rows, dtype=torch.float64)
    err = torch.zeros_like(out)
    # sums of n terms in 32 bits: n * 2^-23 of what is added up in magnitude; x and mid keep 14 bits of
    # their block's largest number, counted here from the row's (bf16 experts: x all, mid 16 bits); exponentials,
    # quotients and weights within 2^-18
    digits = 0.0 if ew.fmt == "bf16" else 2.0 ** -14
    mid_half = 2.0 ** -17 if ew.fmt == "bf16" else 0.0
    for t in range(x.shape[0]):
        for j in range(topk):
            e = int(ids[t, j])
            xd = x[t].double()
            h1, s1 = w1[e] @ xd, (w1[e].abs() @ (xd.abs() + digits * xd.abs().max())) * (xd.numel() * 2.0 ** -23)
            s1 = s1 + w1[e].abs().sum(1) * digits * xd.abs().max()
            if ew.act == "swiglu":
                gate, up = h1[0::2], h1[1::2]
                mid = gate * torch.sigmoid(gate) * up
                d = 1.1 * s1[0::2] * (up.abs() + s1[1::2]) + (gate.abs() + s1[0::2]) * s1[1::2]
            else:
                mid = torch.relu(h1) ** 2
                d = 2 * h1.abs() * s1 + s1 ** 2
            d = d + 2.0 ** -18 * mid.abs()
            d = d + mid_half * (mid.abs() + d) + digits * (mid.abs() + d).max()
            y, a = w2[e] @ mid, w2[e].abs()
            dy = a @ d + (a @ mid.abs()) * (mid.numel() * 2.0 ** -23)
            out[t] += w[t, j] * y
            err[t] += w[t, j] * (dy + 2.0 ** -18 * y.abs())
    err += topk * 2.0 ** -23 * (out.abs() + err)
    return (out if shared is None else out + shared.double()), err


def _check(got, want, err):
    half = torch.finfo(torch.bfloat16).eps / 2
    off = (got.double().cpu() - want).abs() - err - half * (want.abs() + err)
    assert (off <= 0).all(), (float(off.max()), float(want.abs().max()))


CASES = [   # tokens, experts, top-k, hidden, inter, act, fmt, sigmoid, router width
    (1, 8, 2, 256, 128, "swiglu", "mxfp4", False, 0),
    (1, 8, 2, 256, 128, "swiglu", "nvfp4", False, 0),
    (1, 8, 2, 256, 128, "swiglu", "bf16", False, 0),
    (3, 33, 5, 128, 384, "relu2", "mxfp4", True, 96),
    (5, 17, 17, 384, 128, "relu2", "nvfp4", True, 264),
    (4, 40, 3, 48, 24, "swiglu", "bf16", True, 40),
    (16, 9, 9, 256, 192, "swiglu", "mxfp4", False, 0),        # every expert takes all sixteen tokens
    (16, 12, 8, 384, 64, "swiglu", "nvfp4", False, 0),
    (16, 600, 32, 128, 128, "relu2", "mxfp4", True, 0),
    (13, 64, 8, 640, 320, "swiglu", "mxfp4", False, 0),
    (16, 20, 4, 1024, 128, "relu2", "bf16", True, 2048),
    (2, 1, 1, 128, 128, "relu2", "mxfp4", True, 0),
]


@pytest.mark.parametrize("t,e,k,h,inter,act,fmt,sig,wide", [c for c in CASES if c[1] <= 40])
def test_reference_follows_the_definition_cpu(t, e, k, h, inter, act, fmt, sig, wide):
    ew, x, rx, router, bias, sh = _case(t, e, h, act, fmt, inter, wide=wide)
    got = moe.layer_forward(x, router, ew, k, sigmoid=sig, sel_bias=bias if sig else None, scale=1.7, shared=sh, route_x=rx)
    _check(got, *_exact(ew, x, rx, router, k, sig, bias, 1.7, sh))


def test_more_tokens_take_the_grouped_products_cpu():
    ew, x, rx, router, bias, sh = _case(20, 8, 64, "swiglu", "mxfp4", 64)
    got = moe.layer_forward(x, router, ew, 2, shared=sh)
    ids, w = moe.route(x.float() @ router.float().t(), 2)
    assert torch.equal(got, moe.experts_forward(x, ids, w, ew, shared=sh))


def test_refusals_cpu():
    ew, x, rx, router, bias, sh = _case(3, 8, 128, "swiglu", "mxfp4", 64)
    ok = dict(sigmoid=True, sel_bias=bias, shared=sh)
    moe.layer_forward(x, router, ew, 2, **ok)
    for args, kw in (((x.float(), router, ew, 2), ok), ((x[:, :64], router, ew, 2), ok), ((x, router[:7], ew, 2), ok),
                     ((x, router.float(), ew, 2), ok), ((x, router, ew, 0), ok), ((x, router, ew, 9), ok),
                     ((x, router, ew, 2), {**ok, "sigmoid": False}), ((x, router, ew, 2), {**ok, "sel_bias": bias[:5]}),
                     ((x, router, ew, 2), {**ok, "shared": sh[:2]}), ((x, router, ew, 2), {**ok, "route_x": x[:2]}),
                     ((x, router, ew, 2), {**ok, "shared": sh.float()})):
        with pytest.raises(ValueError):
            moe.layer_forward(*args, **kw)


def test_slices_of_mxfp4_experts_cpu():
    ew = _experts(6, 128, 128, "relu2", "mxfp4")
    part = ew.slice(2, 3)
    assert torch.equal(part.dense(1), ew.dense(1)[2:5]) and torch.equal(part.dense(2), ew.dense(2)[2:5])


# ---- kernels


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,inter,act,fmt,sig,wide", CASES)
def test_layer_gpu(t, e, k, h, inter, act, fmt, sig, wide):
    ew, x, rx, router, bias, sh = _case(t, e, h, act, fmt, inter, wide=wide)
    ewg = ew.to("cuda")
    dev = lambda v: None if v is None else v.cuda()      # noqa: E731
    run = lambda **kw: moe.layer_forward(dev(x), dev(router), ewg, k, **{**dict(      # noqa: E731
        sigmoid=sig, sel_bias=dev(bias) if sig else None, scale=1.7, shared=dev(sh), route_x=dev(rx)), **kw})
    got = run()
    _check(got, *_exact(ew, x, rx, router, k, sig, bias, 1.7, sh))
    assert torch.equal(run(), got)
    _check(run(shared=None, renorm=False), *_exact(ew, x, rx, router, k, sig, bias, 1.7, None, renorm=False))
    assert nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
def test_a_token_does_not_depend_on_its_neighbours_gpu(fmt):
    """Rows of a batch give the bits they give alone wherever the experts' order of sums is the same: one expert a token."""
    ew, x, rx, router, bias, sh = _case(16, 8, 256, "swiglu", fmt, 128)
    ewg = ew.to("cuda")
    whole = moe.layer_forward(x.cuda(), router.cuda(), ewg, 1, shared=sh.cuda())
    for i in range(16):
        assert torch.equal(moe.layer_forward(x[i:i + 1].cuda(), router.cuda(), ewg, 1, shared=sh[i:i + 1].cuda()), whole[i:i + 1])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
def test_extreme_rows_gpu(fmt):
    """Rows far outside fp16's range, zeros, and an infinity or a NaN that stays in its row."""
    ew, x, rx, router, bias, sh = _case(6, 8, 256, "relu2", fmt, 128, shared=False)
    router = torch.zeros_like(router)               # every token takes experts 0 and 1 with weight one half
    x[1] = 0
    x[2] *= 2.0 ** 14
    x[3] *= 2.0 ** -20
    got = moe.layer_forward(x.cuda(), router.cuda(), ew.to("cuda"), 2)
    want, err = _exact(ew, x, None, router, 2, False, bias, 1.0, None)
    _check(got, want, err)
    assert (got[1] == 0).all()
    bad = x.clone()
    bad[0, 7], bad[4, 200] = float("inf"), float("nan")
    # the router would see them too: it reads other rows
    again = moe.layer_forward(bad.cuda(), router.cuda(), ew.to("cuda"), 2, route_x=x.cuda())
    keep = [1, 2, 3, 5]
    assert torch.equal(again[keep], got[keep]) and torch.isnan(again[4]).all() and not torch.isfinite(again[0]).any()


@pytest.mark.gpu
def test_ties_go_to_the_lower_expert_gpu():
    ew, x, rx, router, bias, sh = _case(9, 48, 128, "swiglu", "mxfp4", 64, shared=False)
    router[:] = 0
    router[5:40, 3] = 1.0                             # experts 5 .. 39 tie above the rest where x[3] > 0, below where it is < 0
    got = moe.layer_forward(x.cuda(), router.cuda(), ew.to("cuda"), 6)
    ids = torch.stack([torch.arange(5, 11) if x[t, 3] > 0 else torch.tensor([0, 1, 2, 3, 4, 40]) for t in range(9)])
    lg = x.float() @ router.float().t()
    assert torch.equal(moe.route(lg, 6)[0].long(), ids)
    _check(got, *_exact(ew, x, None, router, 6, False, bias, 1.0, None))


@pytest.mark.gpu
def test_nan_logits_keep_the_ids_in_range_gpu():
    ew, x, rx, router, bias, sh = _case(4, 8, 128, "swiglu", "mxfp4", 64)
    router[3, 5] = float("nan")
    got = moe.layer_forward(x.cuda(), router.cuda(), ew.to("cuda"), 8, shared=sh.cuda())
    torch.cuda.synchronize()
    assert got.shape == (4, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_strided_rows_wide_layers_and_outputs_gpu(fmt):
    """Views of wider buffers, aligned and not; and a layer too wide for sixteen tokens in one call."""
    ew, x, rx, router, bias, sh = _case(5, 8, 256, "swiglu", fmt, 64)
    ewg = ew.to("cuda")
    want = moe.layer_forward(x.cuda(), router.cuda(), ewg, 2, shared=sh.cuda())
    for lead, width in ((8, 272), (3, 263)):
        wide = lambda v: torch.zeros(v.shape[0], width, dtype=v.dtype, device="cuda")[:, lead:lead + 256].copy_(v)   # noqa: E731
        assert torch.equal(moe.layer_forward(wide(x), wide(router), ewg, 2, shared=wide(sh)), want)
    ew, x, rx, router, bias, sh = _case(16, 4, 4608, "relu2", fmt, 128, h_out=128, std=0.02)
    assert 8 <= nv.lib().hb_moe_few_tokens(moe._KINDS[fmt], 4608) < 16
    got = moe.layer_forward(x.cuda(), router.cuda(), ew.to("cuda"), 2, shared=sh.cuda())
    _check(got, *_exact(ew, x, None, router, 2, False, bias, 1.0, sh))


@pytest.mark.gpu
def test_empty_and_uncovered_layers_gpu():
    ew, x, rx, router, bias, sh = _case(3, 8, 128, "swiglu", "mxfp4", 64)
    assert moe.layer_forward(x[:0].cuda(), router.cuda(), ew.to("cuda"), 2).shape == (0, 128)
    assert not moe.few_tokens_ok(_experts(4, 128, 96, "swiglu", "mxfp4"), 2)
    assert not moe.few_tokens_ok(_experts(4, 128, 128, "swiglu", "w3"), 2)
    # more tokens: the grouped products, whichever way they are reached
    ew, x, rx, router, bias, sh = _case(40, 8, 256, "swiglu", "mxfp4", 128)
    ewg = ew.to("cuda")
    from hibana_b200.ops import gemm
    ids, w = moe.route(gemm.linear_bf16(x.cuda(), router.cuda(), epilogue=gemm.EPI_STORE_F32), 2)
    assert torch.equal(moe.layer_forward(x.cuda(), router.cuda(), ewg, 2, shared=sh.cuda()),
                       moe.experts_forward(x.cuda(), ids, w, ewg, shared=sh.cuda()))


@pytest.mark.gpu
def test_graphs_and_streams_gpu():
    ew, x, rx, router, bias, sh = _case(7, 16, 256, "swiglu", "mxfp4", 128)
    ewg, r = ew.to("cuda"), router.cuda()
    rows = [torch.randn(7, 256).bfloat16().cuda() for _ in range(4)]
    want = [moe.layer_forward(v, r, ewg, 4) for v in rows]
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for s, v in zip(streams, rows):                   # four calls under way at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                last = moe.layer_forward(v, r, ewg, 4)
            got.append(last)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = [rows[0].clone(), rows[1].clone()]
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(moe.layer_forward(s, r, ewg, 4))
        graphs.append(g)
    static[0].copy_(rows[2])
    static[1].copy_(rows[3])
    torch.cuda.synchronize()
    for s, g in zip(streams, graphs):                 # two captured calls replayed side by side
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[2]) and torch.equal(outs[1], want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,inter,act", [(17, 8, 2, 256, 512, "swiglu"), (37, 16, 4, 288, 128, "relu2"), (300, 8, 2, 128, 256, "swiglu")])
def test_grouped_mxfp4_experts_gpu(t, e, k, h, inter, act):
    """The products behind each other, each from the same quantised input: the first is checked through the second's identity."""
    ew = _experts(e, h, inter, act, "mxfp4", seed=1, h_out=256)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(t, h, generator=g).bfloat16()
    ids, w = moe.route(torch.randn(t, e, generator=g), k)
    shared = torch.randn(t, 256, generator=g).bfloat16()
    ref = moe.experts_forward(x, ids, w, ew, shared=shared).double()
    ewg = ew.to("cuda")
    got = moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ewg, shared=shared.cuda()).double().cpu()
    # a mid value next to a border between two codes may fall on either side, which moves it by up to a third of itself: a few of the
    # `inter` terms of a sum. Their share of an output is bounded in the mean square, not one by one.
    assert (got - ref).norm() <= 2.0 ** -6 * ref.norm()
    again = moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ewg, shared=shared.cuda()).double().cpu()
    assert torch.equal(again, got) and nv.read_status() == 0
    lo = moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ewg, e_lo=0, e_n=e // 2).float()
    hi = moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ewg.slice(e // 2, e // 2), id_base=e // 2).float()
    whole = moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ewg).float()
    # the parts are rounded to bf16 before they meet: 2^-8 of each, and of the sum
    assert ((lo + hi - whole).abs() <= 2.0 ** -8 * (lo.abs() + hi.abs() + whole.abs()) + 1e-6).all()


@pytest.mark.gpu
def test_a_run_of_them_gpu():
    """Projection in MXFP4, a layer of MXFP4 experts, projection: as a block of a model uses them, against the same steps on CPU."""
    from hibana_b200.ops import gemm
    ew, x, rx, router, bias, sh = _case(6, 8, 256, "swiglu", "mxfp4", 128, seed=5)
    g = torch.Generator().manual_seed(9)
    w_in, w_out = (mxfp4.quantize_weight(torch.randn(256, 256, generator=g) * 0.06) for _ in range(2))

    def block(dev, h):
        e = ew.to(dev)
        y = moe.layer_forward(h, router.to(dev), e, 2, shared=sh.to(dev))
        return y, gemm.linear_mxfp4(mxfp4.quantize(y), w_out.to(dev), epilogue=gemm.EPI_RESIDUAL, residual=h)

    h = gemm.linear_mxfp4(mxfp4.quantize(x), w_in)
    hg = gemm.linear_mxfp4(mxfp4.quantize(x.cuda()), w_in.to("cuda")).cpu()
    assert (hg.float() - h.float()).abs().max() <= 2.0 ** -7 * h.float().abs().max()      # one step of bf16 either way
    y, z = block("cpu", h)
    yg, zg = block("cuda", h.cuda())
    assert ((yg.cpu().float() - y.float()).abs() <= 2.0 ** -7 * y.float().abs() + 2.0 ** -9 * y.float().abs().max()).all()
    # what the last projection reads differs by steps of bf16, so some of its codes do
    z2 = gemm.linear_mxfp4(mxfp4.quantize(yg.cpu()), w_out, epilogue=gemm.EPI_RESIDUAL, residual=h)
    assert (zg.cpu().float() - z2.float()).abs().max() <= 2.0 ** -7 * z2.float().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,inter,act", [(129, 4, 2, 256, 320, "swiglu"), (300, 6, 3, 288, 384, "relu2"), (520, 8, 2, 128, 128, "relu2"),
                                               (700, 3, 3, 512, 192, "swiglu"), (129, 40, 1, 96, 128, "swiglu")])
def test_grouped_mxfp4_experts_on_sm_pairs_gpu(t, e, k, h, inter, act):
    """Chunks of 256 rows, the activation quantised in the first product's epilogue; a token with an infinity spoils itself only."""
    ew = _experts(e, h, inter, act, "mxfp4", seed=3, h_out=256)
    assert moe.pair_rows(ew, t) and not moe.pair_rows(ew, 128)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(t, h, generator=g).bfloat16()
    ids, w = moe.route(torch.randn(t, e, generator=g), k)
    shared = torch.randn(t, 256, generator=g).bfloat16()
    ref = moe.experts_forward(x, ids, w, ew, shared=shared).double()
    ewg = ew.to("cuda")
    got = moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ewg, shared=shared.cuda()).double().cpu()
    # (as above: codes of mid next to a border may fall on either side)
    assert (got - ref).norm() <= 2.0 ** -6 * ref.norm()
    assert torch.equal(moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ewg, shared=shared.cuda()).double().cpu(), got)
    bad = x.clone()
    bad[t // 2, 5] = float("inf")
    out = moe.experts_forward(bad.cuda(), ids.cuda(), w.cuda(), ewg, shared=shared.cuda()).double().cpu()
    keep = torch.arange(t) != t // 2
    assert torch.equal(out[keep], got[keep]) and out[t // 2].isnan().all() and nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
def test_dependent_launches_change_nothing_gpu(fmt):
    """A chain in which every kernel reads what the one before wrote, with and without programmatic dependent launches."""
    from hibana_b200.ops import gemm
    ew, x, rx, router, bias, sh = _case(5, 40, 256, "swiglu", fmt, 128, seed=6)
    ew, router, sh = ew.to("cuda"), router.cuda(), sh.cuda()
    g = torch.Generator().manual_seed(7)
    w = mxfp4.quantize_weight((torch.randn(256, 256, generator=g) * 0.06).cuda())

    def chain():
        h = x.cuda()
        for _ in range(12):
            y = moe.layer_forward(h, router, ew, 4, shared=sh)
            h = gemm.linear_mxfp4(mxfp4.quantize(y), w, epilogue=gemm.EPI_RESIDUAL, residual=h, static_weight=True)
            h = h / h.float().abs().amax().clamp_min(1e-6).bfloat16()
        return h

    gemm.set_pdl(0)
    try:
        plain = chain()
    finally:
        gemm.set_pdl(2)
    for _ in range(5):
        assert torch.equal(chain(), plain)
    assert not plain.isnan().any() and nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t", [100, 322])
@pytest.mark.parametrize("act", ["swiglu", "relu2"])
def test_grouped_mxfp4_experts_step_by_step_gpu(t, act):
    """One-CTA tiles and SM pairs against 64 bits from the codes of x on, mid rounded to bf16 and to MXFP4 as the path says."""
    e, k, h, inter = 8, 2, 512, 128
    ew = _experts(e, h, inter, act, "mxfp4", seed=1, h_out=256)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(t, h, generator=g).bfloat16()
    ids, w = moe.route(torch.randn(t, e, generator=g), k)
    got = moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ew.to("cuda")).double().cpu()
    want = torch.zeros_like(got)
    size = torch.zeros_like(got)
    xq = mxfp4.quantize(x).dequantize().double()
    for i in range(e):
        a = xq @ ew.dense(1)[i].double().t()
        mid = torch.relu(a) ** 2 if act == "relu2" else a[:, 0::2] * torch.sigmoid(a[:, 0::2]) * a[:, 1::2]
        y = mxfp4.quantize(mid.bfloat16()).dequantize().double() @ ew.dense(2)[i].double().t()
        for j in range(k):
            sel = ids[:, j] == i
            want[sel] += w[sel, j:j + 1].double() * y[sel]
            size[sel] += w[sel, j:j + 1].double() * y[sel].abs()
    # every expert's output and the sum are rounded to bf16: 2^-8 of each. Where a sum of fc1 lies within 2^-20 of a border between two
    # bf16 numbers and that border is one between two codes, an element of mid moves by up to a third: few rows (2^-12 of the numbers
    # are that near, 128 a row and expert: one row in sixteen), counted here, not bounded.
    off = (got - want).abs() <= 2.0 ** -8 * 1.01 * (size + want.abs()) + 1e-6
    assert off.all(dim=1).float().mean() >= 0.9 and nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,inter,act,fmt", [
    (1, 12, 12, 4640, 1664, "relu2", "nvfp4"),        # two rounds of fc1, the second sparse; more scales than tensor memory holds
    (1, 12, 12, 512, 1664, "relu2", "mxfp4"),
    (2, 20, 10, 256, 2560, "relu2", "bf16"),
    (1, 11, 11, 4640, 1664, "relu2", "nvfp4"),        # one round
    (4, 24, 12, 128, 896, "swiglu", "mxfp4"),         # three or four rounds
])
def test_rounds_of_the_first_product_gpu(t, e, k, h, inter, act, fmt):
    ew, x, rx, router, bias, sh = _case(t, e, h, act, fmt, inter, seed=8, h_out=128)
    got = moe.layer_forward(x.cuda(), router.cuda(), ew.to("cuda"), k, shared=sh.cuda())
    _check(got, *_exact(ew, x, rx, router, k, False, bias, 1.0, sh))
    assert nv.read_status() == 0
