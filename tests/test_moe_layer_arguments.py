"""`moe.layer_forward`: arguments as a caller may hold them, in the few-token and in the grouped form."""
import contextlib

import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200.ops import gemm, moe


def _experts(e, h, inter, act, fmt, h_out=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    n1 = 2 * inter if act == "swiglu" else inter
    return moe.ExpertWeights.create(torch.randn(e, n1, h, generator=g) * 0.05, torch.randn(e, h_out or h, inter, generator=g) * 0.05, act,
                                    fmt, in_amax=5.0, mid_amax=2.0)


def _odd(v, lead=3, pitch=7):
    """The same rows inside a wider buffer, off every boundary."""
    wide = torch.zeros(v.shape[0], lead + v.shape[1] + pitch, dtype=v.dtype, device=v.device)
    return wide[:, lead:lead + v.shape[1]].copy_(v)


def test_both_forms_hand_aligned_rows_to_the_kernels_cpu(monkeypatch):
    """What the kernels of the grouped form get, with the launches taken out: rows and pitches of 16 bytes, a router of whole
    pieces, a contiguous bias."""
    seen = {}

    def linear(x, w, **kw):
        seen["router"] = (x, w)
        return x.float() @ w.float().t()

    def experts(x, ids, w, ew, shared=None):
        seen["rows"] = (x, shared)
        return torch.zeros(x.shape[0], ew.fc2_rows)

    def route(logits, topk, sel_bias=None, **kw):
        seen["bias"] = sel_bias
        return moe.route_ref(logits, topk, sel_bias=sel_bias, **kw)
    monkeypatch.setattr(nv, "use_native", lambda *a: True)
    monkeypatch.setattr(nv, "on_device", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(gemm, "linear_bf16", linear)
    monkeypatch.setattr(moe, "route", route)
    monkeypatch.setattr(moe, "experts_forward", experts)
    ew = _experts(8, 64, 64, "swiglu", "bf16")
    x, rx, router = torch.randn(20, 64).bfloat16(), torch.randn(20, 37).bfloat16(), torch.randn(8, 37).bfloat16()
    bias = torch.randn(8, 5)[:, 2]
    moe.layer_forward(_odd(x), _odd(router), ew, 2, sigmoid=True, sel_bias=bias, shared=_odd(x), route_x=_odd(rx))
    for v in (*seen["router"], *seen["rows"]):
        assert v.data_ptr() % 16 == 0 and v.stride(1) == 1 and v.stride(0) % 8 == 0 and v.shape[1] % 8 == 0
    assert torch.equal(seen["router"][0].float() @ seen["router"][1].float().t(), rx.float() @ router.float().t())
    assert seen["bias"].is_contiguous() and torch.equal(seen["bias"], bias) and torch.equal(seen["rows"][0], x)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
@pytest.mark.parametrize("t", [5, 20, 140])
def test_strided_arguments_gpu(fmt, t):
    """Views off every boundary, an odd router width and a strided bias give the bits of plain tensors, in either form."""
    g = torch.Generator().manual_seed(t)
    ew = _experts(16, 256, 128, "swiglu", fmt).to("cuda")
    x, rx, shared = (torch.randn(t, n, generator=g).bfloat16().cuda() for n in (256, 99, 256))
    router = (torch.randn(16, 99, generator=g) * 0.3).bfloat16().cuda()
    table = torch.randn(16, 5, generator=g).cuda()
    bias = table[:, 2]
    want = moe.layer_forward(x, torch.nn.functional.pad(router, (0, 5)), ew, 3, sigmoid=True, sel_bias=bias.clone(), shared=shared,
                             route_x=torch.nn.functional.pad(rx, (0, 5)))
    got = moe.layer_forward(_odd(x), _odd(router), ew, 3, sigmoid=True, sel_bias=bias, shared=_odd(shared), route_x=_odd(rx))
    assert torch.equal(got, want) and nv.read_status() == 0
    # columns of a transposed buffer
    got = moe.layer_forward(x.t().contiguous().t(), router.t().contiguous().t(), ew, 3, sigmoid=True, sel_bias=bias,
                            shared=shared.t().contiguous().t(), route_x=rx.t().contiguous().t())
    assert torch.equal(got, want) and nv.read_status() == 0


# format, act, hidden, inter, output columns
UNTILED = [("mxfp4", "swiglu", 128, 96, 128), ("mxfp4", "relu2", 128, 128, 64), ("nvfp4", "relu2", 128, 192, 128), ("nvfp4", "swiglu", 144, 64, 128),
           ("bf16", "swiglu", 48, 24, 48)]


@pytest.mark.parametrize("fmt,act,h,inter,h_out", UNTILED)
def test_geometries_the_grouped_products_do_not_tile_cpu(fmt, act, h, inter, h_out):
    with pytest.raises(ValueError, match="multiples of 128"):
        moe.check_grouped(_experts(4, h, inter, act, fmt, h_out=h_out))
    for ok in ("mxfp4", "nvfp4", "bf16", "w3"):
        moe.check_grouped(_experts(4, 128, 128, act, ok))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,act,h,inter,h_out", UNTILED)
def test_untiled_geometries_are_refused_gpu(fmt, act, h, inter, h_out):
    ew = _experts(4, h, inter, act, fmt, h_out=h_out).to("cuda")
    x, router = torch.randn(20, h).bfloat16().cuda(), torch.randn(4, h).bfloat16().cuda()
    for t in (3, 20):
        if moe.few_tokens_per_call(ew, 2, t):          # (bf16 rows of any multiple of eight run in the few-token form)
            assert torch.isfinite(moe.layer_forward(x[:t], router, ew, 2).float()).all()
            continue
        with pytest.raises(ValueError, match="multiples of 128"):
            moe.layer_forward(x[:t], router, ew, 2)
    assert nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 16, 40])
def test_three_bit_layers_are_grouped_ones_gpu(t):
    g = torch.Generator().manual_seed(t)
    ew = _experts(8, 256, 128, "swiglu", "w3").to("cuda")
    x, router, shared = (torch.randn(n, 256, generator=g).bfloat16().cuda() for n in (t, 8, t))
    assert not moe.few_tokens_per_call(ew, 2, t)
    ids, w = moe.route(gemm.linear_bf16(x, router, epilogue=gemm.EPI_STORE_F32), 2)
    assert torch.equal(moe.layer_forward(x, router, ew, 2, shared=shared), moe.experts_forward(x, ids, w, ew, shared=shared))
    assert nv.read_status() == 0


def test_scales_of_nvfp4_experts_are_one_each_cpu():
    """The kernels read a scale at every chosen expert's number: fewer of them are refused, not read past."""
    import dataclasses
    x, router = torch.randn(3, 128).bfloat16(), torch.randn(4, 128).bfloat16()
    for which in ("fc1", "fc2"):
        ew = _experts(4, 128, 128, "relu2", "nvfp4")
        moe.layer_forward(x, router, ew, 2)
        w = getattr(ew, which)
        for scales in (w.gscale[:1], w.gscale[0], w.gscale[:3]):
            setattr(ew, which, dataclasses.replace(w, gscale=scales))
            with pytest.raises(ValueError, match="one scale each"):
                moe.layer_forward(x, router, ew, 2)
