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
