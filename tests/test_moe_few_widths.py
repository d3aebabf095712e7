"""Which widths and token counts take the few-token form: one rule for both devices, for `layer_forward` and for the models."""
import ctypes

import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200 import config as cfgmod
from hibana_b200.models.layers import Init, MoeLayer
from hibana_b200.ops import gemm, moe
from hibana_b200.target import flashnext, scaled
from test_moe_few import _case, _check, _exact


def test_the_rule_is_the_kernels_cpu():
    if not nv.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = ctypes.CDLL(str(nv.LIB_PATH))
    for fmt, kind in moe._KINDS.items():
        for hidden in range(8, 20000, 8):
            assert moe.few_tokens_limit(fmt, hidden) == lib.hb_moe_few_tokens(kind, hidden), (fmt, hidden)


def _wide(fmt, t, h, act="relu2", e=4, k=2):
    return _case(t, e, h, act, fmt, 128, h_out=128, std=0.02)


# width, tokens of one call, tokens of the layer that take it
LIMITS = [("mxfp4", 6144, 6, 12), ("nvfp4", 6144, 6, 12), ("nvfp4", 7168, 3, 6), ("mxfp4", 3584, 16, 16), ("bf16", 5120, 16, 16), ("bf16", 5504, 0, 0)]


@pytest.mark.parametrize("fmt,h,per_call,last", LIMITS)
def test_tokens_of_a_call_cpu(fmt, h, per_call, last):
    ew = moe.ExpertWeights(4, h, 128, "relu2", fmt, *(torch.empty(0),) * 2)
    ew.fc1 = ew.fc2 = type("W", (), {"rows": 512, "shape": (512, 0)})()
    for t in range(0, 20):
        want = 0 if t == 0 or t > last else min(t, per_call)
        assert moe.few_tokens_per_call(ew, 2, t) == want
        if want:
            assert -(-t // want) <= 2


@pytest.mark.parametrize("fmt,h,t", [("mxfp4", 6144, 13), ("bf16", 5504, 1), ("nvfp4", 12288, 1)])
def test_wider_layers_are_grouped_ones_cpu(fmt, h, t):
    ew, x, rx, router, bias, sh = _wide(fmt, t, h)
    ids, w = moe.route(x.float() @ router.float().t(), 2)
    assert moe.few_tokens_ok(ew, 2)
    assert torch.equal(moe.layer_forward(x, router, ew, 2, shared=sh), moe.experts_forward(x, ids, w, ew, shared=sh))


def test_models_ask_the_same_rule_cpu():
    t = scaled(flashnext(), hidden=6144, experts=4, top_k=2, expert_ffn=128, shared_ffn=128, weight_format="mxfp4")
    layer = MoeLayer(t, Init(0, "cpu", init_device="cpu"), "moe")
    assert layer._takes_few(12) and not layer._takes_few(13)      # (the grouped form has its own overlapped path)
    t = scaled(flashnext(), hidden=5504, experts=4, top_k=2, expert_ffn=128, shared_ffn=128, weight_format="bf16")
    layer = MoeLayer(t, Init(0, "cpu", init_device="cpu"), "moe")
    with cfgmod.using(moe_few=True):
        assert not layer._takes_few(1)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,h,t", [("mxfp4", 6144, 16), ("bf16", 5504, 3), ("nvfp4", 7168, 7), ("nvfp4", 12288, 1)])
def test_wider_layers_are_grouped_ones_gpu(fmt, h, t):
    ew, x, rx, router, bias, sh = _wide(fmt, t, h)
    ewg, xg, rg, sg = ew.to("cuda"), x.cuda(), router.cuda(), sh.cuda()
    ids, w = moe.route(gemm.linear_bf16(xg, rg, epilogue=gemm.EPI_STORE_F32), 2)
    assert torch.equal(moe.layer_forward(xg, rg, ewg, 2, shared=sg), moe.experts_forward(xg, ids, w, ewg, shared=sg))
    assert nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,h,t", [("mxfp4", 6144, 6), ("mxfp4", 6144, 12), ("nvfp4", 7168, 5), ("nvfp4", 4096, 16), ("bf16", 5120, 16), ("bf16", 5440, 4),
                                     ("mxfp4", 14336, 2)])
def test_wide_layers_in_one_and_two_calls_gpu(fmt, h, t):
    ew, x, rx, router, bias, sh = _wide(fmt, t, h)
    per_call = moe.few_tokens_per_call(ew, 2, t)
    assert per_call and per_call <= nv.lib().hb_moe_few_tokens(moe._KINDS[fmt], h)
    before = nv.LAUNCHES
    got = moe.layer_forward(x.cuda(), router.cuda(), ew.to("cuda"), 2, shared=sh.cuda())
    assert nv.LAUNCHES - before == 3 * -(-t // per_call)
    _check(got, *_exact(ew, x, None, router, 2, False, bias, 1.0, sh))
    assert nv.read_status() == 0
