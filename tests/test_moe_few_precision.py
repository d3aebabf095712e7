"""What the few-token layer keeps of its activations where a few of them are loud."""
import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200.ops import moe
from test_moe_few import _check, _exact


def _loud(fmt, act, peak, e=6, h=256, inter=384, seed=0):
    """Experts whose inner activation has one loud element, which half of the outputs do not weigh. In that element the second matrix
    holds zeros or ones, both of which every format has."""
    g = torch.Generator().manual_seed(seed)
    n1 = 2 * inter if act == "swiglu" else inter
    fc1 = torch.randn(e, n1, h, generator=g) * 0.05
    fc2 = torch.randn(e, h, inter, generator=g) * 0.05
    rows = slice(14, 16) if act == "swiglu" else slice(7, 8)
    fc1[:, rows] = fc1[:, rows].abs() * peak ** 0.5       # x > 0 below: both factors are large and positive
    fc2[:, :, 7] = torch.zeros(h)
    fc2[:, h // 2:, 7] = 1.0
    x = torch.rand(5, h, generator=g).bfloat16()
    router = (torch.randn(e, h, generator=g) * 0.1).bfloat16()
    return moe.ExpertWeights.create(fc1, fc2, act, fmt), x, router


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
@pytest.mark.parametrize("act", ["swiglu", "relu2"])
def test_the_case_is_what_it_says_cpu(fmt, act):
    ew, x, router = _loud(fmt, act, 1000.0)
    w1, w2 = ew.dense(1).double(), ew.dense(2).double()
    mid = moe._act(x.double() @ w1[0].t(), act)
    assert (w2[:, :128, 7] == 0).all() and (w2[:, 128:, 7] > 0.5).all()
    assert (mid.argmax(-1) == 7).all() and (mid[:, 7] > 100 * mid.abs().mean(-1)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
@pytest.mark.parametrize("act", ["swiglu", "relu2"])
@pytest.mark.parametrize("peak", [1.0, 1e3, 1e5])
def test_loud_inner_activations_gpu(fmt, act, peak):
    ew, x, router = _loud(fmt, act, peak)
    got = moe.layer_forward(x.cuda(), router.cuda(), ew.to("cuda"), 3)
    want, err = _exact(ew, x, None, router, 3, False, torch.zeros(6), 1.0, None)
    _check(got, want, err)                                # (counted from each row's largest number)
    if fmt == "bf16":
        # 16 bits of every number itself: outputs that do not weigh the loud one do not see it. 2^-17 of each of the terms (mid),
        # sums of 256 terms in 32 bits (2^-23 of what is added up in magnitude) in front of an activation that passes on at most three
        # times that, sums of 384 behind it, exponentials and quotients within 2^-18, and the weights, which a shift of the logits
        # by their sums' error moves by twice as much; then the rounding to bf16.
        w1, w2 = ew.dense(1).double(), ew.dense(2).double()
        lg = torch.softmax(x.double() @ router.double().t(), -1)
        w, ids = lg.sort(dim=-1, descending=True, stable=True)
        w, ids = w[:, :3] / w[:, :3].sum(-1, keepdim=True), ids[:, :3]
        size = torch.zeros(5, 128, dtype=torch.float64)
        for t in range(5):
            for j in range(3):
                a1 = w1[ids[t, j]].abs() @ x[t].double()            # magnitudes of fc1's sums
                mag = a1[0::2] * a1[1::2] if act == "swiglu" else a1 ** 2
                mag[7] = 0
                size[t] += w[t, j] * (w2[ids[t, j], :128].abs() @ mag)
        logit = 256 * 2.0 ** -23 * float((x.double().abs() @ router.double().abs().t()).max())
        slack = size * (2.0 ** -17 + (3 * 256 + 384) * 2.0 ** -23 + 3 * 2.0 ** -18 + 2 * logit)
        half = torch.finfo(torch.bfloat16).eps / 2
        assert ((got[:, :128].double().cpu() - want[:, :128]).abs() <= slack + half * (want[:, :128].abs() + slack)).all()
    assert nv.read_status() == 0
