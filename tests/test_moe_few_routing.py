"""Routing of the few-token layer at its edges (NaN and infinite logits), and what a token's neighbours may change."""
import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200.ops import moe
from test_moe_few import _case, _check, _exact


def test_nan_logits_spoil_their_token_cpu():
    ids, w = moe.route(torch.tensor([[0.5, float("nan"), 2.0, float("nan")], [0.0, 3.0, 1.0, 2.0]]), 3)
    assert ids[1].tolist() == [1, 3, 2] and w[0].isnan().all() and not w[1].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("sig", [False, True])
@pytest.mark.parametrize("e", [8, 40, 200, 600])      # the first 64 candidates rank themselves; beyond, ties are found one by one
@pytest.mark.parametrize("fmt", ["mxfp4", "bf16"])
def test_a_nan_logit_spoils_its_token_only_gpu(fmt, e, sig):
    ew, x, rx, router, bias, sh = _case(5, e, 128, "swiglu", fmt, 64, seed=e)
    kw = dict(sigmoid=sig, sel_bias=bias.cuda() if sig else None, shared=sh.cuda())
    ewg = ew.to("cuda")
    clean = moe.layer_forward(x.cuda(), router.cuda(), ewg, 4, route_x=x.cuda(), **kw)
    bad = x.clone()
    bad[3, 17] = float("nan")                             # every logit of token 3
    got = moe.layer_forward(x.cuda(), router.cuda(), ewg, 4, route_x=bad.cuda(), **kw)
    keep = [0, 1, 2, 4]
    assert got[3].isnan().all() and not clean.isnan().any()
    want, err = _exact(ew, x, None, router, 4, sig, bias, 1.0, sh)
    _check(got[keep], want[keep], err[keep])
    router[e - 1, 5] = float("nan")                       # one logit of every token: that expert comes first
    got = moe.layer_forward(x.cuda(), router.cuda(), ewg, 4, **kw)
    assert got.isnan().all() and nv.read_status() == 0


@pytest.mark.gpu
def test_infinite_logits_of_sigmoid_scores_gpu():
    """Sums past the largest float: scores of exactly one and zero, in the order of the bias."""
    ew, x, rx, router, bias, sh = _case(3, 33, 128, "relu2", "mxfp4", 128)
    x = x.abs() + 0.5
    router[:] = 0
    router[4:7] = 3e38
    router[7:20] = -3e38
    got = moe.layer_forward(x.cuda(), router.cuda(), ew.to("cuda"), 6, sigmoid=True, sel_bias=bias.cuda(), shared=sh.cuda())
    _check(got, *_exact(ew, x, None, router, 6, True, bias, 1.0, sh))
    assert nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
@pytest.mark.parametrize("k", [2, 7])
def test_neighbours_change_the_order_of_sums_at_most_gpu(fmt, k):
    """A token's experts are added up in an order that its neighbours take part in. Where they are routed alike the bits are the same;
    elsewhere only the sum over its experts differs: one rounding in 32 bits for each of them and of the cluster's CTAs, then one to bf16
    on each side."""
    ew, x, rx, router, bias, sh = _case(16, 12, 256, "swiglu", fmt, 128, seed=3, shared=False)
    ewg, r, xg = ew.to("cuda"), router.cuda(), x.cuda()
    whole = moe.layer_forward(xg, r, ewg, k).double().cpu()
    alone = torch.cat([moe.layer_forward(xg[i:i + 1], r, ewg, k) for i in range(16)]).double().cpu()
    score = torch.softmax(x.double() @ router.double().t(), -1)
    w, ids = score.sort(dim=-1, descending=True, stable=True)
    w, w1, w2 = w[:, :k] / w[:, :k].sum(-1, keepdim=True), ew.dense(1).double(), ew.dense(2).double()
    size = torch.zeros(16, 256, dtype=torch.float64)
    for t in range(16):
        for j in range(k):
            size[t] += w[t, j] * (w2[ids[t, j]] @ moe._act(w1[ids[t, j]] @ x[t].double(), "swiglu")).abs()
    slack = 1.1 * (k + 16) * 2.0 ** -23 * size            # (a tenth: the kernels' own terms stand a little off these)
    half = torch.finfo(torch.bfloat16).eps / 2
    assert ((whole - alone).abs() <= slack + half * (whole.abs() + alone.abs())).all()
    same = torch.zeros_like(router).cuda()                # every token takes experts 0 .. k - 1, in one entry each
    whole = moe.layer_forward(xg[:8], same, ewg, k)
    assert all(torch.equal(moe.layer_forward(xg[i:i + 1], same, ewg, k), whole[i:i + 1]) for i in range(8))
    assert nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("sig", [False, True])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("t,e", [(3, 8), (3, 200), (300, 200), (3, 600)])      # both routing kernels
def test_route_orders_nan_as_the_plain_form_gpu(t, e, sig, renorm):
    """One NaN logit, a row of them, NaN with either sign: ids and weights of the plain form."""
    lg = torch.randn(t, e, generator=torch.Generator().manual_seed(e))
    lg[0, 5] = float("nan")
    lg[1] = float("nan")
    lg.view(torch.int32)[2, 3] = -1
    ids, w = moe.route(lg.cuda(), 6, sigmoid=sig, renorm=renorm)
    ids_ref, w_ref = moe.route_ref(lg, 6, sigmoid=sig, renorm=renorm)
    assert torch.equal(ids.cpu(), ids_ref) and torch.equal(w.cpu().isnan(), w_ref.isnan())
    # exponential, sum of up to 600 of them, quotients
    ok = ~w_ref.isnan()
    assert ((w.cpu() - w_ref).abs()[ok] <= 2.0 ** -14 * w_ref[ok]).all()
