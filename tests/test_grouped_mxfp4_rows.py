"""Grouped MXFP4 experts, every row of them: from the codes of x on, with what 32-bit sums may do to the codes of the inner activations."""
import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200.ops import moe, mxfp4


def _quantised(v):
    """float64 rows rounded to bf16 and to MXFP4, and their blocks' scales."""
    q = mxfp4.quantize(v.bfloat16())
    return q.dequantize().double(), q.scales()


def _bounds(ew, xq, act):
    """Of every expert: (mid as the path quantises it, how far an element of it may be off), [E, T, inter], and whether a block of a row may
    take either of two scales, [E, T]. The first product's sums
    are exact products added in 32 bits (2^-23 a term of what is added up in magnitude); the activation's exponential and quotient stay
    within 2^-18. An element next to a border between two codes may fall on either side of it."""
    mids, offs, either_of = [], [], []
    for i in range(ew.experts):
        w1 = ew.dense(1)[i].double()
        a, s = xq @ w1.t(), (xq.abs() @ w1.abs().t()) * (xq.shape[1] * 2.0 ** -23)
        if act == "swiglu":
            g, u, sg, su = a[:, 0::2], a[:, 1::2], s[:, 0::2], s[:, 1::2]
            mid, d = g * torch.sigmoid(g) * u, 1.1 * sg * (u.abs() + su) + (g.abs() + sg) * su
        else:
            mid, d = torch.relu(a) ** 2, 2 * a.abs() * s + s ** 2
        d = d + 2.0 ** -18 * mid.abs()
        (at, sc), (lo, sl), (hi, sh) = _quantised(mid), _quantised(mid - d), _quantised(mid + d)
        # blocks whose scale may fall on either side as well: no number moves by more than half of what it is or, below the codes'
        # smallest step, a quarter of the scale's unit
        top = torch.maximum((mid.abs() + d).view(*mid.shape[:1], -1, 32).amax(-1), torch.zeros(()))
        either = (_quantised((mid.abs() + d))[1] != _quantised((mid.abs() - d).clamp_min(0))[1]).repeat_interleave(32, 1)
        off = torch.maximum((hi - at).abs(), (lo - at).abs())
        off = torch.where(either, 0.5 * (mid.abs() + d) + 0.25 * top.repeat_interleave(32, 1), off)
        mids.append(at)
        offs.append(off)
        either_of.append(either.any(1))
    return torch.stack(mids), torch.stack(offs), torch.stack(either_of)


def _case(t, act, e=8, k=2, h=512, inter=128):
    g = torch.Generator().manual_seed(1)
    n1 = 2 * inter if act == "swiglu" else inter
    ew = moe.ExpertWeights.create(torch.randn(e, n1, h, generator=g) * 0.05, torch.randn(e, 256, inter, generator=g) * 0.05, act, "mxfp4")
    x = torch.randn(t, h, generator=g).bfloat16()
    ids, w = moe.route(torch.randn(t, e, generator=g), k)
    xq = mxfp4.quantize(x).dequantize().double()
    mid, off, either = _bounds(ew, xq, act)
    want, allowed = (torch.zeros(t, 256, dtype=torch.float64) for _ in range(2))
    half = torch.finfo(torch.bfloat16).eps / 2
    for i in range(e):
        w2 = ew.dense(2)[i].double()
        y = mid[i] @ w2.t()
        dy = off[i] @ w2.abs().t() + (mid[i].abs() @ w2.abs().t()) * (inter * 2.0 ** -23)
        dy = dy + half * (y.abs() + dy)                   # an expert's output is rounded to bf16
        for j in range(k):
            sel = ids[:, j] == i
            want[sel] += w[sel, j:j + 1].double() * y[sel]
            allowed[sel] += w[sel, j:j + 1].double() * dy[sel]
    allowed = allowed + k * 2.0 ** -23 * (want.abs() + allowed)
    allowed = allowed + half * (want.abs() + allowed)     # and their sum
    return ew, x, ids, w, want, allowed, either.gather(0, ids.t().long()).any(0)


@pytest.mark.parametrize("act", ["swiglu", "relu2"])
def test_the_bound_is_a_narrow_one_cpu(act):
    """The plain form keeps it, and a row that lacks one of its two experts, off by some 0.7 of its norm, does not: half of that is allowed
    at most, but for the few rows with a block that may take either of two scales."""
    ew, x, ids, w, want, allowed, either = _case(100, act)
    got = moe.experts_forward(x, ids, w, ew).double()
    assert ((got - want).abs() <= allowed).all()
    share = allowed.norm(dim=1) / want.norm(dim=1)
    assert (share[~either] < 0.35).all() and float(either.double().mean()) < 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("t", [17, 100, 128, 129, 322])
@pytest.mark.parametrize("act", ["swiglu", "relu2"])
def test_every_row_gpu(t, act):
    """One-CTA tiles (up to 128 tokens) and SM pairs."""
    ew, x, ids, w, want, allowed, _ = _case(t, act)
    got = moe.experts_forward(x.cuda(), ids.cuda(), w.cuda(), ew.to("cuda")).double().cpu()
    off = (got - want).abs() - allowed
    assert (off <= 0).all(), (float(off.max()), float(want.abs().max()))
    assert nv.read_status() == 0
