"""CTAs of the few-token layer leave with nothing in flight: what the source says, and calls in which most CTAs have no work."""
import re
from pathlib import Path

import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200.ops import gemm, moe

SOURCE = (Path(moe.__file__).parent.parent / "csrc" / "moe_few.cu").read_text()


def test_resident_scales_are_copied_only_where_a_unit_waits_for_them_cpu():
    """The copies of B's scales into tensor memory are waited for by the last accumulator's commit, so only a CTA with a unit may issue
    them."""
    guard = re.search(r"if \(([^\n]*)\) \{\n(?:[^\n]*\n){1,4}?\s*tc_commit\(sfb_full\);", SOURCE).group(1)
    assert "u0 < units" in guard and "elect_one()" in guard


def test_a_wait_that_gave_up_anywhere_drains_every_copy_cpu():
    """Any warp can raise the abort flag, so what drains the copies asks for it behind a barrier, does not depend on how the
    loader's own waits ended, and has the rest of the CTA wait for it."""
    tail = SOURCE[SOURCE.index("} else if (SECOND && warp >= 12)"):SOURCE.index("tmem_dealloc(tmem, TMEM_COLS)")]
    assert SOURCE.count("kTimeoutDrain") == tail.count("kTimeoutDrain") == 2            # x's rows and the ring's tiles, in one place
    before, drain = tail.split("if (*abort) {")
    assert before.rstrip().splitlines()[-1].strip() == "__syncthreads();"
    assert drain.index("mbar_wait(x_full") < drain.index("__syncthreads();") and drain.index("mbar_wait(&full[") < drain.index("__syncthreads();")


def _layer(e, h, inter, act, fmt, seed):
    g = torch.Generator().manual_seed(seed)
    n1 = 2 * inter if act == "swiglu" else inter
    ew = moe.ExpertWeights.create(torch.randn(e, n1, h, generator=g) * 0.05, torch.randn(e, h, inter, generator=g) * 0.05, act, fmt)
    return ew.to("cuda"), (torch.randn(e, h, generator=g) * 0.2).bfloat16().cuda(), torch.randn(2, h, generator=g).bfloat16().cuda()


@pytest.mark.gpu
def test_calls_with_fewer_units_than_ctas_gpu():
    """One token and one or two experts: one to four units on 148 CTAs, clusters with more CTAs than entries. Calls of all formats in
    turn, each behind products that use the same tensor memory, give the same bits every time."""
    layers = [_layer(4, 256, 128, "swiglu", fmt, i) for i, fmt in enumerate(("mxfp4", "nvfp4", "bf16"))]
    layers += [_layer(2, 512, 128, "relu2", fmt, i + 3) for i, fmt in enumerate(("mxfp4", "nvfp4"))]
    big = torch.randn(512, 1024, device="cuda").bfloat16()
    first, square = None, None
    for _ in range(40):
        out = []
        for ew, router, x in layers:
            for rows, k in ((1, 1), (1, 2), (2, 1)):
                out.append(moe.layer_forward(x[:rows], router, ew, k))
        y = gemm.linear_bf16(big, big)
        if first is None:
            first, square = out, y
        assert all(torch.equal(a, b) for a, b in zip(out, first)) and torch.equal(y, square)
    assert nv.read_status() == 0
