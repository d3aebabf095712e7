"""The few-token layer reads all it is given behind its wait for the kernels in front: `layer_forward` promises nothing about a router,
an expert scale or a bias being written long ago."""
from pathlib import Path

import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200.ops import basic, gemm, moe

SOURCE = (Path(moe.__file__).parent.parent / "csrc" / "moe_few.cu").read_text()


def test_no_read_only_loads_cpu():
    """Read-only loads may be moved ahead of the wait, and may not be used at all on what a kernel writes that still runs at this
    one's start."""
    for read_only in ("__ldg", "ld.global.nc", "__restrict__"):
        assert read_only not in SOURCE


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
def test_a_router_written_just_before_gpu(fmt):
    """Router rows, x and the shared rows come from kernels of this library launched directly in front, new ones every time, in buffers
    that are used again; bits as with everything written long ago."""
    e, h, inter, k = 64, 512, 128, 4
    g = torch.Generator().manual_seed(1)
    ew = moe.ExpertWeights.create(torch.randn(e, 2 * inter, h, generator=g) * 0.05, torch.randn(e, h, inter, generator=g) * 0.05,
                                  "swiglu", fmt).to("cuda")
    zero = torch.zeros(e, h).bfloat16().cuda()
    routers = [(torch.randn(e, h, generator=g) * 0.2).bfloat16().cuda() for _ in range(6)]
    rows = [torch.randn(5, h, generator=g).bfloat16().cuda() for _ in range(6)]
    want = [moe.layer_forward(x, r, ew, k, shared=x) for x, r in zip(rows, routers)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for x, r in zip(rows, routers):
            router = basic.add(r, zero)                  # (freed behind each call: the next one's lies in the same place)
            got.append(moe.layer_forward(x, router, ew, k, shared=x))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # x straight from a product of products
    a = moe.layer_forward(gemm.linear_bf16(rows[0], gemm.linear_bf16(routers[1].t().contiguous(), routers[2].t().contiguous())),
                          routers[0], ew, k)
    torch.cuda.synchronize()
    mixed = gemm.linear_bf16(routers[1].t().contiguous(), routers[2].t().contiguous())
    x = gemm.linear_bf16(rows[0], mixed)
    torch.cuda.synchronize()
    assert torch.equal(a, moe.layer_forward(x, routers[0], ew, k)) and nv.read_status() == 0
