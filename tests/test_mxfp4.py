"""MXFP4 quantiser, its inverse and the block-scaled product against plain 64-bit computations."""
import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200.ops import gemm, mxfp4

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def _exact_quant(x):
    """(values in 64 bits, scale bytes) of the format's definition, by search: x float64 [M, K] of finite numbers."""
    m, k = x.shape
    b = x.reshape(m, k // 32, 32)
    top = b.abs().amax(-1)
    e = torch.frexp(top).exponent - 1
    byte = torch.where(top > 0, e - 2 + 127, torch.zeros_like(e)).clamp_min(0)
    s = torch.ldexp(torch.ones_like(top), byte - 127)
    a = (b / s.unsqueeze(-1)).abs()
    dist = (a.unsqueeze(-1) - GRID).abs()
    # nearest, an exact tie to the even code: odd codes pay the smallest amount there is
    code = (dist * 2 + torch.tensor([0, 1, 0, 1, 0, 1, 0, 1]) * 1e-300).argmin(-1)
    tie = (dist.gather(-1, (code + 1).clamp_max(7).unsqueeze(-1)).squeeze(-1) == dist.gather(-1, code.unsqueeze(-1)).squeeze(-1))
    code = torch.where(tie & (code % 2 == 1) & (code < 7), code + 1, code)
    q = GRID[code] * torch.where(b < 0, -1.0, 1.0)
    return (q * s.unsqueeze(-1)).view(m, k), byte.to(torch.uint8)


def _rows(m, k, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-6, 7, (m, 1), generator=g).float())
    return x.to(dtype)


def _edge_rows(dtype):
    """Every boundary between codes and its neighbours, powers of two, zeros, the smallest and largest numbers."""
    vals = []
    for s in (2.0 ** -8, 1.0, 2.0 ** 5):
        for v in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.96875, 4.0, 0.0):
            vals += [4.0 * s, v * s, -v * s, v * s * (1 + 2 ** -7), v * s * (1 - 2 ** -8)] + [0.0] * 27
    tiny, huge = (2.0 ** -24, 60000.0) if dtype == torch.float16 else (2.0 ** -133, 3e38)
    for v in (tiny, 3 * tiny, huge, 0.0):
        vals += [v, -v / 2] + [v / 3] * 30
    return torch.tensor(vals, dtype=torch.float64).float().to(dtype).view(-1, 32 * 5) if len(vals) % 160 == 0 else \
        torch.tensor(vals, dtype=torch.float64).float().to(dtype).view(-1, 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_reference_follows_the_definition_cpu(dtype):
    for x in (_rows(7, 96, dtype=dtype), _edge_rows(dtype)):
        t = mxfp4.quantize(x)
        want, byte = _exact_quant(x.double())
        assert torch.equal(t.scales(), byte)
        assert torch.equal(mxfp4.dequantize(t, torch.float32).double(), want)


def test_non_finite_blocks_become_nan_cpu():
    x = torch.ones(3, 64)
    x[0, 3], x[1, 40], x[2, 63] = float("inf"), float("nan"), -float("inf")
    t = mxfp4.quantize(x)
    assert t.scales().tolist() == [[255, 125], [125, 255], [125, 255]]
    d = mxfp4.dequantize(t, torch.float32)
    assert torch.isnan(d[0, :32]).all() and torch.equal(d[0, 32:], torch.ones(32))
    assert torch.isnan(d[1, 32:]).all() and torch.equal(d[1, :32], torch.ones(32))


def test_blocks_of_a_checkpoint_cpu():
    g = torch.Generator().manual_seed(1)
    packed = torch.randint(0, 256, (130, 3, 16), generator=g, dtype=torch.uint8)
    scales = torch.randint(100, 140, (130, 3), generator=g, dtype=torch.uint8)
    t = mxfp4.from_blocks(packed, scales)
    assert (t.rows, t.k, t.ka) == (130, 96, 2) and torch.equal(t.scales(), scales)
    assert t.sf.shape == (2, 2, 512)
    low = packed.flatten(1).int() & 15
    want = GRID[low.long() & 7] * torch.where(low > 7, -1.0, 1.0) * torch.ldexp(torch.ones(130, 3).double(), scales.int() - 127
                                                                               ).repeat_interleave(16, 1)
    assert torch.equal(t.dequantize()[:, 0::2].double(), want)
    # a misaligned view is moved, not handed on
    flat = torch.zeros(130 * 48 + 1, dtype=torch.uint8)
    flat[1:] = packed.flatten()
    assert mxfp4.from_blocks(flat[1:].view(130, 48), scales).q.data_ptr() % 16 == 0


def test_refusals_cpu():
    for bad in (torch.zeros(2, 48), torch.zeros(2, 0), torch.zeros(64), torch.zeros(2, 64, dtype=torch.float64),
                torch.zeros(64, 4).t()):
        with pytest.raises(ValueError):
            mxfp4.quantize(bad)
    with pytest.raises(ValueError):
        mxfp4.from_blocks(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 3, dtype=torch.uint8))
    with pytest.raises(ValueError):
        mxfp4.from_blocks(torch.zeros(4, 32), torch.zeros(4, 2, dtype=torch.uint8))
    x, w = mxfp4.quantize(torch.ones(3, 64)), mxfp4.quantize(torch.ones(5, 64))
    with pytest.raises(ValueError):
        mxfp4.dequantize(x, torch.float64)
    for kw in ({"epilogue": gemm.EPI_SILU_MUL}, {"epilogue": gemm.EPI_RELU2}, {"residual": torch.zeros(3, 5).bfloat16()},
               {"epilogue": gemm.EPI_RESIDUAL}, {"epilogue": gemm.EPI_RESIDUAL, "residual": torch.zeros(3, 4).bfloat16()}):
        with pytest.raises(ValueError):
            gemm.linear_mxfp4(x, w, **kw)
    with pytest.raises(ValueError):
        gemm.linear_mxfp4(mxfp4.quantize(torch.ones(3, 96)), w)


def test_product_reference_cpu():
    x, w = mxfp4.quantize(_rows(5, 96)), mxfp4.quantize(_rows(6, 96, 1))
    acc = x.dequantize() @ w.dequantize().t()
    assert torch.equal(gemm.linear_mxfp4(x, w), acc.bfloat16())
    res = torch.randn(5, 6).bfloat16()
    assert torch.equal(gemm.linear_mxfp4(x, w, epilogue=gemm.EPI_RESIDUAL, residual=res), (acc + res.float()).bfloat16())


# ---- kernels


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 5120), (3, 96), (130, 160), (33, 1056), (257, 2688)])
def test_quantiser_gpu(dtype, m, k):
    x = _rows(m, k, dtype=dtype)
    t = mxfp4.quantize(x.cuda())
    want, byte = _exact_quant(x.double())
    assert torch.equal(t.scales().cpu(), byte)
    assert torch.equal(mxfp4.dequantize(t, torch.float32).cpu().double(), want)
    assert torch.equal(mxfp4.dequantize(t).cpu().double(), want)               # two significant bits: exact in bf16
    assert torch.equal(mxfp4.dequantize(t, torch.float16).cpu(), want.to(torch.float16))
    # groups that pad the last K tile hold a finite scale
    rb = t.sf.shape[0]
    full = t.sf.view(rb, t.ka, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, t.ka * 4)
    assert int(full[:m, k // 32:].sum()) == 0
    # rows of a wider buffer, aligned and not
    for lead in (8, 1):
        buf = torch.zeros(m, k + lead + 3, dtype=dtype, device="cuda")
        buf[:, lead:lead + k] = x.cuda()
        s = mxfp4.quantize(buf[:, lead:lead + k])
        assert torch.equal(s.q, t.q) and torch.equal(s.scales(), t.scales())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantiser_edges_gpu(dtype):
    x = _edge_rows(dtype)
    t = mxfp4.quantize(x.cuda())
    want, byte = _exact_quant(x.double())
    assert torch.equal(t.scales().cpu(), byte) and torch.equal(mxfp4.dequantize(t, torch.float32).cpu().double(), want)
    bad = torch.ones(3, 64, dtype=dtype)
    bad[0, 3], bad[1, 40], bad[2, 63] = float("inf"), float("nan"), -float("inf")
    t = mxfp4.quantize(bad.cuda())
    assert torch.equal(t.scales().cpu(), mxfp4.quantize(bad).scales())
    assert torch.equal(torch.isnan(mxfp4.dequantize(t)).cpu(), torch.isnan(mxfp4.dequantize(mxfp4.quantize(bad))))
    empty = mxfp4.quantize(torch.empty(0, 64, dtype=dtype, device="cuda"))
    assert mxfp4.dequantize(empty).shape == (0, 64)


@pytest.mark.gpu
def test_every_code_and_scale_gpu():
    packed = torch.arange(256, dtype=torch.uint8).repeat(256, 1)              # K = 512, every pair of codes
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 16)    # row r: scale byte r
    t = mxfp4.from_blocks(packed, scales)
    got = mxfp4.dequantize(t.to("cuda"), torch.float32).cpu()
    want = mxfp4.dequantize(t, torch.float32)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(1.0, 2.0, 3.0), want.nan_to_num(1.0, 2.0, 3.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantiser_into_a_sorted_buffer_gpu(dtype):
    x = _rows(3, 160).to(dtype).cuda()
    pos = torch.tensor([4, -1, 0, 130, 2, 11], dtype=torch.int32, device="cuda")
    plain = mxfp4.quantize(x)
    t = mxfp4.quantize_pairs(x, pos, 2, 131)
    for p, r in enumerate(pos.tolist()):
        assert r < 0 or (torch.equal(t.q[r], plain.q[p // 2]) and torch.equal(t.scales()[r], plain.scales()[p // 2]))
    wide = torch.zeros(131, 160, dtype=dtype, device="cuda")
    wide[[4, 0, 130, 2, 11]] = x[[0, 1, 1, 2, 2]]
    u = mxfp4.quantize_pairs(wide, pos, 0, 131)
    for r in (4, 0, 130, 2, 11):
        assert torch.equal(u.q[r], t.q[r]) and torch.equal(u.scales()[r], t.scales()[r])


def _product_case(m, n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = mxfp4.quantize(_rows(m, k, seed).cuda())
    packed = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    w = mxfp4.from_blocks(packed.cuda(), torch.randint(117, 123, (n, k // 32), generator=g, dtype=torch.uint8).cuda())
    xd, wd = x.dequantize().double(), w.dequantize().double()
    # products of two e2m1 numbers are exact; the sums round in 32 bits at most once per term, relative to what has been
    # added up in magnitude (2^-23: the tensor core may cut instead of rounding)
    acc, slack = xd @ wd.t(), (xd.abs() @ wd.abs().t()) * k * 2.0 ** -23
    return x, w, acc, slack


SHAPES = [(1, 16, 32), (1, 384, 288), (5, 130, 512), (17, 250, 1056), (64, 512, 2048), (100, 136, 640), (200, 384, 256),
          (256, 1040, 1312), (257, 264, 512), (300, 520, 288), (301, 100, 96), (513, 1024, 2688), (700, 77, 320)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_gpu(m, n, k):
    x, w, acc, slack = _product_case(m, n, k)
    half = torch.finfo(torch.bfloat16).eps / 2
    got = gemm.linear_mxfp4(x, w)
    assert ((got.double() - acc).abs() <= slack + half * (acc.abs() + slack)).all()
    assert torch.equal(gemm.linear_mxfp4(x, w), got)
    f32 = gemm.linear_mxfp4(x, w, epilogue=gemm.EPI_STORE_F32)
    assert f32.dtype == torch.float32 and ((f32.double() - acc).abs() <= slack).all()
    res = torch.randn(m, n, device="cuda").bfloat16()
    got = gemm.linear_mxfp4(x, w, epilogue=gemm.EPI_RESIDUAL, residual=res)
    want = acc + res.double()        # the product may be rounded to bf16 once before the sum is
    assert ((got.double() - want).abs() <= slack + half * (acc.abs() + slack) * (1 + half) + half * (want.abs() + slack)).all()
    wide = torch.full((m, n + 24), 7.0, dtype=torch.bfloat16, device="cuda")      # a view of a wider buffer as output
    gemm.linear_mxfp4(x, w, out=wide[:, 8:8 + n])
    assert torch.equal(wide[:, 8:8 + n], gemm.linear_mxfp4(x, w)) and (wide[:, :8] == 7).all() and (wide[:, 8 + n:] == 7).all()
    wide_res = torch.randn(m, n + 8, device="cuda").bfloat16()[:, :n]                # and a residual of another stride
    assert torch.equal(gemm.linear_mxfp4(x, w, epilogue=gemm.EPI_RESIDUAL, residual=wide_res),
                       gemm.linear_mxfp4(x, w, epilogue=gemm.EPI_RESIDUAL, residual=wide_res.contiguous()))
    if n % 2 == 0:
        g, u, sg, su = acc[:, 0::2], acc[:, 1::2], slack[:, 0::2], slack[:, 1::2]
        want = g * torch.sigmoid(g) * u
        # |silu'| <= 1.1; exponential, sum and quotient of the epilogue within 2^-20 of the value
        err = 1.1 * sg * (u.abs() + su) + (g.abs() + sg) * su + 2.0 ** -20 * (want.abs() + sg * su)
        got = gemm.linear_mxfp4(x, w, epilogue=gemm.EPI_SILU_MUL).double()
        assert got.shape == (m, n // 2) and ((got - want).abs() <= err + half * (want.abs() + err)).all()
    assert nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 300])
def test_product_nan_scales_stay_in_their_rows_gpu(m):
    x, w, acc, slack = _product_case(m, 264, 512, seed=3)
    sfx = x.scales()
    sfx[1, 3] = 255
    bad = mxfp4.from_blocks(x.q, sfx)
    got, clean = gemm.linear_mxfp4(bad, w), gemm.linear_mxfp4(x, w)
    assert torch.isnan(got[1]).all()
    keep = torch.arange(m, device="cuda") != 1
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.gpu
def test_product_in_a_graph_and_on_another_stream_gpu():
    rows = _rows(40, 512, 4).cuda()
    w = _product_case(1, 384, 512)[1]
    want = gemm.linear_mxfp4(mxfp4.quantize(rows), w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gemm.linear_mxfp4(mxfp4.quantize(rows), w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    static = torch.zeros_like(rows)
    gemm.linear_mxfp4(mxfp4.quantize(static), w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = gemm.linear_mxfp4(mxfp4.quantize(static), w)
    for seed in (5, 6):
        r = _rows(40, 512, seed).cuda()
        static.copy_(r)
        g.replay()
        assert torch.equal(out, gemm.linear_mxfp4(mxfp4.quantize(r), w))


def test_row_number_refusals_cpu():
    with pytest.raises(ValueError):                    # (expert-sorted buffers are the GPU's)
        mxfp4.quantize_pairs(torch.randn(4, 64).bfloat16(), torch.arange(4, dtype=torch.int32), 1, 4)


@pytest.mark.gpu
def test_row_number_refusals_gpu():
    x = torch.randn(4, 64, device="cuda").bfloat16()
    pos = torch.arange(8, dtype=torch.int32, device="cuda")
    for args in ((pos.long(), 2, 8), (pos.cpu(), 2, 8), (pos[::2], 1, 4), (pos, 1, 8), (pos, 3, 8), (pos, 0, 5), (pos, -1, 4), (pos, 2, -1)):
        with pytest.raises(ValueError):
            mxfp4.quantize_pairs(x, *args)
    assert mxfp4.quantize_pairs(x[:0], pos[:0], 2, 0).rows == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantiser_alignments_gpu(dtype):
    """Rows that start on 32-, 16- and 4- or 2-byte boundaries, at every length of the last piece of a row."""
    for k in (32, 480, 512, 992, 1024, 1056, 1568):
        base = _rows(6, k + 64, seed=k).to(dtype)
        for offset in (0, 1, 4, 8, 16):
            for pad in (0, 1, 4, 8, 16):
                view = torch.as_strided(base.cuda().flatten(), (5, k), (k + pad, 1), offset)
                want = mxfp4.quantize(torch.as_strided(base.flatten(), (5, k), (k + pad, 1), offset))
                got = mxfp4.quantize(view)
                assert torch.equal(got.q.cpu(), want.q) and torch.equal(got.scales().cpu(), want.scales()), (k, offset, pad)
                # blocks that pad the last K tile read as zero
                assert not mxfp4.unswizzle_sf(got.sf, 5, got.ka * 4)[:, k // 32:].any()


def test_row_numbers_are_bounded_in_the_kernel_cpu():
    """Row numbers live on the device, so the kernel itself keeps them inside the buffers, ahead of any use."""
    from pathlib import Path
    source = (Path(mxfp4.__file__).parent.parent / "csrc" / "mxfp4.cu").read_text()
    body = source[source.index("dst = dst_rows[row];"):]
    assert body.splitlines()[1].strip() == "if (static_cast<uint32_t>(dst) >= static_cast<uint32_t>(dst_count)) return;"


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 2])
def test_row_numbers_past_the_buffer_are_left_out_gpu(topk):
    x = _rows(6, 160).cuda()
    n = 6 * topk if topk else 7
    pos = torch.tensor([4, 6, -1, 2 ** 31 - 1, 1, -2 ** 31, 5, 7, 2 ** 20, 0, 128, 3][:n], dtype=torch.int32, device="cuda")
    plain = mxfp4.quantize(x)
    out = mxfp4.quantize_pairs(x, pos, topk, 6)
    for p, r in enumerate(pos.tolist()):
        src = p // topk if topk else r
        assert not 0 <= r < 6 or (torch.equal(out.q[r], plain.q[src]) and torch.equal(out.scales()[r], plain.scales()[src]))
