"""MXFP4 weights in the layers and models: linears, shards, checkpoints, decoders; the few-token layer inside `MoeLayer`."""
import dataclasses

import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200 import config as cfgmod
from hibana_b200.engine.executor import Executor
from hibana_b200.engine.request import SamplingParams
from hibana_b200.models.dense import DenseModel
from hibana_b200.models.hybrid import HybridModel
from hibana_b200.models.layers import Init, MoeLayer
from hibana_b200.models.linear import Linear, norm_linear
from hibana_b200.ops import gemm, moe, mxfp4, nvfp4
from hibana_b200.target import dense_tiny, flashnext, nemotron, scaled, tiny_hybrid_moe
from hibana_b200.weights import checkpoint, modelopt, snapshot
from hibana_b200.weights import nemotron_layout as nl


def _prompts(vocab, n=3, length=20, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (length,), generator=g).tolist() for _ in range(n)]


def _tokens(model, prompts, n=6, **kw):
    ex = Executor(model, max_batch=4, max_ctx=128, use_graphs=kw.get("use_graphs", False))
    if kw.get("use_graphs"):
        ex.capture_graphs()
    return [r.output_ids for r in ex.generate_batch(prompts, SamplingParams(max_tokens=n))]


def _moe_target(fmt, latent=False, act="swiglu"):
    return scaled(nemotron() if latent else flashnext(), hidden=256, experts=16, top_k=4, expert_ffn=128, shared_ffn=128,
                  weight_format=fmt, moe_act=act, **({"latent": 128} if latent else {}))


def _layer(fmt, device="cpu", **kw):
    t = _moe_target(fmt, **kw)
    return t, MoeLayer(t, Init(0, device, init_device="cpu"), "moe")


# ---- linears
def test_linear_follows_its_parts_cpu():
    g = torch.Generator().manual_seed(0)
    w, x = torch.randn(96, 64, generator=g) * 0.1, torch.randn(5, 64, generator=g).bfloat16()
    res = torch.randn(5, 96, generator=g).bfloat16()
    lin = Linear(w, "mxfp4", name="l")
    ref = mxfp4.quantize(x).dequantize() @ mxfp4.quantize(w).dequantize().t()
    assert torch.equal(lin(x), ref.bfloat16())
    assert torch.equal(lin(x, epilogue=gemm.EPI_RESIDUAL, residual=res), (ref + res.float()).bfloat16())
    assert lin(x, epilogue=gemm.EPI_SILU_MUL).shape == (5, 48)
    assert torch.equal(lin.dequantized(), mxfp4.quantize(w).dequantize()) and lin.nbytes() < w.numel()
    q = lin(x, requant=torch.tensor([0.01]))
    assert isinstance(q, nvfp4.Nvfp4Tensor) and q.k == 96
    y = norm_linear(x, x.clone(), torch.ones(64).bfloat16(), 1e-6, lin)
    assert y.shape == (5, 96) and not lin.takes_gemv(1)
    with pytest.raises(ValueError):
        Linear(w[:, :40], "mxfp4")


def test_shards_are_slices_cpu():
    g = torch.Generator().manual_seed(1)
    w = torch.randn(160, 320, generator=g)
    full = Linear(w, "mxfp4").dequantized()
    assert torch.equal(Linear.sharded(w, "mxfp4", rows=slice(32, 97)).dequantized(), full[32:97])
    assert torch.equal(Linear.sharded(w, "mxfp4", cols=slice(96, 224)).dequantized(), full[:, 96:224])
    sel = torch.tensor([5, 1, 150, 151])
    assert torch.equal(Linear.sharded(w, "mxfp4", rows=sel).dequantized(), full[sel])
    with pytest.raises(ValueError):
        Linear.sharded(w, "mxfp4", cols=slice(16, 64))


def test_tensor_parallel_shards_cpu():
    t = scaled(dense_tiny(), weight_format="mxfp4")
    full = DenseModel(t, "cpu", seed=0)
    shards = [DenseModel.sharded(t, 2, r, "cpu", seed=0) for r in range(2)]
    assert torch.equal(torch.cat([s.layers[0].o.dequantized() for s in shards], 1), full.layers[0].o.dequantized())
    assert torch.equal(torch.cat([s.layers[1].gate_up.dequantized() for s in shards], 0), full.layers[1].gate_up.dequantized())


# ---- checkpoints
@pytest.mark.parametrize("hf", [False, True])
def test_checkpoint_round_trip_cpu(tmp_path, hf):
    t = scaled(dense_tiny(), weight_format="mxfp4")
    model = DenseModel(t, "cpu", seed=0)
    checkpoint.save_dense(model, str(tmp_path), layers_per_file=1, hf_layout=hf)
    loaded = checkpoint.load_dense(t, str(tmp_path))
    for a, b in zip(model.linears(), loaded.linears()):
        assert b.fmt == "mxfp4" and torch.equal(a.wq.q, b.wq.q) and torch.equal(a.wq.scales(), b.wq.scales())
    ref, shard = DenseModel.sharded(t, 2, 1, "cpu", seed=0), checkpoint.load_dense(t, str(tmp_path), tp=2, rank=1)
    for a, b in zip(ref.linears(), shard.linears()):
        assert torch.equal(a.wq.q, b.wq.q) and torch.equal(a.wq.scales(), b.wq.scales())
    prompts = _prompts(t.vocab, 2)
    assert _tokens(model, prompts, 4) == _tokens(loaded, prompts, 4)


def test_checkpoint_refusals_cpu():
    w = mxfp4.quantize(torch.randn(8, 64))
    tensors = {"a.weight": w.q, "a.weight_scale": w.scales(), "b.weight": w.q[:4], "b.weight_scale": w.scales()[:4]}
    assert modelopt.is_mxfp4(tensors, "a") and modelopt.load_mxfp4(tensors, ["a", "b"]).rows == 12
    with pytest.raises(ValueError):
        modelopt.load_mxfp4(tensors, ["a", "b"], interleave=True)
    with pytest.raises(ValueError):
        modelopt.load_mxfp4(tensors, ["a"], cols=slice(0, 16))


def test_nemotron_layout_round_trip_cpu(tmp_path):
    base = nemotron()
    t = scaled(base, hidden=256, vocab=512, q_heads=4, kv_heads=2, head_dim=64, mamba_heads=8, mamba_head_dim=32,
               mamba_state=64, mamba_groups=2, experts=8, top_k=3, expert_ffn=128, shared_ffn=128, latent=128,
               weight_format="mxfp4", kv_dtype="bf16", mtp_layers=0, max_context=512)
    t = dataclasses.replace(t, layers=base.layers[:9])
    model = HybridModel(t, "cpu", seed=3)
    other = nl.load(t, nl.save(model, tmp_path / "ckpt", blocks_per_file=4), "cpu", seed=99)
    a, b = nl.tensors_of(model), nl.tensors_of(other)
    assert a.keys() == b.keys() and all(torch.equal(a[k], b[k]) for k in a)
    prompts = _prompts(t.vocab, 2, 24)
    assert _tokens(model, prompts, 4) == _tokens(other, prompts, 4)


def test_snapshot_round_trip_cpu(tmp_path):
    t = scaled(tiny_hybrid_moe(), weight_format="mxfp4", expert_ffn=128)
    model, other = HybridModel(t, "cpu", seed=0), HybridModel(t, "cpu", seed=9)
    snapshot.save_state(model, str(tmp_path))
    snapshot.load_state(other, str(tmp_path))
    prompts = _prompts(t.vocab, 2)
    assert _tokens(model, prompts, 4) == _tokens(other, prompts, 4)


# ---- the few-token form inside MoeLayer
def test_which_calls_take_the_few_token_form_cpu():
    _, mx = _layer("mxfp4")
    _, nvf = _layer("nvfp4")
    assert mx._takes_few(1) and mx._takes_few(moe.FEW_TOKENS) and not mx._takes_few(moe.FEW_TOKENS + 1) and not mx._takes_few(0)
    assert not nvf._takes_few(4)                       # what ran before stays on its path
    with cfgmod.using(moe_few=True):
        assert nvf._takes_few(4)
    for off in ({"stable_numerics": True}, {"expert_budget": 8}):
        with cfgmod.using(**off):
            assert not mx._takes_few(4)
    mx.attach_w3()
    assert not mx._takes_few(4)                        # the 3-bit decode copy is what was asked for


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("fmt", ["bf16", "nvfp4", "mxfp4"])
def test_few_token_layer_agrees_with_the_grouped_one_cpu(fmt, latent):
    t, layer = _layer(fmt, latent=latent, act="relu2" if latent else "swiglu")
    x = torch.randn(4, t.hidden, generator=torch.Generator().manual_seed(2)).bfloat16()
    with cfgmod.using(moe_few=True):
        few = layer.forward(x).float()
    with cfgmod.using(stable_numerics=True):
        ref = layer.forward(x).float()
    # one quantisation of x and one of mid apart: 2^-3 at most of each number for e2m1 between 2 and 6, far less in the norm
    assert (few - ref).norm() <= (0.01 if fmt == "bf16" else 0.3) * ref.norm()


def test_all_to_all_refuses_mxfp4_cpu():
    from hibana_b200.parallel.ep import ExpertParallel
    with pytest.raises(ValueError, match="mxfp4"):
        ExpertParallel.create(0, 2, torch.device("cpu"), tokens=4, topk=2, experts=8, hidden=128, fmt="mxfp4")


def test_models_run_cpu():
    for t, cls in ((scaled(dense_tiny(), weight_format="mxfp4"), DenseModel),
                   (scaled(tiny_hybrid_moe(), weight_format="mxfp4", expert_ffn=128), HybridModel)):
        out = _tokens(cls(t, "cpu", seed=0), _prompts(t.vocab), 4)
        assert all(len(o) == 4 for o in out)


# ---- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 7, 64, 129])
def test_linear_gpu(rows):
    g = torch.Generator().manual_seed(0)
    w, x = torch.randn(256, 320, generator=g) * 0.1, torch.randn(rows, 320, generator=g).bfloat16()
    cpu, gpu = Linear(w, "mxfp4"), Linear(w, "mxfp4").to("cuda")
    res = torch.randn(rows, 256, generator=g).bfloat16()
    for kw in ({}, {"epilogue": gemm.EPI_RESIDUAL}, {"epilogue": gemm.EPI_SILU_MUL}, {"epilogue": gemm.EPI_STORE_F32}):
        r = {"residual": res} if kw.get("epilogue") == gemm.EPI_RESIDUAL else {}
        a = cpu(x, **kw, **r).float()
        b = gpu(x.cuda(), **kw, **{k: v.cuda() for k, v in r.items()}).float().cpu()
        # the operands are the same bits; sums of 320 products in fp32 either way, then one rounding to bf16 (2^-8 of the
        # value) that may fall on either side, and for SiLU a product of two such sums
        tol = 2 ** -7 * a.abs() + 320 * 2 ** -23 * 40
        assert ((a - b).abs() <= tol).all()
    y = norm_linear(x.cuda(), res.cuda()[:, :1].expand(rows, 320).contiguous(), torch.ones(320).bfloat16().cuda(), 1e-6, gpu)
    assert y.shape == (rows, 256) and nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("fmt", ["bf16", "nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 5, 16])
def test_moe_layer_gpu_matches_cpu(fmt, latent, rows):
    act = "relu2" if latent else "swiglu"
    t, cpu = _layer(fmt, latent=latent, act=act)
    _, gpu = _layer(fmt, "cuda", latent=latent, act=act)
    x = torch.randn(rows, t.hidden, generator=torch.Generator().manual_seed(3)).bfloat16()
    with cfgmod.using(moe_few=True):
        a = cpu.forward(x).float()
        before = nv.LAUNCHES
        b = gpu.forward(x.cuda()).float().cpu()
        assert nv.LAUNCHES > before
        with cfgmod.using(moe_few=True, overlap_rows=0):
            c = gpu.forward(x.cuda()).float().cpu()
    assert torch.equal(b, c)                           # beside the side stream or not
    assert (a - b).abs().max() <= 3e-2 * a.abs().max() + 1e-3 and nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,few", [("mxfp4", False), ("nvfp4", True)])
def test_decoders_gpu(fmt, few):
    """Prefill and decode through the engine: captured graphs give the eager tokens. (The layers are held to the CPU's numbers
    above; argmaxes of random weights' nearly flat logits have no bound of their own.)"""
    targets = [(scaled(tiny_hybrid_moe(), weight_format=fmt, expert_ffn=128), HybridModel)]
    if fmt == "mxfp4":
        targets.append((scaled(dense_tiny(), weight_format=fmt), DenseModel))
    for t, cls in targets:
        with cfgmod.using(moe_few=few):
            prompts = _prompts(t.vocab, 3, 33)
            gpu = cls(t, "cuda", seed=0, init_device="cpu")
            eager = _tokens(gpu, prompts, 10)
            assert _tokens(gpu, prompts, 10, use_graphs=True) == eager
            assert all(len(e) == 10 for e in eager) and nv.read_status() == 0


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "bf16"])
def test_calibration_sees_the_rows_of_short_prompts_cpu(fmt):
    """Chunks of up to sixteen rows count like any others: every (token, choice) pair, once."""
    from hibana_b200.weights import calibrate_model as cm
    t = scaled(tiny_hybrid_moe(), weight_format=fmt, expert_ffn=128, mtp_layers=0, mtp_depth=0)
    model = HybridModel(t, "cpu", seed=0)
    samples = _prompts(t.vocab, 3, 9) + _prompts(t.vocab, 1, 40)
    with cfgmod.using(moe_few=True):
        cov = cm.capture(model, samples, max_batch=1)
    layers = cm.expert_layers(model)
    assert layers and set(cov.experts.rows) == set(layers)
    for name, layer in layers.items():
        assert int(cov.experts.rows[name].sum()) == sum(map(len, samples)) * t.top_k
        assert not layer.calibrating


@pytest.mark.gpu
@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("fmt", ["bf16", "nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 5, 16])
def test_moe_layer_gpu_is_its_parts(fmt, latent, rows):
    """The model's layer is the bits of its parts called one by one: `layer_forward` (held to 64 bits where that is tested) on the latent
    or the hidden rows, routed on the hidden ones, and the shared expert, added inside the layer or behind the up-projection."""
    from hibana_b200.ops import basic
    t, layer = _layer(fmt, "cuda", latent=latent, act="relu2" if latent else "swiglu")
    x = torch.randn(rows, t.hidden, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    with cfgmod.using(moe_few=True):
        got = layer.forward(x)
        shared = layer.shared.forward(x)
    kw = dict(sigmoid=t.router == "sigmoid", sel_bias=layer.sel_bias, scale=t.router_scale)
    if latent:
        y = moe.layer_forward(layer.fc1_latent(x), layer.router.weight, layer.experts, t.top_k, route_x=x, **kw)
        want = basic.add(layer.fc2_latent(y), shared)
    else:
        want = moe.layer_forward(x, layer.router.weight, layer.experts, t.top_k, shared=shared, **kw)
    assert torch.equal(got, want) and nv.read_status() == 0
