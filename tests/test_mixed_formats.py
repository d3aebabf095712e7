"""Dense models whose projections are stored in formats of their own."""
import itertools

import pytest
import torch

from hibana_b200 import _native as nv
from hibana_b200 import config as cfgmod
from hibana_b200.cache.kv_pool import KvPool
from hibana_b200.engine.context import PREFILL, ForwardContext
from hibana_b200.engine.executor import Executor
from hibana_b200.engine.request import SamplingParams
from hibana_b200.models.dense import DenseModel
from hibana_b200.models.linear import Linear
from hibana_b200.target import dense_tiny


def _mixed(formats, device="cpu", per_layer=None):
    """dense_tiny with its projections in `formats` (one a part; `per_layer` overrides them by layer)."""
    model = DenseModel(dense_tiny(), device, seed=0, init_device="cpu")
    for i, layer in enumerate(model.layers):
        for part, fmt in {**formats, **(per_layer or {}).get(i, {})}.items():
            lin = getattr(layer, part)
            setattr(layer, part, Linear(lin.dequantized(), fmt, name=lin.name))
    return model


def _run(model, graphs=False, n=4):
    ex = Executor(model, max_batch=4, max_ctx=128, use_graphs=graphs)
    if graphs:
        ex.capture_graphs()
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, model.target.vocab, (m,), generator=g).tolist() for m in (5, 20, 33)]
    return [r.output_ids for r in ex.generate_batch(prompts, SamplingParams(max_tokens=n, ignore_eos=True))]


def test_only_an_nvfp4_down_projection_is_handed_nvfp4_rows_cpu():
    for fmt, other in itertools.product(("bf16", "nvfp4", "mxfp4"), repeat=2):
        layer = _mixed({"down": fmt, "gate_up": other}).layers[0]
        for fused in (False, True):
            got = DenseModel._requants_down(layer, 4, True, fused)
            assert got == (fmt == "nvfp4" and (fused or other == "nvfp4")), (fmt, other, fused)
        layer.down.calibrating = True
        assert not DenseModel._requants_down(layer, 4, True, True)


class _Ranks:
    """A communicator of one rank that offers the sequence-parallel chain."""
    sp_rows, sp_hidden = 256, 256

    def sp_ok(self, rows, hidden):
        return True

    def fits(self, rows, hidden):
        return False

    def all_reduce(self, x):
        return x


class _Chain(Exception):
    pass


def _prefill(model):
    """Whether a prefill runs the sequence-parallel chain."""
    t = model.target
    pool = KvPool(model.kv_layers, 64, t.kv_heads, t.head_dim, device="cpu")
    ctx = ForwardContext(PREFILL, torch.arange(6, dtype=torch.int32), torch.arange(1, 7, dtype=torch.int32),
                         torch.arange(1, 7, dtype=torch.int32).view(1, 6), torch.tensor([6], dtype=torch.int32),
                         q_indptr=torch.tensor([0, 6], dtype=torch.int32), max_rows=6, max_ctx_host=6, comm=_Ranks())

    def chain(*args):
        raise _Chain
    model.forward_sp = chain
    try:
        out = model.forward(torch.arange(6), ctx, pool)
    except _Chain:
        return True
    assert torch.isfinite(out.float()).all()
    return False


def test_the_sequence_parallel_chain_takes_layers_it_can_carry_cpu():
    assert _prefill(_mixed({})) and _prefill(_mixed({"qkv": "bf16", "down": "bf16"}))
    for part in ("qkv", "o", "gate_up", "down"):
        assert not _prefill(_mixed({part: "mxfp4"}))
        assert not _prefill(_mixed({}, per_layer={1: {part: "mxfp4"}}))
    model = _mixed({"qkv": "bf16"})
    model.layers[1].gate_up.calibrating = True           # (its range is recorded by the plain forward)
    assert not _prefill(model)


@pytest.mark.gpu
@pytest.mark.parametrize("down", ["bf16", "mxfp4"])
@pytest.mark.parametrize("gate_up", ["nvfp4", "mxfp4"])
def test_nvfp4_attention_beside_another_mlp_gpu(down, gate_up):
    model = _mixed({"qkv": "nvfp4", "o": "nvfp4", "gate_up": gate_up, "down": down}, "cuda")
    eager = _run(model)
    assert all(len(e) == 4 for e in eager) and _run(model, graphs=True) == eager and nv.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("part,fmt,layer", [("down", "mxfp4", 0), ("o", "bf16", 1), ("down", "bf16", 1), ("qkv", "mxfp4", 1), ("gate_up", "bf16", 0)])
def test_few_row_decode_of_mixed_layers_gpu(part, fmt, layer):
    """The few-row decode path (setting `gemv`) hands NVFP4 rows to o_proj and down, so it runs where all of those are NVFP4."""
    model = _mixed({}, "cuda", {layer: {part: fmt}})
    with cfgmod.using(gemv=True):
        ran = []
        whole = model._forward_few_rows
        model._forward_few_rows = lambda *a: ran.append(1) or whole(*a)
        eager = _run(model)
        assert all(len(e) == 4 for e in eager) and bool(ran) == (part in ("qkv", "gate_up"))
        assert _run(model, graphs=True) == eager and nv.read_status() == 0
