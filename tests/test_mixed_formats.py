"""Dense models whose projections are stored in formats of their own."""
import itertools

import pytest
import torch

from hibana_b200 import _native as nv
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


@pytest.mark.gpu
@pytest.mark.parametrize("down", ["bf16", "mxfp4"])
@pytest.mark.parametrize("gate_up", ["nvfp4", "mxfp4"])
def test_nvfp4_attention_beside_another_mlp_gpu(down, gate_up):
    model = _mixed({"qkv": "nvfp4", "o": "nvfp4", "gate_up": gate_up, "down": down}, "cuda")
    eager = _run(model)
    assert all(len(e) == 4 for e in eager) and _run(model, graphs=True) == eager and nv.read_status() == 0
