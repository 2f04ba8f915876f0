"""The Roformers' ``int8`` precision, layer by layer: broken and vanishing weights, and the forward against the same 8-bit
arithmetic written out in PyTorch."""
import os

import numpy as np
import pytest
import torch

from conftest import CONFIGS


def _model(model_type, cfg):
    from sesa.utils import get_model_from_config
    from sesa.weights import synth_model_state
    m, c = get_model_from_config(model_type, os.path.join(CONFIGS, cfg))
    return m, c, synth_model_state(m, affine="random", seed=0)


def _forward(m, state, x):
    m.load_state_dict(state, strict=True)
    return m.set_precision("int8")(x).cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["to_qkv.weight", "to_out.0.weight", "net.1.weight", "net.4.weight"])
def test_int8_broken_and_vanishing_weights(name):
    """A NaN or infinite weight shows in the output, as in the other precisions; a row too small for a scale counts as 0."""
    m, c, state = _model("bs_roformer", "config_bs_roformer_small.yaml")
    x = 0.1 * torch.randn(1, 2, c.audio.chunk_size, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    key = next(k for k in state if k.endswith(name) and k.startswith("layers.1.0."))
    assert bool(torch.isfinite(_forward(m, state, x)).all())
    for bad in (float("nan"), float("inf")):
        broken = {k: v.clone() for k, v in state.items()}
        broken[key][3, 5] = bad
        assert bool(torch.isnan(_forward(m, broken, x)).any())
        assert bool(torch.isnan(m.set_precision("fp16")(x)).any())
    out = []
    for size in (0.0, 1e-38, 1e-37):
        small = {k: v.clone() for k, v in state.items()}
        small[key][3] = size * torch.sign(small[key][3])
        out.append(_forward(m, small, x))
    assert bool(torch.isfinite(out[0]).all()) and torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])
