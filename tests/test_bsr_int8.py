"""The Roformers' ``int8`` precision (SESA_PREC_I8: the layers on sesa_norm_residual, sesa_linear_i8, sesa_rope_axes and
sesa_attention_packed) against the reference's outputs, and how a user reaches it.

Tolerance: rounding a row of normal values to 8 bits on one scale moves it by (largest / 127) / sqrt(12) of its rms, about
1 % with the largest at 4.5 rms; a product has two such operands (1.45 %).  A layer's two blocks have two products each
on the way to the residual stream, so the stream is off by about 2 x 1.45 % of itself (errors of different blocks are
independent), and what later blocks make of that error is at most as much again: 5.8 %.
"""
import os

import numpy as np
import pytest
import torch

from conftest import CONFIGS

REL = 4 * 0.0145


def _model(model_type, cfg, affine="random"):
    from sesa.utils import get_model_from_config
    from sesa.weights import synth_model_state
    m, c = get_model_from_config(model_type, os.path.join(CONFIGS, cfg))
    m.load_state_dict(synth_model_state(m, affine=affine, seed=0), strict=True)
    return m, c


def test_int8_is_a_precision_of_the_roformers_only():
    for mt, cfg, has in (("bs_roformer", "config_bs_roformer_small.yaml", True),
                         ("mel_band_roformer", "config_mel_band_roformer_small.yaml", True),
                         ("scnet", "config_scnet_small.yaml", False)):
        m, c = _model(mt, cfg) if has else (__import__("sesa.utils", fromlist=["x"]).get_model_from_config(
            mt, os.path.join(CONFIGS, cfg)))
        if has:
            small = m.workspace_bytes(1, c.audio.chunk_size)
            assert m.set_precision("int8").workspace_bytes(1, c.audio.chunk_size) > small   # 8-bit rows, positions
        else:
            with pytest.raises(ValueError):
                m.set_precision("int8")


def test_command_line_names_a_precision():
    from sesa.inference import build_parser
    assert build_parser().parse_args(["--config_path", "c"]).precision is None
    assert build_parser().parse_args(["--config_path", "c", "--precision", "int8"]).precision == "int8"


@pytest.mark.gpu
@pytest.mark.parametrize("model_type,cfg,fixture", [
    ("bs_roformer", "config_bs_roformer_small.yaml", "bsr_small.npz"),
    ("mel_band_roformer", "config_mel_band_roformer_small.yaml", "mbr_small.npz"),
    ("bs_roformer", "config_bs_roformer_vocals.yaml", "bsr_full_chunk.npz"),
    ("mel_band_roformer", "config_mel_band_roformer_vocals.yaml", "mbr_full_chunk.npz")])
def test_int8_forward_near_reference(golden, model_type, cfg, fixture):
    from sesa.backend import create_inference_session
    g = golden(fixture)
    m, _ = _model(model_type, cfg, str(g["affine"]) if "affine" in g.files else "random")
    be = create_inference_session(m, device="cuda:0", precision="int8")
    assert m.precision == "int8"
    y = be(torch.from_numpy(g["x"]).to("cuda:0")).cpu().numpy().astype(np.float64)
    ref = g["y"].astype(np.float64)
    rel = float(np.linalg.norm(y - ref) / np.linalg.norm(ref))
    print(f"{fixture} int8: rel {rel:.4f}, rms {np.sqrt(np.mean((y - ref) ** 2)):.3e}")
    assert y.shape == ref.shape and rel <= REL


@pytest.mark.gpu
def test_int8_forward_streams_and_graph():
    """The same bits on two streams at once, and from a replayed graph among eager forwards."""
    m, c = _model("bs_roformer", "config_bs_roformer_small.yaml")
    m.set_precision("int8")
    xs = [0.1 * torch.randn(2, 2, c.audio.chunk_size, generator=torch.Generator("cuda").manual_seed(s), device="cuda")
          for s in (1, 2)]
    want = [m(x).clone() for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for st, x in zip(streams, xs):
        with torch.cuda.stream(st):
            got.append(m(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    hold = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(hold)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        out = m(hold)
    for i in range(4):
        hold.copy_(xs[i % 2])
        gr.replay()
        eager = m(xs[i % 2])
        torch.cuda.synchronize()
        assert torch.equal(out, want[i % 2]) and torch.equal(eager, want[i % 2])
