"""Models with their default settings (a step is a CUDA graph) on a context that runs on
torch's default stream, which cannot itself be captured."""
import pytest
import torch

import dcpp_b200
import flux2_oracle as fo
from dcpp_b200 import synth

pytestmark = pytest.mark.gpu


@pytest.fixture
def on_default():
    own = dcpp_b200.Context(0)
    own.use_current_stream()
    yield own
    own.close()


def flux2(ctx, graph):
    c = synth.Flux2Cfg(num_layers=1, num_single_layers=1, num_attention_heads=2, joint_attention_dim=64, in_channels=32,
                       guidance_embeds=False)
    m = dcpp_b200.Flux2Model(ctx, c)
    m.load_params(synth.make_params(c, fo.GGML_Q8_0, seed=41))
    m.prepare(1, 16, 8, **graph)
    hid, enc, iid, tid = synth.make_inputs(c, 1, 4, 4, 8, seed=42)
    outs = []
    for t in (0.5, 0.25):
        out = torch.empty_like(hid)
        m.forward(hid, enc, torch.tensor([t]), iid, tid, out)
        outs.append(out)
        m.denoise_step(hid, enc, torch.tensor([t]), -0.25, iid, tid, out2 := torch.empty_like(hid))
        outs.append(out2)
    return m, outs


def qwen3(ctx, graph):
    c = synth.Qwen3Cfg(vocab_size=100, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4,
                       num_key_value_heads=2)
    m = dcpp_b200.Qwen3Model(ctx, c)
    m.load_params(synth.make_qwen3_params(c, dcpp_b200.TYPE_Q8_0, seed=3))
    m.prepare(1, 40, (), **graph)
    outs = []
    for seed in (4, 5):
        out = torch.empty(1, 40, c.hidden_size)
        m.forward(synth.make_qwen3_ids(c, 1, 40, seed=seed).contiguous(), out, None)
        outs.append(out)
    return m, outs


def vae(ctx, graph):
    c = synth.VAECfg(block_out_channels=(64, 64), layers_per_block=1)
    m = dcpp_b200.VAEModel(ctx, c)
    m.load_params(synth.make_vae_params(c, seed=11))
    m.prepare(1, 4, 4, **graph)
    outs = []
    for seed in (3, 4):
        img = torch.empty(1, c.out_channels, 16, 16)
        m.decode(synth.make_vae_latents(c, 1, 4, 4, seed=seed), img)
        outs.append(img)
    return m, outs


@pytest.mark.parametrize("model", [flux2, qwen3, vae])
def test_model_on_the_default_stream(ctx, on_default, model):
    """Graph captured and replayed on the default stream: the results of a context on a
    stream of its own, step by step."""
    plain, want = model(ctx, dict(use_graph=False))
    m, got = model(on_default, {})
    on_default.synchronize()
    try:
        for a, b in zip(got, want):
            assert torch.isfinite(a).all() and torch.equal(a, b)
    finally:
        m.close()
        plain.close()


def test_default_stream_keeps_the_order_of_work(on_default):
    """Device tensors that torch fills on the default stream just before a call, the
    result read by torch just after it."""
    c = synth.Qwen3Cfg(vocab_size=100, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4,
                       num_key_value_heads=2)
    m = dcpp_b200.Qwen3Model(on_default, c)
    m.load_params(synth.make_qwen3_params(c, dcpp_b200.TYPE_Q8_0, seed=3))
    m.prepare(1, 40)
    ids = [synth.make_qwen3_ids(c, 1, 40, seed=s).contiguous() for s in range(4)]
    want = []
    for i in ids:
        out = torch.empty(1, 40, c.hidden_size)
        m.forward(i, out, None)
        on_default.synchronize()
        want.append(out.clone())
    out = torch.empty(1, 40, c.hidden_size, device="cuda")
    got = []
    for i in ids:
        torch.cuda._sleep(2_000_000)  # about a millisecond on the stream
        x = i.cuda(non_blocking=True)
        out.fill_(7.0)
        m.forward(x, out, None)
        got.append(out.clone())
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    m.close()
