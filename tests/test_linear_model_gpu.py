"""The hybrid model with linear-attention mixers and layer norms: training, and
the mixer's prompt and decode paths against each other."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def _mod():
    importlib.import_module("gateddeltanet-2_b200")
    from gdn2_b200 import model
    return model


@pytest.mark.parametrize("decay", ["token", "fixed", "none"])
def test_mixer_prompt_and_decode_agree(gdn2, decay):
    torch.manual_seed(0)
    layer = gdn2.LinearAttention(hidden_size=256, head_dim=64, num_heads=2, num_v_heads=4, decay=decay,
                                 layer_idx=0).cuda().bfloat16().eval()
    if decay == "token":  # the decay's own parameters stay in fp32
        layer.A_log.data, layer.dt_bias.data = layer.A_log.data.float(), layer.dt_bias.data.float()
    x = torch.randn(2, 80, 256, device="cuda").bfloat16()
    with torch.no_grad():
        whole = layer(x)[0].float()
        cache = gdn2.LayerCache()
        parts = [layer(x[:, :70], past_key_values=cache, use_cache=True)[0]]
        for t in range(70, 80):
            parts.append(layer(x[:, t:t + 1], past_key_values=cache, use_cache=True)[0])
    got = torch.cat(parts, 1).float()
    assert cache.seen_tokens == 80
    # both sides round q, k, v, o, the norm's and the gate's output to bf16 in other GEMM shapes
    assert (got - whole).norm() <= 1e-2 * whole.norm()


def test_small_model_trains(gdn2):
    m = _mod()
    cfg = m.HybridConfig(vocab_size=512, n_layer=2, n_embd=256, n_head=2, intermediate_size=512, local_window=64,
                         block_size=256, mixer="linear", norm="layer")
    torch.manual_seed(1)
    model = m.GPT(cfg).cuda()
    model.init_weights()
    assert isinstance(model.transformer.h[0].attn, gdn2.LinearAttention)
    assert isinstance(model.transformer.ln_f, gdn2.LayerNorm)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3, fused=True)
    idx = torch.randint(0, cfg.vocab_size, (2, 200), device="cuda")
    tgt = torch.randint(0, cfg.vocab_size, (2, 200), device="cuda")
    losses = []
    for step in range(40):
        losses.append(float(m.train_step(model, opt, idx, tgt)))
        if step == 0:
            for n, p in model.named_parameters():
                assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, n
    assert losses[-1] < 0.5 * losses[0], losses


def test_config_refusals(gdn2):
    m = _mod()
    with pytest.raises(ValueError):
        m.HybridConfig(mixer="other")
    with pytest.raises(ValueError):
        m.HybridConfig(norm="other")
    with pytest.raises(ValueError):
        gdn2.LinearAttention(decay="other")
