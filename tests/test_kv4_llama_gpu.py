"""The 4-bit page cache inside the Llama tower (RMSNorm, q | k | v in blocks, rotary over the whole head): what tests/test_kv4_model_gpu.py checks of the other towers."""
import pytest
import torch

import _parity as P
import test_kv4_model_gpu as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=[64, 128])
def tower(request):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from unimp_amd.flamingo import Flamingo
    from unimp_amd.lm import LlamaConfig, build_lm
    from unimp_amd.synthetic import TokenLayout
    from unimp_amd.vit import CLIPStub, VisionTransformer
    cfg = dict(P.TINY_OPT)
    layout = TokenLayout(cfg["base_vocab"], cfg["n_items"], 16)
    torch.manual_seed(0)
    with torch.device("cuda"):
        lm = build_lm(LlamaConfig(vocab_size=layout.vocab, hidden_size=2 * request.param, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                                  max_position_embeddings=256))
        m = Flamingo(CLIPStub(VisionTransformer(**cfg["vit"])), lm, layout.eoc, layout.media, vis_dim=cfg["vit"]["width"], cross_attn_every_n_layers=1)
    for n, p in m.named_parameters():
        if p.dim() >= 2 and "latents" not in n:
            torch.nn.init.normal_(p, std=0.06)
        if n.endswith("_gate"):
            torch.nn.init.constant_(p, 0.5)
    return cfg, m.to(torch.bfloat16).eval(), layout


def test_generate(tower):
    M.test_generate(tower)


def test_step_logits_are_those_of_rounded_keys_and_values(tower, monkeypatch):
    M.test_step_logits_are_those_of_rounded_keys_and_values(tower, monkeypatch)
