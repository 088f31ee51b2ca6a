"""One prompt and several take the same scaled rotation."""
import pytest
import torch

from mojodiffusion_b200.llm import PagedKVCache, Qwen3Decoder, SamplerConfig, paged_prefill, paged_step
from mojodiffusion_b200.models.text.qwen3 import Qwen3Config, Qwen3Encoder


def _decoder(scaling):
    torch.manual_seed(0)
    cfg = Qwen3Config(vocab_size=97, hidden_size=64, intermediate_size=128, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=16, rope_theta=10000.0, rope_scaling=scaling)
    return cfg, Qwen3Decoder(Qwen3Encoder(cfg, torch.float32, "cpu"))


@pytest.mark.parametrize("scaling", [None, (4.0, 64, 32.0, 1.0), (16.0, 16384, 32.0, 1.0)], ids=["none", "short", "long"])
def test_dense_and_paged_decoding_follow_the_encoder(scaling):
    cfg, dec = _decoder(scaling)
    text = [(7 * i + 3) % 97 for i in range(80)]
    dense, cache = dec.prefill(torch.tensor([text]), 90)
    pages = PagedKVCache(cfg, 8, torch.float32, page_size=16)
    paged = paged_prefill(dec.enc, pages, [0], [text])
    for new in (5, 90, 2):
        want = dec.enc(torch.tensor([text]), final_norm=False)[0, -1]
        torch.testing.assert_close(dense[0], want, atol=3e-5, rtol=0)
        torch.testing.assert_close(paged[0], want, atol=3e-5, rtol=0)
        text.append(new)
        dense, paged = dec.decode_step(torch.tensor([new]), cache), paged_step(dec.enc, pages, [0], torch.tensor([new]))
    prompts = [text[:70], text[10:30]]
    assert dec.generate_batch(prompts, 6, SamplerConfig(temperature=0.0)) == [dec.generate(p, 6, SamplerConfig(temperature=0.0)) for p in prompts]
