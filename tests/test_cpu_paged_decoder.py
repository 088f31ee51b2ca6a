"""Generation for several prompts over pages: the replies of one prompt at a time, pages taken and given back."""
import io

import pytest
import torch

from mojodiffusion_b200.llm import PagedKVCache, Qwen3Decoder, SamplerConfig, paged_prefill, paged_step
from mojodiffusion_b200.models.text.qwen3 import Qwen3Config, Qwen3Encoder

PROMPTS = [[5, 17, 3, 88, 42, 9], [1], [7] * 70, [2, 3, 4]]


def _tiny(**more):
    torch.manual_seed(0)
    cfg = Qwen3Config(**(dict(vocab_size=97, hidden_size=64, intermediate_size=128, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=16, rope_theta=10000.0) | more))
    return cfg, Qwen3Encoder(cfg, torch.float32, "cpu")


@pytest.mark.parametrize("more", [{}, dict(qk_norm=False, qkv_bias=True)], ids=["norm", "bias"])
def test_prefill_and_steps_match_the_full_stack(more):
    cfg, enc = _tiny(**more)
    cache = PagedKVCache(cfg, 20, torch.float32, page_size=16)
    hidden = paged_prefill(enc, cache, [3, 0, 8, 1], PROMPTS)
    texts = [list(p) for p in PROMPTS]
    for step in range(4):
        for h, t in zip(hidden, texts):
            want = enc(torch.tensor([t]), final_norm=False)[0, -1]
            assert torch.allclose(h, want, atol=3e-5), step
        new = [(11 * step + 5 * i) % 97 for i in range(4)]
        for t, n in zip(texts, new):
            t.append(n)
        hidden = paged_step(enc, cache, [3, 0, 8, 1], torch.tensor(new))
    assert [cache.lengths[s] for s in (3, 0, 8, 1)] == [len(t) for t in texts]


def test_hooked_norms_run():
    cfg, enc = _tiny()
    dec = Qwen3Decoder(enc)
    plain = dec.generate_batch(PROMPTS, 3, SamplerConfig(temperature=0.0))
    seen = []
    handle = enc.model.layers[0].self_attn.q_norm.register_forward_hook(lambda m, a, o: seen.append(1))
    assert dec.generate_batch(PROMPTS, 3, SamplerConfig(temperature=0.0)) == plain and len(seen) == 3
    handle.remove()


@pytest.mark.parametrize("sampler", [SamplerConfig(temperature=0.0), SamplerConfig(temperature=0.8, top_k=20, top_p=0.9, seed=7)], ids=["greedy", "sampled"])
def test_generate_batch_is_generate_for_each(sampler):
    cfg, enc = _tiny()
    dec = Qwen3Decoder(enc)
    alone = [dec.generate(p, 6, sampler) for p in PROMPTS]
    assert dec.generate_batch(PROMPTS, 6, sampler) == alone
    eos = (alone[0][2], alone[3][0])
    assert dec.generate_batch(PROMPTS, 6, sampler, eos) == [dec.generate(p, 6, sampler, eos) for p in PROMPTS]
    assert dec.generate_batch([], 4) == [] and dec.generate_batch([[1]], 0) == [[]]
    with pytest.raises(ValueError):
        dec.generate_batch([[1], []], 4)


def test_pages_are_taken_and_given_back():
    cfg, enc = _tiny()
    dec = Qwen3Decoder(enc)
    cache = PagedKVCache(cfg, 8, torch.float32, page_size=16)
    want = dec.generate_batch(PROMPTS, 5, SamplerConfig(temperature=0.0))
    for _ in range(2):                                       # the second time in pages that hold what was there
        assert dec.generate_batch(PROMPTS, 5, SamplerConfig(temperature=0.0), cache=cache) == want
        assert sorted(cache.free) == list(range(8)) and not cache.pages and not cache.lengths
    with pytest.raises(RuntimeError, match="full"):
        dec.generate_batch(PROMPTS + [[1] * 40], 5, cache=cache)
    assert sorted(cache.free) == list(range(8))
    with pytest.raises(RuntimeError, match="full"):          # while decoding
        dec.generate_batch([[1] * 16] * 5, 5, cache=cache)
    assert sorted(cache.free) == list(range(8))


def test_eight_bits_stay_near():
    """e4m3 keeps 3 bits behind the point: keys and values are off by 2^-4 of their size at most, independently, and a softmax of scores that are off by d weighs values by factors
    of e^d at most. Here scores are small (untrained weights), so a layer's attention is off by less than 2^-3 of the size of its values; the logits by less than that of theirs."""
    cfg, enc = _tiny()
    dec = Qwen3Decoder(enc)
    caches = [PagedKVCache(cfg, 20, t, page_size=16) for t in (torch.float32, torch.float8_e4m3fn)]
    for c in caches:
        paged_prefill(enc, c, [0, 1, 2, 3], PROMPTS)
    for token in (4, 50, 9):
        a, b = (dec.logits(paged_step(enc, c, [0, 1, 2, 3], torch.full((4,), token))) for c in caches)
        assert not torch.equal(a, b)
        assert float((a - b).norm() / a.norm()) < 2 ** -3


def test_magic_prompt_lines(tmp_path, monkeypatch, capsys):
    from mojodiffusion_b200.captioner import magic_prompt as M

    reply = tmp_path / "reply.txt"
    reply.write_text('{"high_level_description": "a red house", "compositional_deconstruction": {"background": "sky", "elements": []}}')
    one = M.magic_prompt(f"stub:{reply}", "1:1", "a house")
    monkeypatch.setattr("sys.stdin", io.StringIO("a house\n\nanother house\n"))
    assert M.main(["--lines", f"stub:{reply}", "1:1"]) == 0
    assert capsys.readouterr().out == f"{one}\n{one}\n"
