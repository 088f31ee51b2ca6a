"""The pool of pages behind a batch of prompts: its tables of angles, and pages after an error."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from mojodiffusion_b200.llm import PagedKVCache, Qwen3Decoder, SamplerConfig, paged_prefill, paged_step
from mojodiffusion_b200.models.text.qwen3 import Qwen3Config, Qwen3Encoder


def _tiny(**more):
    torch.manual_seed(0)
    cfg = Qwen3Config(**(dict(vocab_size=97, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=16, rope_theta=10000.0) | more))
    return cfg, Qwen3Encoder(cfg, torch.float32, "cpu")


def test_angles_are_kept_from_step_to_step():
    cfg, enc = _tiny()
    cache = PagedKVCache(cfg, 30, torch.float32, page_size=16)
    paged_prefill(enc, cache, [0], [[1] * 70])
    tables = []
    for _ in range(70):                                        # from 71 positions to 140
        paged_step(enc, cache, [0], torch.tensor([3]))
        if not tables or cache.angles(1)[0] is not tables[-1]:
            tables.append(cache.angles(1)[0])
    assert [t.shape[0] for t in tables] == [128, 256]
    inv = 1.0 / 10000.0 ** (torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    angle = torch.arange(256, dtype=torch.float64)[:, None] * inv.float().double()
    for t, want in zip(cache.angles(200), (angle.cos(), angle.sin())):
        assert torch.equal(t, want.float())


def test_a_prefill_that_fails_takes_no_pages():
    cfg, enc = _tiny()
    cache = PagedKVCache(cfg, 8, torch.float32, page_size=16)
    paged_prefill(enc, cache, [0], [[1] * 20])
    cache.reserve(4, 16)                                       # a new sequence with a page already

    def state():
        return list(cache.free), {s: list(p) for s, p in cache.pages.items()}, dict(cache.lengths)

    before = state()
    with pytest.raises(RuntimeError, match="full"):            # five pages are left, the first two prompts take four
        paged_prefill(enc, cache, [1, 4, 2], [[1] * 32, [2] * 40, [3] * 70])
    assert state() == before
    hook = enc.model.layers[1].mlp.register_forward_hook(_fail)
    with pytest.raises(ArithmeticError):                       # in the model
        paged_prefill(enc, cache, [1, 4], [[1] * 32, [2] * 40])
    hook.remove()
    assert state() == before
    again = paged_prefill(enc, cache, [1, 4], [[1] * 32, [2] * 40])
    other = PagedKVCache(cfg, 8, torch.float32, page_size=16)
    assert torch.equal(again, paged_prefill(enc, other, [1, 4], [[1] * 32, [2] * 40]))
    for s in (0, 1, 4):
        cache.release(s)
    assert sorted(cache.free) == list(range(8)) and not cache.pages and not cache.lengths


def _fail(*_):
    raise ArithmeticError


def test_eight_bits_and_a_cache_of_another_type():
    cfg, enc = _tiny()
    dec = Qwen3Decoder(enc)
    eight, wide = (PagedKVCache(cfg, 8, t, page_size=16) for t in (torch.float8_e4m3fn, torch.float32))
    greedy = SamplerConfig(temperature=0.0)
    want = dec.generate_batch([[1, 2], [3]], 3, greedy, cache=eight)
    assert dec.generate_batch([[1, 2], [3]], 3, greedy, cache=eight, eight_bits=True) == want
    with pytest.raises(ValueError, match="eight_bits"):
        dec.generate_batch([[1, 2], [3]], 3, greedy, cache=wide, eight_bits=True)


def test_reports_of_kernels_end_the_generation(monkeypatch):
    """``ops.check_status`` is asked before tokens are drawn; its error gives the pages back."""
    cfg, enc = _tiny()
    cache, asked = PagedKVCache(cfg, 8, torch.float32, page_size=16), []

    def status(like):
        asked.append(like.shape)
        if len(asked) == 3:
            raise RuntimeError("TIMEOUT")

    monkeypatch.setattr(O, "check_status", status)
    with pytest.raises(RuntimeError, match="TIMEOUT"):
        Qwen3Decoder(enc).generate_batch([[1, 2], [3]], 6, SamplerConfig(temperature=0.0), cache=cache)
    assert asked == [(2, 64)] * 3 and sorted(cache.free) == list(range(8)) and not cache.pages
