"""Replies for many prompts at once on the GPU: the output head over any number of rows."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from mojodiffusion_b200.llm import PagedKVCache, Qwen3Decoder, SamplerConfig, paged_prefill, paged_step
from test_gpu_paged_decoder import _model

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows", [1, 8, 9, 33, 130])
@pytest.mark.parametrize("vocabulary", [97, 20000])
@torch.no_grad()
def test_logits_of_many_rows(rows, vocabulary):
    """Sums of 256 exact products in fp32: 256 additions, each off by 2^-23 of the sum of sizes at most (2^-24 where it rounds to nearest). The table is not copied to fp32."""
    cfg, enc, _ = _model(vocab_size=vocabulary)
    dec = Qwen3Decoder(enc)
    hidden = torch.randn(rows, 256, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    dec.logits(hidden)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = dec.logits(hidden)
    table = vocabulary * 256 * 2
    assert torch.cuda.max_memory_allocated() - before < rows * vocabulary * 4 + rows * 256 * 16 + table // 2 + (1 << 20)
    h, w = enc.model.norm(hidden).double(), enc.model.embed_tokens.weight.double()
    assert got.dtype == torch.float32 and got.shape == (rows, vocabulary)
    assert float(((got.double() - h @ w.t()).abs() - 256 * 2.0 ** -23 * (h.abs() @ w.abs().t())).max()) <= 0
    O.check_status()


def test_a_dozen_prompts():
    """More sequences than the few-row kernels take: every sequence's hidden state is as near to the fp32 stack's as the encoder's own run of it (with the room for chance of the
    tests of four prompts), and a batch gives a reply of the wanted length for each prompt."""
    cfg, enc, wide = _model()
    prompts = [[(7 * i + j) % 97 for j in range(1 + 9 * i)] for i in range(12)]
    cache = PagedKVCache(cfg, 40, torch.bfloat16, DEV)
    numbers = list(range(12))
    hidden = paged_prefill(enc, cache, numbers, prompts)
    new = [(5 * i + 3) % 97 for i in range(12)]
    hidden = paged_step(enc, cache, numbers, torch.tensor(new, device=DEV))
    texts = [p + [n] for p, n in zip(prompts, new)]
    want = torch.cat([wide(torch.tensor([t]), final_norm=False)[:, -1] for t in texts]).to(DEV).double()
    rows = torch.cat([enc(torch.tensor([t], device=DEV), final_norm=False)[:, -1] for t in texts]).double()
    assert float((hidden.double() - want).norm()) < 1.25 * float((rows - want).norm())
    replies = Qwen3Decoder(enc).generate_batch(prompts, 5, SamplerConfig(temperature=0.0))
    assert [len(r) for r in replies] == [5] * 12
    O.check_status()


def test_a_page_that_is_not_there_ends_the_generation():
    class Wrong(PagedKVCache):
        def table(self, sequences):
            return super().table(sequences) + (1000 if max(self.lengths[s] for s in sequences) > 5 else 0)

    cfg, enc, _ = _model()
    cache = Wrong(cfg, 8, torch.bfloat16, DEV)
    with pytest.raises(RuntimeError, match="BOUNDS"):
        Qwen3Decoder(enc).generate_batch([[1, 2], [3]], 9, SamplerConfig(temperature=0.0), cache=cache)
    assert sorted(cache.free) == list(range(8))
    O.check_status()
