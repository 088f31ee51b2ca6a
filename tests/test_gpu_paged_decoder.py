"""Paged caches as a decoder uses them: prompts and steps of a model, captured steps, other streams."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from mojodiffusion_b200.llm import PagedKVCache, Qwen3Decoder, SamplerConfig, paged_prefill, paged_step
from mojodiffusion_b200.models.text.qwen3 import Qwen3Config, Qwen3Encoder
from paged_oracle import angles, pool

pytestmark = pytest.mark.gpu
DEV = "cuda"
PROMPTS = [[5, 17, 3, 88, 42, 9], [1], [7, 8] * 65, list(range(64))]


def _model(**more):
    torch.manual_seed(0)
    cfg = Qwen3Config(**(dict(vocab_size=97, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=64, rope_theta=10000.0) | more))
    enc = Qwen3Encoder(cfg, torch.bfloat16, DEV)
    with torch.no_grad():
        enc.model.embed_tokens.weight.normal_(0, 1)
        for p in enc.parameters():
            if p.dim() == 2 and p.shape[0] != 97:
                p.normal_(0, p.shape[1] ** -0.5)
    wide = Qwen3Encoder(cfg, torch.float32, "cpu")
    wide.load_state_dict({n: t.float() for n, t in enc.state_dict().items()})
    return cfg, enc, wide


def _off(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("more", [{}, dict(qk_norm=False, qkv_bias=True), dict(head_dim=128), dict(num_attention_heads=6)], ids=["norm", "bias", "128", "three"])
def test_prefill_and_steps_are_as_near_as_the_whole_stack(more):
    """Against the same weights in fp32. The paged path rounds queries, keys and outputs no more often than the encoder's run of the whole text in bf16; 1.25 leaves room for
    chance over 256 x 4 values."""
    cfg, enc, wide = _model(**more)
    cache = PagedKVCache(cfg, 20, torch.bfloat16, DEV)
    hidden = paged_prefill(enc, cache, [3, 0, 8, 1], PROMPTS)
    texts = [list(p) for p in PROMPTS]
    for step in range(4):
        want = torch.cat([wide(torch.tensor([t]), final_norm=False)[:, -1] for t in texts]).to(DEV)
        rows = torch.cat([enc(torch.tensor([t], device=DEV), final_norm=False)[:, -1] for t in texts])
        assert _off(hidden, want) < 1.25 * _off(rows, want), step
        new = [(11 * step + 5 * i) % 97 for i in range(4)]
        for t, n in zip(texts, new):
            t.append(n)
        hidden = paged_step(enc, cache, [3, 0, 8, 1], torch.tensor(new, device=DEV))
    O.check_status()


def test_generation_over_eight_bits():
    cfg, enc, _ = _model()
    dec = Qwen3Decoder(enc)
    cache = PagedKVCache(cfg, 30, torch.float8_e4m3fn, DEV)
    first = dec.generate_batch(PROMPTS, 70, SamplerConfig(temperature=0.0), cache=cache)
    assert [len(r) for r in first] == [70] * 4 and len(cache.free) == 30
    # pages of earlier sequences hold what they held; scales start anew
    assert dec.generate_batch(PROMPTS, 70, SamplerConfig(temperature=0.0), cache=cache) == first
    assert dec.generate_batch(PROMPTS, 70, SamplerConfig(temperature=0.0), eight_bits=True) == first
    O.check_status()


def _step_inputs(B=3, H=8, G=2, D=128, P=16, most=200):
    g = torch.Generator(device=DEV).manual_seed(5)
    (kp, ks), (vp, vs) = pool(B * most // P + B, G, P, D, True, DEV, 0), pool(B * most // P + B, G, P, D, True, DEV, 1)
    table = torch.randperm(kp.shape[0], generator=g, device=DEV)[:B * (most // P + 1)].view(B, -1).int()
    cos, sin = angles(most, D, DEV)
    qkv = torch.randn(B, H + 2 * G, D, generator=g, device=DEV).bfloat16()
    return qkv, (H, G), kp, vp, ks, vs, table, cos, sin


def _step(qkv, heads, kp, vp, ks, vs, table, cos, sin, start):
    q, k, v = qkv.split([heads[0], heads[1], heads[1]], 1)
    q = O.paged_append(k, v, kp, vp, table, start, cos, sin, k_scale=ks, v_scale=vs, q=q)
    return O.paged_attention(q[:, None], kp, vp, table, start + 1, k_scale=ks, v_scale=vs)[:, 0]


def test_captured_steps_follow_lengths_and_share_a_pool():
    """Two graphs captured from one pool of workspaces, replayed in turn with other lengths and rows, give what eager calls give."""
    a, b = _step_inputs(), _step_inputs(B=2, H=4, G=4, D=64, P=64)
    eager = [[t.clone() if isinstance(t, torch.Tensor) else t for t in x] for x in (a, b)]
    starts = [torch.zeros(x[0].shape[0], dtype=torch.int32, device=DEV) for x in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, s in zip((a, b), starts):
            _step(*x, s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, handle = [], [], torch.cuda.graph_pool_handle()
    for x, s in zip((a, b), starts):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=handle):
            outs.append(_step(*x, s))
        graphs.append(graph)
    g = torch.Generator(device=DEV).manual_seed(9)
    for n in range(40):
        for x, y, s, graph, out in zip((a, b), eager, starts, graphs, outs):
            rows = torch.randn(x[0].shape, generator=g, device=DEV).bfloat16() * (1 + n % 3)
            x[0].copy_(rows)
            y[0].copy_(rows)
            graph.replay()
            got = out.clone()
            want = _step(*y, s)
            assert torch.equal(got, want), n
            for t, u in zip(x[2:6], y[2:6]):
                assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))
            s += 1 + torch.arange(s.numel(), device=DEV, dtype=torch.int32)
    O.check_status()


def test_streams_at_once():
    """Calls on several streams at the same time, each on its own pages."""
    inputs = [_step_inputs(B=2 + i) for i in range(3)]
    starts = [torch.full((x[0].shape[0],), 150, dtype=torch.int32, device=DEV) for x in inputs]
    want = [_step(*x, s) for x, s in zip(inputs, starts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(20):
        got = []
        for x, s, st in zip(inputs, starts, streams):
            with torch.cuda.stream(st):
                got.append(_step(*x, s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    O.check_status()


def test_captured_training_step_of_packed_sequences():
    g = torch.Generator(device=DEV).manual_seed(3)
    cu = torch.tensor([0, 30, 170, 171], dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(171, n, 64, generator=g, device=DEV).bfloat16().requires_grad_() for n in (4, 2, 2))
    grad = torch.randn(171, 4, 64, generator=g, device=DEV).bfloat16()

    def step():
        out = O.packed_attention(q, k, v, cu)
        return (out, *torch.autograd.grad(out, [q, k, v], grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for lengths in ([30, 140, 1], [0, 171, 0], [100, 0, 50]):
        cu.copy_(torch.tensor([sum(lengths[:i]) for i in range(4)], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
    O.check_status()
