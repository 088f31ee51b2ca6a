"""Window attention and attention with relative position buckets: the torch statements, the rules and the refusals."""
import math

import pytest
import torch

from mojodiffusion_b200 import ops as O
from mojodiffusion_b200.models.text.t5 import relative_bucket
from mojodiffusion_b200.ops import reference as ref
from text_attention_oracle import bucket, oracle, seen_by


def _normal(*shape, seed, dtype=torch.float64):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


CASES = [
    (1, 1, 1, 2, 1, None, 0, None, 0, False),
    (2, 9, 9, 4, 2, 3, 0, None, 0, True),
    (2, 9, 9, 4, 2, 3, 2, [9, 4], 0, False),
    (3, 5, 20, 3, 3, 6, 1, [20, 0, 7], [15, -5, 2], True),
    (3, 5, 20, 3, 3, 6, 0, [20, 0, 7], [15, -5, 12], False),
    (1, 4, 11, 4, 1, None, 0, None, 7, True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_window_attention_and_its_gradients(case):
    """fp64: rounding errors of sums of at most 20 x 8 terms of size 10, far below 1e-12."""
    B, Sq, Skv, H, G, window, sinks, kv_len, q_start, logits = case
    q, k, v = (_normal(B, s, h, 8, seed=i).requires_grad_() for i, (s, h) in enumerate(((Sq, H), (Skv, G), (Skv, G))))
    n = torch.tensor(kv_len, dtype=torch.int32) if kv_len is not None else None
    at = torch.tensor(q_start, dtype=torch.int32) if isinstance(q_start, list) else q_start
    sink = _normal(H, seed=5).requires_grad_() if logits else None
    grad = _normal(B, Sq, H, 8, seed=6)
    value, _ = oracle(q, k, v, 8 ** -0.5, seen_by(Sq, Skv, B, window, sinks, n, at), grad, sink)
    out = O.window_attention(q, k, v, window, sinks, kv_len=n, q_start=at, sink_logits=sink)
    got = torch.autograd.grad(out, [q, k, v] + ([sink] if logits else []), grad)
    for name, t in zip(("out", "dq", "dk", "dv", "dsink"), (out, *got)):
        assert float((t - value[name]).abs().max()) < 1e-12, name
    leaves = [q, k, v] + ([sink] if logits else [])
    assert torch.autograd.gradcheck(lambda q, k, v, *s: O.window_attention(q, k, v, window, sinks, kv_len=n, q_start=at, sink_logits=s[0] if s else None), leaves)


@pytest.mark.parametrize("buckets,distance,kv_len", [(32, 128, None), (8, 10, [30, 7]), (4, 3, [0, 30])])
def test_relative_attention_and_its_gradients(buckets, distance, kv_len):
    B, S, H = 2, 30, 4
    q, k, v = (_normal(B, S, H, 8, seed=i).requires_grad_() for i in range(3))
    table, grad = _normal(buckets, H, seed=5).requires_grad_(), _normal(B, S, H, 8, seed=6)
    n = torch.tensor(kv_len, dtype=torch.int32) if kv_len is not None else None
    value, _ = oracle(q, k, v, 0.5, seen_by(S, S, B, kv_len=n, causal=False), grad, table=table, max_distance=distance)
    out = O.relative_attention(q, k, v, table, distance, 0.5, kv_len=n)
    for name, t in zip(("out", "dq", "dk", "dv", "dtable"), (out, *torch.autograd.grad(out, [q, k, v, table], grad))):
        assert float((t - value[name]).abs().max()) < 1e-12, name
    assert torch.autograd.gradcheck(lambda *a: O.relative_attention(*a, distance, 0.5, kv_len=n), [t[:, :6].detach().requires_grad_() for t in (q, k, v)] + [table])


@pytest.mark.parametrize("buckets,distance", [(32, 128), (64, 256), (16, 100), (8, 3), (4, 2), (6, 50), (128, 1024), (32, 9)])
def test_buckets(buckets, distance):
    rel = torch.arange(-distance - 300, distance + 301)
    got = ref.relative_bucket(rel, buckets, distance)
    assert got.tolist() == [bucket(int(r), buckets, distance) for r in rel]
    if (buckets, distance) in ((32, 128), (64, 256), (16, 100)):             # where fp32 logarithms round to the same side of every border
        assert torch.equal(got, relative_bucket(rel, buckets, distance))


def test_unseen_keys_are_not_read():
    q, k, v = (_normal(2, s, 2, 8, seed=s, dtype=torch.float32) for s in (3, 20, 20))
    v = _normal(2, 20, 2, 8, seed=9, dtype=torch.float32)
    n, at = torch.tensor([18, 9], dtype=torch.int32), torch.tensor([15, 6], dtype=torch.int32)
    want = O.window_attention(q, k, v, 3, 1, kv_len=n, q_start=at)
    hidden = ~seen_by(3, 20, 2, 3, 1, n, at).any(1)[:, :, None, None]
    for bad in (math.nan, math.inf):
        leaves = [t.requires_grad_() for t in (q.clone(), k.masked_fill(hidden, bad), v.masked_fill(hidden, bad))]
        out = O.window_attention(*leaves, 3, 1, kv_len=n, q_start=at)
        assert torch.equal(out, want)
        out.sum().backward()
        assert all(torch.isfinite(t.grad).all() for t in leaves)


def test_outputs_and_empty_inputs():
    q, k = _normal(2, 5, 4, 8, seed=1, dtype=torch.bfloat16), _normal(2, 5, 2, 8, seed=2, dtype=torch.bfloat16)
    table = _normal(32, 4, seed=3, dtype=torch.bfloat16)
    out = torch.empty_like(q)
    assert O.window_attention(q, k, k, 2, out=out) is out and torch.equal(out, O.window_attention(q, k, k, 2))
    assert O.relative_attention(q, q, q, table, out=out) is out and torch.equal(out, O.relative_attention(q, q, q, table))
    assert O.window_attention(q[:0], k[:0], k[:0]).shape == (0, 5, 4, 8)
    assert O.window_attention(q[:, :0], k, k).shape == (2, 0, 4, 8)
    assert float(O.window_attention(q, k[:, :0], k[:, :0]).abs().max()) == 0


def test_refusals():
    q, k = _normal(2, 5, 4, 8, seed=1, dtype=torch.float32), _normal(2, 5, 2, 8, seed=2, dtype=torch.float32)
    table = _normal(32, 4, seed=3, dtype=torch.float32)
    w, r = O.window_attention, O.relative_attention
    ints = lambda *v: torch.tensor(v, dtype=torch.int32)
    for call in (lambda: w(q[0], k, k), lambda: w(q, k, k[:, :4]), lambda: w(q, k[:1], k[:1]), lambda: w(q, k[..., :4], k[..., :4]), lambda: w(q[:, :, :3], k, k),
                 lambda: w(q, k.double(), k.double()), lambda: w(q.long(), k.long(), k.long()), lambda: w(q, k, k, 0), lambda: w(q, k, k, -1), lambda: w(q, k, k, 2.0),
                 lambda: w(q, k, k, True), lambda: w(q, k, k, 2, -1), lambda: w(q, k, k, 2, None), lambda: w(q, k, k, kv_len=ints(1)), lambda: w(q, k, k, kv_len=torch.tensor([1, 2])),
                 lambda: w(q, k, k, q_start=ints(1, 2, 3)), lambda: w(q, k, k, q_start=1.0), lambda: w(q, k, k, q_start=torch.tensor([1, 2])),
                 lambda: w(q, k, k, sink_logits=_normal(2, seed=1)), lambda: w(q, k, k, sink_logits=torch.ones(4, dtype=torch.long)), lambda: w(q, k, k, out=q[:, :2]),
                 lambda: w(q, k, k, out=torch.empty_like(q, dtype=torch.float64)), lambda: w(q, k[:, :, :0], k[:, :, :0]),
                 lambda: r(q, q, q, table[:, :3]), lambda: r(q, q, q, table[:31]), lambda: r(q, q, q, table[:2]), lambda: r(q, q, q, table[0]), lambda: r(q, q, q, table.long()),
                 lambda: r(q, q, q, table, 8), lambda: r(q, q, q, table, 100.0), lambda: r(q, q, q, table, kv_len=ints(1)), lambda: r(q, q, q, table, out=q[:1]), lambda: r(q, k, k, table)):
        with pytest.raises(ValueError):
            call()


def test_prefix_lengths():
    assert O.prefix_lengths(torch.tensor([[1, 1, 0], [0, 0, 0], [1, 1, 1]])).tolist() == [2, 0, 3]
    assert O.prefix_lengths(torch.tensor([[True, False]])).dtype == torch.int32
    assert O.prefix_lengths(torch.tensor([[0, 1]])) is None and O.prefix_lengths(torch.tensor([[1, 1], [1, 1], [0, 1]])) is None


@pytest.mark.parametrize("per_layer", [False, True])
def test_t5_encoder_with_fused_attention(per_layer):
    """fp32, two layers of width 16: the separate operations and the fused one differ by fp32 roundings only (sums of at most 24 terms of size 1: 1e-5)."""
    from mojodiffusion_b200.models.text.t5 import T5Config, T5Encoder

    torch.manual_seed(0)
    cfg = T5Config(vocab_size=50, d_model=16, d_kv=8, d_ff=24, num_layers=2, num_heads=2, relative_attention_num_buckets=8, relative_attention_max_distance=10, per_layer_bias=per_layer)
    enc = T5Encoder(cfg)
    ids = torch.randint(0, 50, (3, 23))
    for mask in (None, (torch.arange(23)[None] < torch.tensor([23, 7, 15])[:, None]).long(), torch.cat((torch.zeros(3, 4), torch.ones(3, 19)), 1)):
        cfg.fused_attention = False
        want = enc(ids, mask)
        cfg.fused_attention = True
        kept = mask.bool() if mask is not None else torch.ones_like(ids, dtype=torch.bool)
        assert float((enc(ids, mask) - want)[kept].abs().max()) < 1e-5


def test_gpt_oss_encoder_with_fused_attention():
    from mojodiffusion_b200.models.text.gpt_oss import GptOssConfig, GptOssEncoder

    torch.manual_seed(0)
    cfg = GptOssConfig(vocab_size=50, hidden_size=16, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=8, intermediate_size=16, num_local_experts=4,
                       num_experts_per_tok=2, sliding_window=5)
    enc = GptOssEncoder(cfg)
    for l in enc.layers:
        torch.nn.init.normal_(l.self_attn.sinks)
    ids = torch.randint(0, 50, (2, 17))
    for mask in (None, (torch.arange(17)[None] < torch.tensor([17, 6])[:, None]).long(), torch.cat((torch.zeros(2, 3), torch.ones(2, 14)), 1)):
        cfg.fused_attention = False
        want = enc.layer_states(ids, mask)
        cfg.fused_attention = True
        kept = mask.bool() if mask is not None else torch.ones_like(ids, dtype=torch.bool)
        for a, b in zip(enc.layer_states(ids, mask), want):
            assert float((a - b)[kept].abs().max()) < 1e-5
