"""Window attention and attention with relative position buckets on the GPU, against their definitions in 64 bits."""
import math

import pytest
import torch

from mojodiffusion_b200 import ops as O
from text_attention_oracle import FINE, HALF, bucket, check, oracle, seen_by

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(*shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _inputs(B, Sq, Skv, H, G, D, seed=0):
    return _normal(B, Sq, H, D, seed=seed), _normal(B, Skv, G, D, seed=seed + 1), _normal(B, Skv, G, D, seed=seed + 2)


# B, Sq, Skv, H, Hkv, Dh, window, sinks, kv_len, q_start, sink logits
WINDOW = [
    (1, 1, 1, 4, 4, 64, None, 0, None, 0, False),
    (1, 1, 1, 8, 1, 128, 1, 0, None, 0, True),
    (2, 77, 77, 4, 2, 64, None, 0, None, 0, False),
    (1, 128, 128, 2, 2, 128, None, 0, None, 0, False),
    (1, 129, 129, 6, 2, 128, 128, 0, None, 0, False),
    (1, 300, 300, 8, 2, 64, 128, 0, None, 0, True),
    (2, 257, 257, 4, 4, 64, 1, 0, None, 0, False),
    (2, 257, 257, 4, 4, 64, 5, 3, None, 0, True),
    (1, 700, 700, 4, 1, 64, 100, 130, None, 0, False),
    (1, 700, 700, 2, 1, 128, 64, 4, None, 0, False),
    (1, 513, 513, 3, 1, 64, 200, 1, None, 0, False),
    (3, 200, 200, 4, 2, 128, 50, 2, [200, 0, 61], 0, False),            # a sequence without keys; padded rows far behind their window
    (3, 200, 200, 4, 2, 64, 50, 0, [133, 1, 20], 0, True),              # rows whose window lies behind kv_len: only the sink logit is left
    (2, 40, 333, 4, 2, 64, 100, 4, [333, 200], [293, 160], False),      # parts of prompts behind a cache
    (2, 150, 600, 4, 4, 128, 130, 0, [600, 300], [450, 150], True),
    (2, 33, 500, 6, 2, 128, None, 0, [500, 33], [467, 0], False),
    (2, 64, 300, 4, 2, 64, 20, 4, None, [-30, 290], False),             # rows before the first key, and behind the last
    (4, 1, 700, 8, 2, 128, None, 0, [700, 1, 0, 353], [699, 0, -1, 352], False),
    (4, 1, 700, 8, 1, 64, 128, 4, [700, 1, 0, 353], [699, 0, -1, 352], True),
    (2, 1, 2000, 16, 2, 64, 1000, 0, [2000, 1234], [1999, 1233], True),
    (3, 5, 400, 8, 2, 128, 100, 4, [400, 5, 77], [395, 0, 72], False),
    (2, 7, 900, 28, 4, 128, 300, 1, [900, 17], [893, 10], False),
    (2, 3, 900, 5, 5, 64, None, 0, [900, 3], [897, 0], True),
    (1, 8, 260, 64, 8, 64, 17, 200, [258], [250], False),
    (2, 16, 130, 4, 4, 64, 1 << 40, 1 << 40, None, 114, False),         # bounds beyond 32 bits
]


@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_window_attention(case):
    B, Sq, Skv, H, G, D, window, sinks, kv_len, q_start, logits = case
    q, k, v = _inputs(B, Sq, Skv, H, G, D)
    n = _ints(kv_len) if kv_len is not None else None
    at = _ints(q_start) if isinstance(q_start, list) else q_start
    sink = _normal(H, seed=9) if logits else None
    seen = seen_by(Sq, Skv, B, window, sinks, n, at)
    value, bound = oracle(q, k, v, D ** -0.5, seen, sink=sink)
    out = O.window_attention(q, k, v, window, sinks, kv_len=n, q_start=at, sink_logits=sink)
    check(dict(out=out), value, bound, str(case))


@pytest.mark.parametrize("case", [c for c in WINDOW if c[1] >= 7 or c[0] == 1], ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_window_attention_gradients(case):
    B, Sq, Skv, H, G, D, window, sinks, kv_len, q_start, logits = case
    q, k, v = (t.requires_grad_() for t in _inputs(B, Sq, Skv, H, G, D, seed=20))
    n = _ints(kv_len) if kv_len is not None else None
    at = _ints(q_start) if isinstance(q_start, list) else q_start
    sink = _normal(H, seed=29).requires_grad_() if logits else None
    grad = _normal(B, Sq, H, D, seed=30)
    value, bound = oracle(q, k, v, D ** -0.5, seen_by(Sq, Skv, B, window, sinks, n, at), grad, sink)
    out = O.window_attention(q, k, v, window, sinks, kv_len=n, q_start=at, sink_logits=sink)
    got = torch.autograd.grad(out, [q, k, v] + ([sink] if logits else []), grad)
    check(dict(zip(("out", "dq", "dk", "dv", "dsink"), (out, *got))), value, bound, str(case))


# B, S, H, H, Dh, buckets, max_distance, kv_len, fp32 table
RELATIVE = [
    (1, 1, 4, 4, 64, 32, 128, None, False),
    (2, 77, 4, 4, 64, 32, 128, [77, 40], False),
    (1, 128, 3, 3, 64, 32, 128, None, False),
    (1, 300, 2, 2, 128, 32, 128, None, True),
    (3, 257, 2, 2, 64, 32, 128, [257, 0, 129], False),
    (1, 600, 4, 4, 64, 32, 128, None, False),
    (2, 190, 2, 2, 64, 64, 200, [11, 190], False),
    (1, 333, 2, 2, 128, 8, 3, None, False),
    (1, 150, 2, 2, 64, 4, 100, None, True),
    (1, 1300, 1, 1, 64, 64, 560, None, False),          # the last bucket begins at 502
    (1, 520, 2, 2, 128, 32, 385, [519], False),         # at 238
    (1, 200, 2, 2, 128, 32, 1000, None, False),         # at 547: the torch statement
    (1, 260, 2, 2, 64, 32, 9, None, False),             # all borders at one distance
    (1, 1100, 1, 1, 64, 6, 60, None, False),            # shared blocks of keys behind an odd number of sums of the table
    (1, 1100, 1, 1, 128, 10, 100, [1000], True),
    (1, 200, 2, 2, 64, 66, 128, None, False),           # more buckets than the kernels keep: the torch statement
]


@pytest.mark.parametrize("case", RELATIVE, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_relative_attention(case):
    B, S, H, G, D, buckets, distance, kv_len, wide = case
    q, k, v = _normal(B, S, H, D, seed=40, scale=D ** -0.5), _normal(B, S, G, D, seed=41), _normal(B, S, G, D, seed=42)
    table = _normal(buckets, H, seed=43, dtype=torch.float32 if wide else torch.bfloat16)
    n = _ints(kv_len) if kv_len is not None else None
    grad = _normal(B, S, H, D, seed=44)
    value, bound = oracle(q, k, v, 1.0, seen_by(S, S, B, kv_len=n, causal=False), grad, table=table, max_distance=distance)
    check(dict(out=O.relative_attention(q, k, v, table, distance, kv_len=n)), value, bound, str(case))
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = O.relative_attention(q, k, v, table, distance, kv_len=n)
    got = torch.autograd.grad(out, leaves, grad)
    assert got[3].dtype == table.dtype
    check(dict(zip(("out", "dq", "dk", "dv", "dtable"), (out, *got))), value, bound, str(case))


def test_relative_attention_rectangle():
    q, k, v = _normal(2, 50, 2, 64, seed=1, scale=0.125), _normal(2, 170, 2, 64, seed=2), _normal(2, 170, 2, 64, seed=3)
    table, grad = _normal(32, 2, seed=4), _normal(2, 50, 2, 64, seed=5)
    value, bound = oracle(q, k, v, 0.7, seen_by(50, 170, 2, causal=False), grad, table=table)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = O.relative_attention(q, k, v, table, scale=0.7)
    check(dict(zip(("out", "dq", "dk", "dv", "dtable"), (out, *torch.autograd.grad(out, leaves, grad)))), value, bound, "rectangle")


@pytest.mark.parametrize("Sq", [1, 90])
def test_lengths_and_positions_out_of_range(Sq):
    """Lengths below zero and beyond the keys, positions at the ends of 32 bits: what they say, without wrapping."""
    B, Skv, H, G, D = 4, 200, 4, 2, 64
    q, k, v = (t.requires_grad_() for t in _inputs(B, Sq, Skv, H, G, D, seed=50))
    grad = _normal(B, Sq, H, D, seed=53)
    for n, at in (([-5, 200, 2**31 - 1, -2**31], [100, 2**31 - 1, 110, 100]), ([200, 200, 150, 200], [-2**31, -2**31 + 5, 2**31 - 9, -1])):
        near = torch.tensor(at).clamp(-2**30, 2**30)                       # the oracle counts in 64 bits; nothing changes beyond
        for window, sinks in ((None, 0), (50, 3)):
            seen = seen_by(Sq, Skv, B, window, sinks, torch.tensor(n), near)
            value, bound = oracle(q, k, v, D ** -0.5, seen, grad)
            out = O.window_attention(q, k, v, window, sinks, kv_len=_ints(n), q_start=_ints(at))
            check(dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, [q, k, v], grad)))), value, bound, f"{n} {at} {window}")
            with torch.no_grad():
                check(dict(out=O.window_attention(q, k, v, window, sinks, kv_len=_ints(n), q_start=_ints(at))), value, bound, f"{n} {at} {window} step")


@pytest.mark.parametrize("Sq", [1, 90])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_unseen_keys_may_hold_anything(Sq, bad):
    """Behind kv_len, and between the first tokens and the windows: neither the output nor a gradient of what is seen changes."""
    B, Skv, H, G, D, window, sinks = 2, 700, 4, 2, 128, 60, 3
    q, k, v = _inputs(B, Sq, Skv, H, G, D, seed=60)
    n = _ints([600, 430])
    at = n - Sq
    sink = _normal(H, seed=63)
    grad = _normal(B, Sq, H, D, seed=64)
    seen = seen_by(Sq, Skv, B, window, sinks, n, at)
    value, bound = oracle(q, k, v, D ** -0.5, seen, grad, sink)
    hidden = ~seen.any(1).to(DEV)[:, :, None, None]
    k, v = k.masked_fill(hidden, bad), v.masked_fill(hidden, bad)
    with torch.no_grad():
        check(dict(out=O.window_attention(q, k, v, window, sinks, kv_len=n, q_start=at, sink_logits=sink)), value, bound, "forward")
    leaves = [t.requires_grad_() for t in (q, k, v, sink)]
    out = O.window_attention(q, k, v, window, sinks, kv_len=n, q_start=at, sink_logits=sink)
    check(dict(zip(("out", "dq", "dk", "dv", "dsink"), (out, *torch.autograd.grad(out, leaves, grad)))), value, bound, "gradients")


def test_sink_logits_at_the_ends():
    """-inf: as without; very large: the row is (nearly) empty; fp32 logits."""
    q, k, v = _inputs(1, 140, 140, 3, 3, 64, seed=70)
    sink = torch.tensor([-math.inf, 200.0, -200.0], device=DEV)
    out = O.window_attention(q, k, v, 50, 2, sink_logits=sink)
    plain = O.window_attention(q, k, v, 50, 2)
    assert torch.equal(out[:, :, 0], plain[:, :, 0]) and torch.equal(out[:, :, 2], plain[:, :, 2])
    assert float(out[:, :, 1].abs().max()) < 1e-30
    value, bound = oracle(q, k, v, 0.125, seen_by(140, 140, 1, 50, 2), sink=sink)
    check(dict(out=out), value, bound, "sink logits")


def test_large_scores_move_the_maximum():
    """Scores that grow along the keys: the running maximum is raised again and again, and a key takes the whole row."""
    q, k, v = _inputs(1, 400, 400, 2, 2, 64, seed=75)
    q = (q.float().abs() + 0.5).bfloat16()
    k = (torch.arange(400, device=DEV)[None, :, None, None] / 40.0 + 0.1 * k.float()).bfloat16()
    seen = seen_by(400, 400, 1, 300, 0)
    value, _ = oracle(q, k, v, 0.125, seen)
    out = O.window_attention(q, k, v, 300)
    # scores up to 100, so exponents up to 144 with steps of 2^-17 of fp32, from products up to 10: relative 3e-4 of a probability
    assert float((out.double() - value["out"]).abs().max()) <= (2 * 2.0 ** -8 + 1e-3) * float(v.abs().max())


def test_table_gradient_keeps_what_rounding_the_output_left():
    """Scores that are all equal (p = 1 before the division, also in bf16) over values whose mean no bf16 number holds: o is off by 2^-9 in every element, in
    the same direction, so that delta = do . o would be off by 64 * 2^-9 = 0.125 in every row. The bound is what is left without that rounding: FINE for
    the sums and exponentials in o, delta and ds each, and HALF twice for the rest of o that is kept in bf16; 0.08 of a row."""
    S, H, D = 512, 2, 64
    q, k = torch.zeros(1, S, H, D, device=DEV, dtype=torch.bfloat16), _normal(1, S, H, D, seed=60)
    v = torch.where(torch.arange(S, device=DEV) % 4 == 3, 1 + 2.0 ** -7, 1.0).to(torch.bfloat16)[None, :, None, None].expand(1, S, H, D).contiguous()
    grad = torch.ones_like(q)
    table = torch.zeros(32, H, device=DEV, requires_grad=True)
    got, = torch.autograd.grad(O.relative_attention(q, k, v, table), [table], grad)
    dp = D * v[0, :, 0, 0].double()
    delta = dp.mean()
    ds = ((dp - delta) / S).expand(S, S)
    off = (FINE * delta + HALF ** 2 * delta + FINE * (dp.abs() + delta + (dp - delta).abs())) / S
    which = torch.tensor([[bucket(j - i, 32, 128) for j in range(S)] for i in range(S)], device=DEV)
    want, bound = (torch.zeros(32, device=DEV, dtype=torch.float64).index_add_(0, which.flatten(), t.expand(S, S).flatten()) for t in (ds, off))
    assert bool(((got.double() - want[:, None]).abs() <= bound[:, None]).all())


def test_sink_gradient_keeps_what_rounding_the_output_left():
    """As above, with o off by 2^-8 (127 of 256 values are 1 + 2^-7): d_sink = -sum p_sink delta would be off by 0.0039 relative. The bound is FINE for
    p_sink, o and delta each, and HALF twice: 0.0012."""
    S, H, D = 512, 4, 64
    q, k = torch.zeros(1, S, H, D, device=DEV, dtype=torch.bfloat16), _normal(1, S, 2, D, seed=61)
    v = torch.where(torch.arange(S, device=DEV) % 256 < 127, 1 + 2.0 ** -7, 1.0).to(torch.bfloat16)[None, :, None, None].expand(1, S, 2, D).contiguous()
    sink = torch.full((H,), -4.0, device=DEV, requires_grad=True)
    got, = torch.autograd.grad(O.window_attention(q, k, v, q_start=S, sink_logits=sink), [sink], torch.ones_like(q))
    others = S * math.exp(4.0)                                           # of the keys, for one of the sink
    want = -S / (others + 1) * D * float(v[0, :, 0, 0].double().mean()) * others / (others + 1)
    assert bool(((got.double() - want).abs() <= (3 * FINE + HALF ** 2) * abs(want)).all())


def test_switched_off_buckets():
    q, k, v = _normal(1, 140, 2, 64, seed=80, scale=0.125), _normal(1, 140, 2, 64, seed=81), _normal(1, 140, 2, 64, seed=82)
    table, grad = _normal(32, 2, seed=83), _normal(1, 140, 2, 64, seed=84)
    table[16:, 0] = -math.inf                # head 0 does not look ahead
    table[:16, 1] = -math.inf                # head 1 looks ahead only: the last query sees nothing
    value, bound = oracle(q, k, v, 1.0, seen_by(140, 140, 1, causal=False), grad, table=table)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = O.relative_attention(q, k, v, table)
    got = dict(zip(("out", "dq", "dk", "dv", "dtable"), (out, *torch.autograd.grad(out, leaves, grad))))
    assert float(out[0, -1, 1].abs().max()) == 0 and float(got["dq"][0, -1, 1].abs().max()) == 0
    check(got, value, bound, "buckets off")


LAYOUTS = {
    "packed projection": lambda B, S, H, D, s: _normal(B, S, 3 * H * D, seed=s)[..., H * D:2 * H * D].unflatten(-1, (H, D)),
    "heads first": lambda B, S, H, D, s: _normal(B, H, S, D, seed=s).transpose(1, 2),
    "sequence first": lambda B, S, H, D, s: _normal(S, B, H, D, seed=s).transpose(0, 1),
    "part of a cache": lambda B, S, H, D, s: _normal(B + 1, H, S + 13, D, seed=s)[1:, :, 5:5 + S].transpose(1, 2),
    "off 16 bytes": lambda B, S, H, D, s: _normal(B, S, H, D + 1, seed=s)[..., 1:],
    "elements apart": lambda B, S, H, D, s: _normal(B, S, H, D, 2, seed=s)[..., 0],
    "one for the batch": lambda B, S, H, D, s: _normal(1, S, H, D, seed=s).expand(B, S, H, D),
    "one head for all": lambda B, S, H, D, s: _normal(B, S, 1, D, seed=s).expand(B, S, H, D),
}


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("Sq", [1, 150])
def test_layouts(layout, Sq):
    B, Skv, H, G, D = 2, 150, 4, 2, 64
    make = LAYOUTS[layout]
    q, k, v = make(B, Sq, H, D, 90), make(B, Skv, G, D, 91), make(B, Skv, G, D, 92)
    at = Skv - Sq
    value, bound = oracle(q, k, v, D ** -0.5, seen_by(Sq, Skv, B, 40, 3, None, at))
    check(dict(out=O.window_attention(q, k, v, 40, 3, q_start=at)), value, bound, layout)
    table = _normal(32, 2 * H, seed=93)[:, ::2]
    k, v = make(B, Skv, H, D, 94), make(B, Skv, H, D, 95)
    value, bound = oracle(q, k, v, D ** -0.5, seen_by(Sq, Skv, B, causal=False), table=table)
    check(dict(out=O.relative_attention(q, k, v, table, scale=D ** -0.5)), value, bound, layout)


def test_gradients_of_broadcast_inputs():
    """A key / value head that all sequences share, a gradient that is one number for all elements, and sums over the expanded batch."""
    B, S, H, D = 3, 140, 4, 64
    q = _normal(B, S, H, D, seed=100).requires_grad_()
    k0, v0 = _normal(1, S, 1, D, seed=101).requires_grad_(), _normal(1, S, 1, D, seed=102).requires_grad_()
    k, v = k0.expand(B, S, 1, D), v0.expand(B, S, 1, D)
    grad = torch.ones(1, 1, 1, 1, device=DEV, dtype=torch.bfloat16).expand(B, S, H, D)
    value, bound = oracle(q, k, v, D ** -0.5, seen_by(S, S, B, 33, 2), grad)
    out = O.window_attention(q, k, v, 33, 2)
    dq, dk, dv = torch.autograd.grad(out, [q, k0, v0], grad)
    check(dict(out=out, dq=dq), value, bound, "broadcast")
    half = torch.finfo(torch.bfloat16).eps / 2
    for got, name in ((dk, "dk"), (dv, "dv")):
        want, off = value[name].sum(0, keepdim=True), bound[name].sum(0, keepdim=True)
        assert bool(((got.double() - want).abs() <= off * (1 + half) + 2 * half * value[name].abs().sum(0, keepdim=True)).all())     # torch adds the sequences in bf16


def test_out_buffers():
    B, S, H, G, D = 2, 150, 4, 2, 64
    q, k, v = _inputs(B, S, S, H, G, D, seed=110)
    want = O.window_attention(q, k, v, 40, 3)
    wide = torch.full((B, S + 2, H, 2 * D), 7.0, device=DEV, dtype=torch.bfloat16)
    for out in (wide[:, 1:-1, :, D:], torch.empty(B, H, S, D, device=DEV, dtype=torch.bfloat16).transpose(1, 2),
                torch.empty(B, S, H, D + 1, device=DEV, dtype=torch.bfloat16)[..., 1:], q.clone()):
        assert O.window_attention(q, k, v, 40, 3, out=out) is out
        assert torch.equal(out, want)
    assert bool((wide[:, 0] == 7).all() and (wide[:, -1] == 7).all() and (wide[..., :D] == 7).all())
    q2 = q.clone()
    O.window_attention(q2, k, v, 40, 3, out=q2)                      # over its own input
    assert torch.equal(q2, want)
    step = O.window_attention(q[:, -1:], k, v, 40, 3, q_start=S - 1)
    row = wide[:, 1:2, :, :D]
    O.window_attention(q[:, -1:], k, v, 40, 3, q_start=S - 1, out=row)
    assert torch.equal(row, step) and bool((wide[:, 0] == 7).all())


def test_the_same_bits_every_time():
    q, k, v = (t.requires_grad_() for t in _inputs(2, 700, 700, 8, 2, 64, seed=120))
    q2, k2 = (_normal(2, 700, 8, 64, seed=i).requires_grad_() for i in (127, 128))
    grad, table, sink = _normal(2, 700, 8, 64, seed=124), _normal(32, 8, seed=125).requires_grad_(), _normal(8, seed=126).requires_grad_()

    def both():
        a = O.window_attention(q, k, v, 100, 4, sink_logits=sink)
        b = O.relative_attention(q, q2, k2, table, scale=0.125)
        return [a, b, *torch.autograd.grad(a, [q, k, v, sink], grad), *torch.autograd.grad(b, [q, q2, k2, table], grad)]

    first = both()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, both()))


def test_a_batch_changes_no_sequence():
    """The rows of a sequence are the same bits alone and in a batch, whatever the others hold."""
    q, k, v = _inputs(3, 200, 200, 4, 2, 64, seed=130)
    n = _ints([200, 150, 33])
    out = O.window_attention(q, k, v, 70, 3, kv_len=n)
    for b in range(3):
        assert torch.equal(out[b:b + 1], O.window_attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], 70, 3, kv_len=n[b:b + 1]))


def test_prompt_parts_and_steps_agree():
    """A prompt in one call; its first part, its second part behind the cache, then tokens one by one and a few at once over the cache."""
    B, S, H, G, D, window, sinks = 2, 400, 8, 2, 64, 90, 4
    q, k, v = _inputs(B, S, S, H, G, D, seed=140)
    sink = _normal(H, seed=143)
    value, bound = oracle(q, k, v, D ** -0.5, seen_by(S, S, B, window, sinks), sink=sink)
    cache_k, cache_v = (torch.full((B, G, 512, D), math.nan, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    parts, lo = [], 0
    for hi in (150, 385, 386, 387, 388, 393, 400):
        cache_k[:, :, lo:hi], cache_v[:, :, lo:hi] = k[:, lo:hi].transpose(1, 2), v[:, lo:hi].transpose(1, 2)
        parts.append(O.window_attention(q[:, lo:hi], cache_k.transpose(1, 2), cache_v.transpose(1, 2), window, sinks,
                                        kv_len=_ints([hi] * B), q_start=_ints([lo] * B), sink_logits=sink))
        lo = hi
    check(dict(out=torch.cat(parts, 1)), value, bound, "parts")
    check(dict(out=O.window_attention(q, k, v, window, sinks, sink_logits=sink)), value, bound, "whole")


def test_streams_and_graphs():
    """Calls on two streams at once, and two captured graphs that are replayed in turn with new inputs, share nothing."""
    sets = [_inputs(1, 1, 900, 8, 2, 64, seed=150 + 10 * i) + _inputs(2, 260, 260, 4, 4, 64, seed=200 + 10 * i) for i in range(2)]
    table = _normal(32, 4, seed=250)
    lens = [_ints([900]), _ints([500])]

    def call(i):
        q, k, v, q2, k2, v2 = sets[i]
        return (O.window_attention(q, k, v, 300, 4, kv_len=lens[i], q_start=lens[i] - 1), O.relative_attention(q2, k2, v2, table, scale=0.125),
                O.window_attention(q2, k2, v2, 60, 1))

    want = [call(0), call(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            for _ in range(5):
                out = call(i)
            got.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(i))
        graphs.append(g)
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(outs, want) for a, b in zip(x, y))
    lens[0].fill_(321)
    sets[0][0].mul_(2)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], call(0)))


def test_captured_training_step():
    """Forward and backward in one graph, replayed with other inputs."""
    q, k, v = (t.requires_grad_() for t in _inputs(1, 200, 200, 4, 2, 64, seed=300))
    sink, grad = _normal(4, seed=303).requires_grad_(), _normal(1, 200, 4, 64, seed=304)
    step = lambda: torch.autograd.grad(O.window_attention(q, k, v, 50, 2, sink_logits=sink), [q, k, v, sink], grad)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    with torch.no_grad():
        k.mul_(0.5)
        grad.mul_(2)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements: 2^21 + 4096 positions of 8 heads of 128 (4.3 GB), read at its end."""
    T, G, D = (1 << 21) + 4096, 8, 128
    cache = torch.zeros(1, T, G, D, device=DEV, dtype=torch.bfloat16)
    cache[:, :8] = _normal(1, 8, G, D, seed=310)
    cache[:, -2500:] = _normal(1, 2500, G, D, seed=311)
    for Sq in (1, 200):
        q = _normal(1, Sq, 16, D, seed=312)
        out = O.window_attention(q, cache, cache, 2000, 8, q_start=T - Sq)
        small = torch.cat((cache[:, :8], cache[:, -2500:]), 1)
        seen = seen_by(Sq, 2508, 1, 2000, 8, None, 2508 - Sq)
        value, bound = oracle(q, small, small, D ** -0.5, seen)
        check(dict(out=out), value, bound, f"end of a long cache, {Sq}")


def test_other_types_and_widths_take_the_torch_statement():
    for dtype, D, tol in ((torch.float16, 64, 2e-3), (torch.float32, 128, 1e-5), (torch.bfloat16, 96, 2e-2)):
        q, k, v = (_normal(1, 20, h, D, seed=320 + i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
        value, _ = oracle(q, k, v, D ** -0.5, seen_by(20, 20, 1, 6, 1))
        assert float((O.window_attention(q, k, v, 6, 1).double() - value["out"]).abs().max()) < tol
        table = _normal(16, 4, seed=330, dtype=dtype)
        value, _ = oracle(q, q, q, 0.1, seen_by(20, 20, 1, causal=False), table=table, max_distance=20)
        assert float((O.relative_attention(q, q, q, table, 20, 0.1).double() - value["out"]).abs().max()) < tol


def test_scales_the_kernels_do_not_take():
    """Zero and negative scales: the torch statement."""
    q, k, v = _inputs(1, 20, 20, 4, 4, 64, seed=335)
    table = _normal(32, 4, seed=336)
    for scale in (0.0, -0.2):
        value, bound = oracle(q, k, v, scale, seen_by(20, 20, 1, 6, 1))
        check(dict(out=O.window_attention(q, k, v, 6, 1, scale)), value, bound, "window")
        value, bound = oracle(q, k, v, scale, seen_by(20, 20, 1, causal=False), table=table)
        check(dict(out=O.relative_attention(q, k, v, table, scale=scale)), value, bound, "relative")


def test_nothing_to_do():
    q, k = _normal(0, 3, 4, 64, seed=1), _normal(0, 3, 2, 64, seed=1)
    assert O.window_attention(q, k, k).shape == (0, 3, 4, 64)
    q, k = _normal(1, 0, 4, 64, seed=1), _normal(1, 3, 2, 64, seed=1)
    assert O.window_attention(q, k, k).shape == (1, 0, 4, 64)
    q, k = _normal(1, 3, 4, 64, seed=1), _normal(1, 0, 2, 64, seed=1)
    assert float(O.window_attention(q, k, k).abs().max()) == 0
    k = _normal(1, 0, 4, 64, seed=1)
    table = _normal(32, 4, seed=2)
    assert float(O.relative_attention(q, k, k, table).abs().max()) == 0
    leaves = [t.requires_grad_() for t in (q, k, table)]
    got = torch.autograd.grad(O.relative_attention(q, k, k, table).sum(), leaves)
    assert [g.shape for g in got] == [t.shape for t in leaves] and all(float(g.abs().sum()) == 0 for g in got)


def test_refusals():
    q, k = _normal(2, 5, 4, 64, seed=1), _normal(2, 5, 2, 64, seed=2)
    table = _normal(32, 4, seed=3)
    w, r = O.window_attention, O.relative_attention
    leaf = lambda t: t.clone().requires_grad_()
    calls = [lambda q, k: w(q[0], k, k), lambda q, k: w(q, k, k[:, :4]), lambda q, k: w(q, k[:1], k[:1]), lambda q, k: w(q, k[..., :32], k[..., :32]),
             lambda q, k: w(q[:, :, :3], k, k), lambda q, k: w(q, k.float(), k.float()), lambda q, k: w(q, k.cpu(), k.cpu()), lambda q, k: w(q, k, k, 0),
             lambda q, k: w(q, k, k, 2.0), lambda q, k: w(q, k, k, 2, -1), lambda q, k: w(q, k, k, kv_len=_ints([1])), lambda q, k: w(q, k, k, kv_len=_ints([1, 2]).long()),
             lambda q, k: w(q, k, k, kv_len=_ints([1, 2]).cpu()), lambda q, k: w(q, k, k, q_start=_ints([1, 2, 3])), lambda q, k: w(q, k, k, q_start=1.0),
             lambda q, k: w(q, k, k, q_start=_ints([1, 2]).long()), lambda q, k: w(q, k, k, sink_logits=_normal(2, seed=1)),
             lambda q, k: w(q, k, k, sink_logits=torch.ones(4, dtype=torch.long, device=DEV)), lambda q, k: w(q, k, k, sink_logits=_normal(4, seed=1).cpu()),
             lambda q, k: w(q, k, k, out=torch.empty_like(q)[:, :2]), lambda q, k: w(q, k, k, out=torch.empty_like(q, dtype=torch.float32)),
             lambda q, k: w(q, k, k, out=torch.empty_like(q, device="cpu")), lambda q, k: w(q, k[:, :, :0], k[:, :, :0]),
             lambda q, k: r(q, q, q, table[:, :3]), lambda q, k: r(q, q, q, table[:31]), lambda q, k: r(q, q, q, table[:2]), lambda q, k: r(q, q, q, table[0]),
             lambda q, k: r(q, q, q, table.long()), lambda q, k: r(q, q, q, table.cpu()), lambda q, k: r(q, q, q, table, 8), lambda q, k: r(q, q, q, table, 100.0),
             lambda q, k: r(q, q, q, table, kv_len=_ints([1])), lambda q, k: r(q, q, q, table, out=torch.empty_like(q)[:1]), lambda q, k: r(q, k, k, table)]
    for i, call in enumerate(calls):
        for grad in (False, True):
            with pytest.raises(ValueError):
                call(leaf(q), leaf(k)) if grad else call(q, k)
                pytest.fail(f"call {i} went through")
    o = w(leaf(q), k, k)
    g, = torch.autograd.grad(o, [o.grad_fn.next_functions[0][0].variable], torch.ones_like(o), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                       # differentiable once


def test_native_refusals():
    """What the C++ entries check by themselves, on the host, before a launch."""
    q, k, v = _inputs(2, 8, 8, 4, 2, 64, seed=340)
    table = _normal(32, 4, seed=1)
    relative = lambda b, k=q, t=table: torch.ops.mdb200.relative_attention(q, k, k, t, b, 1.0, None, None)
    relative([32, 8, 9])
    for bad in (lambda: relative([32, 8, 9], k), lambda: relative([16, 4, 9]), lambda: relative([32]), lambda: relative([32, 8] + [9] * 40), lambda: relative([32, 8, 5000]),
                lambda: relative([32, 8, 20, 10]), lambda: relative([32, 16]), lambda: relative([32, 0, 9]), lambda: relative([66, 8, 9], t=_normal(66, 4, seed=1)),
                lambda: relative([32, 8, 9], t=_normal(32, 4, seed=1, dtype=torch.float16)),
                lambda: torch.ops.mdb200.window_attention(q, k, v, 0, 0, 1.0, None, 0, None, None, None),
                lambda: torch.ops.mdb200.window_attention(q, k, v, 4, -1, 1.0, None, 0, None, None, None),
                lambda: torch.ops.mdb200.window_attention(q, k, v, 4, 0, 0.0, None, 0, None, None, None),
                lambda: torch.ops.mdb200.window_attention(q, k, v, 4, 0, math.nan, None, 0, None, None, None)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


def test_encoders_with_fused_attention():
    """Both text encoders in bf16: the fused form launches its kernels and gives what the separate operations give, up to the rounding of their bf16 scores,
    bias and probabilities (2^-8 of a score of size 4 is 1.6 % of a probability: 5 % of the norm leaves room for two layers)."""
    from mojodiffusion_b200.models.text.gpt_oss import GptOssConfig, GptOssEncoder
    from mojodiffusion_b200.models.text.t5 import T5Config, T5Encoder

    torch.manual_seed(0)
    t5 = T5Config(vocab_size=100, d_model=256, d_ff=512, num_layers=2, num_heads=4)
    oss = GptOssConfig(vocab_size=100, hidden_size=256, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2, intermediate_size=128, num_local_experts=4,
                       num_experts_per_tok=2, sliding_window=16)
    ids = torch.randint(0, 100, (2, 70), device=DEV)
    mask = (torch.arange(70, device=DEV)[None] < _ints([70, 31])[:, None]).long()
    for cfg, enc in ((t5, T5Encoder(t5, torch.bfloat16, DEV)), (oss, GptOssEncoder(oss, torch.bfloat16, DEV))):
        want = enc(ids, mask)
        cfg.fused_attention = True
        before = torch.ops.mdb200.launch_count()
        got = enc(ids, mask)
        assert torch.ops.mdb200.launch_count() > before
        kept = mask.bool()
        assert float((got.float() - want.float())[kept].norm() / want.float()[kept].norm()) < 0.05
