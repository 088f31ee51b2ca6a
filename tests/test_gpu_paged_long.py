"""Attention over pages where a CTA has many tiles of several sequences, and its join in captured graphs and on several streams."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from paged_oracle import angles, dense, pool, table_of
from test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
LENGTHS = [20000, 0, 17, 13001, 9999, 128, 16384, 12345, 1000, 19991]


# about 92600 positions: 735 tiles of 128 keys for each of 8 or 16 key heads, on 296 or 444 CTAs
@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("Sq,H,G,D,P", [(1, 16, 8, 128, 16), (1, 16, 8, 128, 64), (5, 16, 8, 128, 16), (1, 16, 16, 64, 16), (5, 16, 16, 64, 64), (3, 32, 8, 64, 128), (2, 24, 8, 128, 32)], ids=lambda x: str(x))
def test_many_tiles_to_a_cta(Sq, H, G, D, P, eight):
    width = max(LENGTHS) // P + 2
    pages = sum(-(-n // P) for n in LENGTHS) + 1
    table = table_of(LENGTHS, P, pages, width)
    (kp, ks), (vp, vs) = pool(pages, G, P, D, eight, DEV, 1), pool(pages, G, P, D, eight, DEV, 2)
    q = torch.randn(len(LENGTHS), Sq, H, D, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(torch.bfloat16)
    # scores with a spread of 2: references are raised now and then along a sequence
    q *= 2
    n = torch.tensor(LENGTHS, dtype=torch.int32, device=DEV)
    out = O.paged_attention(q, kp, vp, table.to(DEV), n, k_scale=ks, v_scale=vs)
    for b, length in enumerate(LENGTHS):
        if not length:
            assert not out[b].any()
            continue
        kd, vd = (dense(p, s, table[b:b + 1], [length], length) for p, s in ((kp, ks), (vp, vs)))
        check_attention(out[b:b + 1], q[b:b + 1], kd, vd, [length], f"sequence {b}")
    O.check_status()


def _step_inputs(B, H, G, D, P, most):
    g = torch.Generator(device=DEV).manual_seed(5)
    width = most // P + 1
    (kp, ks), (vp, vs) = pool(B * width + 1, G, P, D, True, DEV, 0), pool(B * width + 1, G, P, D, True, DEV, 1)
    table = torch.randperm(kp.shape[0], generator=g, device=DEV)[:B * width].view(B, width).int()
    cos, sin = angles(most + 8, D, DEV)
    qkv = torch.randn(B, H + 2 * G, D, generator=g, device=DEV).bfloat16()
    return qkv, (H, G), kp, vp, ks, vs, table, cos, sin


def _step(qkv, heads, kp, vp, ks, vs, table, cos, sin, start):
    q, k, v = qkv.split([heads[0], heads[1], heads[1]], 1)
    q = O.paged_append(k, v, kp, vp, table, start, cos, sin, k_scale=ks, v_scale=vs, q=q)
    return O.paged_attention(q[:, None], kp, vp, table, start + 1, k_scale=ks, v_scale=vs)[:, 0]


def _starts(x, most, first=0):
    B = x[0].shape[0]
    return torch.tensor([first + (most - first - 1) * i // max(B - 1, 1) for i in range(B)], dtype=torch.int32, device=DEV)


def test_captured_steps_with_parts_to_join_share_a_pool():
    """Two graphs, captured from one pool of workspaces and replayed in turn, one with many parts to a row: what eager calls give, whatever the lengths are at the replay."""
    a, b = _step_inputs(5, 8, 2, 128, 16, 4000), _step_inputs(1, 4, 4, 64, 64, 60000)
    eager = [[t.clone() if isinstance(t, torch.Tensor) else t for t in x] for x in (a, b)]
    starts = [_starts(a, 3000), _starts(b, 100, 90)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, s in zip((a, b), starts):
            _step(*[t.clone() if isinstance(t, torch.Tensor) else t for t in x], s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, handle = [], [], torch.cuda.graph_pool_handle()
    for x, s in zip((a, b), starts):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=handle):
            outs.append(_step(*x, s))
        graphs.append(graph)
    g = torch.Generator(device=DEV).manual_seed(9)
    for n in range(30):
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
            s += 1 + (1990 if s is starts[1] else 30) * torch.ones_like(s)
    O.check_status()


def test_streams_at_once_with_parts_to_join():
    inputs = [_step_inputs(1 + 2 * i, 8, 2, 128 if i % 2 else 64, 32, 3000 + 9000 * (2 - i)) for i in range(3)]
    starts = [_starts(x, 2900) for x in inputs]
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
