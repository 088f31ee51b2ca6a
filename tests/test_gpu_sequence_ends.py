"""Ends of packed sequences that fall, or lie outside the rows: an append keeps sequences disjoint and within the rows, attention has none where they fall; such calls are reported."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from paged_oracle import angles, pool

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(torch.bfloat16)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def held(cu, T):
    """The largest end so far, none beyond the last one, all within T rows."""
    cu = [min(max(c, 0), T) for c in cu]
    return [min(max(cu[:i + 1]), cu[-1]) for i in range(len(cu))]


# of 60 rows
ENDS = [[0, 40, 10, 60], [0, 40, 10], [50, 20, 60], [60, 0], [30, 40, 20, 25, 50], [0, 60, 0, 60, 0, 60], list(range(0, 40)) + [5] * 30 + [55, 60], [7 * i % 61 for i in range(1500)] + [50]]
OUTSIDE = [[-5, 30, 70], [70, 80, 90], [0, 1 << 30], [-(1 << 31), 20, 60]]


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("D,P", [(64, 16), (128, 32), (64, 64)])
@pytest.mark.parametrize("cu", ENDS + OUTSIDE, ids=lambda c: str(c[:6]).replace(" ", ""))
def test_append(cu, D, P, eight):
    T, H, G, B = 60, 4, 2, len(cu) - 1
    width = 80 // P + 1
    q, k, v = (_normal(T, n, D, seed=n) for n in (H, G, G))
    start = _ints([(7 * b) % 19 for b in range(B)])
    table = torch.arange(B * width, dtype=torch.int32, device=DEV).view(B, width)
    cos, sin = angles(100, D, DEV)
    O.check_status()
    found = []
    for ends in (held(cu, T), cu):
        (kp, ks), (vp, vs) = pool(B * width, G, P, D, eight, DEV, 2), pool(B * width, G, P, D, eight, DEV, 3)
        out, keys = O.paged_append(k, v, kp, vp, table, start, cos, sin, cu_seqlens=_ints(ends), k_scale=ks, v_scale=vs, q=q, keys=True)
        (kp2, ks2), (vp2, vs2) = pool(B * width, G, P, D, eight, DEV, 2), pool(B * width, G, P, D, eight, DEV, 3)
        if ends is cu:
            with pytest.raises(RuntimeError, match="BOUNDS"):
                O.check_status()
        O.check_status()
        assert O.paged_append(k, v, kp2, vp2, table, start, cos, sin, cu_seqlens=_ints(ends), k_scale=ks2, v_scale=vs2) is None
        if ends is cu:
            with pytest.raises(RuntimeError, match="BOUNDS"):
                O.check_status()
        found.append([t.view(torch.uint8) for t in (out, keys, kp, vp, ks, vs, kp2, vp2, ks2, vs2) if t is not None])
    for a, b in zip(*found):
        assert torch.equal(a, b)


@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (4, 2, 128), (3, 1, 128)])
@pytest.mark.parametrize("scale", [1, 9])
@pytest.mark.parametrize("cu", ENDS + OUTSIDE, ids=lambda c: str(c[:6]).replace(" ", ""))
def test_packed_attention(cu, scale, H, G, D):
    T = 60 * scale                                              # with 9, sequences of several tiles
    cu = [c * scale if abs(c) < 1 << 20 else c for c in cu]
    q, k, v, grad, sink = _normal(T, H, D, seed=1), _normal(T, G, D, seed=2), _normal(T, G, D, seed=3), _normal(T, H, D, seed=4), _normal(H, seed=5)
    O.check_status()

    inside = [min(max(c, 0), T) for c in cu]
    falls = inside != sorted(inside)

    def reports(bad):
        if bad:
            with pytest.raises(RuntimeError, match="BOUNDS"):
                O.check_status()
        O.check_status()

    found = []
    for ends in (inside, cu):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, sink)]
        with torch.no_grad():
            alone = O.packed_attention(*leaves[:3], _ints(ends), sink_logits=leaves[3])
        reports(falls)
        out = O.packed_attention(*leaves[:3], _ints(ends), sink_logits=leaves[3])
        reports(falls)
        grads = torch.autograd.grad(out, leaves, grad)
        reports(falls)
        found.append((alone, out, *grads))
    for a, b in zip(*found):
        assert torch.equal(a, b) and torch.isfinite(b).all()
        assert not (falls and b.any())


@pytest.mark.parametrize("B", [20, 45])
def test_captured_training_step_follows_the_ends(B):
    """A captured step replayed with other ends, falling ones among them: what an eager call gives."""
    T, H, G, D = 700, 4, 2, 128
    q, k, v, grad = (_normal(T, n, D, seed=n + i) for i, n in enumerate((H, G, G, H)))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV)

    def step():
        out = O.packed_attention(*leaves, cu)
        return (out.detach(), *torch.autograd.grad(out, leaves, grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    O.check_status()
    g = torch.Generator().manual_seed(3)
    for n in range(12):
        ends = torch.sort(torch.randint(0, T + 1, (B + 1,), generator=g)).values.int()
        if n % 4 == 1:
            ends = torch.where(torch.rand(B + 1, generator=g) < 0.7, 650, ends).sort().values.int()      # a long one and short ones
        if n % 4 == 3:
            ends[B // 2] = 0
            ends[0] = 1
        cu.copy_(ends)
        graph.replay()
        if n % 4 == 3:
            with pytest.raises(RuntimeError, match="BOUNDS"):
                O.check_status()
        O.check_status()
        want = step()
        if n % 4 == 3:
            with pytest.raises(RuntimeError, match="BOUNDS"):
                O.check_status()
        for a, b in zip(got, want):
            assert torch.equal(a, b), n


def test_many_sequences_on_several_streams():
    """Each call has its own list of units."""
    cases = []
    for i in range(3):
        lengths = [(j * (7 + i)) % 60 for j in range(40 + 300 * i)]
        cu = _ints([sum(lengths[:j]) for j in range(len(lengths) + 1)])
        cases.append((*(_normal(sum(lengths), n, 64, seed=10 * i + n) for n in (4, 2)), _normal(sum(lengths), 2, 64, seed=10 * i + 9), cu))
    want = [O.packed_attention(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        got = []
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(O.packed_attention(*c))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    O.check_status()
