"""Attention over packed sequences in its torch statement, and what the entry point refuses."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from packed_oracle import packed_oracle


def _ints(v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("cu,spare,window,logits", [([0, 1], 0, None, False), ([0, 5, 5, 12], 3, None, True), ([2, 9, 10], 0, 3, False), ([0, 0], 4, None, True), ([0], 2, None, False)],
                         ids=lambda x: str(x).replace(" ", ""))
def test_values_and_gradients(cu, spare, window, logits):
    g = torch.Generator().manual_seed(0)
    T, H, G, D = cu[-1] + spare, 4, 2, 8
    normal = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
    q, k, v, sink = normal(T, H, D), normal(T, G, D), normal(T, G, D), normal(H) if logits else None
    grad = torch.randn(T, H, D, generator=g, dtype=torch.float64)
    out = O.packed_attention(q, k, v, _ints(cu), window, sink_logits=sink)
    value, _ = packed_oracle(q, k, v, cu, D ** -0.5, window, grad, sink)
    torch.testing.assert_close(out, value["out"])
    leaves = [q, k, v] + ([sink] if logits else [])
    got = torch.autograd.grad(out, leaves, grad, allow_unused=True)
    for n, t in zip(("dq", "dk", "dv", "dsink"), got):
        torch.testing.assert_close(t if t is not None else torch.zeros_like(value[n]), value[n])
    if T and cu[-1] > cu[0]:
        assert torch.autograd.gradcheck(lambda *x: O.packed_attention(x[0], x[1], x[2], _ints(cu), window, sink_logits=x[3] if logits else None), leaves, eps=1e-6, atol=1e-6, fast_mode=True)


BAD = [
    dict(q=lambda a: a["q"][None]), dict(k=lambda a: a["k"][:3]), dict(v=lambda a: a["v"][:, :1]), dict(k=lambda a: a["k"][:, :, :4], v=lambda a: a["v"][:, :, :4]), dict(q=lambda a: a["q"][:, :3]),
    dict(q=lambda a: a["q"].double()), dict(cu_seqlens=lambda a: a["cu_seqlens"].long()), dict(cu_seqlens=lambda a: _ints([])), dict(cu_seqlens=lambda a: _ints([[0, 3]])), dict(window=lambda a: 0),
    dict(window=lambda a: 2.0), dict(sink_logits=lambda a: torch.zeros(3)), dict(cu_seqlens=lambda a: _ints([0, 8])), dict(cu_seqlens=lambda a: _ints([0, 5, 3])), dict(cu_seqlens=lambda a: _ints([-1, 5])),
]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_refuses(i):
    a = dict(q=torch.randn(7, 4, 8), k=torch.randn(7, 2, 8), v=torch.randn(7, 2, 8), cu_seqlens=_ints([0, 3, 7]))
    assert O.packed_attention(**a).shape == (7, 4, 8)
    with pytest.raises(ValueError):
        O.packed_attention(**(a | {n: f(a) for n, f in BAD[i].items()}))
