"""The language models' attention at its edges on the GPU: long streams."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from text_attention_oracle import check, oracle, seen_by

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(*shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _inputs(B, Sq, Skv, H, G, D, seed):
    return _normal(B, Sq, H, D, seed=seed), _normal(B, Skv, G, D, seed=seed + 1), _normal(B, Skv, G, D, seed=seed + 2)


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_of_long_streams(D):
    """Several hundred CTAs that stream up to 24 tiles for each of two heads, again and again: no wait runs out, and the bits stay."""
    B, S, H, G = 2, 1500, 24, 12
    q, k, v = (t.requires_grad_() for t in _inputs(B, S, S, H, G, D, seed=400))
    grad = _normal(B, S, H, D, seed=403)
    value, bound = oracle(q, k, v, D ** -0.5, seen_by(S, S, B), grad)
    step = lambda: dict(zip(("out", "dq", "dk", "dv"), (out := O.window_attention(q, k, v), *torch.autograd.grad(out, [q, k, v], grad))))
    first = step()
    check(first, value, bound, f"{D}")
    for _ in range(20):
        assert all(torch.equal(t, first[name]) for name, t in step().items())
    O.check_status(q)
