"""How the gradients of a packed sequence are rounded does not depend on what is packed with it."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from packed_oracle import packed_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _run(rows, lengths, H, G, window, sink):
    cu = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    leaves = [t.clone().requires_grad_() for t in rows[:3]] + ([sink.clone().requires_grad_()] if sink is not None else [])
    out = O.packed_attention(*leaves[:3], torch.tensor(cu, dtype=torch.int32, device=DEV), window, sink_logits=leaves[3] if sink is not None else None)
    return out, torch.autograd.grad(out, leaves, rows[3]), cu


# A result rounded to bf16 once is off by 2^-8 of itself at most, and by 2^-8 / sqrt(12) * sqrt(4/3) = 2^-9.6 on average (mantissas evenly spread: 0.0013; up to 0.0017 as they
# lie nearer to 1). Terms that are rounded to bf16 as well would add as much again, and more for differences of nearly equal terms: 0.0024 to 0.0030.
@pytest.mark.parametrize("short,window", [([2, 3] * 11, None), ([200, 30, 3, 250], None), ([256, 129], 300), ([130, 7], 100)], ids=lambda x: str(x)[:16].replace(" ", ""))
@pytest.mark.parametrize("beside", [[2000], [700, 1500]], ids=lambda x: str(x).replace(" ", ""))
@pytest.mark.parametrize("logits", [False, True])
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (8, 2, 128), (3, 1, 128)])
def test_short_sequences_beside_long_ones(H, G, D, logits, beside, short, window):
    g = torch.Generator(device=DEV).manual_seed(1)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    n, T = sum(short), sum(short) + sum(beside)
    rows = [normal(T, h, D) for h in (H, G, G, H)]
    sink = normal(H) if logits else None
    alone = _run([t[:n] for t in rows], short, H, G, window, sink)
    first = _run(rows, short + beside, H, G, window, sink)
    turned = [torch.cat((t[n:], t[:n])) for t in rows]
    last = _run(turned, beside + short, H, G, window, sink)
    value, _ = packed_oracle(*[t[:n] for t in rows[:3]], alone[2], D ** -0.5, window, rows[3][:n], sink)
    for got, part in ((alone, slice(0, n)), (first, slice(0, n)), (last, slice(T - n, T))):
        assert torch.equal(got[0][part], alone[0]) and torch.equal(got[1][0][part], alone[1][0])      # dk and dv may be added up from other parts
        for name, t in zip(("out", "dq", "dk", "dv"), (got[0], *got[1][:3])):
            want = value[name]
            assert float((t[part].detach().double() - want).norm() / want.norm()) < 0.0019, name
    O.check_status()
