"""Attention over packed sequences on the GPU, against its definition in 64 bits."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from packed_oracle import packed_oracle
from text_attention_oracle import check

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(*shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _ends(lengths, first=0):
    return [first + sum(lengths[:i]) for i in range(len(lengths) + 1)]


# lengths, H, Hkv, Dh, window, sink logits, rows before the first and behind the last sequence
CASES = [
    ([1], 4, 4, 64, None, False, 0, 0),
    ([1, 0, 2], 2, 1, 128, None, True, 0, 3),
    ([77, 20, 128, 5], 4, 2, 64, None, False, 0, 0),
    ([77, 20, 128, 5], 4, 2, 128, None, False, 2, 60),
    ([300, 129, 64], 8, 2, 64, 128, True, 0, 0),
    ([300, 129, 64], 6, 2, 128, 100, False, 0, 1),          # three heads to a group: 256 rows of one head at a time
    ([257, 1, 513], 3, 3, 64, None, True, 5, 0),
    ([700, 130], 2, 1, 128, 1, False, 0, 0),
    ([700, 130], 7, 1, 128, 200, True, 0, 0),
    ([0, 0, 900, 0], 4, 4, 64, None, False, 0, 0),
    ([1300], 4, 2, 128, None, False, 0, 130),
    ([n % 50 + (n % 7 == 0) * 140 for n in range(33)], 4, 2, 64, None, True, 0, 2),         # more sequences than lanes
    ([n % 50 + (n % 7 == 0) * 140 for n in range(70)], 2, 2, 128, 64, False, 1, 2),
    ([0] * 40 + [200, 3], 4, 1, 64, None, False, 0, 0),
    ([4] * 200, 3, 1, 64, None, False, 0, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "")[:20] for x in c))
def test_values_and_gradients(case):
    lengths, H, G, D, window, logits, before, spare = case
    cu = _ends(lengths, before)
    T = cu[-1] + spare
    rows = _normal(T, H + 2 * G, D, seed=1)                      # as a projection leaves them
    grad = _normal(T, H, D, seed=2)
    for lo, hi in ((0, before), (cu[-1], T)):                    # rows of no sequence may hold anything
        rows[lo:hi] = torch.nan
        grad[lo:hi] = torch.nan
    q, k, v = (t.detach().requires_grad_() for t in rows.split([H, G, G], 1))
    sink = _normal(H, seed=3).requires_grad_() if logits else None
    clean = lambda t: torch.nan_to_num(t.detach())
    value, bound = packed_oracle(clean(q), clean(k), clean(v), cu, D ** -0.5, window, clean(grad), sink)
    with torch.no_grad():
        alone = O.packed_attention(q, k, v, _ints(cu), window, sink_logits=sink)
    check(dict(out=alone), dict(out=value["out"]), dict(out=bound["out"]), f"{case} without gradients")
    out = O.packed_attention(q, k, v, _ints(cu), window, sink_logits=sink)
    assert not alone[:before].any() and not alone[cu[-1]:].any()
    for lo, hi in zip(cu[:-1], cu[1:]):         # rows of few keys may keep more of the probabilities when a backward pass follows; the others have the same bits
        assert window is not None and window <= 256 or torch.equal(out[lo + 256:hi], alone[lo + 256:hi])
    got = dict(zip(("dq", "dk", "dv", "dsink"), torch.autograd.grad(out, [q, k, v] + ([sink] if logits else []), grad)))
    check(dict(out=out) | got, value, bound, str(case))
    for t in (out, got["dq"], got["dk"], got["dv"]):
        assert not t[:before].any() and not t[cu[-1]:].any()
    O.check_status()


@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (4, 2, 128), (3, 1, 128)])
def test_sequences_do_not_see_one_another(H, G, D):
    """A sequence of NaN leaves the others' values and gradients as they were, bit for bit."""
    lengths = [40, 100, 30, 500, 7]
    cu = _ends(lengths)
    q, k, v, grad = _normal(cu[-1], H, D, seed=1), _normal(cu[-1], G, D, seed=2), _normal(cu[-1], G, D, seed=3), _normal(cu[-1], H, D, seed=4)

    def run(bad):
        t = [x.clone() for x in (q, k, v, grad)]
        if bad is not None:
            for x in t:
                x[cu[bad]:cu[bad + 1]] = torch.nan
        t[:3] = [x.requires_grad_() for x in t[:3]]
        out = O.packed_attention(*t[:3], _ints(cu))
        return out, *torch.autograd.grad(out, t[:3], t[3])

    good = run(None)
    for bad in range(len(lengths)):
        for a, b in zip(good, run(bad)):
            for i, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
                if i == bad:
                    assert torch.isnan(b[lo:hi]).all()
                else:
                    assert torch.equal(a[lo:hi], b[lo:hi]), (bad, i)


def test_same_as_a_padded_batch():
    """A sequence's bits do not depend on what is packed with it, and equal those of window_attention."""
    lengths, H, G, D = [77, 300, 128], 4, 2, 128
    cu = _ends(lengths)
    q, k, v = _normal(cu[-1], H, D, seed=1), _normal(cu[-1], G, D, seed=2), _normal(cu[-1], G, D, seed=3)
    out = O.packed_attention(q, k, v, _ints(cu))
    for lo, hi in zip(cu[:-1], cu[1:]):
        assert torch.equal(O.packed_attention(q[lo:hi], k[lo:hi], v[lo:hi], _ints([0, hi - lo])), out[lo:hi])
        assert torch.equal(O.window_attention(q[None, lo:hi], k[None, lo:hi], v[None, lo:hi])[0], out[lo:hi])


def test_refuses_what_the_cpu_refuses():
    from test_cpu_packed_attention import BAD

    a = dict(q=_normal(7, 4, 64, seed=0), k=_normal(7, 2, 64, seed=1), v=_normal(7, 2, 64, seed=2), cu_seqlens=_ints([0, 3, 7]))
    O.packed_attention(**a)
    for bad in BAD[:12]:
        with pytest.raises(ValueError):
            O.packed_attention(**(a | {n: (x := f(a)).to(DEV) if isinstance(x := f(a), torch.Tensor) else x for n, f in bad.items()}))
    with pytest.raises(ValueError):
        O.packed_attention(**(a | dict(cu_seqlens=a["cu_seqlens"].cpu())))
    # lengths that lie outside the rows are held within them: nothing outside is read
    good = O.packed_attention(a["q"], a["k"], a["v"], _ints([0, 3, 7]))
    assert torch.equal(O.packed_attention(a["q"], a["k"], a["v"], _ints([-4, 3, 1000])), good)
    out = O.packed_attention(a["q"].requires_grad_(), a["k"], a["v"], a["cu_seqlens"])
    d, = torch.autograd.grad(out.sum(), a["q"], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()


def test_more_than_32_bits_of_elements():
    """2400 sequences whose rows reach beyond 2^31 elements: the last ones as by themselves."""
    B, n, H, G, D = 2400, 131, 64, 1, 128
    T = B * n
    assert T * H * D > 1 << 31
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV) * n
    q = torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEV)
    k, v = _normal(T, G, D, seed=2), _normal(T, G, D, seed=3)
    grad = torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEV)
    last = slice(T - 3 * n, T)
    q[last], grad[last] = _normal(3 * n, H, D, seed=1), _normal(3 * n, H, D, seed=4)

    def run(rows, cu):
        x = [t[rows].clone().requires_grad_() for t in (q, k, v)]
        out = O.packed_attention(*x, cu)
        return out, *torch.autograd.grad(out, x, grad[rows])

    small = run(last, _ints([0, n, 2 * n, 3 * n]))
    large = run(slice(0, T), cu)
    with torch.no_grad():
        alone = O.packed_attention(q, k, v, cu)[last]
        assert torch.equal(alone, O.packed_attention(q[last], k[last], v[last], _ints([0, n, 2 * n, 3 * n])))
    # few blocks of keys are shared by several CTAs, many are not: the sums of dk and dv are added in another order
    assert torch.equal(small[0], large[0][last]) and torch.equal(small[1], large[1][last])
    value, bound = packed_oracle(q[last], k[last], v[last], [0, n, 2 * n, 3 * n], D ** -0.5, None, grad[last])
    check(dict(zip(("out", "dq", "dk", "dv"), (t[last] for t in large))), value, bound, "far")
    O.check_status()
