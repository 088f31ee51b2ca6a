"""Paged caches in their torch statements, the refusals of their entry points, and bad pages."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from paged_oracle import angles, check_append, dense, pool, table_of
from text_attention_oracle import oracle, seen_by


def _ints(v):
    return torch.tensor(v, dtype=torch.int32)


# B's starts and lengths, H, Hkv, D, P, 8 bits, norm, rows behind the last sequence
APPEND = [
    ([0], [1], 2, 1, 64, 16, True, True, 0),
    ([5, 0, 16, 31], [1, 1, 1, 1], 4, 2, 128, 16, True, False, 0),
    ([0, 7, 3], [33, 0, 20], 4, 4, 64, 16, True, True, 3),
    ([30, 0], [70, 5], 6, 2, 64, 32, False, True, 0),
    ([15, 16, 17, 0], [1, 17, 2, 48], 2, 2, 16, 16, True, False, 1),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_append(case):
    start, lengths, H, G, D, P, eight, norm, spare = case
    g = torch.Generator().manual_seed(1)
    cu = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    T = cu[-1] + spare
    q, k, v = (torch.randn(T, n, D, generator=g).to(torch.bfloat16) for n in (H, G, G))
    ends = [a + b for a, b in zip(start, lengths)]
    width = max(ends) // P + 2
    pages = sum(-(-n // P) for n in ends) + 2
    table = table_of(ends, P, pages, width)
    (kp, ks), (vp, vs) = pool(pages, G, P, D, eight, "cpu", 2), pool(pages, G, P, D, eight, "cpu", 3)
    cos, sin = angles(max(ends) + 1, D, "cpu")
    qn, kn = ((1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16) for _ in range(2)) if norm else (None, None)
    before = [None if t is None else t.clone() for t in (kp, vp, ks, vs)]
    packed = None if lengths == [1] * len(lengths) and spare == 0 else _ints(cu)
    out = O.paged_append(k, v, kp, vp, table, _ints(start), cos, sin, cu_seqlens=packed, k_scale=ks, v_scale=vs, q=q, q_norm=qn, k_norm=kn)
    check_append(before, (kp, vp, ks, vs), out, k, v, q, table, start, cu, cos, sin, qn, kn, 1e-6, str(case))


def test_append_rows_of_no_sequence():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(9, n, 16, generator=g) for n in (2, 1, 1))
    q[[0, 1, 8]] = k[[0, 1, 8]] = torch.nan
    (kp, ks), (vp, vs) = pool(2, 1, 16, 16, True, "cpu", 2), pool(2, 1, 16, 16, True, "cpu", 3)
    cos, sin = angles(20, 16, "cpu")
    out, keys = O.paged_append(k, v, kp, vp, _ints([[1], [0]]), _ints([0, 3]), cos, sin, cu_seqlens=_ints([2, 5, 8]), k_scale=ks, v_scale=vs, q=q, keys=True)
    for t in (out, keys):
        assert not t[:2].any() and not t[8:].any() and torch.isfinite(t).all() and t[2:8].all()


def test_append_scale_values():
    """Zeros, values at the border of a scale, infinities and NaN; a larger token later, and a new owner of a page."""
    P, D = 16, 16
    kp, ks = torch.zeros(2, 1, P, D).to(torch.float8_e4m3fn), torch.full((2, 1), 200, dtype=torch.uint8)
    vp, vs = kp.clone(), ks.clone()
    cos, sin = torch.ones(40, D // 2), torch.zeros(40, D // 2)
    table = _ints([[1, 0]])

    def put(values, at):
        x = torch.zeros(1, 1, D)
        x[0, 0, :len(values)] = torch.tensor(values)
        O.paged_append(x, x, kp, vp, table, _ints([at]), cos, sin, k_scale=ks, v_scale=vs)

    put([0.0], 0)
    assert int(ks[1]) == 1 and int(vs[1]) == 1 and int(ks[0]) == 200           # the page's old scale does not count
    put([448.0, 2.0 ** -9, 1e-12], 1)
    assert int(ks[1]) == 127 and kp[1, 0, 1, :3].float().tolist() == [448.0, 2.0 ** -9, 0.0]
    put([449.0, float("inf"), float("-inf"), float("nan")], 2)
    assert int(ks[1]) == 128 and kp[1, 0, 2, 0].float() == 224.0 and torch.isnan(kp[1, 0, 2, 1:4].float()).all()
    assert kp[1, 0, 1, :2].float().tolist() == [224.0, 0.0]                     # half a step below the least: to even
    put([3e38], 3)
    assert int(ks[1]) == 127 + 120 and float(kp[1, 0, 3, 0].float() * 2.0 ** 120) == pytest.approx(3e38, rel=2 ** -4)


ATTENTION = [
    ([1], 1, 2, 1, 16, 16, True),
    ([5, 0, 40], 1, 4, 2, 64, 16, True),
    ([17, 2, 33], 3, 4, 4, 16, 32, False),
    ([70, 64], 40, 6, 2, 16, 16, True),
]


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_attention(case):
    lengths, Sq, H, G, D, P, eight = case
    width = max(lengths) // P + 2
    pages = sum(-(-n // P) for n in lengths) + 1
    table = table_of(lengths, P, pages, width)
    (kp, ks), (vp, vs) = pool(pages, G, P, D, eight, "cpu", 4), pool(pages, G, P, D, eight, "cpu", 5)
    q = torch.randn(len(lengths), Sq, H, D, generator=torch.Generator().manual_seed(6))
    kp, vp = (kp, vp) if eight else (kp.float(), vp.float())
    kd, vd = (dense(p, s, table, lengths, max(lengths)) for p, s in ((kp, ks), (vp, vs)))
    n = _ints(lengths)
    value, _ = oracle(q, kd, vd, D ** -0.5, seen_by(Sq, max(lengths), len(lengths), None, 0, n, n - Sq))
    # slots behind the ends may hold anything
    for b, length in enumerate(lengths):
        if length % P:
            kp[table[b, length // P], :, length % P:] = torch.nan
            vp[table[b, length // P], :, length % P:] = torch.nan
    out = O.paged_attention(q, kp, vp, table, n, k_scale=ks, v_scale=vs)
    torch.testing.assert_close(out.double(), value["out"], rtol=1e-5, atol=1e-5)
    if max(lengths) > 5:                                  # max_len cuts
        cut = n.clamp(max=5)
        torch.testing.assert_close(O.paged_attention(q, kp, vp, table, n, k_scale=ks, v_scale=vs, max_len=5), O.paged_attention(q, kp, vp, table, cut, k_scale=ks, v_scale=vs))


def _append_args():
    P, G, D, T = 16, 2, 16, 3
    k = torch.randn(T, G, D)
    (kp, ks), (vp, vs) = pool(4, G, P, D, True, "cpu", 0), pool(4, G, P, D, True, "cpu", 1)
    cos, sin = angles(64, D, "cpu")
    return dict(k=k, v=k.clone(), k_pages=kp, v_pages=vp, block_table=_ints([[0, 1], [2, 3]]), start=_ints([0, 5]), cos=cos, sin=sin, cu_seqlens=_ints([0, 1, 3]),
                k_scale=ks, v_scale=vs, q=torch.randn(T, 4, D))


BAD_APPEND = [
    dict(k=lambda a: a["k"][0]), dict(v=lambda a: a["v"][:2]), dict(v=lambda a: a["v"].double()), dict(start=lambda a: a["start"].long()), dict(start=lambda a: a["start"][:1]),
    dict(cu_seqlens=lambda a: None), dict(cu_seqlens=lambda a: _ints([0, 3])), dict(cu_seqlens=lambda a: a["cu_seqlens"].long()), dict(k_scale=lambda a: None),
    dict(k_scale=lambda a: a["k_scale"].float()), dict(v_scale=lambda a: a["v_scale"][:1]), dict(k_pages=lambda a: a["k_pages"].float()), dict(k_pages=lambda a: a["k_pages"][:, :1]),
    dict(k_pages=lambda a: a["k_pages"].transpose(2, 3)), dict(block_table=lambda a: a["block_table"].long()), dict(block_table=lambda a: a["block_table"][:1]), dict(cos=lambda a: a["cos"][:, :4]),
    dict(cos=lambda a: a["cos"].double()), dict(q=lambda a: a["q"][:, :3]), dict(q=lambda a: a["q"][:2]), dict(q=lambda a: a["q"].double()), dict(q_norm=lambda a: torch.ones(3)),
    dict(k_norm=lambda a: torch.ones(16, dtype=torch.int32)), dict(q=lambda a: None, q_norm=lambda a: torch.ones(16)), dict(k=lambda a: a["k"].clone().requires_grad_()),
    # positions without a page, page numbers outside the pool, rows outside the tensor
    dict(start=lambda a: _ints([0, 31])), dict(start=lambda a: _ints([-1, 5])), dict(block_table=lambda a: _ints([[0, 1], [4, 3]])), dict(block_table=lambda a: _ints([[-1, 1], [2, 3]])),
    dict(cu_seqlens=lambda a: _ints([0, 1, 4])), dict(cu_seqlens=lambda a: _ints([0, 2, 1])), dict(cos=lambda a: a["cos"][:6], sin=lambda a: a["sin"][:6]),
]


@pytest.mark.parametrize("i", range(len(BAD_APPEND)))
def test_append_refuses(i):
    args = _append_args()
    assert O.paged_append(**_append_args()).shape == args["q"].shape
    args.update({n: f(args) for n, f in BAD_APPEND[i].items()})
    with pytest.raises(ValueError):
        O.paged_append(**args)


BAD_ATTENTION = [
    dict(q=lambda a: a["q"][0]), dict(q=lambda a: a["q"][:, :, :3]), dict(q=lambda a: a["q"][:1]), dict(q=lambda a: a["q"].int()), dict(kv_len=lambda a: a["kv_len"].long()), dict(kv_len=lambda a: a["kv_len"][:1]),
    dict(k_scale=lambda a: None), dict(max_len=lambda a: -1), dict(max_len=lambda a: 2.0), dict(scale=lambda a: 0.0), dict(scale=lambda a: -1.0), dict(scale=lambda a: float("nan")),
    dict(q=lambda a: a["q"].clone().requires_grad_()), dict(kv_len=lambda a: _ints([33, 2])), dict(block_table=lambda a: _ints([[0, 9], [2, 3]])), dict(k_pages=lambda a: a["k_pages"][..., :8]),
]


@pytest.mark.parametrize("i", range(len(BAD_ATTENTION)))
def test_attention_refuses(i):
    a = _append_args()
    args = {n: a[n] for n in ("k_pages", "v_pages", "block_table", "k_scale", "v_scale")} | dict(q=torch.randn(2, 1, 4, 16), kv_len=_ints([20, 2]))
    assert O.paged_attention(**args).shape == args["q"].shape
    args.update({n: f(args) for n, f in BAD_ATTENTION[i].items()})
    if i == 13:       # beyond the table: cut at what it has room for
        torch.testing.assert_close(O.paged_attention(**args), O.paged_attention(**(args | dict(kv_len=_ints([32, 2])))))
        return
    with pytest.raises(ValueError):
        O.paged_attention(**args)
