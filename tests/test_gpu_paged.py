"""Paged caches on the GPU, against their definitions in 64 bits."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from paged_oracle import angles, check_append, dense, pool, table_of
from text_attention_oracle import FINE, HALF, oracle, seen_by

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(*shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# starts, lengths, H, Hkv, Dh, P, 8 bits, norm, rows behind the last sequence
APPEND = [
    ([0], [1], 2, 1, 64, 16, True, True, 0),
    ([300], [1], 16, 8, 128, 64, True, True, 0),
    ([300], [1], 28, 4, 128, 64, False, True, 0),
    (list(range(0, 130, 2)), [1] * 65, 8, 2, 128, 32, True, False, 0),
    (list(range(0, 130, 2)), [1] * 65, 8, 2, 64, 16, True, True, 0),
    ([5, 0, 64], [200, 1, 64], 4, 4, 128, 64, True, True, 5),
    ([5, 0, 64], [200, 1, 64], 4, 2, 128, 128, True, False, 0),
    ([0, 7, 3, 0], [33, 0, 20, 0], 4, 4, 64, 16, True, True, 3),
    ([100, 127, 0], [300, 2, 128], 2, 1, 64, 128, True, True, 1),
    ([30, 0], [70, 5], 6, 2, 64, 32, False, True, 0),
    ([30, 0], [170, 257], 6, 2, 128, 128, False, False, 70),
    ([15, 16, 17, 0], [1, 17, 2, 48], 2, 2, 128, 16, True, False, 1),
    ([i % 37 for i in range(70)], [i % 5 for i in range(70)], 3, 1, 64, 16, True, True, 2),
]


def _append_inputs(case, seed=1):
    start, lengths, H, G, D, P, eight, norm, spare = case
    cu = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    T = cu[-1] + spare
    rows = _normal(T, H + 2 * G, D, seed=seed)                  # as a projection leaves them
    q, k, v = rows.split([H, G, G], 1)
    q[cu[-1]:] = torch.nan                                       # rows of no sequence are not read
    k[cu[-1]:] = torch.nan
    ends = [a + b for a, b in zip(start, lengths)]
    width = max(ends) // P + 2
    pages = sum(-(-n // P) for n in ends) + 2
    (kp, ks), (vp, vs) = pool(pages, G, P, D, eight, DEV, 2), pool(pages, G, P, D, eight, DEV, 3)
    cos, sin = angles(max(ends) + 1, D, DEV)
    w = [(1 + 0.2 * torch.randn(D, generator=torch.Generator().manual_seed(i))).to(torch.bfloat16) for i in range(2)] if norm else [None, None]
    return q, k, v, cu, kp, vp, ks, vs, table_of(ends, P, pages, width), cos, sin, *w


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace(" ", "")[:24] for x in c))
def test_append(case):
    start, lengths, *_, spare = case
    q, k, v, cu, kp, vp, ks, vs, table, cos, sin, qn, kn = _append_inputs(case)
    before = [None if t is None else t.clone() for t in (kp, vp, ks, vs)]
    single = lengths == [1] * len(lengths) and spare == 0
    on = lambda w: None if w is None else w.to(DEV)
    out = O.paged_append(k, v, kp, vp, table.to(DEV), _ints(start), cos, sin, cu_seqlens=None if single else _ints(cu), k_scale=ks, v_scale=vs, q=q, q_norm=on(qn), k_norm=on(kn))
    check_append(before, (kp, vp, ks, vs), out, k, v, q, table, start, cu, cos, sin, qn, kn, 1e-6, str(case))
    O.check_status()
    if single:                                                   # the same rows, with their lengths given
        again = [None if t is None else t.clone() for t in before]
        out2 = O.paged_append(k, v, again[0], again[1], table.to(DEV), _ints(start), cos, sin, cu_seqlens=_ints(cu), k_scale=again[2], v_scale=again[3], q=q, q_norm=on(qn), k_norm=on(kn))
        assert torch.equal(out, out2)
        for a, b in zip(again, (kp, vp, ks, vs)):
            assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # without queries, and with weights in fp32; with the keys
    again = [None if t is None else t.clone() for t in before]
    none, keys = O.paged_append(k, v, again[0], again[1], table.to(DEV), _ints(start), cos, sin, cu_seqlens=None if single else _ints(cu), k_scale=again[2], v_scale=again[3],
                                k_norm=None if kn is None else on(kn).float(), keys=True)
    assert none is None
    check_append(before, again, None, k, v, None, table, start, cu, cos, sin, None, kn, 1e-6, str(case), k_out=keys)
    for a, b in zip(again, (kp, vp, ks, vs)):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("eight", [True, False])
def test_append_rows_of_no_sequence(eight):
    q, k, v = (_normal(90, n, 64, seed=n) for n in (6, 2, 2))
    for t in (q, k, v):
        t[:20] = t[75:] = torch.nan
    (kp, ks), (vp, vs) = pool(6, 2, 16, 64, eight, DEV, 2), pool(6, 2, 16, 64, eight, DEV, 3)
    cos, sin = angles(60, 64, DEV)
    out, keys = O.paged_append(k, v, kp, vp, _ints([[1, 2, 4, 0], [0, 3, 0, 0]]), _ints([0, 3]), cos, sin, cu_seqlens=_ints([20, 60, 75]), k_scale=ks, v_scale=vs, q=q, keys=True)
    for t in (out, keys):
        assert not t[:20].any() and not t[75:].any() and torch.isfinite(t).all()
    part = O.paged_append(k[20:75], v[20:75], kp, vp, _ints([[1, 2, 4, 0], [0, 3, 0, 0]]), _ints([0, 3]), cos, sin, cu_seqlens=_ints([0, 40, 55]), k_scale=ks, v_scale=vs, q=q[20:75], keys=True)
    assert torch.equal(part[0], out[20:75]) and torch.equal(part[1], keys[20:75])
    O.check_status()


def test_append_values_that_are_not_finite_and_later_larger_ones():
    P, D, G = 16, 64, 2
    (kp, ks), (vp, vs) = pool(3, G, P, D, True, DEV, 0), pool(3, G, P, D, True, DEV, 1)
    cos, sin = angles(40, D, DEV)
    table, start = _ints([[2, 0]]), 0
    for n, (scale, put) in enumerate([(1e-3, {}), (1.0, {3: float("inf"), 40: float("nan")}), (50.0, {0: float("-inf")}), (0.0, {}), (2e30, {}), (1e-30, {})]):
        rows = 3 if n % 2 else 4
        k, v = (_normal(rows, G, D, seed=10 * n + i) * scale for i in range(2))
        for at, x in put.items():
            v[1, 1, at] = x
        before = [t.clone() for t in (kp, vp, ks, vs)]
        O.paged_append(k, v, kp, vp, table, _ints([start]), cos, sin, cu_seqlens=_ints([0, rows]), k_scale=ks, v_scale=vs)
        check_append(before, (kp, vp, ks, vs), None, k, v, None, table.cpu(), [start], [0, rows], cos, sin, None, None, 1e-6, str(n))
        start += rows
    O.check_status()


# lengths, Sq, H, Hkv, Dh, P, 8 bits
ATTENTION = [
    ([1], 1, 2, 1, 64, 16, True),
    ([1, 0, 16], 1, 4, 4, 128, 16, True),
    ([300], 1, 16, 8, 128, 64, True),
    ([300], 1, 16, 8, 128, 64, False),
    ([5, 0, 640, 63, 64, 65], 1, 8, 2, 64, 16, True),
    ([5, 0, 640, 63, 64, 65], 1, 8, 1, 128, 32, False),
    ([3000, 17, 1025], 1, 28, 4, 128, 64, True),
    ([3000, 17, 1025], 1, 12, 12, 64, 128, True),
    ([n * 7 for n in range(70)], 1, 8, 2, 128, 32, True),
    ([n * 7 for n in range(70)], 2, 4, 2, 64, 64, False),
    ([4, 200, 129], 5, 16, 2, 64, 16, True),          # fewer positions than queries: rows before the first one
    ([8, 700], 8, 64, 8, 128, 64, True),
    ([8, 700], 7, 28, 4, 128, 16, False),
    ([40, 300, 20], 20, 16, 2, 64, 32, True),         # parts of prompts
    ([200, 131], 130, 6, 2, 128, 64, True),
    ([500, 77], 70, 4, 4, 64, 16, False),
    ([1, 0], 33, 8, 2, 128, 128, True),
]


def _attention_inputs(case, seed=4):
    lengths, Sq, H, G, D, P, eight = case
    width = max(lengths) // P + 2
    pages = max(1, sum(-(-n // P) for n in lengths)) + 1
    table = table_of(lengths, P, pages, width)
    (kp, ks), (vp, vs) = pool(pages, G, P, D, eight, DEV, seed), pool(pages, G, P, D, eight, DEV, seed + 1)
    q = _normal(len(lengths), Sq, H, D, seed=seed + 2)
    kd, vd = (dense(p, s, table, lengths, max(lengths)) for p, s in ((kp, ks), (vp, vs)))
    for b, n in enumerate(lengths):                              # slots behind the ends may hold anything
        if n % P:
            kp[int(table[b, n // P]), :, n % P:] = torch.nan
            vp[int(table[b, n // P]), :, n % P:] = torch.nan
    return q, kp, vp, ks, vs, table.to(DEV), kd, vd


def check_attention(out, q, kd, vd, lengths, name):
    """One rounding of the output, and one of the probabilities: to bf16 at most (HALF and FINE: see ``text_attention_oracle``)."""
    B, Sq, H, D = q.shape
    n = _ints(lengths)
    value, bound = oracle(q, kd, vd, D ** -0.5, seen_by(Sq, max(lengths), B, None, 0, n, n - Sq))
    assert torch.isfinite(out).all(), name
    off = (out.double() - value["out"]).abs() - bound["out"]
    assert float(off.max()) <= 1e-30, f"{name}: {float(off.max()):.3g} outside"


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(str(x).replace(" ", "")[:24] for x in c))
def test_attention(case):
    lengths, *_ = case
    q, kp, vp, ks, vs, table, kd, vd = _attention_inputs(case)
    out = O.paged_attention(q, kp, vp, table, _ints(lengths), k_scale=ks, v_scale=vs)
    check_attention(out, q, kd, vd, lengths, str(case))
    bounded = O.paged_attention(q, kp, vp, table, _ints(lengths), k_scale=ks, v_scale=vs, max_len=max(lengths))
    if (max(lengths) <= 512) == (table.shape[1] * kp.shape[2] <= 512):
        assert torch.equal(bounded, out)
    else:       # up to 512 positions a sequence's keys are not shared out, so the sums of one result are added in another order: the same bounds, not the same bits
        check_attention(bounded, q, kd, vd, lengths, str(case))
    strided = torch.stack((q, q), 3)[:, :, :, 0]
    assert torch.equal(O.paged_attention(strided.transpose(1, 2).contiguous().transpose(1, 2), kp, vp, table, _ints(lengths), k_scale=ks, v_scale=vs), out)
    assert torch.equal(O.paged_attention(strided, kp, vp, table, _ints(lengths), k_scale=ks, v_scale=vs), out)
    O.check_status()


def test_attention_max_len_cuts():
    case = ([300, 40, 90], 1, 8, 2, 128, 32, True)
    q, kp, vp, ks, vs, table, kd, vd = _attention_inputs(case)
    out = O.paged_attention(q, kp, vp, table, _ints(case[0]), k_scale=ks, v_scale=vs, max_len=77)
    check_attention(out, q, kd[:, :77], vd[:, :77], [min(n, 77) for n in case[0]], "cut")
    assert not O.paged_attention(q, kp, vp, table, _ints(case[0]), k_scale=ks, v_scale=vs, max_len=0).any()


def test_reports_pages_that_are_not_there():
    """What has no page is skipped and reported; nothing else is written."""
    P, D, G = 16, 64, 2
    (kp, ks), (vp, vs) = pool(4, G, P, D, True, DEV, 0), pool(4, G, P, D, True, DEV, 1)
    cos, sin = angles(64, D, DEV)
    k, v = _normal(2, G, D, seed=2), _normal(2, G, D, seed=3)
    before = [t.clone() for t in (kp, vp, ks, vs)]
    O.check_status()
    for table, start, c, s in (([[4, 1], [-1, 3]], [3, 3], cos, sin), ([[0, 1], [2, 3]], [32, 1 << 30], cos, sin), ([[0, 1], [2, 3]], [5, 9], cos[:5], sin[:5]), ([[0, 1], [2, 3]], [-1, -(1 << 31)], cos, sin)):
        for cu in (None, _ints([0, 1, 2])):
            out = O.paged_append(k, v, kp, vp, _ints(table), _ints(start), c, s, cu_seqlens=cu, k_scale=ks, v_scale=vs, q=k)
            for a, b in zip(before, (kp, vp, ks, vs)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert not out.any()
            with pytest.raises(RuntimeError, match="BOUNDS"):
                O.check_status()
            assert not O.paged_append(k, v, kp, vp, _ints(table), _ints(start), c, s, cu_seqlens=cu, k_scale=ks, v_scale=vs, keys=True)[1].any()
            with pytest.raises(RuntimeError, match="BOUNDS"):
                O.check_status()
    q = _normal(2, 1, 4, D, seed=5)
    good = O.paged_attention(q, kp, vp, _ints([[0, 1], [2, 3]]), _ints([20, 20]), k_scale=ks, v_scale=vs)
    out = O.paged_attention(q, kp, vp, _ints([[0, 1], [2, 77]]), _ints([20, 20]), k_scale=ks, v_scale=vs)
    assert torch.equal(out[0], good[0])
    with pytest.raises(RuntimeError, match="BOUNDS"):
        O.check_status()
    O.check_status()


def test_empty_calls():
    P, D, G = 16, 64, 2
    (kp, ks), (vp, vs) = pool(4, G, P, D, True, DEV, 0), pool(4, G, P, D, True, DEV, 1)
    cos, sin = angles(8, D, DEV)
    none = torch.empty(0, G, D, dtype=torch.bfloat16, device=DEV)
    table0 = torch.empty(0, 3, dtype=torch.int32, device=DEV)
    assert O.paged_append(none, none, kp, vp, table0, _ints([]), cos, sin, k_scale=ks, v_scale=vs, q=none).shape == none.shape
    rows = torch.full((3, G, D), torch.nan, dtype=torch.bfloat16, device=DEV)
    assert not O.paged_append(rows, rows, kp, vp, table0, _ints([]), cos, sin, cu_seqlens=_ints([0]), k_scale=ks, v_scale=vs, q=rows).any()
    assert not O.paged_append(rows, rows, kp, vp, _ints([[0], [1]]), _ints([3, 4]), cos, sin, cu_seqlens=_ints([0, 0, 0]), k_scale=ks, v_scale=vs, q=rows).any()
    assert O.paged_attention(torch.empty(2, 0, 4, D, dtype=torch.bfloat16, device=DEV), kp, vp, _ints([[0], [1]]), _ints([3, 4]), k_scale=ks, v_scale=vs).shape == (2, 0, 4, D)
    assert not O.paged_attention(_normal(2, 1, 4, D, seed=0), kp, vp, _ints([[9], [9]]), _ints([0, -5]), k_scale=ks, v_scale=vs).any()
    assert not O.paged_attention(_normal(2, 40, 4, D, seed=0), kp, vp, torch.empty(2, 0, dtype=torch.int32, device=DEV), _ints([3, 5]), k_scale=ks, v_scale=vs).any()
    O.check_status()


def test_refuses_what_the_cpu_refuses():
    """The calls that the torch statements refuse for their arguments, and layouts that the kernels do not take."""
    from test_cpu_paged import BAD_APPEND, BAD_ATTENTION

    P, G, D, T = 16, 2, 64, 3
    k = _normal(T, G, D, seed=0)
    (kp, ks), (vp, vs) = pool(4, G, P, D, True, DEV, 0), pool(4, G, P, D, True, DEV, 1)
    cos, sin = angles(64, D, DEV)
    base = dict(k=k, v=k.clone(), k_pages=kp, v_pages=vp, block_table=_ints([[0, 1], [2, 3]]), start=_ints([0, 5]), cos=cos, sin=sin, cu_seqlens=_ints([0, 1, 3]), k_scale=ks, v_scale=vs, q=_normal(T, 4, D, seed=1))
    O.paged_append(**base)
    before = [t.clone() for t in (kp, vp, ks, vs)]
    move = lambda t: t.to(DEV) if isinstance(t, torch.Tensor) else t
    wide = torch.zeros(4, G, P, 2 * D, device=DEV).to(torch.float8_e4m3fn)
    for bad in BAD_APPEND[:25] + [dict(k_pages=lambda a: wide[..., :D], v_pages=lambda a: wide[..., :D]), dict(start=lambda a: a["start"].cpu()), dict(q=lambda a: a["q"].cpu()), dict(cos=lambda a: a["cos"].cpu())]:
        with pytest.raises(ValueError):
            O.paged_append(**(base | {n: move(f(base)) if "cpu" not in f.__code__.co_names else f(base) for n, f in bad.items()}))
    base = {n: base[n] for n in ("k_pages", "v_pages", "block_table", "k_scale", "v_scale")} | dict(q=_normal(2, 1, 4, D, seed=2), kv_len=_ints([20, 2]))
    for i, bad in enumerate(BAD_ATTENTION):
        if i not in (13, 14):                                # those are page numbers and lengths, not arguments
            with pytest.raises(ValueError):
                O.paged_attention(**(base | {n: move(f(base)) for n, f in bad.items()}))
    for a, b in zip(before, (kp, vp, ks, vs)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    O.check_status()


@pytest.mark.parametrize("eight", [True, False])
def test_pools_inside_larger_ones(eight):
    """Keys and values of one page next to one another, and scales in a larger array: strides of pages and heads of any size."""
    P, D, G, H, N = 32, 64, 2, 6, 8
    (kp, ks), (vp, vs) = pool(N, G, P, D, eight, DEV, 2), pool(N, G, P, D, eight, DEV, 3)
    both = torch.zeros(N, G, 3, P, D, device=DEV).to(kp.dtype)
    both[:, :, 0], both[:, :, 2] = kp, vp
    scales = torch.zeros(N, 2 * G + 3, dtype=torch.uint8, device=DEV)
    if eight:
        scales[:, 1:1 + G], scales[:, G + 2:2 * G + 2] = ks, vs
    inner = (both[:, :, 0], both[:, :, 2], *((scales[:, 1:1 + G], scales[:, G + 2:2 * G + 2]) if eight else (None, None)))
    cos, sin = angles(200, D, DEV)
    table, start = _ints([[3, 1, 0, 0], [2, 7, 5, 4]]), [20, 60]
    q, k, v = (_normal(50, n, D, seed=n) for n in (H, G, G))
    want = O.paged_append(k, v, kp, vp, table, _ints(start), cos, sin, cu_seqlens=_ints([0, 30, 50]), k_scale=ks, v_scale=vs, q=q)
    got = O.paged_append(k, v, inner[0], inner[1], table, _ints(start), cos, sin, cu_seqlens=_ints([0, 30, 50]), k_scale=inner[2], v_scale=inner[3], q=q)
    assert torch.equal(got, want)
    for a, b in zip(inner, (kp, vp, ks, vs)):
        assert a is None or torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))
    assert not both[:, :, 1].float().any()
    for Sq in (1, 3, 30):
        x = _normal(2, Sq, H, D, seed=9)
        a = O.paged_attention(x, kp, vp, table, _ints([50, 80]), k_scale=ks, v_scale=vs)
        assert torch.equal(O.paged_attention(x, inner[0], inner[1], table, _ints([50, 80]), k_scale=inner[2], v_scale=inner[3]), a)
    O.check_status()


@pytest.mark.parametrize("eight", [True, False])
def test_pools_of_more_than_32_bits(eight):
    """Pages whose elements lie beyond 2^31."""
    P, D, G, H = 64, 128, 2, 8
    N = (1 << 31) // (G * P * D) + 70
    big = [torch.empty(N, G, P, D, dtype=torch.float8_e4m3fn if eight else torch.bfloat16, device=DEV) for _ in range(2)]
    scales = [torch.ones(N, G, dtype=torch.uint8, device=DEV) if eight else None for _ in range(2)]
    (kp, ks), (vp, vs) = pool(6, G, P, D, eight, DEV, 2), pool(6, G, P, D, eight, DEV, 3)
    far = torch.tensor([N - 1, N - 2, 3, N - 60, 0, N - 9], device=DEV)
    for t, s, p, c in zip(big, scales, (kp, vp), (ks, vs)):
        t.view(torch.uint8).index_copy_(0, far, p.view(torch.uint8))
        if eight:
            s[far] = c
    near, distant = _ints([[0, 1, 2], [3, 4, 5]]), far.int().view(2, 3)
    cos, sin = angles(200, D, DEV)
    q, k, v = (_normal(90, n, D, seed=n) for n in (H, G, G))
    calls = [(near, kp, vp, ks, vs), (distant, *big, *scales)]
    got = [O.paged_append(k, v, p, w, table, _ints([30, 100]), cos, sin, cu_seqlens=_ints([0, 40, 90]), k_scale=c, v_scale=d, q=q) for table, p, w, c, d in calls]
    assert torch.equal(*got)
    got = [O.paged_append(k[:2], v[:2], p, w, table, _ints([70, 150]), cos, sin, k_scale=c, v_scale=d, q=q[:2]) for table, p, w, c, d in calls]
    assert torch.equal(*got)
    for t, p in zip((*big, *scales), (kp, vp, ks, vs)):
        assert t is None or torch.equal(t.view(torch.uint8)[far], p.view(torch.uint8))
    for Sq in (1, 5, 40):
        x = _normal(2, Sq, H, D, seed=9)
        got = [O.paged_attention(x, p, w, table, _ints([71, 151]), k_scale=c, v_scale=d) for table, p, w, c, d in calls]
        assert torch.equal(*got)
    O.check_status()


def test_parts_of_prompts_report_pages_that_are_not_there():
    P, D, G = 16, 64, 2
    (kp, ks), (vp, vs) = pool(4, G, P, D, True, DEV, 0), pool(4, G, P, D, True, DEV, 1)
    q = _normal(2, 40, 4, D, seed=5)
    good = O.paged_attention(q, kp, vp, _ints([[0, 1], [2, 3]]), _ints([20, 20]), k_scale=ks, v_scale=vs)
    out = O.paged_attention(q, kp, vp, _ints([[0, 1], [2, -3]]), _ints([20, 20]), k_scale=ks, v_scale=vs)
    assert torch.equal(out[0], good[0])
    with pytest.raises(RuntimeError, match="BOUNDS"):
        O.check_status()
