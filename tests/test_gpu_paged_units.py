"""Attention over pages of 8 bits whose units of values lie far apart, against the definition in 64 bits."""
import pytest
import torch

from mojodiffusion_b200 import ops as O
from paged_oracle import dense, pool, table_of
from test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def _inputs(lengths, Sq, H, G, D, P, seed=0):
    width = max(lengths) // P + 2
    pages = sum(-(-n // P) for n in lengths) + 1
    table = table_of(lengths, P, pages, width)
    (kp, ks), (vp, vs) = pool(pages, G, P, D, True, DEV, seed), pool(pages, G, P, D, True, DEV, seed + 1)
    return table, kp, ks, vp, vs, pages


def _run(q, kp, ks, vp, vs, table, lengths, name):
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out = O.paged_attention(q, kp, vp, table.to(DEV), n, k_scale=ks, v_scale=vs)
    kd, vd = (dense(p, s, table, lengths, max(lengths)) for p, s in ((kp, ks), (vp, vs)))
    check_attention(out, q, kd, vd, lengths, name)
    O.check_status()


# Queries are 1 + noise of 0.1 and keys +-size with noise, so that a row's score of the pages it prefers is 2 size sqrt(D) above the other's: with 4 the others' weight
# is below 2^-92, with 1.3 and heads of 128 about 2^-42, with 0.9 about 2^-29. Scores are sums of 128 products of 7 at most, off by 128 * 2^-23 * 900 * 0.088 = 0.0012 in fp32, so a
# probability by 0.0012 beside the 2^-11 of its rounding to f16 and so is the divisor: together below the 2^-8 that the bound gives a probability.
@pytest.mark.parametrize("size", [4.0, 1.3, 0.9])
@pytest.mark.parametrize("large", ["first", "last", "between"])
@pytest.mark.parametrize("lengths,Sq,H,G,D,P", [([100, 300], 1, 4, 2, 128, 16), ([400], 5, 4, 2, 64, 64), ([900, 130], 1, 8, 2, 64, 32), ([3000], 3, 6, 2, 128, 128), ([1200], 16, 4, 2, 64, 16), ([700], 40, 4, 2, 128, 64)],
                         ids=lambda x: str(x).replace(" ", ""))
def test_units_of_values_far_apart(lengths, Sq, H, G, D, P, large, size):
    """Pages with units 2^30 larger, whose keys the queries hardly see, before, behind and between those that they see."""
    table, kp, ks, vp, vs, pages = _inputs(lengths, Sq, H, G, D, P)
    far = torch.zeros(pages, dtype=torch.bool)
    for b, n in enumerate(lengths):
        count = -(-n // P)
        for i in range(count):
            far[int(table[b, i])] = {"first": i < (count + 1) // 2, "last": i >= count // 2, "between": i % 3 == 1}[large] and count > 1
    sign = torch.where(far, -1.0, 1.0).to(DEV)[:, None, None, None]
    kp.copy_(((sign * size + 0.05 * _normal(*kp.shape, seed=3)) * 32).to(kp.dtype))
    ks.fill_(127 - 5)
    vs.copy_(torch.where(far.to(DEV)[:, None], 150, 120).expand_as(vs))
    q = (1 + 0.1 * _normal(len(lengths), Sq, H, D, seed=4)).to(torch.bfloat16)
    _run(q, kp, ks, vp, vs, table, lengths, f"{large} {size}")


@pytest.mark.parametrize("lengths,Sq,H,G,D,P", [([100, 5, 0], 1, 4, 2, 128, 16), ([500], 4, 4, 2, 64, 32), ([5000, 700], 1, 8, 4, 128, 16), ([2000, 33], 7, 4, 2, 64, 64)], ids=lambda x: str(x).replace(" ", ""))
def test_units_of_all_sizes(lengths, Sq, H, G, D, P):
    """Units drawn from 2^-60 to 2^60: the largest values seen make up the output, wherever they are."""
    table, kp, ks, vp, vs, _ = _inputs(lengths, Sq, H, G, D, P, seed=5)
    vs.copy_(torch.randint(67, 188, vs.shape, generator=torch.Generator().manual_seed(6), dtype=torch.uint8))
    q = _normal(len(lengths), Sq, H, D, seed=7).to(torch.bfloat16)
    _run(q, kp, ks, vp, vs, table, lengths, "all sizes")


@pytest.mark.parametrize("first,then", [(0, 120), (120, 0), (0, 200), (1, 240), (240, 1), (0, 1)])
@pytest.mark.parametrize("D,P,length", [(128, 16, 90), (64, 64, 700)])
def test_least_and_largest_bytes(D, P, length, first, then):
    """A byte of 0 stands for 2^-127: beside any other page what it holds counts for nothing. Values of 448 * 2^113 are within the range of bf16."""
    table, kp, ks, vp, vs, pages = _inputs([length], 1, 4, 2, D, P, seed=8)
    count = -(-length // P)
    for i in range(count):
        vs[int(table[0, i])] = first if i < (count + 1) // 2 else then
    q = _normal(1, 1, 4, D, seed=9).to(torch.bfloat16)
    _run(q, kp, ks, vp, vs, table, [length], f"{first} {then}")
