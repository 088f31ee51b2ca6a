"""The language models' attention at its edges on the GPU: long streams, scores that are not numbers."""
import math

import pytest
import torch

from mojodiffusion_b200 import ops as O
from mojodiffusion_b200.ops import reference as ref
from text_attention_oracle import FINE, HALF, check, oracle, seen_by

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


BAD = [("key", math.nan), ("key", math.inf), ("query", math.nan), ("query", math.inf)]


def _with_bad_places(bad, B, Sq, Skv, H, G, D, seed):
    """One bad element in one query or in one of sixteen neighbouring keys, a sequence of the batch for each."""
    q, k, v = _inputs(B, Sq, Skv, H, G, D, seed=seed)
    what, value = bad
    for b in range(B):
        if what == "key":
            k[b, 20 + b, :, 5] = value
        else:
            q[b, b % Sq, :, 5] = value
    return q, k, v


def _check_bad(got, want, name):
    """Not a number where the definition in 64 bits is not; elsewhere near it: the products' terms of size 4 and the roundings of outputs of size 1 to 4."""
    lost = torch.isnan(want)
    wrong = int((torch.isnan(got) != lost).sum())
    assert int(lost.sum()) > 0 and wrong == 0, f"{name}: {wrong} values of {lost.numel()}, {int(lost.sum())} of which are lost"
    worst = float(torch.where(lost, 0.0, got.double() - want).abs().max())
    assert worst <= 2 * HALF * 4 + 4 * FINE, f"{name}: {worst}"


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,starts", [(60, 10), (3, 40), (1, 35)])
def test_window_scores_that_are_not_numbers(Sq, starts, D, bad):
    """A prompt and a few tokens over a cache: a query with a score of NaN or +inf among the keys that it sees has no result, and nobody else loses one."""
    B, Skv, H, G, window = 16, 70, 4, 2, 18
    q, k, v = _with_bad_places(bad, B, Sq, Skv, H, G, D, seed=410)
    at = torch.arange(B, device=DEV, dtype=torch.int32) + starts - 10
    want = ref.window_attention(q.double(), k.double(), v.double(), window, 2, q_start=at)
    _check_bad(O.window_attention(q, k, v, window, 2, q_start=at), want, f"{bad} {Sq} {D}")


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("D", [64, 128])
def test_relative_scores_that_are_not_numbers(D, bad):
    B, S, H = 16, 200, 2
    q, k, v = _with_bad_places(bad, B, S, S, H, H, D, seed=420)
    q = q * D ** -0.5
    n = torch.tensor([17 + 5 * b for b in range(B)], dtype=torch.int32, device=DEV)      # some do not reach the bad key
    table = _normal(32, H, seed=423)
    want = ref.relative_attention(q.double(), k.double(), v.double(), table.double(), kv_len=n)
    _check_bad(O.relative_attention(q, k, v, table, kv_len=n), want, f"{bad} {D}")


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_of_scores_that_are_not_numbers(D):
    """The row of a bad query has no gradients, nor have the keys and values that it sees; those of other rows and of keys that no row near it sees are kept."""
    S, H, G, window, bad = 600, 4, 2, 20, 250
    q, k, v = _inputs(1, S, S, H, G, D, seed=430)
    grad = _normal(1, S, H, D, seed=433)
    clean = torch.autograd.grad(O.window_attention(*(leaves := [t.clone().requires_grad_() for t in (q, k, v)]), window), leaves, grad)
    q[:, bad, :, 3] = math.nan
    leaves = [t.requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(O.window_attention(*leaves, window), leaves, grad)
    others = torch.arange(S, device=DEV) != bad
    same = torch.equal(dq[:, others], clean[0][:, others])
    assert same and bool(torch.isnan(dq[:, bad]).all())
    for got, want in ((dk, clean[1]), (dv, clean[2])):
        assert bool(torch.isnan(got[:, bad - window + 1:bad + 1]).all())
        for far in (slice(0, bad - 128 - window), slice(bad + 128 + window, S)):
            same = torch.equal(got[:, far], want[:, far])
            assert same


@pytest.mark.parametrize("case", [(2, 1500, 1800, 4, 2, 64, 100, 300, [300, 100], [1800, 1300]), (2, 1500, 1800, 4, 2, 128, 100, 300, [300, 100], [1800, 1300]),
                                  (1, 900, 1500, 6, 2, 128, 130, 700, [500], [1399]), (1, 1200, 1200, 4, 4, 64, 50, 1199, [0], [1200]),
                                  (4, 700, 700, 32, 32, 128, 100, 600, [0, 0, 3, -9], [700, 650, 700, 0])], ids=str)
def test_gradients_of_many_first_keys(case):
    """Blocks of first keys whose later queries go to slices, with lengths and positions of their own; the last case has enough blocks without them."""
    B, Sq, Skv, H, G, D, window, sinks, at, n = case
    q, k, v = (t.requires_grad_() for t in _inputs(B, Sq, Skv, H, G, D, seed=440))
    at, n = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in (at, n))
    grad = _normal(B, Sq, H, D, seed=443)
    value, bound = oracle(q, k, v, D ** -0.5, seen_by(Sq, Skv, B, window, sinks, n.cpu(), at.cpu()), grad)
    out = O.window_attention(q, k, v, window, sinks, kv_len=n, q_start=at)
    check(dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, [q, k, v], grad)))), value, bound, str(case))


def _backward_memory(window, sinks, B, S, H, G, D):
    q, k, v = (t.requires_grad_() for t in _inputs(B, S, S, H, G, D, seed=450))
    out = O.window_attention(q, k, v, window, sinks)
    grad = _normal(B, S, H, D, seed=453)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(out, [q, k, v], grad)
    torch.cuda.synchronize()
    return grads, torch.cuda.max_memory_allocated() - before - sum(t.nbytes for t in grads)


def test_workspace_of_many_first_keys():
    """160 MB at most, beside the gradients and 4 bytes for each row of each head; and as many first keys as keys are no window at all."""
    B, S, H, G, D = 1, 8192, 32, 8, 128
    _, extra = _backward_memory(256, 2048, B, S, H, G, D)
    assert extra <= 160e6 + 4 * B * S * H
    plain, none = _backward_memory(None, 0, B, S, H, G, D)
    for sinks in (S, 1 << 40):
        grads, extra = _backward_memory(128, sinks, B, S, H, G, D)
        same = all(torch.equal(a, b) for a, b in zip(grads, plain))
        assert same and extra <= none


def _calls_with_out():
    q, k, v = _inputs(2, 150, 150, 4, 2, 64, seed=460)
    table = _normal(32, 4, seed=463)
    few = q[:, :1].contiguous()
    return {"prompt": (q, lambda out: O.window_attention(q, k, v, 40, 3, out=out)), "few": (few, lambda out: O.window_attention(few, k, v, 40, 3, q_start=149, out=out)),
            "relative": (q, lambda out: O.relative_attention(q, q, q, table, scale=0.125, out=out))}


@pytest.mark.parametrize("which", ["prompt", "few", "relative"])
def test_an_output_buffer_is_an_in_place_operation(which):
    """What autograd has to know: a tensor that another node saved has changed, and a leaf that requires a gradient is not written."""
    like, call = _calls_with_out()[which]
    want = call(torch.empty_like(like)).clone()
    buffer, weight = torch.ones_like(like), torch.ones_like(like, requires_grad=True)
    loss = (weight * buffer).sum()
    version = buffer._version
    assert call(buffer) is buffer and buffer._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    leaf = torch.ones_like(like, requires_grad=True)
    with pytest.raises(RuntimeError, match="leaf"):
        call(leaf)
    assert float(leaf.detach().min()) == 1
    with torch.no_grad():
        assert call(leaf) is leaf
    same = torch.equal(leaf.detach(), want)
    assert same
    part = (weight * 2)[:, :]                        # a view of a result with a history: its own gradient ends here
    out = call(part)
    grad, = torch.autograd.grad(out.sum(), weight)
    same = torch.equal(out.detach(), want)
    assert same and float(grad.abs().max()) == 0
    with torch.inference_mode():
        frozen = torch.empty_like(like)
        call(frozen)
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        call(frozen)


@pytest.mark.parametrize("scale", [1e-50, 1e-40, 2.0 ** -126, 2.0 ** 127])
def test_scales_at_the_ends_of_fp32(scale):
    """Scales below fp32's normal numbers go to the torch statement. Small ones make all scores equal, large ones leave the largest score's key alone."""
    q, k, v = (t.requires_grad_() for t in _inputs(1, 70, 70, 4, 2, 64, seed=470))
    with torch.no_grad():
        k[..., 1:], q[..., 1:], q[..., 0] = 0, 0, 1                # scores are single numbers, all different
        k[0, :, :, 0] = (torch.arange(70, device=DEV)[:, None] + 1.0) * (0.015625 if scale < 1 else -0.015625)
        table = torch.zeros(32, 4, device=DEV)
        k4 = k.repeat_interleave(2, 2)
        for name, out in (("window", O.window_attention(q, k, v, scale=scale)), ("relative", O.relative_attention(q, k4, v.repeat_interleave(2, 2), table, scale=scale))):
            vh = v.double().repeat_interleave(2, 2)
            if scale < 1:
                want = vh.cumsum(1) / torch.arange(1, 71, device=DEV)[None, :, None, None] if name == "window" else vh.mean(1, keepdim=True).expand_as(vh)
            else:
                want = vh[:, :1].expand_as(vh)
            worst = float((out.double() - want).abs().max())
            assert worst <= 2 * HALF * 4 + 4 * FINE, f"{name} {worst}"
    out = O.window_attention(q, k, v, scale=scale)
    assert all(bool(torch.isfinite(t).all()) for t in torch.autograd.grad(out.sum(), [q, k, v]))


@pytest.mark.parametrize("scale", [1e39, 1e300])
def test_scales_beyond_fp32(scale):
    """The torch statement, whose fp32 scores are infinite."""
    q, k, v = _inputs(1, 70, 70, 4, 4, 64, seed=475)
    table = _normal(32, 4, seed=478)
    for got, want in ((O.window_attention(q, k, v, 20, scale=scale), ref.window_attention(q, k, v, 20, scale=scale)),
                      (O.relative_attention(q, k, v, table, scale=scale), ref.relative_attention(q, k, v, table, scale=scale))):
        same = torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        assert same


@pytest.mark.parametrize("B,H", [(65535, 1), (65536, 1), (1, 65535), (1, 65536)])
def test_many_sequences_and_heads(B, H):
    """To the ends of a grid, and beyond them by the torch statement; forward and backward."""
    q, k, v = (t.requires_grad_() for t in _inputs(B, 2, 3, H, H, 64, seed=480))
    grad, table = _normal(B, 2, H, 64, seed=483), _normal(4, H, seed=484)
    for call, seen in ((lambda: O.window_attention(q, k, v, 2, q_start=1), seen_by(2, 3, 1, 2, 0, None, 1)),
                       (lambda: O.relative_attention(q, k, v, table, 2, scale=0.125), seen_by(2, 3, 1, causal=False))):
        relative = bool(seen.all())
        value, bound = oracle(q, k, v, 0.125, seen.expand(B, 2, 3), grad, table=table if relative else None, max_distance=2)
        with torch.no_grad():
            check(dict(out=call()), value, bound, "no gradient")
        out = call()
        check(dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, [q, k, v], grad)))), value, bound, "gradients")


@pytest.mark.parametrize("H,G,D,window", [(64, 8, 64, 128), (64, 8, 64, None), (4, 4, 128, 3)])
def test_a_prompt_padded_to_other_lengths(H, G, D, window):
    """The tokens of a prompt are the same bits whatever the length that it is padded to, with or without a gradient."""
    q, k, v = _inputs(1, 300, 300, H, G, D, seed=490)
    sink, n = _normal(H, seed=493), torch.tensor([5], dtype=torch.int32, device=DEV)
    want = O.window_attention(q, k, v, window, kv_len=n, sink_logits=sink)[:, :5]
    for S in (5, 8, 9, 64, 65, 130):
        for grad in (False, True):
            got = O.window_attention(q[:, :S].clone().requires_grad_(grad), k[:, :S], v[:, :S], window, kv_len=n, sink_logits=sink)[:, :5]
            same = torch.equal(got.detach(), want)
            assert same, f"{S} {grad}"
